"""GPU: attention at the shapes where the cut of the work changes, against its definition in 64 bits (bounds: policy_reference.py)."""
import importlib
import math

import pytest
import torch

from tests import policy_reference as ref
from tests.test_gpu_policy_ops import DT, _allowed, _close, _gen, _qkv

pytestmark = pytest.mark.gpu


def _pkg():
    return importlib.import_module("online-3d-bpp-pct_amd")


def _check(shape, dtype, kind, seed, train=True):
    b, lq, lk, h, hk, d = shape
    q, k, v, do = _qkv(shape, dtype, seed)
    mask, lengths, allowed = _allowed(kind, b, lk, seed)
    bad = ~allowed.cuda()
    k[bad] = math.nan  # what is not allowed does not matter
    v[bad] = math.inf
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = _pkg().cross_attention(q, k, v, key_mask=mask, key_lengths=lengths)
    got = (out.detach(),) + (torch.autograd.grad(out, leaves, do) if train else ())
    want, bound = ref.attention(q, k.detach().nan_to_num(0, 0, 0), v.detach().nan_to_num(0, 0, 0), allowed, 1 / math.sqrt(d), do if train else None)
    for name, g, w, e in zip(("out", "dq", "dk", "dv"), got, want, bound):
        _close(g, w, e, (name, shape, kind))


# 64 heads and more of at most 512 keys, of which some are not allowed: the key gradient's workgroups are numbered by dies, with
# places left over where the heads are not a multiple of 8, several tiles of keys, and (the last) several parts of the queries
BY_DIE = [(67, 9, 131, 1, 1, 32), (33, 5, 300, 2, 2, 64), (13, 3, 512, 5, 5, 16), (71, 40, 97, 2, 1, 128), (66, 300, 300, 2, 1, 16)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind", ["lengths", "column", "both"])
@pytest.mark.parametrize("shape", BY_DIE, ids=str)
def test_heads_numbered_by_die(shape, kind, dtype):
    _check(shape, dtype, kind, 40)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1, 1, 768, 1, 1, 64), (1, 3, 5000, 1, 1, 8), (1, 1, 16384, 3, 3, 128), (1, 5, 3000, 1, 1, 40), (1, 1, 2048, 1, 1, 16)], ids=str)
def test_an_odd_number_of_partial_rows(shape, dtype):
    _check(shape, dtype, "none", 41, train=False)
    _check(shape, dtype, "lengths", 42, train=False)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("lq,lk", [(1, 1), (40, 70), (5, 33), (130, 3), (64, 64), (3, 2500), (300, 9)], ids=str)
def test_infinite_values_and_gradients_stay_in_their_columns(lq, lk, dtype):
    """an allowed key's infinite value makes its column infinite where it weighs, and so does the output's gradient in dv: at the
    first, an inner and the last place, behind which a tile is filled up"""
    d = 40
    q, k, v, do = _qkv((2, lq, lk, 2, 1, d), dtype, 43)
    out = _pkg().cross_attention(q, k, v)
    for at in sorted({0, lk // 2, lk - 1}):
        w = v.clone()
        w[1, at, 0, 7] = math.inf
        w[1, at, 0, 8] = -math.inf
        got = _pkg().cross_attention(q, k, w)
        assert (got[1, :, :, 7] == math.inf).all() and (got[1, :, :, 8] == -math.inf).all(), at
        keep = [i for i in range(d) if i not in (7, 8)]
        assert torch.equal(got[0], out[0]) and torch.equal(got[1][..., keep], out[1][..., keep]), at
    leaf = v.clone().requires_grad_(True)
    want, = torch.autograd.grad(_pkg().cross_attention(q, k, leaf), [leaf], do)
    for at in sorted({0, lq // 2, lq - 1}):
        g = do.clone()
        g[1, at, 1, 7] = -math.inf
        leaf = v.clone().requires_grad_(True)
        got, = torch.autograd.grad(_pkg().cross_attention(q, k, leaf), [leaf], g)
        keep = [i for i in range(d) if i != 7]
        assert (got[1, :, 0, 7] == -math.inf).all(), at
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][..., keep], want[1][..., keep]), at


# 8 wavefronts to a workgroup in the forward, in dq, in dk and dv; lengths that would make 5 to 7, and just not 8
CUTS = [(16, 1024, 70, 4, 4, 64), (64, 1024, 70, 1, 1, 128), (64, 40, 1024, 1, 1, 128), (64, 1100, 35, 1, 1, 64), (64, 1023, 9, 2, 1, 104), (32, 130, 1300, 2, 2, 120)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", CUTS, ids=str)
def test_long_rows_and_keys_of_many_heads(shape, dtype):
    _check(shape, dtype, "none", 44)
    _check(shape, dtype, "lengths", 45)
