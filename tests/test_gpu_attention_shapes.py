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
