"""GPU: the policy operators as parts of a program -- saved tensors that are moved, inputs that are written over, several calls and
captured ones."""
import importlib
import math

import pytest
import torch

from tests import policy_reference as ref
from tests.test_gpu_policy_ops import _close, _gen, _logits, _qkv

pytestmark = pytest.mark.gpu


def _pkg():
    return importlib.import_module("online-3d-bpp-pct_amd")


def _column(n, v, seed):
    wide = torch.zeros(n, 131, 9)
    wide[:, 80:80 + v, 8] = (torch.rand(n, v, generator=_gen(seed)) < 0.5).float()
    wide[::5, 80:80 + v, 8] = 0
    return wide.cuda()[:, 80:80 + v, 8]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gradients_with_saved_tensors_on_the_cpu(dtype):
    pk = _pkg()
    ids = torch.randint(-1, 50, (64, 2), generator=_gen(1)).cuda()
    for mask in (_column(64, 50, 2), torch.arange(64).cuda()[:, None] % 3 != 0, torch.arange(50).cuda()[None] % 7 != 0, None):
        def run():
            x = _logits(64, 50, dtype, 3).requires_grad_(True)
            o = pk.action_log_probs(x, ids, mask=mask, top=4)
            return x, [o.log_probs, o.entropy, o.top_log_probs]
        d = [torch.randn(64, k, generator=_gen(k)).cuda().squeeze(1) for k in (2, 1, 4)]
        x, outs = run()
        want, = torch.autograd.grad(outs, [x], d)
        with torch.autograd.graph.save_on_cpu():
            x, outs = run()
        got, = torch.autograd.grad(outs, [x], d)
        assert torch.equal(got, want)
    q, k, v, do = _qkv((3, 9, 70, 4, 2, 40), dtype, 4)
    mask = _column(3, 50, 5)[:, :1] != torch.ones(1, 70).cuda()
    mask[:, 0] = True
    wide = torch.stack([k, v], 2)  # k and v as slices of one tensor
    run = lambda: (lambda l: (l, pk.cross_attention(*l, key_mask=mask)))(
        [q.clone().requires_grad_(True), wide[:, :, 0].detach().requires_grad_(True), wide[:, :, 1].detach().requires_grad_(True)])
    leaves, out = run()
    want = torch.autograd.grad(out, leaves, do)
    with torch.autograd.graph.save_on_cpu():
        leaves, out = run()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, do), want))


def test_an_evaluation_outlives_the_next_rollout():
    """collect writes actions and observations of the slots; a gradient that is taken after it is that of the steps evaluated"""
    pk = _pkg()
    items = [(a, b, c) for a in range(1, 6) for b in range(1, 6) for c in range(1, 6)]
    env = pk.PctVecEnv(24, setting=2, item_set=items, internal_node_holder=80, leaf_node_holder=50, seed=9)
    env.reset()
    slots = pk.RolloutSlots(5, 24, (131 * 9,), 1.0, "cuda")
    weights = torch.randn(9, generator=_gen(1)).cuda()
    policy = lambda nodes: nodes[:, 80:130] @ weights
    torch.manual_seed(3)
    pk.collect(env, policy, slots)
    logits = torch.randn(120, 50, generator=_gen(2)).cuda().requires_grad_(True)
    d = [torch.randn(120, 1, generator=_gen(3)).cuda(), torch.randn(120, generator=_gen(4)).cuda()]
    res = slots.evaluate(logits)
    want, = torch.autograd.grad([res.log_probs, res.entropy], [logits], d)
    with torch.no_grad():
        plain = slots.evaluate(logits)
    assert all(torch.equal(a.detach(), b) for a, b in zip(res[:2], plain[:2]))
    res = slots.evaluate(logits)
    before = slots.actions.clone(), slots.obs.clone()
    slots.after_update()
    pk.collect(env, policy, slots)
    assert not torch.equal(before[0], slots.actions) and not torch.equal(before[1], slots.obs)
    got, = torch.autograd.grad([res.log_probs, res.entropy], [logits], d)
    assert torch.equal(got, want)


def test_lengths_may_change_after_the_forward_pass():
    pk = _pkg()
    q, k, v, do = _qkv((4, 20, 130, 2, 1, 32), "bf16", 14)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    lengths = torch.tensor([130, 0, 77, 1]).cuda()
    for mask in (None, (torch.rand(4, 130, generator=_gen(5)) < 0.5).cuda()):
        want = torch.autograd.grad(pk.cross_attention(q, k, v, key_mask=mask, key_lengths=lengths), leaves, do)
        own = lengths.clone()
        out = pk.cross_attention(q, k, v, key_mask=mask, key_lengths=own)
        own.fill_(130)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, do), want))
