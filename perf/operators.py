"""The policy operators next to the environment: what is timed, and what their outputs are compared with.

Three operators a policy runs between the observation and `RolloutSlots.step_env`:

* `pick`     -- choose one leaf per env from masked logits (`pct_amd.pick_actions`): the index, its log-probability and
                the entropy of the row.  The noise of a sampled choice is an input.
* `logprobs` -- the log-probabilities of given choices, the entropy and the best alternatives
                (`pct_amd.action_log_probs`), forward and, for training, backward.
* `attend`   -- attention of one set of nodes to another of a different length (`pct_amd.cross_attention`), forward and,
                for training, backward.

`own` selects who computes them: the framework's kernels or, where it is false, elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

I_NODES, L_LEAVES = 80, 50  # the environment's default holders: 80 placed boxes, 50 leaves, 1 item to place
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _package():
    import importlib
    return importlib.import_module("pct_amd")


# ---------------------------------------------------------------------------------------------------------------- cases

def _pick(rows, choices, dtype, mask, noise, **kw):
    return dict(op="pick", rows=rows, choices=choices, dtype=dtype, mask=mask, noise=noise, **kw)


def _logprobs(rows, choices, dtype, mask, given, top, train, **kw):
    return dict(op="logprobs", rows=rows, choices=choices, dtype=dtype, mask=mask, given=given, top=top, train=train, **kw)


def _attend(batch, q_len, k_len, heads, kv_heads, dim, dtype, keys, train, **kw):
    return dict(op="attend", batch=batch, q_len=q_len, k_len=k_len, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                keys=keys, train=train, **kw)


def listed():
    return [
        # 64 workers, the trainer's own default: one choice among 50 leaves each.  Nothing but latency.
        _pick(64, 50, "fp32", "nodes", True, name="pick_64x50"),
        # one step of the benchmark's batch of 4096 environments
        _pick(4096, 50, "fp32", "nodes", True, name="pick_4096x50"),
        # the update after a rollout of 5 steps of 4096 environments: log-probabilities, entropy and their gradient
        _logprobs(20480, 50, "fp32", "nodes", 1, 0, True, name="logprobs_train_20480x50"),
        # serving: a few rows over a long list of choices, with the 20 best alternatives
        _logprobs(16, 131072, "bf16", "none", 1, 20, False, name="logprobs_16x131072_top20"),
        # training over a long list of choices: one pass over memory each way
        _logprobs(8192, 65536, "bf16", "none", 1, 0, True, name="logprobs_train_8192x65536"),
        # odd sizes, a mask over single choices, several given choices and alternatives that carry gradients too
        _logprobs(1237, 30011, "fp16", "bool", 3, 5, True, name="logprobs_train_1237x30011_top5"),
        # the leaves of 64 environments attend to all of their nodes: latency
        _attend(64, 50, 131, 1, 1, 64, "fp32", "nodes", False, name="attend_64x50x131"),
        # every node to every node of 4096 environments, in the trainer's type, with gradients
        _attend(4096, 131, 131, 1, 1, 64, "fp32", "nodes", True, name="attend_train_4096x131x131"),
        # the wide configuration: 200 leaves to 401 nodes of 2048 environments, 4 heads
        _attend(2048, 200, 401, 4, 4, 32, "bf16", "nodes", True, name="attend_train_2048x200x401"),
        # single queries against long states, shared heads, ragged lengths: serving
        _attend(16, 1, 16384, 32, 8, 128, "bf16", "lengths", False, name="attend_16x1x16384"),
        # long sequences on both sides, training: matrix products
        _attend(4, 2048, 4096, 16, 16, 128, "bf16", "none", True, name="attend_train_4x2048x4096"),
        # odd lengths, shared heads, a head size between two powers of two, ragged lengths of which one is zero
        _attend(3, 517, 1999, 12, 4, 80, "fp16", "lengths", True, name="attend_train_3x517x1999"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pick", "logprobs", "attend"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("pick", "logprobs"):
        while True:
            rows, choices = _log_int(rng, 1, 32768), _log_int(rng, 1, 131072)
            if rows * choices <= (1 << 27):
                break
        mask = rng.choice(["none", "bool", "lowest"] + (["nodes"] if choices <= 400 else []))
        if op == "pick":
            return _pick(rows, choices, dtype, mask, rng.random() < 0.7)
        return _logprobs(rows, choices, dtype, mask, rng.randint(1, 4), rng.choice([0, 0, 1, rng.randint(2, 32)]),
                         rng.random() < 0.6)
    kv_heads = rng.choice([1, 1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128])
    train = rng.random() < 0.6
    while True:
        batch, q_len, k_len = _log_int(rng, 1, 4096), _log_int(rng, 1, 4096), _log_int(rng, 1, 16384)
        cost = batch * heads * q_len * k_len * (3 if train else 1)
        if cost * dim <= (1 << 36) and cost <= (1 << 30) and batch * max(q_len * heads, k_len * kv_heads) * dim <= (1 << 28):
            break
    keys = rng.choice(["none", "lengths", "bool"] + (["nodes"] if k_len <= 401 else []))
    return _attend(batch, q_len, k_len, heads, kv_heads, dim, dtype, keys, train)


# --------------------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 11)
    return g


def _nodes(rows, placed, leaves, g):
    """Observations as the environment lays them out: [rows, placed + leaves + 1, 9] float32, column 8 saying which rows
    hold a node.  A share of the placed boxes' rows is in use, any number of leaves (none in one row of sixteen), and
    the item to place always."""
    total = placed + leaves + 1
    obs = torch.rand(rows, total, 9, generator=g, device="cuda") * 10
    n_box = (torch.rand(rows, 1, generator=g, device="cuda") * (0.35 * placed + 1)).long()
    n_leaf = (torch.rand(rows, 1, generator=g, device="cuda") * (leaves + 1)).long()
    n_leaf = torch.where(torch.rand(rows, 1, generator=g, device="cuda") < 1 / 16, torch.zeros_like(n_leaf), n_leaf)
    pos = torch.arange(total, device="cuda").unsqueeze(0)
    used = (pos < n_box) | ((pos >= placed) & (pos < placed + n_leaf)) | (pos == total - 1)
    obs[:, :, 8] = used.float()
    return obs * used.unsqueeze(2).float()


def _split(total):
    """how many of `total` nodes are placed boxes and how many leaves, in the environment's proportion"""
    placed = (total - 1) * I_NODES // (I_NODES + L_LEAVES)
    return placed, total - 1 - placed


def _choice_inputs(case, g):
    rows, choices, dtype = case["rows"], case["choices"], _DT[case["dtype"]]
    logits = torch.randn(rows, choices, generator=g, device="cuda", dtype=torch.float32).mul_(2.5).to(dtype)
    mask = None
    if case["mask"] == "nodes":
        # the leaves' own column of the observations: a view with the observation's strides
        mask = _nodes(rows, I_NODES, choices, g)[:, I_NODES:I_NODES + choices, 8]
    elif case["mask"] == "bool":
        mask = torch.rand(rows, choices, generator=g, device="cuda") < 0.6
        mask[:: 97] = False  # some rows have no choice at all
    elif case["mask"] == "lowest":
        # masked by value: the type's lowest number in some places, minus infinity in others
        where = torch.rand(rows, choices, generator=g, device="cuda")
        logits.masked_fill_(where < 0.2, torch.finfo(dtype).min).masked_fill_(where > 0.9, -math.inf)
    return logits, mask


def prepare(case, seed):
    g = _gen(seed)
    dtype = _DT[case["dtype"]]
    state = dict(case=case)
    if case["op"] in ("pick", "logprobs"):
        rows, choices = case["rows"], case["choices"]
        state["logits"], state["mask"] = _choice_inputs(case, g)
        if case["op"] == "pick":
            state["noise"] = None
            if case["noise"]:  # Gumbel noise: the argument of the maximum is then a sample
                u = torch.rand(rows, choices, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
                state["noise"] = u.log_().neg_().log_().neg_()
        else:
            state["given"] = torch.randint(0, choices, (rows, case["given"]), generator=g, device="cuda")
            if case["train"]:
                state["logits"].requires_grad_(True)
                state["d_given"] = torch.randn(rows, case["given"], generator=g, device="cuda")
                state["d_entropy"] = torch.randn(rows, generator=g, device="cuda") * 0.01
                if case["top"]:
                    state["d_top"] = torch.randn(rows, case["top"], generator=g, device="cuda") * 0.1
        return state
    b, lq, lk, h, hk, d = (case[n] for n in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim"))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    state["q"], state["k"], state["v"] = normal(b, lq, h, d), normal(b, lk, hk, d), normal(b, lk, hk, d)
    state["key_mask"] = state["key_lengths"] = None
    if case["keys"] == "nodes":
        state["key_mask"] = _nodes(b, *_split(lk), g)[:, :, 8]
    elif case["keys"] == "bool":
        state["key_mask"] = torch.rand(b, lk, generator=g, device="cuda") < 0.6
    elif case["keys"] == "lengths":
        # between half of the states and all of them; one of three or more has none
        n = (lk * (0.5 + 0.5 * torch.rand(b, generator=g, device="cuda"))).round().to(torch.int32)
        if case["train"] and b >= 3:
            n[1] = 0
        state["key_lengths"] = n
    if case["train"]:
        for name in ("q", "k", "v"):
            state[name].requires_grad_(True)
        state["d_out"] = normal(b, lq, h, d)
    return state


# ------------------------------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if case["op"] == "pick":
        return _pick_own(state) if own else _pick_plain(state)
    if case["op"] == "logprobs":
        return _logprobs_own(state) if own else _logprobs_plain(state)
    return _attend_own(state) if own else _attend_plain(state)


def _pick_own(state):
    out = _package().pick_actions(state["logits"], mask=state["mask"], noise=state["noise"])
    return dict(actions=out.actions, log_probs=out.log_probs, entropy=out.entropy)


def _logprobs_own(state):
    case = state["case"]
    out = _package().action_log_probs(state["logits"], state["given"], mask=state["mask"], top=case["top"])
    res = dict(log_probs=out.log_probs, entropy=out.entropy)
    if case["top"]:
        res.update(top_log_probs=out.top_log_probs, top_actions=out.top_actions)
    if case["train"]:
        outs, grads = [out.log_probs, out.entropy], [state["d_given"], state["d_entropy"]]
        if case["top"]:
            outs.append(out.top_log_probs)
            grads.append(state["d_top"])
        res["d_logits"], = torch.autograd.grad(outs, [state["logits"]], grads)
    return {k: v.detach() for k, v in res.items()}


def _attend_own(state):
    q, k, v = state["q"], state["k"], state["v"]
    out = _package().cross_attention(q, k, v, key_mask=state["key_mask"], key_lengths=state["key_lengths"])
    res = dict(out=out.detach())
    if state["case"]["train"]:
        res["d_q"], res["d_k"], res["d_v"] = torch.autograd.grad(out, (q, k, v), state["d_out"])
    return res


def _choice_terms(logits, mask):
    """allowed, whether a row allows anything, log-probabilities of the allowed choices, probabilities, entropy: in 32 bits"""
    x = logits.detach().float()
    allowed = x != -math.inf
    if mask is not None:
        allowed = allowed & (mask != 0)
    some = allowed.any(1)
    x = x.masked_fill(~allowed, -math.inf)
    top = torch.where(some, x.amax(1), torch.zeros_like(x[:, 0]))
    x = x - top.unsqueeze(1)
    e = x.exp()
    total = torch.where(some, e.sum(1), torch.ones_like(top))
    log_total = total.log()
    p = e / total.unsqueeze(1)
    entropy = log_total - (p * x.masked_fill(~allowed, 0.0)).sum(1)
    return allowed, some, x - log_total.unsqueeze(1), p, torch.where(some, entropy, torch.zeros_like(entropy))


def _order_keys(x, allowed):
    """whole numbers in the order of the values, the lower index first among equal ones; below all others where not allowed"""
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    pos = torch.arange(x.shape[1], device=x.device)
    return torch.where(allowed, (key << 32) + (0xFFFFFFFF - pos), torch.full_like(key, -(1 << 63)))


def _pick_plain(state):
    x = state["logits"].float()
    allowed, some, log_p, _, entropy = _choice_terms(state["logits"], state["mask"])
    if state["noise"] is not None:
        x = x + state["noise"]
    actions = torch.where(some, _order_keys(x, allowed).argmax(1), torch.zeros_like(some, dtype=torch.long)).unsqueeze(1)
    log_probs = torch.where(some.unsqueeze(1), log_p.gather(1, actions), torch.zeros_like(entropy).unsqueeze(1))
    return dict(actions=actions, log_probs=log_probs, entropy=entropy)


def _logprobs_plain(state):
    case, logits, given = state["case"], state["logits"], state["given"]
    allowed, some, log_p, p, entropy = _choice_terms(logits, state["mask"])
    log_probs = log_p.gather(1, given).masked_fill(~some.unsqueeze(1), 0.0)
    res = dict(log_probs=log_probs, entropy=entropy)
    best = None
    if case["top"]:
        keys = _order_keys(logits.detach().float(), allowed)
        n = min(case["top"], keys.shape[1])
        value, best = keys.topk(n, dim=1)
        found = value != -(1 << 63)
        alt = torch.where(found, log_p.gather(1, best), torch.full_like(value, -math.inf, dtype=torch.float32))
        best = torch.where(found, best, torch.full_like(best, -1))
        if n < case["top"]:
            more = case["top"] - n
            alt = torch.nn.functional.pad(alt, (0, more), value=-math.inf)
            best = torch.nn.functional.pad(best, (0, more), value=-1)
        res.update(top_log_probs=alt, top_actions=best)
    if case["train"]:
        # d logit_j = sum over given g of d_g (1[j = g] - p_j)  -  d_entropy p_j (log p_j + entropy)
        ids, d = given, state["d_given"]
        d = torch.where(allowed.gather(1, ids), d, torch.zeros_like(d))
        if best is not None:
            ids = torch.cat([ids, best.clamp(min=0)], 1)
            d = torch.cat([d, torch.where(best >= 0, state["d_top"], torch.zeros_like(state["d_top"]))], 1)
        slope = log_p.masked_fill(~allowed, 0.0) + entropy.unsqueeze(1)
        grad = -p * (d.sum(1, keepdim=True) + state["d_entropy"].unsqueeze(1) * slope)
        grad = grad.scatter_add(1, ids, d)
        grad = grad.masked_fill(~allowed, 0.0)
        res["d_logits"] = grad.to(logits.dtype)
    return res


def _allowed_keys(state):
    """[batch, k_len] truth values, or None where every key is allowed"""
    case, allowed = state["case"], None
    if state["key_mask"] is not None:
        allowed = state["key_mask"] != 0
    if state["key_lengths"] is not None:
        short = torch.arange(case["k_len"], device="cuda").unsqueeze(0) < state["key_lengths"].unsqueeze(1)
        allowed = short if allowed is None else allowed & short
    return allowed


def _attend_plain(state):
    case = state["case"]
    b, lq, lk, h, hk, d = (case[n] for n in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim"))
    dtype, groups, scale = state["q"].dtype, h // hk, 1.0 / math.sqrt(d)
    allowed = _allowed_keys(state)

    def heads_first(x, n):  # [b, l, n, d] -> [b, kv heads, (l, heads that share one), d] in 32 bits
        x = x.detach().float().view(b, -1, hk, n // hk, d)
        return x.permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d).contiguous()

    def back(x, n):
        return x.view(b, hk, -1, n // hk, d).permute(0, 2, 1, 3, 4).reshape(b, -1, n, d).to(dtype).contiguous()

    q, k, v = heads_first(state["q"], h), heads_first(state["k"], hk), heads_first(state["v"], hk)
    if allowed is not None:
        keep = allowed.view(b, 1, lk, 1)
        k, v = k.masked_fill(~keep, 0.0), v.masked_fill(~keep, 0.0)
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    if allowed is not None:
        p.masked_fill_(~allowed.view(b, 1, 1, lk), -math.inf)
        top = p.amax(3, keepdim=True)
        p.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
        total = p.sum(3, keepdim=True)
        p.div_(total.masked_fill_(total == 0, 1.0))
    else:
        p.sub_(p.amax(3, keepdim=True)).exp_()
        p.div_(p.sum(3, keepdim=True))
    o = torch.matmul(p, v)
    res = dict(out=back(o, h))
    if case["train"]:
        do = heads_first(state["d_out"], h)
        res["d_v"] = back(torch.matmul(p.transpose(2, 3).contiguous(), do), hk)
        ds = torch.matmul(do, v.transpose(2, 3).contiguous()).sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(scale)
        res["d_q"] = back(torch.matmul(ds, k), h)
        res["d_k"] = back(torch.matmul(ds.transpose(2, 3).contiguous(), q), hk)
        res = {n: res[n] for n in ("out", "d_q", "d_k", "d_v")}
    return res


# ---------------------------------------------------------------------------------------------------------------- work

def _used_share(placed, leaves):
    """the mean share of an observation's nodes in use"""
    return (0.35 * placed / 2 + leaves / 2 * 15 / 16 + 1) / (placed + leaves + 1)


def work(case):
    n = _SIZE[case["dtype"]]
    if case["op"] in ("pick", "logprobs"):
        cells = case["rows"] * case["choices"]
        bytes_ = cells * n
        bytes_ += cells * {"none": 0, "lowest": 0, "bool": 1, "nodes": 4}[case["mask"]]
        flops = 6 * cells
        if case["op"] == "pick":
            bytes_ += (4 * cells if case["noise"] else 0) + case["rows"] * 16
        else:
            bytes_ += case["rows"] * (case["given"] * 12 + 4 + case["top"] * 12)
            if case["train"]:
                # the gradient reads the logits once more: it is asked for after the log-probabilities were given out
                bytes_ += 2 * cells * n + case["rows"] * 4 * (case["given"] + case["top"] + 1)
                flops += 6 * cells
        return {"bytes": bytes_, "flops": flops}
    b, lq, lk, h, hk, d = (case[n_] for n_ in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim"))
    share = {"none": 1.0, "bool": 0.6, "lengths": 0.75, "nodes": _used_share(*_split(lk))}[case["keys"]]
    if case["keys"] == "lengths" and case["train"] and b >= 3:
        share *= (b - 1) / b
    rows_q, rows_k = b * lq * h * d, b * lk * hk * d
    bytes_ = (2 * rows_q + 2 * rows_k * share) * n
    flops = 4 * b * h * lq * lk * share * d
    if case["train"]:
        bytes_ += (4 * rows_q + 2 * rows_k * share + 2 * rows_k) * n
        flops += 10 * b * h * lq * lk * share * d
    return {"bytes": int(bytes_), "flops": int(flops)}


# --------------------------------------------------------------------------------------------------------------- exact

def _exact_choice(state, lo, hi):
    case = state["case"]
    raw = state["logits"].detach()[lo:hi]
    x = raw.double()
    ok = torch.isfinite(x)
    if state["mask"] is not None:
        ok &= state["mask"][lo:hi].bool()
    empty = ~ok.any(dim=1)
    x = torch.where(ok, x, torch.tensor(-math.inf, dtype=torch.float64, device=x.device))
    lse = torch.logsumexp(x, dim=1)
    lp = torch.where(ok, x - lse[:, None], torch.tensor(-math.inf, dtype=torch.float64, device=x.device))
    prob = torch.where(ok, lp.exp(), torch.zeros_like(lp))
    ent = -(prob * torch.where(ok, lp, torch.zeros_like(lp))).sum(dim=1)
    ent[empty] = 0.0
    if case["op"] == "pick":
        score = raw.float()
        if state["noise"] is not None:
            score = score + state["noise"][lo:hi]
        best = score.masked_fill(~ok, -math.inf)
        rank = best == best.amax(dim=1, keepdim=True)
        rank &= ok
        idx = torch.where(empty, 0, rank.to(torch.uint8).argmax(dim=1))
        chosen = lp.gather(1, idx[:, None])
        chosen[empty] = 0.0
        return dict(actions=idx[:, None], log_probs=chosen, entropy=ent)
    given = state["given"][lo:hi]
    chosen = lp.gather(1, given)
    chosen[empty] = 0.0
    out = dict(log_probs=chosen, entropy=ent)
    weights = []
    if case["top"]:
        count = case["top"]
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :count]
        alt = lp.gather(1, order)
        order = torch.where(torch.isinf(alt), -1, order)
        alt = torch.where(order < 0, -math.inf, alt)
        lack = count - order.shape[1]
        if lack:
            order = torch.cat([order, order.new_full((order.shape[0], lack), -1)], 1)
            alt = torch.cat([alt, alt.new_full((alt.shape[0], lack), -math.inf)], 1)
        out.update(top_log_probs=alt, top_actions=order)
        weights = [(order, "d_top")]
    if case["train"]:
        grad = -state["d_entropy"][lo:hi].double()[:, None] * prob * (torch.where(ok, lp, torch.zeros_like(lp)) + ent[:, None])
        for ids, name in [(given, "d_given")] + weights:
            for c in range(ids.shape[1]):
                j = ids[:, c:c + 1]
                w = state[name][lo:hi, c:c + 1].double()
                w = torch.where((j >= 0) & ok.gather(1, j.clamp(min=0)), w, torch.zeros_like(w))
                grad -= prob * w
                grad.scatter_add_(1, j.clamp(min=0), w)
        out["d_logits"] = torch.where(ok, grad, torch.zeros_like(grad))
    return out


def _exact_attend(state):
    case = state["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    outs = {n: torch.zeros(state[m].shape, dtype=torch.float64, device="cuda")
            for n, m in (("out", "q"), ("d_q", "q"), ("d_k", "k"), ("d_v", "v")) if n == "out" or case["train"]}
    allowed = _allowed_keys(state)
    if case["batch"] * max(1, hk) <= 256:
        spans = [(i, i + 1) for i in range(case["batch"])]
    else:
        step = max(1, (1 << 26) // (case["q_len"] * case["k_len"] * h))
        spans = [(i, min(i + step, case["batch"])) for i in range(0, case["batch"], step)]
    for lo, hi in spans:
        for head in range(h):
            kv = head * hk // h
            q, k, v = (state[n].detach()[lo:hi, :, j].double() for n, j in (("q", head), ("k", kv), ("v", kv)))
            s = torch.matmul(q, k.mT.contiguous()) / math.sqrt(d)
            if allowed is not None:
                use = allowed[lo:hi, None, :]
                s = torch.where(use, s, torch.full_like(s, -math.inf))
                p = torch.softmax(s, dim=2)
                p = torch.where(use, p, torch.zeros_like(p))  # a row with nothing allowed is zero, not NaN
            else:
                p = torch.softmax(s, dim=2)
            o = torch.matmul(p, v)
            outs["out"][lo:hi, :, head] = o
            if case["train"]:
                do = state["d_out"][lo:hi, :, head].double()
                outs["d_v"][lo:hi, :, kv] += torch.matmul(p.mT.contiguous(), do)
                dp = torch.matmul(do, v.mT.contiguous())
                ds = p * (dp - (p * dp).sum(dim=2, keepdim=True)) / math.sqrt(d)
                outs["d_q"][lo:hi, :, head] = torch.matmul(ds, k)
                outs["d_k"][lo:hi, :, kv] += torch.matmul(ds.mT.contiguous(), q)
    return outs


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attend":
        if case["batch"] * case["heads"] * case["q_len"] * case["k_len"] * case["dim"] > (1 << 38):
            return None
        return _exact_attend(state)
    if case["rows"] * case["choices"] > (1 << 30):
        return None
    step = max(1, (1 << 26) // case["choices"])
    parts = [_exact_choice(state, lo, min(lo + step, case["rows"])) for lo in range(0, case["rows"], step)]
    return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
