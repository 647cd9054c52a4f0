"""The operators a policy runs between an observation and `RolloutSlots.step_env`, as hand-written kernels behind
include/pct_policy.h:

* `pick_actions`      one choice per row from masked logits -- with Gumbel noise a sample, without the best -- with its
                      log-probability and the row's entropy (distributions.py's Categorical .sample() / .mode() and
                      .log_probs(), in one launch);
* `action_log_probs`  the log-probabilities of given choices, the entropy and the best alternatives, differentiable with
                      respect to the logits (what evaluate_actions needs, model.py / train_tools.py);
* `cross_attention`   softmax attention of one set of nodes to another of a different length, with a key mask or key lengths
                      and shared key/value heads, differentiable with respect to q, k and v.

All of them run on the current stream of the tensors' device, allocate outputs and workspaces from torch's allocator (so
they can be captured into a graph) and never synchronise.  A tensor that another stream is still writing, or is handed to
another stream for reuse, is the caller's to order (wait_stream, record_stream), as with torch's own operators.  To capture a
backward pass, let no eager graph of the same leaves live: their accumulation nodes remember the stream they were made on.
Tensors on the CPU are refused: there is no CPU path.
"""
import collections
import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .vec_env import PctEnvError

PickedActions = collections.namedtuple("PickedActions", "actions log_probs entropy")
ActionLogProbs = collections.namedtuple("ActionLogProbs", "log_probs entropy top_log_probs top_actions")

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MASK = {torch.bool: 1, torch.uint8: 1, torch.int8: 1, torch.float16: 2, torch.bfloat16: 2, torch.float32: 3, torch.int32: 4}
_INTS = (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8)
MAX_GIVEN = MAX_TOP = 64

try:  # the handle alone, without a Stream object around it
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


class _Choice(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("dtype", ctypes.c_int32), ("rows", ctypes.c_int32), ("choices", ctypes.c_int32),
                ("logits", ctypes.c_void_p), ("logits_row", ctypes.c_int64), ("mask", ctypes.c_void_p), ("mask_row", ctypes.c_int64),
                ("mask_col", ctypes.c_int64), ("mask_type", ctypes.c_int32), ("given_count", ctypes.c_int32), ("given", ctypes.c_void_p),
                ("top", ctypes.c_int32), ("pad", ctypes.c_int32), ("noise", ctypes.c_void_p), ("noise_row", ctypes.c_int64),
                ("actions", ctypes.c_void_p), ("log_probs", ctypes.c_void_p), ("entropy", ctypes.c_void_p),
                ("top_log_probs", ctypes.c_void_p), ("top_actions", ctypes.c_void_p), ("stats", ctypes.c_void_p),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64)]


class _ChoiceGrad(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("dtype", ctypes.c_int32), ("rows", ctypes.c_int32), ("choices", ctypes.c_int32),
                ("logits", ctypes.c_void_p), ("logits_row", ctypes.c_int64), ("mask", ctypes.c_void_p), ("mask_row", ctypes.c_int64),
                ("mask_col", ctypes.c_int64), ("mask_type", ctypes.c_int32), ("given_count", ctypes.c_int32), ("given", ctypes.c_void_p),
                ("top", ctypes.c_int32), ("pad", ctypes.c_int32), ("top_actions", ctypes.c_void_p), ("stats", ctypes.c_void_p),
                ("d_log_probs", ctypes.c_void_p), ("d_entropy", ctypes.c_void_p), ("d_top_log_probs", ctypes.c_void_p),
                ("d_logits", ctypes.c_void_p)]


_CHOICE_SIZE, _GRAD_SIZE = ctypes.sizeof(_Choice), ctypes.sizeof(_ChoiceGrad)


class _Attention(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("dtype", ctypes.c_int32), ("batch", ctypes.c_int32), ("q_len", ctypes.c_int32),
                ("k_len", ctypes.c_int32), ("heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("dim", ctypes.c_int32),
                ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("q_stride", ctypes.c_int64 * 3), ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
                ("key_mask", ctypes.c_void_p), ("mask_row", ctypes.c_int64), ("mask_col", ctypes.c_int64),
                ("mask_type", ctypes.c_int32), ("lengths_type", ctypes.c_int32), ("key_lengths", ctypes.c_void_p),
                ("scale", ctypes.c_float), ("pad", ctypes.c_int32), ("out", ctypes.c_void_p), ("stats", ctypes.c_void_p),
                ("key_list", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64),
                ("d_out", ctypes.c_void_p), ("d_out_stride", ctypes.c_int64 * 3), ("d_q", ctypes.c_void_p),
                ("d_k", ctypes.c_void_p), ("d_v", ctypes.c_void_p)]


_ATTENTION_SIZE = ctypes.sizeof(_Attention)

_L = None


def _library():
    global _L
    if _L is None:
        L = _lib.load()
        i32, vp = ctypes.c_int32, ctypes.c_void_p
        L.pct_choice_workspace.argtypes = [i32, i32, i32]
        L.pct_choice_workspace.restype = ctypes.c_int64
        L.pct_attend_workspace.argtypes = [vp, i32]
        L.pct_attend_workspace.restype = ctypes.c_int64
        for f in (L.pct_choice_pick, L.pct_choice_log_probs, L.pct_choice_backward, L.pct_attend, L.pct_attend_backward):
            f.argtypes = [vp, vp]
            f.restype = ctypes.c_int
        _L = L
    return _L


def _call(fn, args, device):
    """one C call on the device's current stream, with that device current"""
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = fn(ctypes.addressof(args), torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = fn(ctypes.addressof(args), _raw_stream(index))
    if rc:
        _lib.check(rc)


def _once_differentiable(backward):
    """torch's once_differentiable, but only where a graph of the backward pass is being made"""
    guarded = torch.autograd.function.once_differentiable(backward)

    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return wrapper


def _on_gpu(name, *tensors):
    dev = tensors[0].device
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device != dev):
            if not t.is_cuda:
                raise PctEnvError("%s runs on an AMD GPU only (a tensor is on %s); there is no CPU path" % (name, t.device))
            raise ValueError("%s: tensors on %s and on %s" % (name, dev, t.device))
    return dev


def _no_tangents(name, *tensors):
    """the kernels differentiate backward only: a forward-mode derivative would be lost on the way"""
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("%s: forward-mode derivatives are not implemented" % name)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _whole(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _rows_of(x):
    """x with unit stride along the last dimension (itself where it has it)"""
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


def _mask_of(name, mask, shape):
    """a mask that broadcasts to `shape`, expanded to it (or None)"""
    if mask is None:
        return None
    if mask.dtype not in _MASK:
        raise TypeError("%s: the mask must be bool, uint8, int8, int32 or a 16 / 32-bit float, not %s" % (name, mask.dtype))
    if mask.shape != shape:
        if mask.dim() > 2 or any(a != 1 and a != b for a, b in zip(reversed(mask.shape), reversed(shape))):
            raise ValueError("%s: a mask of shape %s does not fit %s" % (name, tuple(mask.shape), tuple(shape)))
        mask = mask.expand(shape)
    return mask


def _mask_fields(mask):
    """address, strides and type of the tensor at hand: a saved mask may come back laid out in another way"""
    return (None, 0, 0, 0) if mask is None else (mask.data_ptr(), mask.stride(0), mask.stride(1), _MASK[mask.dtype])


def _check_logits(name, logits):
    if logits.dim() != 2:
        raise ValueError("%s: logits must be [rows, choices], not %s" % (name, tuple(logits.shape)))
    if logits.dtype not in _DTYPE:
        raise TypeError("%s: logits must be float32, bfloat16 or float16, not %s" % (name, logits.dtype))
    if logits.shape[1] < 1:
        raise ValueError("%s: at least one choice is needed" % name)
    if logits.shape[0] >= 1 << 31 or logits.shape[1] >= 1 << 31:
        raise ValueError("%s: rows and choices must be below 2^31" % name)


def _out(name, t, shape, dtype, x):
    if t is None:
        return x.new_empty(shape, dtype=dtype)  # (a microsecond less than torch.empty with a device)
    dev = x.device
    if t.dtype != dtype or t.device != dev or t.numel() != math.prod(shape) or not t.is_contiguous():
        raise ValueError("%s must be a contiguous %s tensor of %s on %s" % (name, dtype, tuple(shape), dev))
    return t


def pick_actions(logits, mask=None, noise=None, actions_out=None, log_probs_out=None):
    """One choice per row of `logits` [N, V]: `argmax(float32(logits) + noise)` over the allowed choices, the lowest index
    among equal ones; returns `PickedActions(actions int64 [N, 1], log_probs float32 [N, 1], entropy float32 [N])`, where the
    log-probability and the entropy are those of softmax(logits) over the allowed choices (without the noise).

    A choice is allowed where `mask` [N, V] (or broadcast to it; any strides: the observation's own mask column will do) is
    not zero and its logit is not -inf.  With Gumbel noise (float32 [N, V], -log(-log(u))) the choice is a sample; without,
    the mode.  A row that allows nothing picks 0 with log-probability and entropy 0.  Results carry no gradient.
    `actions_out` / `log_probs_out`: contiguous int64 / float32 tensors of N elements to write to."""
    _check_logits("pick_actions", logits)
    n, v = logits.shape
    x = _rows_of(logits)
    mask = _mask_of("pick_actions", mask, logits.shape)
    if noise is not None:
        if noise.dtype != torch.float32 or noise.shape != logits.shape:
            raise ValueError("pick_actions: noise must be float32 of the logits' shape")
        noise = _rows_of(noise)
    dev = _on_gpu("pick_actions", logits, mask, noise, actions_out, log_probs_out)
    actions = _out("actions_out", actions_out, (n, 1), torch.int64, x)
    log_probs = _out("log_probs_out", log_probs_out, (n, 1), torch.float32, x)
    entropy = x.new_empty(n, dtype=torch.float32)
    if n:
        L = _library()
        ws_bytes = L.pct_choice_workspace(n, v, 0)
        ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
        c = _Choice(_CHOICE_SIZE, _DTYPE[x.dtype], n, v, x.data_ptr(), x.stride(0), *_mask_fields(mask), 0, None,
                    0, 0, _ptr(noise), noise.stride(0) if noise is not None else 0, actions.data_ptr(), log_probs.data_ptr(),
                    entropy.data_ptr(), None, None, None, _ptr(ws), ws_bytes)
        _call(L.pct_choice_pick, c, dev)
        for t in (actions_out, log_probs_out):
            if t is not None:  # written in place: a graph that has saved it says so instead of reading the new values
                torch.autograd.graph.increment_version(t)
    return PickedActions(actions, log_probs, entropy)


def _log_probs_forward(x, given, mask, top, want_stats):
    n, v = x.shape
    dev = x.device
    g = given.shape[1]
    log_probs = x.new_empty((n, g), dtype=torch.float32)
    entropy = x.new_empty(n, dtype=torch.float32)
    top_log_probs = x.new_empty((n, top), dtype=torch.float32) if top else None
    top_actions = x.new_empty((n, top), dtype=torch.int64) if top else None
    stats = x.new_empty((n, 4), dtype=torch.float32) if want_stats else None
    if n:
        L = _library()
        ws_bytes = L.pct_choice_workspace(n, v, top)
        ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
        c = _Choice(_CHOICE_SIZE, _DTYPE[x.dtype], n, v, x.data_ptr(), x.stride(0), *_mask_fields(mask),
                    g, given.data_ptr(), top, 0, None, 0, None, log_probs.data_ptr(), entropy.data_ptr(), _ptr(top_log_probs),
                    _ptr(top_actions), _ptr(stats), _ptr(ws), ws_bytes)
        _call(L.pct_choice_log_probs, c, dev)
    return log_probs, entropy, top_log_probs, top_actions, stats


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, given, mask, top):
        x = _rows_of(logits)
        log_probs, entropy, top_log_probs, top_actions, stats = _log_probs_forward(x, given, mask, top, True)
        ctx.save_for_backward(x, given, mask, top_actions, stats)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_actions)
            return log_probs, entropy, top_log_probs, top_actions
        return log_probs, entropy

    @staticmethod
    @_once_differentiable
    def backward(ctx, d_log_probs, d_entropy, d_top=None, _=None):
        x, given, mask, top_actions, stats = ctx.saved_tensors  # (hooks on saved tensors may have laid them out anew)
        x, given, top_actions, stats = _rows_of(x), _whole(given), _whole(top_actions), _whole(stats)
        n, v = x.shape
        dx = x.new_empty((n, v))
        if n:
            d_log_probs, d_entropy, d_top = _whole(d_log_probs), _whole(d_entropy), _whole(d_top)
            c = _ChoiceGrad(_GRAD_SIZE, _DTYPE[x.dtype], n, v, x.data_ptr(), x.stride(0), *_mask_fields(mask),
                            given.shape[1], given.data_ptr(), 0 if top_actions is None else top_actions.shape[1], 0, _ptr(top_actions),
                            stats.data_ptr(), _ptr(d_log_probs), _ptr(d_entropy), _ptr(d_top), dx.data_ptr())
            _call(_library().pct_choice_backward, c, x.device)
        return dx, None, None, None


def action_log_probs(logits, actions, mask=None, top=0):
    """Log-probabilities of given choices under softmax(logits) over the allowed choices (`pick_actions` says which), the
    entropy of each row and, with `top` = K (at most 64), its K best choices.  Returns `ActionLogProbs(log_probs, entropy [N],
    top_log_probs [N, K] or None, top_actions int64 [N, K] or None)`, the log-probabilities float32 and in the shape of
    `actions`, integers [N] or [N, G], G at most 64.  Differentiable with respect to `logits` (once, backward).

    An id of -1 stands for "none": log-probability 0, no gradient.  A choice that is not allowed has -inf and takes no
    gradient; an id outside of [-1, V) has NaN.  A row that allows nothing has log-probabilities and entropy 0 and a zero
    gradient.  Alternatives come in falling order, the lower index first among equal logits; where fewer than K choices are
    allowed the rest is -inf with action -1.  The backward pass reads the logits and the mask again: neither may have been
    written over by then.  The actions may: where a gradient can be asked for, a copy of them is kept."""
    _check_logits("action_log_probs", logits)
    n = logits.shape[0]
    if actions.dtype not in _INTS:
        raise TypeError("action_log_probs: actions must be integers, not %s" % actions.dtype)
    if actions.dim() not in (1, 2) or actions.shape[0] != n:
        raise ValueError("action_log_probs: actions must be [N] or [N, G] for %d rows, not %s" % (n, tuple(actions.shape)))
    given = actions if actions.dim() == 2 else actions.unsqueeze(1)
    if given.shape[1] > MAX_GIVEN:
        raise ValueError("action_log_probs: at most %d actions to a row" % MAX_GIVEN)
    top = int(top)
    if not 0 <= top <= MAX_TOP:
        raise ValueError("action_log_probs: top must be 0 .. %d" % MAX_TOP)
    mask = _mask_of("action_log_probs", mask, logits.shape)
    _on_gpu("action_log_probs", logits, actions, mask)
    _no_tangents("action_log_probs", logits)
    taped = torch.is_grad_enabled() and logits.requires_grad
    if given.dtype != torch.int64 or not given.is_contiguous():
        given = given.to(torch.int64).contiguous()
    elif taped:  # (the caller's own, a rollout's slots for instance, which kernels write without telling torch)
        given = given.clone()
    if taped:
        res = _LogProbs.apply(logits, given, mask, top)
    else:
        res = _log_probs_forward(_rows_of(logits), given, mask, top, False)
    return ActionLogProbs(res[0] if actions.dim() == 2 else res[0].squeeze(1), res[1], res[2] if top else None, res[3] if top else None)


def _attention_rows(x):
    """x [batch, length, heads, dim] as the kernels read it -- unit stride along dim, every row on a 16-byte boundary -- itself
    where it is so, else a copy"""
    if x.data_ptr() % 16 == 0:
        if x.is_contiguous():
            return x
        per = 16 // x.element_size()
        if (x.stride(3) == 1 or x.shape[3] == 1) and not any(x.stride(i) % per for i in range(3) if x.shape[i] > 1):
            return x
    return x.contiguous() if not x.is_contiguous() else x.clone()


_Strides = ctypes.c_int64 * 3


def _strides(x):
    s, n = x.stride(), x.shape
    # (the stride of a dimension of one element is arbitrary)
    return _Strides(s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


def _attention_struct(q, k, v, mask, lengths, scale, out, stats, key_list):
    """mask: address, row stride, column stride, type; the backward reads key_list alone, and says so with any address and type"""
    b, lq, h, d = q.shape
    return _Attention(_ATTENTION_SIZE, _DTYPE[q.dtype], b, lq, k.shape[1], h, k.shape[2], d, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                      _strides(q), _strides(k), _strides(v), *mask,
                      0 if lengths is None else lengths.element_size(), _ptr(lengths), scale, 0, out.data_ptr(), _ptr(stats), _ptr(key_list))


def _workspace(L, a, backward, like):
    a.workspace_bytes = L.pct_attend_workspace(ctypes.addressof(a), backward)
    if not a.workspace_bytes:
        return None
    ws = like.new_empty(a.workspace_bytes, dtype=torch.uint8)
    a.workspace = ws.data_ptr()
    return ws


def _attend_forward(q, k, v, mask, lengths, scale, want_stats):
    b, lq, h, d = q.shape
    dev, hk = q.device, k.shape[2]
    out = q.new_empty((b, lq, h, d))
    stats = q.new_empty(b * lq * h * 2, dtype=torch.float32) if want_stats else None
    key_list = q.new_empty((b, k.shape[1] + 1), dtype=torch.int32) if mask is not None else None
    if b and lq:
        L = _library()
        a = _attention_struct(q, k, v, _mask_fields(mask), lengths, scale, out, stats, key_list)
        ws = _workspace(L, a, 0, q)  # noqa: F841  (held until the call has been enqueued)
        _call(L.pct_attend, a, dev)
    return out, stats, key_list


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, lengths, scale):
        q, k, v = _attention_rows(q), _attention_rows(k), _attention_rows(v)
        out, stats, key_list = _attend_forward(q, k, v, mask, lengths, scale, True)
        # (the backward reads the list the forward made of the mask and the lengths, or the lengths alone, never the mask)
        ctx.save_for_backward(q, k, v, None if key_list is not None else lengths, out, stats, key_list)
        ctx.scale = scale
        return out

    @staticmethod
    @_once_differentiable
    def backward(ctx, d_out):
        q, k, v, lengths, out, stats, key_list = ctx.saved_tensors
        q, k, v, d_out = _attention_rows(q), _attention_rows(k), _attention_rows(v), _attention_rows(d_out)
        lengths, out, stats, key_list = _whole(lengths), _whole(out), _whole(stats), _whole(key_list)
        dev = q.device
        d_q, d_k, d_v = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        if q.shape[0]:
            L = _library()
            a = _attention_struct(q, k, v, (_ptr(key_list), 0, 0, 4), lengths, ctx.scale, out, stats, key_list)
            a.d_out, a.d_out_stride = d_out.data_ptr(), _strides(d_out)
            a.d_q, a.d_k, a.d_v = d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr()
            ws = _workspace(L, a, 1, q)  # noqa: F841
            _call(L.pct_attend_backward, a, dev)
        return d_q, d_k, d_v, None, None, None


def cross_attention(q, k, v, key_mask=None, key_lengths=None, scale=None):
    """softmax(scale q k^T) v over the allowed keys of each batch: q [B, Lq, H, D], k and v [B, Lk, Hk, D], one of float32,
    bfloat16 and float16; H a multiple of Hk (H / Hk heads in a row share a key/value head), D a multiple of 8 up to 128; any
    lengths.  Returns [B, Lq, H, D] (contiguous), differentiable with respect to q, k and v (once, backward).

    Key j of batch b is allowed where `key_mask` [B, Lk] (any strides: the observation's mask column will do) is not zero and
    j < `key_lengths`[b] (int32 or int64 [B]; values outside of [0, Lk] count as the nearer end).  What stands in keys and
    values that are not allowed does not matter, NaN included.  A batch that allows no key gives zeros and takes no gradient.
    Lk, and Lq * H / Hk, are below 2^29, and a call is refused whose launch would hold more than 2^32 threads (some 2^26
    heads times groups of 32 rows).  The mask and the lengths may be written over once the call has returned, in its stream's
    order: the backward pass reads what was made of them.
    Scores, sums and statistics are float32; in 16-bit types the weights and the scores' gradients are rounded to the type before they
    are multiplied with v, k, q and the output's gradient, as the results are.
    `scale` is positive, 1 / sqrt(D) if not given.  q, k, v and the output's gradient are read where they are if their rows
    are contiguous and start on 16 bytes, else from a copy."""
    name = "cross_attention"
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("%s: q must be [B, Lq, H, D], k and v [B, Lk, Hk, D]; got %s, %s, %s" % (name, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    if k.shape[0] != b or k.shape[3] != d or h < 1 or hk < 1 or h % hk:
        raise ValueError("%s: q %s does not go with k %s (H must be a multiple of Hk)" % (name, tuple(q.shape), tuple(k.shape)))
    if q.dtype not in _DTYPE or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("%s: q, k and v must share one of float32, bfloat16, float16; got %s, %s, %s" % (name, q.dtype, k.dtype, v.dtype))
    if d % 8 or not 8 <= d <= 128:
        raise ValueError("%s: D must be a multiple of 8 up to 128, not %d" % (name, d))
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError("%s: scale must be positive and finite" % name)
    if key_lengths is not None:
        if key_lengths.dtype not in (torch.int32, torch.int64) or key_lengths.shape != (b,):
            raise ValueError("%s: key_lengths must be int32 or int64 [B]" % name)
        key_lengths = key_lengths.contiguous()
    mask = _mask_of(name, key_mask, torch.Size((b, lk)))
    _on_gpu(name, q, k, v, key_mask, key_lengths)
    _no_tangents(name, q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if key_lengths is not None and mask is None:
            key_lengths = key_lengths.clone()  # (the backward reads them again)
        return _CrossAttention.apply(q, k, v, mask, key_lengths, scale)
    return _attend_forward(_attention_rows(q), _attention_rows(k), _attention_rows(v), mask, key_lengths, scale, False)[0]
