"""Attention over ordered series: the moving window and the moving average with weights that come from
the data (device tensors in, device tensors out, as the rest of `tempo_amd.ops`, which exports these).

`ops.ema` and `ops.lookback` weigh or list the rows before a row by their distance alone.  The two
operators here weigh them by how well their keys fit the row's query:

* `decay_attention`: S_i = exp(log_decay) S_{i-1} + k_i v_i^T, out_i = scale S_i^T q_i, a moving average of
  k v^T for each head (with q = k = 1 it is the untruncated `ema` divided by exp_factor);
* `window_attention`: softmax attention over a row's last `window` rows (itself included) and the first
  `sinks` rows of its series.

Rows are in (key, ts) order, one series after the other (`ops.sort_order`), and `offsets` -- int64 on the
device, `series_offsets(key, n_keys)` -- says where each series starts; rows before the first or behind the last
offset belong to no series and get zeros.  q, k and v are [rows, heads, dim] in bfloat16 or float32 with a
contiguous innermost dimension and any other strides (slices of one projection's output need no copy).  Both
are differentiable in q, k and v (decay_attention in `state` too); `*_grad` are the backward passes by
themselves, for programs that do not use autograd or capture a training step into a graph; forward-mode
differentiation is refused.  `*_step` add one row to each of some slots of kept state.  Calls do not wait for the device.
"""
import contextlib
import ctypes as C

import torch
from torch.autograd import forward_ad

from ._lib import (CacheRef, DecayAttentionArgs, DecayAttentionStepArgs, RowsRef, WindowAttentionArgs,
                   WindowAttentionStepArgs, WindowCacheWriteArgs, check, lib)

_TYPES = {torch.bfloat16: 0, torch.float32: 1}
_MOST = 2 ** 31 - 65536  # series: the library is told their number in 32 bits, and compares with others beside it


def _on_device(t, name, device=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA (ROCm) tensor; tempo_amd has no CPU path")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _rows_check(t, name, like=None, n=None, heads=None, dim=None):
    """[rows, heads, dim], innermost dimension contiguous; type and device of `like`.  Returns the rows to hand on: a copy
    where they overlap in memory (a broadcast row) or lie 2^22 elements or more apart."""
    if isinstance(t, torch.Tensor) and t.dim() == 3 and t.is_cuda and t.dtype in _TYPES:
        # the usual case, asked for at once: small calls are bound by their host part
        (rows, h, d), (row, _, last) = t.shape, t.stride()
        if last == 1 and 0 < h <= 65536 and 0 < d <= 128 and (rows <= 1 or d <= row < 2 ** 22):
            if like is None:
                return t
            if rows == n and heads in (None, h) and dim in (None, d) and t.dtype is like.dtype and t.device == like.device:
                return t
    _on_device(t, name, None if like is None else like.device)
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be bfloat16 or float32, got {t.dtype}")
    if like is not None and t.dtype != like.dtype:
        raise TypeError(f"{name} must have dtype {like.dtype}, got {t.dtype}")
    if t.dim() != 3:
        raise ValueError(f"{name} must be [rows, heads, dim], got {t.dim()} dimensions")
    for what, have, want in (("rows", t.shape[0], n), ("heads", t.shape[1], heads), ("elements a head", t.shape[2], dim)):
        if want is not None and have != want:
            raise ValueError(f"{name} has {have} {what}, expected {want}")
    if t.shape[1] < 1 or t.shape[2] < 1:
        raise ValueError(f"{name} needs at least one head and one element")
    if t.shape[1] > 65536 or t.shape[2] > 128:  # (asked here too: the library is told them in 32 bits)
        raise NotImplementedError(f"{name} has {t.shape[1]} heads of {t.shape[2]} elements, limited to 65536 of 128")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name} must be contiguous in its innermost dimension")
    return t if t.shape[0] <= 1 or t.shape[2] <= t.stride(0) < 2 ** 22 else t.contiguous()


def _plain_check(t, name, dtype, shape, device):
    _on_device(t, name, device)
    if t.dtype != dtype:
        raise TypeError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _offsets_check(offsets, device):
    if offsets is None:
        return 1
    _on_device(offsets, "offsets", device)
    if offsets.dtype != torch.int64 or offsets.dim() != 1 or not offsets.is_contiguous() or offsets.numel() < 1:
        raise ValueError("offsets must be a contiguous int64 vector of at least one element")
    if offsets.numel() > _MOST:
        raise ValueError(f"offsets of {offsets.numel() - 1} series, at most {_MOST - 1}")
    return offsets.numel() - 1


def _scale(scale, dim):
    return float(dim) ** -0.5 if scale is None else float(scale)


def _ref(t):
    row, head, _ = t.stride()
    return RowsRef(t.data_ptr(), row, head)


def _p(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _current(device):
    """The device's context, entered only where it is not the current one already."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _workspace(nbytes, device):
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def _no_tangent(*tensors):
    """Forward-mode differentiation: the kernels would drop the tangents without a word."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("attention over series has no forward-mode derivative")


def _changed(*tensors):
    """Tells autograd that a call writes them: a backward pass that saved one of them raises instead of reading what is
    there by then."""
    torch.autograd.graph.increment_version(tensors)


def _int_arg(value, name, low, most):
    """An integer >= low; what is above `most` is handed on as that."""
    if isinstance(value, bool) or int(value) != value or value < low:
        raise ValueError(f"{name} must be an integer >= {low}")
    return min(int(value), most)


def series_offsets(key, n_keys):
    """Where each series of a table in (key, ts) order starts: int64 [n_keys + 1] on the device, from the
    key column (int32, ids in [0, n_keys))."""
    from . import ops
    with _current(_on_device(key, "key").device):
        counts = ops.key_counts(key, n_keys)
        offsets = torch.zeros(n_keys + 1, dtype=torch.int64, device=counts.device)
        torch.cumsum(counts, 0, out=offsets[1:])
    return offsets


# ---- linear attention with a decay for each head -------------------------------------------------

def _decay_args(q, k, v, log_decay, offsets, scale, state):
    q = _rows_check(q, "q")
    n, heads, dk = q.shape
    k = _rows_check(k, "k", q, n, heads, dk)
    v = _rows_check(v, "v", q, n, heads)
    dv = v.shape[2]
    _plain_check(log_decay, "log_decay", torch.float32, (heads,), q.device)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("log_decay has no gradient: detach it")
    n_series = _offsets_check(offsets, q.device)
    if state is not None:
        _plain_check(state, "state", torch.float32, (n_series, heads, dk, dv), q.device)
    a = DecayAttentionArgs(n=n, n_series=n_series, offsets=_p(offsets), type=_TYPES[q.dtype], heads=heads, dim_k=dk,
                           dim_v=dv, scale=_scale(scale, dk), log_decay=log_decay.data_ptr(), q=_ref(q), k=_ref(k),
                           v=_ref(v), state_in=_p(state))
    a.held = (q, k, v)  # (copies live as long as the pointers to them)
    return a, n_series


def _decay_call(fn, a, device):
    with _current(device):
        ws = _workspace(lib().tmp_decay_attention_workspace_bytes(C.byref(a)), device)
        check(getattr(lib(), fn)(C.byref(a), ws.data_ptr(), ws.numel(), _stream(device)), fn)


def _decay_forward(q, k, v, log_decay, offsets, scale, state, return_state):
    a, n_series = _decay_args(q, k, v, log_decay, offsets, scale, state)
    out = q.new_empty((q.shape[0], q.shape[1], v.shape[2]))
    last = None
    if return_state:
        last = torch.empty((n_series, q.shape[1], q.shape[2], v.shape[2]), dtype=torch.float32, device=q.device)
    a.out, a.state_out = _ref(out), _p(last)
    _decay_call("tmp_decay_attention", a, q.device)
    return out, last


def decay_attention_grad(dout, q, k, v, log_decay, offsets=None, scale=None, state=None, dstate=None, return_dstate=False):
    """Backward of `decay_attention`: (dq, dk, dv), and with return_dstate the gradient of `state` behind them.
    dout: gradient of out; dstate: gradient of the returned state, if that was used."""
    _no_tangent(dout, q, k, v, log_decay, state, dstate)
    a, n_series = _decay_args(q, k, v, log_decay, offsets, scale, state)
    n, heads, dk = q.shape
    dv = v.shape[2]
    dout = _rows_check(dout, "dout", q, n, heads, dv)
    if dstate is not None:
        _plain_check(dstate, "dstate", torch.float32, (n_series, heads, dk, dv), q.device)
    gq, gk = (torch.empty((n, heads, dk), dtype=q.dtype, device=q.device) for _ in range(2))
    gv = torch.empty((n, heads, dv), dtype=q.dtype, device=q.device)
    gs = torch.empty((n_series, heads, dk, dv), dtype=torch.float32, device=q.device) if return_dstate else None
    a.dout, a.dq, a.dk, a.dv = _ref(dout), _ref(gq), _ref(gk), _ref(gv)
    a.dstate_out, a.dstate_in = _p(dstate), _p(gs)
    _decay_call("tmp_decay_attention_grad", a, q.device)
    return (gq, gk, gv, gs) if return_dstate else (gq, gk, gv)


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, offsets, scale, state, return_state):
        out, last = _decay_forward(q, k, v, log_decay, offsets, scale, state, return_state)
        ctx.save_for_backward(q, k, v, log_decay, offsets, state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, last) if return_state else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dstate=None):
        q, k, v, log_decay, offsets, state = ctx.saved_tensors
        if dout is None:
            dout = torch.zeros((q.shape[0], q.shape[1], v.shape[2]), dtype=q.dtype, device=q.device)
        want = ctx.needs_input_grad[6]
        grads = decay_attention_grad(dout.contiguous(), q, k, v, log_decay, offsets, ctx.scale, state,
                                     None if dstate is None else dstate.contiguous(), want)
        return grads[0], grads[1], grads[2], None, None, None, grads[3] if want else None, None


def decay_attention(q, k, v, log_decay, offsets=None, scale=None, state=None, return_state=False):
    """Linear attention with a decay for each head over whole series (beside `ops.ema`).

    q, k [n, heads, dk], v [n, heads, dv]; log_decay float32 [heads], <= 0 (-inf: a row sees itself alone), without a
    gradient: detached, or under no_grad;
    scale defaults to dk ** -0.5 and must be positive.  state float32 [n_series, heads, dk, dv]: what the
    rows before this call left (None: nothing); return_state hands back the same for the call that goes on, or
    for `decay_attention_step`.  Returns out [n, heads, dv], or (out, state)."""
    _no_tangent(q, k, v, log_decay, state)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v, state, log_decay)):
        if isinstance(log_decay, torch.Tensor) and log_decay.requires_grad:  # (asked here: within forward() gradients are off)
            raise ValueError("log_decay has no gradient: detach it")
        return _DecayAttention.apply(q, k, v, log_decay, offsets, scale, state, bool(return_state))
    out, last = _decay_forward(q, k, v, log_decay, offsets, scale, state, return_state)
    return (out, last) if return_state else out


def _slots_check(slots, n, n_slots, device):
    if n_slots >= 2 ** 31:
        raise ValueError(f"{n_slots} slots, at most {2 ** 31 - 1}: the library is told their number in 32 bits")
    if slots is None:
        if n != n_slots:
            raise ValueError(f"{n} rows for {n_slots} slots: slots must say which")
        return
    _plain_check(slots, "slots", torch.int32, (n,), device)


def _no_grad(*tensors):
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("an argument requires a gradient; a step has none (use the form over whole series)")


def decay_attention_step(q, k, v, log_decay, state, slots=None, scale=None):
    """One new row for each of some series: q, k [b, heads, dk], v [b, heads, dv]; state float32 [n_slots, heads,
    dk, dv], changed in place; slots int32 [b] (None: row i is slot i).  A row whose slot is out of range or named
    by an earlier row changes nothing and results in NaN; with slots b is at most 65536.  Returns out [b, heads, dv]."""
    _no_tangent(q, k, v, log_decay, state)
    q = _rows_check(q, "q")
    n, heads, dk = q.shape
    k = _rows_check(k, "k", q, n, heads, dk)
    v = _rows_check(v, "v", q, n, heads)
    dv = v.shape[2]
    _plain_check(log_decay, "log_decay", torch.float32, (heads,), q.device)
    _on_device(state, "state", q.device)
    if state.dim() != 4:
        raise ValueError("state must be [n_slots, heads, dk, dv]")
    _plain_check(state, "state", torch.float32, (state.shape[0], heads, dk, dv), q.device)
    _slots_check(slots, n, state.shape[0], q.device)
    _no_grad(q, k, v, state, log_decay)
    out = q.new_empty((n, heads, dv))
    a = DecayAttentionStepArgs(n=n, n_slots=state.shape[0], slots=_p(slots), type=_TYPES[q.dtype], heads=heads, dim_k=dk,
                               dim_v=dv, scale=_scale(scale, dk), log_decay=log_decay.data_ptr(), q=_ref(q), k=_ref(k),
                               v=_ref(v), out=_ref(out), state=state.data_ptr())
    _changed(state)
    with _current(q.device):
        check(lib().tmp_decay_attention_step(C.byref(a), _stream(q.device)), "tmp_decay_attention_step")
    return out


# ---- attention over a sliding window -------------------------------------------------------------

def _window_args(q, k, v, window, sinks, offsets, scale):
    q = _rows_check(q, "q")
    n, heads, dk = q.shape
    k = _rows_check(k, "k", q, n, None, dk)
    kv = k.shape[1]
    v = _rows_check(v, "v", q, n, kv)
    if heads % kv:
        raise ValueError(f"{heads} query heads cannot share {kv} key/value heads")
    n_series = _offsets_check(offsets, q.device)
    a = WindowAttentionArgs(n=n, n_series=n_series, offsets=_p(offsets), type=_TYPES[q.dtype], heads=heads, kv_heads=kv,
                            dim_k=dk, dim_v=v.shape[2], window=_int_arg(window, "window", 1, 2 ** 62),
                            sinks=_int_arg(sinks, "sinks", 0, 2 ** 31 - 1), scale=_scale(scale, dk), q=_ref(q), k=_ref(k), v=_ref(v))
    a.held = (q, k, v)
    return a


def _window_forward(q, k, v, window, sinks, offsets, scale, return_lse):
    a = _window_args(q, k, v, window, sinks, offsets, scale)
    out = q.new_empty((q.shape[0], q.shape[1], v.shape[2]))
    lse = torch.empty((q.shape[0], q.shape[1]), dtype=torch.float32, device=q.device) if return_lse else None
    a.out, a.lse = _ref(out), _p(lse)
    with _current(q.device):
        check(lib().tmp_window_attention(C.byref(a), _stream(q.device)), "tmp_window_attention")
    return out, lse


def window_attention_grad(dout, q, k, v, out, lse, window, sinks=0, offsets=None, scale=None):
    """Backward of `window_attention`: (dq, dk, dv) from dout and what the forward returned (out, lse)."""
    _no_tangent(dout, q, k, v, out, lse)
    a = _window_args(q, k, v, window, sinks, offsets, scale)
    n, heads, dv = q.shape[0], q.shape[1], v.shape[2]
    dout = _rows_check(dout, "dout", q, n, heads, dv)
    out = _rows_check(out, "out", q, n, heads, dv)
    _plain_check(lse, "lse", torch.float32, (n, heads), q.device)
    gq, gk, gv = (torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v))
    a.out, a.lse, a.dout, a.dq, a.dk, a.dv = _ref(out), lse.data_ptr(), _ref(dout), _ref(gq), _ref(gk), _ref(gv)
    with _current(q.device):
        ws = _workspace(lib().tmp_window_attention_grad_workspace_bytes(C.byref(a)), q.device)
        check(lib().tmp_window_attention_grad(C.byref(a), ws.data_ptr(), ws.numel(), _stream(q.device)),
              "tmp_window_attention_grad")
    return gq, gk, gv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, offsets, scale):
        out, lse = _window_forward(q, k, v, window, sinks, offsets, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, offsets)
        ctx.how = (window, sinks, scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, out, lse, offsets = ctx.saved_tensors
        window, sinks, scale = ctx.how
        return window_attention_grad(dout.contiguous(), q, k, v, out, lse, window, sinks, offsets, scale) + (None,) * 4


def window_attention(q, k, v, window, sinks=0, offsets=None, scale=None, return_lse=False):
    """Softmax attention over a sliding window of each series (beside `ops.lookback`).

    q [n, heads, dk], k [n, kv_heads, dk], v [n, kv_heads, dv]; consecutive query heads share a key/value head.  Row
    i sees rows j <= i of its series with j > i - window, and the series' first `sinks` rows.  scale defaults to
    dk ** -0.5 and must be positive.  Returns out [n, heads, dv], with return_lse also the log of the sum of
    exponentials of each row's scores, float32 [n, heads] (-inf for rows of no series; no gradient)."""
    _no_tangent(q, k, v)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v)):
        out, lse = _WindowAttention.apply(q, k, v, window, sinks, offsets, scale)
    else:
        out, lse = _window_forward(q, k, v, window, sinks, offsets, scale, return_lse)
    return (out, lse) if return_lse else out


def _caches_check(k_cache, v_cache, length, sinks, like, kv_heads, dk, dv):
    """(n_slots, window, sinks) of a pair of caches [n_slots, window + sinks, kv_heads, dim]."""
    for t, name, dim in ((k_cache, "k_cache", dk), (v_cache, "v_cache", dv)):
        _on_device(t, name, like.device)
        if t.dtype != like.dtype:
            raise TypeError(f"{name} must have dtype {like.dtype}, got {t.dtype}")
        if t.dim() != 4 or t.shape[2:] != (kv_heads, dim):
            raise ValueError(f"{name} must be [n_slots, window + sinks, {kv_heads}, {dim}], got {tuple(t.shape)}")
        if dim > 1 and t.stride(3) != 1:
            raise ValueError(f"{name} must be contiguous in its innermost dimension")
        if 0 in t.stride() and any(t.shape[i] > 1 and t.stride(i) == 0 for i in range(3)):
            raise ValueError(f"{name} must not repeat its rows (expanded tensor)")
    if k_cache.shape[:2] != v_cache.shape[:2]:
        raise ValueError("k_cache and v_cache must have the same slots and rows")
    sinks = _int_arg(sinks, "sinks", 0, 2 ** 31 - 1)
    window = k_cache.shape[1] - sinks
    if window >= 2 ** 30:
        raise ValueError(f"a cache of {k_cache.shape[1]} rows: its window must be below 2^30")
    if window < 1:
        raise ValueError(f"a cache of {k_cache.shape[1]} rows has no window behind {sinks} sinks")
    _plain_check(length, "length", torch.int64, (k_cache.shape[0],), like.device)
    return k_cache.shape[0], window, sinks


def _cache_ref(t):
    return CacheRef(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def window_cache_write(k, v, k_cache, v_cache, length, sinks=0, offsets=None, slots=None):
    """Fills cache slots from whole series: after `window_attention` over k, v [n, kv_heads, dim], slot slots[s] (None:
    s) holds what `window_attention_step` needs of series s, in place of what it held.  k_cache, v_cache [n_slots,
    window + sinks, kv_heads, dim]; length int64 [n_slots]: rows seen by each slot."""
    _no_tangent(k, v, k_cache, v_cache)
    k = _rows_check(k, "k")
    n, kv, dk = k.shape
    v = _rows_check(v, "v", k, n, kv)
    dv = v.shape[2]
    n_series = _offsets_check(offsets, k.device)
    n_slots, window, sinks = _caches_check(k_cache, v_cache, length, sinks, k, kv, dk, dv)
    _slots_check(slots, n_series, n_slots, k.device)
    _no_grad(k_cache, v_cache)
    a = WindowCacheWriteArgs(n=n, n_series=n_series, offsets=_p(offsets), n_slots=n_slots, slots=_p(slots),
                             type=_TYPES[k.dtype], kv_heads=kv, dim_k=dk, dim_v=dv, window=window, sinks=sinks, k=_ref(k),
                             v=_ref(v), k_cache=_cache_ref(k_cache), v_cache=_cache_ref(v_cache), length=length.data_ptr())
    _changed(k_cache, v_cache, length)
    with _current(k.device):
        check(lib().tmp_window_cache_write(C.byref(a), _stream(k.device)), "tmp_window_cache_write")


def window_attention_step(q, k, v, k_cache, v_cache, length, sinks=0, slots=None, scale=None):
    """One new row for each of some series: adds k, v [b, kv_heads, dim] to the caches (in place, length counts
    it) and attends with q [b, heads, dk] over the slot's last `window` rows, the new one included, and its first
    `sinks`.  The caches' number of rows is window + sinks.  slots int32 [b] (None: row i is slot i); a row whose slot is
    out of range or named by an earlier row changes nothing and results in NaN; with slots b is at most 65536.  Returns
    out [b, heads, dv]."""
    _no_tangent(q, k, v, k_cache, v_cache)
    q = _rows_check(q, "q")
    n, heads, dk = q.shape
    k = _rows_check(k, "k", q, n, None, dk)
    kv = k.shape[1]
    v = _rows_check(v, "v", q, n, kv)
    dv = v.shape[2]
    if heads % kv:
        raise ValueError(f"{heads} query heads cannot share {kv} key/value heads")
    n_slots, window, sinks = _caches_check(k_cache, v_cache, length, sinks, q, kv, dk, dv)
    _slots_check(slots, n, n_slots, q.device)
    _no_grad(q, k, v, k_cache, v_cache)
    out = q.new_empty((n, heads, dv))
    a = WindowAttentionStepArgs(n=n, n_slots=n_slots, slots=_p(slots), type=_TYPES[q.dtype], heads=heads, kv_heads=kv,
                                dim_k=dk, dim_v=dv, window=window, sinks=sinks, scale=_scale(scale, dk), q=_ref(q), k=_ref(k),
                                v=_ref(v), out=_ref(out), k_cache=_cache_ref(k_cache), v_cache=_cache_ref(v_cache),
                                length=length.data_ptr())
    _changed(k_cache, v_cache, length)
    with _current(q.device):
        ws = _workspace(lib().tmp_window_attention_step_workspace_bytes(C.byref(a)), q.device)
        check(lib().tmp_window_attention_step(C.byref(a), ws.data_ptr(), ws.numel(), _stream(q.device)),
              "tmp_window_attention_step")
    return out
