"""Causal linear attention with a decay for each head, beside the exact attention of flash_attn_interface: the same
tensor layouts (batch, seqlen, nheads, headdim) or packed (total, nheads, headdim), shared K/V heads, dtypes and errors.

A head of queries holds a state S of headdim x headdim_v values. With l = exp(-decay[head]),
    S_t = l S_{t-1} + k_t v_t^T,     o_t = scale q_t^T S_t = scale sum_{s<=t} l^(t-s) (q_t . k_s) v_s.

    linear_attn_func         dense batches, with gradients; states in and out
    linear_attn_varlen_func  packed batches, with gradients; states in and out
    linear_attn_with_state   serving: the states of a pool updated in place, one new token or many per sequence

States and sums are kept in fp32. Head dims up to 256 each (values may be wider or narrower than keys; one that is no multiple of 8
is zero-padded). decay is (nheads) or (batch, nheads), as the slopes that flash_attn_func takes for its biases:
at least 0, 0 for no decay, infinity for a head that sees only the token itself; like those it gets no gradient.
What is no number (or infinite) in a row of k or v makes the outputs of its heads so (in v: of its column) from that row on, in a row
of q that row's only; rows before it and other sequences keep their bits.
Tensors that carry a tangent (forward-mode differentiation) are refused.
All calls capture into HIP graphs; a captured backward pass wants leaves that no eager graph still holds, because torch's own
accumulation would run on that graph's stream.
"""
import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _C, _lib
from .flash_attn_interface import (MAX_HEAD_DIM, _DTYPES, _aligned, _as_index, _kernel_width, _no_tangents, _place, _plans, _remember, _sig,
                                   _with_width)

# Rows per sequence up to which linear_attn_with_state goes token by token: a step takes 1 us a row and more, a pass by chunks 18 us or the
# states' bytes. bf16, heads of 128, steps / chunks: one sequence x 32 heads, 16 rows 15 / 18 us, 24 rows 20 / 18; 8 x 16, 16 rows 17 / 18,
# 24 rows 24 / 18; 48 x 16 heads of 64, 12 rows 19 / 18. Many states are through earlier by chunks: 48 x 64, 4 rows 82 / 78, 8 rows 106 / 78.
STEP_ROWS = 16


def _rows(t):
    """t itself where the kernels can read it in place, else a copy: aligned rows that do not overlap (an expanded sequence)."""
    return _aligned(t) if t.shape[-3] <= 1 or t.stride(-3) >= t.shape[-1] else t.clone(memory_format=torch.contiguous_format)


def _check(q, k, v, decay, packed, scale):
    """What every call has to satisfy; (decay in fp32, scale)."""
    if not q.is_cuda:
        raise ValueError("fable_attn: tensors must be on the GPU (q.is_cuda == False)")
    if q.dtype not in _DTYPES:
        raise ValueError(f"fable_attn: dtype {q.dtype} is not supported; use fp16, bf16 or fp32")
    dims = 3 if packed else 4
    if q.dim() != dims or k.dim() != dims or v.dim() != dims:
        raise ValueError(f"fable_attn: q, k, v must be (batch, seqlen, nheads, headdim), or (total, nheads, headdim) with "
                         f"cu_seqlens; got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if q.shape[-2] == 0 or k.shape[-2] == 0 or q.shape[-2] % k.shape[-2]:
        raise ValueError(f"fable_attn: nheads_q={q.shape[-2]} is not a multiple of nheads_k={k.shape[-2]} (GQA)")
    if k.shape[-1] != q.shape[-1]:
        raise ValueError(f"fable_attn: q and k must share a head_dim, got {q.shape[-1]} and {k.shape[-1]}")
    if max(q.shape[-1], v.shape[-1]) > MAX_HEAD_DIM or min(q.shape[-1], v.shape[-1]) < 1:
        raise ValueError(f"fable_attn: head_dim={q.shape[-1]} and {v.shape[-1]}: 1 to {MAX_HEAD_DIM}")
    if not torch.is_tensor(decay):
        raise TypeError(f"fable_attn: decay must be a tensor (nheads) or (batch, nheads), got {type(decay)}")
    if decay.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("fable_attn: decay gets no gradient; pass decay.detach()")
    if decay.dtype != torch.float32 or decay.requires_grad or not decay.is_contiguous():
        decay = decay.detach().to(torch.float32).contiguous()
    return decay, float(q.shape[-1] ** -0.5 if scale is None else scale)


def _forward(q, k, v, decay, scale, cu, most, state, final, idx=None):
    """_C.linear_fwd; the parameters that the first call of a signature came to are kept per thread, and later ones fill in
    addresses."""
    key = (_place(q), _place(k), _place(v), _sig(decay), scale, _sig(cu), most, _sig(state), _sig(final), _sig(idx))
    plans = _plans("linear_plans")
    plan = plans.get(key)
    qp, kp, vp, sp, dev = q.data_ptr(), k.data_ptr(), v.data_ptr(), state.data_ptr() if state is not None else 0, q.get_device()
    if plan is None or (qp | kp | vp | sp) & 15 or dev != torch._C._cuda_getDevice():
        out, ws, p, dt, need = _C.linear_fwd(q, k, v, decay, scale, cu, most, state, final, idx)
        if p.batch:
            _remember(plans, key, (p, dt, need, out.shape, out.stride()))
        return out, ws
    p, dt, need, shape, strides = plan
    out = torch.empty_strided(shape, strides, dtype=q.dtype, device=q.device)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    p.q, p.k, p.v, p.o, p.decay = qp, kp, vp, out.data_ptr(), decay.data_ptr()
    p.state_in, p.state_out = sp or None, final.data_ptr() if final is not None else None
    if cu is not None:
        p.cu = cu.data_ptr()
    if idx is not None:
        p.slots = idx.data_ptr()
    _lib.check(_C._L.fable_linear_attn_fwd(p, dt, ws.data_ptr() if need else None, need, torch._C._cuda_getCurrentRawStream(dev)),
               "fable_linear_attn_fwd")
    return out, ws


def _backward(dout, q, k, v, decay, scale, cu, most, state, dfinal, want, seg):
    """_C.linear_bwd, planned as _forward."""
    key = (_place(dout), _place(q), _place(k), _place(v), _sig(decay), scale, _sig(cu), most, _sig(state), _sig(dfinal), want, seg is None)
    plans = _plans("linear_bwd_plans")
    plan = plans.get(key)
    dp, qp, kp, vp, dev = dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), q.get_device()
    if plan is None or (dp | qp | kp | vp) & 15 or dev != torch._C._cuda_getDevice():
        dq, dk, dv, dstate, p, dt, need = _C.linear_bwd(dout, q, k, v, decay, scale, cu, most, state, dfinal, want, seg)
        if p.batch:
            _remember(plans, key, (p, dt, need, dq.stride(), dk.stride(), dv.stride()))
        return dq, dk, dv, dstate
    p, dt, need, qs, ks, vs = plan
    device = q.device
    dq = torch.empty_strided(q.shape, qs, dtype=q.dtype, device=device)
    dk = torch.empty_strided(k.shape, ks, dtype=q.dtype, device=device)
    dv = torch.empty_strided(v.shape, vs, dtype=q.dtype, device=device)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    dstate = torch.empty((p.batch, p.NH, p.DK, p.DV), dtype=torch.float32, device=device) if want else None
    ptr = lambda t: t.data_ptr() if t is not None else None
    p.dout, p.q, p.k, p.v, p.dq, p.dk, p.dv, p.decay = dp, qp, kp, vp, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), decay.data_ptr()
    p.state_in, p.dstate_out, p.dstate_in, p.seg_states, p.cu = ptr(state), ptr(dfinal), ptr(dstate), ptr(seg), ptr(cu)
    _lib.check(_C._L.fable_linear_attn_bwd(p, dt, ptr(ws), need, torch._C._cuda_getCurrentRawStream(dev)), "fable_linear_attn_bwd")
    return dq, dk, dv, dstate


class _LinearAttention(torch.autograd.Function):
    """Forward and backward of one dense (pack None) or packed (pack = (cu_seqlens, max_seqlen)) batch."""

    @staticmethod
    def forward(ctx, pack, scale, want, q, k, v, decay, state):
        cu, most = pack if pack is not None else (None, 0)
        batch = cu.numel() - 1 if cu is not None else q.shape[0]
        final = torch.empty((batch, q.shape[-2], q.shape[-1], v.shape[-1]), dtype=torch.float32, device=q.device) if want else None
        out, seg = _forward(q, k, v, decay, scale, cu, most, state, final)
        ctx.scale, ctx.most = scale, most
        ctx.save_for_backward(q, k, v, decay, state, cu, seg)
        ctx.set_materialize_grads(False)
        return (out, final) if want else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal=None):
        q, k, v, decay, state, cu, seg = ctx.saved_tensors
        if dout is None and dfinal is None:
            return None, None, None, None, None, None, None, None
        dout = q.new_zeros((*q.shape[:-1], v.shape[-1])) if dout is None else _rows(dout)
        dq, dk, dv, dstate = _backward(dout, q, k, v, decay, ctx.scale, cu, ctx.most, state,
                                       _aligned(dfinal, dense=True) if dfinal is not None else None, ctx.needs_input_grad[7], seg)
        return None, None, None, dq, dk, dv, None, dstate


def _attend(pack, q, k, v, decay, scale, state, want):
    if fwAD._current_level >= 0:
        _no_tangents(q, k, v, decay, state)
    batch = pack[0].numel() - 1 if pack is not None else q.shape[0]
    decay, scale = _check(q, k, v, decay, pack is not None, scale)
    dk, dv = q.shape[-1], v.shape[-1]
    if state is not None:
        if tuple(state.shape) != (batch, q.shape[-2], dk, dv) or state.dtype != torch.float32 or state.device != q.device:
            raise ValueError(f"fable_attn: initial_state must be float32 {(batch, q.shape[-2], dk, dv)} on q's device, got "
                             f"{state.dtype} {tuple(state.shape)}")
    wk, wv = _kernel_width(dk, q.dtype), _kernel_width(dv, q.dtype)
    padded = wk != dk or wv != dv
    if state is not None:
        state = _aligned(torch.nn.functional.pad(state, (0, wv - dv, 0, wk - dk)) if padded else state, dense=True)
    q, k, v = _rows(_with_width(q, wk)), _rows(_with_width(k, wk)), _rows(_with_width(v, wv))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)):
        res = _LinearAttention.apply(pack, scale, want, q, k, v, decay, state)
        out, final = res if want else (res, None)
    else:
        cu, most = pack if pack is not None else (None, 0)
        final = torch.empty((batch, q.shape[-2], wk, wv), dtype=torch.float32, device=q.device) if want else None
        out, _ = _forward(q, k, v, decay, scale, cu, most, state, final)
    if wv != dv:
        out = out[..., :dv].contiguous()
    if not want:
        return out
    return out, (final[..., :dk, :dv].contiguous() if padded else final)


def linear_attn_func(q, k, v, decay, scale=None, initial_state=None, return_final_state=False):
    """Linear attention of q (batch, seqlen, nheads, d), k (batch, seqlen, nheads_k, d) and v (batch, seqlen, nheads_k, dv),
    causal, with a decay per head of q. scale: d^-0.5 by default. initial_state: float32 (batch, nheads, d, dv), the state before the first
    token (zeros by default). Returns out (batch, seqlen, nheads, dv), or (out, final_state) with the state
    behind the last token, from which the next call goes on. Gradients flow to q, k, v and initial_state, also through
    final_state; results are reproducible bit for bit."""
    return _attend(None, q, k, v, decay, scale, initial_state, return_final_state)


def linear_attn_varlen_func(q, k, v, cu_seqlens, max_seqlen, decay, scale=None, initial_state=None, return_final_state=False):
    """linear_attn_func of packed sequences: q (total, nheads, d), k and v (total, nheads_k, ...), cu_seqlens int32 (batch+1);
    states are (batch, nheads, d, dv). max_seqlen sizes the launch (a longer sequence is served, more
    slowly). Sequences may be empty: their state passes through. Rows of no sequence come back as zeros, as do their gradients."""
    cu = cu_seqlens if cu_seqlens.dtype == torch.int32 and cu_seqlens.device == q.device and cu_seqlens.is_contiguous() else _as_index(cu_seqlens, q.device)
    return _attend((cu, int(max_seqlen)), q, k, v, decay, scale, initial_state, return_final_state)


def _step_fast(plan, q, k, v, state, decay, idx, cu):
    """One call of a planned signature, or None when an address is not aligned or the device is not current (the general path
    serves it)."""
    p, dt, dev, shape, strides = plan
    qp, kp, vp, sp = q.data_ptr(), k.data_ptr(), v.data_ptr(), state.data_ptr()
    if (qp | kp | vp | sp) & 15 or dev != torch._C._cuda_getDevice():
        return None
    out = torch.empty_strided(shape, strides, dtype=q.dtype, device=q.device)
    p.q, p.k, p.v, p.o, p.state_in, p.state_out, p.decay = qp, kp, vp, out.data_ptr(), sp, sp, decay.data_ptr()
    if idx is not None:
        p.slots = idx.data_ptr()
    if cu is not None:
        p.cu = cu.data_ptr()
    increment_version(state)                   # (a graph that holds the pool for its backward pass sees that it changed)
    _lib.check(_C._L.fable_linear_attn_step(p, dt, torch._C._cuda_getCurrentRawStream(dev)), "fable_linear_attn_step")
    return out


def linear_attn_with_state(q, k, v, state, decay, state_idx=None, scale=None, cu_seqlens=None, max_seqlen=None):
    """Serving: new tokens q, k, v (batch, seqlen_new, nheads, ...), or packed (total, nheads, ...) with cu_seqlens int32 (batch+1) and
    max_seqlen (default: total), go on from the states of a pool, float32 (num_states, nheads, d, dv), which are
    updated in place (autograd sees that as any change in place). state_idx int32 (batch): the state of each sequence (default: its
    own number); an entry outside the pool names no sequence (a padded batch): its rows of out are zeros and no state changes. Two
    sequences of one call must not name one state; a new request starts from a state that the caller has zeroed. Returns out as
    linear_attn_func. Up to 16 new tokens per sequence (by max_seqlen where packed) run token by token, each state read and written
    once; more run by chunks. Head dims are multiples of 8. There is no gradient: where one is asked for, run it under torch.no_grad()."""
    if fwAD._current_level >= 0:
        _no_tangents(q, k, v, state, decay)
    key, plans, asks = None, _plans("linear_step_plans"), False
    scale = None if scale is None else float(scale)
    max_seqlen = None if max_seqlen is None else int(max_seqlen)
    try:
        key = (_place(q), _place(k), _place(v), _place(state), _sig(decay), _sig(state_idx), _sig(cu_seqlens), scale, max_seqlen)
        plan = plans.get(key)
        asks = q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad or decay.requires_grad
    except (AttributeError, TypeError, ValueError, RuntimeError):   # not tensors, or no key
        key = plan = None
    if asks and torch.is_grad_enabled():
        raise NotImplementedError("fable_attn: linear_attn_with_state has no gradient; run it under torch.no_grad()")
    if plan is not None:
        out = _step_fast(plan, q, k, v, state, decay, state_idx, cu_seqlens)
        if out is not None:
            return out
    return _with_state(key, plans, q, k, v, state, decay, state_idx, scale, cu_seqlens, max_seqlen)


@torch.no_grad()
def _with_state(key, plans, q, k, v, state, decay, state_idx, scale, cu_seqlens, max_seqlen):
    """linear_attn_with_state with all checks and conversions; remembers the launch where nothing was converted."""
    if not torch.is_tensor(state) or state.dim() != 4 or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("fable_attn: state must be a contiguous float32 tensor (num_states, nheads, headdim, headdim_v)")
    packed = cu_seqlens is not None
    fp32, scale = _check(q, k, v, decay, packed, scale)
    if q.shape[-1] % 8 or v.shape[-1] % 8:
        raise NotImplementedError(f"fable_attn: states are updated in place for head dims that are multiples of 8, got {q.shape[-1]} and {v.shape[-1]}")
    dev = q.device
    cu = _as_index(cu_seqlens, dev) if packed else None
    most = (q.shape[0] if max_seqlen is None else max_seqlen) if packed else q.shape[1]
    idx = _as_index(state_idx, dev) if state_idx is not None else None
    given = (q, k, v, decay, cu_seqlens, state_idx)
    q, k, v = _rows(q), _rows(k), _rows(v)
    if most > STEP_ROWS:
        out = _forward(q, k, v, fp32, scale, cu, most, state, state, idx)[0]
        increment_version(state)
        return out
    out, p, dt = _C.linear_step(q, k, v, state, fp32, scale, cu, most, idx)
    increment_version(state)
    used = (q, k, v, fp32, cu, idx)
    if key is not None and p.batch and all(a is b for a, b in zip(given, used)):
        _remember(plans, key, (p, dt, dev.index, out.shape, out.stride()))   # nothing was converted: the next call may fill in its addresses
    return out
