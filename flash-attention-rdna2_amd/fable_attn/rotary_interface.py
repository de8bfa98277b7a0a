"""Rotary positions outside a cache call: queries and keys turned by the rows of two tables, with gradients, for
training and for prompts (flash_attn_with_kvcache and flash_attn_append_kvcache turn by the same tables where
they write a cache), and the tables, scaled for contexts longer than the trained ones.

    flash_attn_rotary_func    q and k of a padded or packed batch
    flash_attn_rotary_tables  cosines and sines of all positions
"""
import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable

from . import _C, _lib
from .flash_attn_interface import _DTYPES, _as_index, _no_tangents, _place, _plans, _remember, _sig


def _flat(t):
    """t with a contiguous head dim."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _index(t, dev):
    """t as the kernels read it: int32, contiguous, on dev."""
    return t if t.dtype == torch.int32 and t.device == dev and t.is_contiguous() else _as_index(t, dev)


def _turn(q, k, cos, sin, interleaved, cu, start, conj):
    """One launch; the parameters that the first one of a signature came to are kept per thread, and later ones fill in addresses."""
    key = (_place(q), _place(k), _sig(cos), _sig(sin), _sig(cu), _sig(start), interleaved, conj)
    plans = _plans("rotary_plans")
    plan = plans.get(key)
    dev = q.get_device()
    qp, kp = q.data_ptr(), k.data_ptr() if k is not None else 0
    if plan is None or (qp | kp) & 15 != plan[4] or dev != torch._C._cuda_getDevice():
        qo, ko, p, dt = _C.rotary(q, k, cos, sin, interleaved, cu, start, conj)
        if q.numel():
            _remember(plans, key, (p, dt, qo.stride(), ko.stride() if ko is not None else None, (qp | kp) & 15))
        return qo, ko
    p, dt, qs, ks, _ = plan
    qo = torch.empty_strided(q.shape, qs, dtype=q.dtype, device=q.device)
    p.q, p.q_out, p.cos, p.sin = qp, qo.data_ptr(), cos.data_ptr(), sin.data_ptr()
    ko = None
    if k is not None:
        ko = torch.empty_strided(k.shape, ks, dtype=k.dtype, device=k.device)
        p.k, p.k_out = kp, ko.data_ptr()
    if cu is not None:
        p.cu = cu.data_ptr()
    if start is not None:
        p.start = start.data_ptr()
    _lib.check(_C._L.fable_attn_rotary(p, dt, torch._C._cuda_getCurrentRawStream(dev)), "fable_attn_rotary")
    return qo, ko


class _Rotary(torch.autograd.Function):
    """The rotation is orthogonal but for the tables' amplitude: the gradients go back turned the other way."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, interleaved, cu, start):
        ctx.save_for_backward(cos, sin, cu, start)
        ctx.interleaved = interleaved
        ctx.set_materialize_grads(False)
        qo, ko = _turn(q, k, cos, sin, interleaved, cu, start, False)
        if k is None:
            return qo
        # (one launch turns both; what needs no gradient asks for none further on either)
        needs = ctx.needs_input_grad
        if not (needs[0] and needs[1]):
            ctx.mark_non_differentiable(ko if needs[0] else qo)
        return qo, ko

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        cos, sin, cu, start = ctx.saved_tensors
        one, two = (dq, dk) if dq is not None else (dk, None)
        if one is None:
            return (None,) * 7
        one, two = _turn(_flat(one), _flat(two) if two is not None else None, cos, sin, ctx.interleaved, cu, start, True)
        return (one, two, None, None, None, None, None) if dq is not None else (None, one, None, None, None, None, None)


def flash_attn_rotary_func(q, k, rotary_cos, rotary_sin, *, rotary_interleaved=True, rotary_seqlens=None, cu_seqlens=None):
    """q (batch, seqlen, nheads, d) and k (batch, seqlen, nheads_k, d; may be None), or packed (total, nheads, d) with
    cu_seqlens int32 (batch+1), turned in fp32 and rounded once. rotary_cos, rotary_sin: (rows, rotary_dim / 2), rotary_dim at most d; the
    columns behind it are copied. Token t of sequence b has row rotary_seqlens[b] + t (an int or int32 (batch); default 0), the last
    row serving those past it, as in flash_attn_append_kvcache. rotary_interleaved: pairs are columns 2 i and 2 i + 1,
    else i and i + rotary_dim / 2. Returns (q, k), or q alone without a k, in new tensors; rows of no sequence come back as zeros.
    Gradients flow to q and k; tensors that carry a tangent (forward-mode differentiation) are refused."""
    if not q.is_cuda:
        raise ValueError("fable_attn: tensors must be on the GPU (q.is_cuda == False)")
    if q.dtype not in _DTYPES:
        raise ValueError(f"fable_attn: dtype {q.dtype} is not supported; use fp16, bf16 or fp32")
    if q.dim() != (4 if cu_seqlens is None else 3):
        raise ValueError(f"fable_attn: q must be (batch, seqlen, nheads, headdim), or (total, nheads, headdim) with cu_seqlens; "
                         f"got {tuple(q.shape)}")
    if fwAD._current_level >= 0:
        _no_tangents(q, k, rotary_cos, rotary_sin)
    grad = torch.is_grad_enabled()
    if grad and (rotary_cos.requires_grad or rotary_sin.requires_grad):
        raise NotImplementedError("fable_attn: rotary tables get no gradient; pass them detached")
    dev = q.device
    cos, sin, cu, start = rotary_cos, rotary_sin, cu_seqlens, rotary_seqlens
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or not (cos.is_contiguous() and sin.is_contiguous()):
        cos, sin = cos.detach().to(torch.float32).contiguous(), sin.detach().to(torch.float32).contiguous()
    if cu is not None:
        cu = _index(cu, dev)
    if isinstance(start, int):
        batch = q.shape[0] if cu is None else cu.numel() - 1
        start = torch.full((batch,), start, dtype=torch.int32, device=dev) if start else None
    elif start is not None:
        start = _index(start, dev)
    q, k = _flat(q), _flat(k) if k is not None else None
    if grad and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, cos, sin, bool(rotary_interleaved), cu, start)
    qo, ko = _turn(q, k, cos, sin, bool(rotary_interleaved), cu, start, False)
    return (qo, ko) if k is not None else qo


def flash_attn_rotary_tables(seqlen, rotary_dim, *, base=10000.0, factor=1.0, original_seqlen=None, low_turns=1.0, high_turns=32.0,
                             amplitude=1.0, start=0, device=None):
    """(cos, sin) in fp32, (seqlen, rotary_dim / 2), of positions start, start + 1, ...: pair i turns by f_i = base^(-2 i /
    rotary_dim) per position, angles formed in 64 bits. For a context `factor` times longer than the trained one, f_i becomes f_i
    (keep + (1 - keep) / factor): without original_seqlen keep is 0 (all positions are divided by the factor); with it
    a pair that turns r times over that length has keep = (r - low_turns) / (high_turns - low_turns), between 0 and 1. The tables are
    multiplied by amplitude."""
    seqlen, rotary_dim, start = int(seqlen), int(rotary_dim), int(start)
    if seqlen < 0 or start < 0:
        raise ValueError(f"fable_attn: seqlen={seqlen}, start={start}: at least 0")
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > 8192:
        raise ValueError(f"fable_attn: rotary_dim={rotary_dim}: an even number of 2 to 8192")
    if not 0 < base < float("inf") or not factor > 0:
        raise ValueError(f"fable_attn: base={base}, factor={factor}: above 0, the base finite")
    if original_seqlen is not None and not (original_seqlen > 0 and high_turns > low_turns):
        raise ValueError(f"fable_attn: original_seqlen={original_seqlen}, low_turns={low_turns}, high_turns={high_turns}: "
                         "a length above 0, high_turns above low_turns")
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    else:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"fable_attn: tables are made on the GPU (device={device})")
    return _C.rotary_tables(seqlen, start, rotary_dim // 2, float(base), float(factor), float(original_seqlen or 0), float(low_turns),
                            float(high_turns), float(amplitude), device)
