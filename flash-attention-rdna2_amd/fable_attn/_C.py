"""Host glue between torch tensors and the C-ABI launchers (the reference's `_C` module).

Mirrors the functions of the reference's pybind module (package/csrc/dispatch.cpp:35-231,
bound at :239-268) with the same names, argument order and meaning:
    fwd(q, k, v, scale, causal, win_left, win_right, softcap, alibi, dropout_p, seed,
        attn_chunk=0, out=None) -> (out, lse)
    bwd(dout, q, k, v, out, lse, scale, causal, win_left, win_right, softcap, alibi,
        dropout_p, seed, ds_max_bytes=None) -> (dq, dk, dv)
    bwd_varlen(dout, q, k, v, out, lse, cu_q, cu_k, max_sq, max_sk, scale, causal, win_left,
               win_right, softcap, alibi, dropout_p, seed, seqused_q=None, seqused_k=None,
               ds_max_bytes=None)
        -> (dq, dk, dv)   (no counterpart in the reference's _C: native varlen backward)
    fwd_varlen(q, k, v, cu_q, cu_k, max_sq, max_sk, scale, causal, win_left, win_right,
               softcap, alibi, dropout_p, seed, attn_chunk=0, seqused_q=None,
               seqused_k=None, return_lse=False) -> out  (or (out, lse) when return_lse)
    fwd_paged(q, k_cache, v_cache, block_table, cu_q, cu_k, max_sq, scale, causal, win_left, win_right,
              softcap, alibi, attn_chunk=0, seqused_q=None, seqused_k=None) -> out or None
        (no counterpart in the reference's _C: packed prompts over a paged cache)
    dec(q, k_cache, v_cache, block_table, cache_seqlens, new_k, new_v, rotary_cos,
        rotary_sin, rotary_interleaved, scale, window, num_splits, cache_leftpad=None,
        return_lse=False, softcap=0.0, alibi=None, rotary_dim=0, rotary_pos=None) -> (out, lse)
    combine(out_partial, lse_partial, out_dtype) -> out
Without counterparts there: dec8 and fwd_paged8 (caches held in 8 bits), append (packed or padded new
tokens into a cache) and gather (cached rows as a packed batch).
Tensor checks raise RuntimeError as TORCH_CHECK does there. torch only allocates outputs and
workspaces and supplies the current stream; all compute is in libfable_attn_hip.so. There is
no fallback: if the library is missing, importing this module raises ImportError.

Backward dS workspace: for fp16/bf16 at every head dim the backward can store dS once and
form dQ = dS.K from it (FableBwdParams.ds_ws) instead of recomputing S and dP in its dQ kernel. The
workspace holds 2 bytes per visible (query, key) pair of every q head, in 32x32 tiles (about half
of B*Hq*SQ*SK*2 bytes under a causal mask; packed varlen batches keep the rectangle of the longest
sequences); bwd/bwd_varlen allocate it when it is at most `ds_max_bytes` (default
BWD_DS_MAX_BYTES, 16 GiB, or the environment variable FABLE_ATTN_BWD_DS_MAX_BYTES) and fall back
to the recomputing path when the allocation fails. Both paths give the same gradients to
rounding.
"""
import contextlib
import ctypes
import os

import torch

from . import _lib
from ._lib import FableBwdParams, CombineParams, FableDecParams, FableFwdParams, Strides

_L = _lib.load()

BWD_DS_MAX_BYTES = int(os.environ.get("FABLE_ATTN_BWD_DS_MAX_BYTES", 16 << 30))


def _ds_workspace(p, dtype, device, ds_max_bytes):
    """Attach a dS workspace to FableBwdParams p when the library has a path for it and it fits the
    cap; returns the tensor (kept alive by the caller until the launch is enqueued)."""
    cap = BWD_DS_MAX_BYTES if ds_max_bytes is None else int(ds_max_bytes)
    need = int(_L.fable_attn_bwd_ds_bytes(p, dtype))
    if need <= 0 or need > cap:
        return None
    try:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
    except torch.cuda.OutOfMemoryError:
        return None  # the recomputing path needs no workspace
    if ws.data_ptr() % 16:  # (the caching allocator aligns; an unaligned buffer is not used)
        return None
    p.ds_ws, p.ds_ws_bytes = ws.data_ptr(), need
    return ws


def _req(cond, msg):
    if not cond:
        raise RuntimeError("fable_attn: " + msg)


def _dt(t):
    if t.dtype == torch.float16:
        return _lib.FA_F16
    if t.dtype == torch.bfloat16:
        return _lib.FA_BF16
    if t.dtype == torch.float32:
        return _lib.FA_F32
    raise RuntimeError(f"fable_attn: dtype {t.dtype} not supported")


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _on(dev):
    """The device context of a launch: a no-op when dev is already current (the common case;
    entering torch.cuda.device costs microseconds per call)."""
    if dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _stream(t):
    """The current stream of t's device as a raw handle (the torch call that returns the handle
    directly costs a fraction of building a Stream object; the public call is the fallback)."""
    try:
        return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(t.device.index))
    except AttributeError:
        return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _bhs(t):
    """(b, h, s) element strides of a [B,H,S,D] view."""
    return Strides(t.stride(0), t.stride(1), t.stride(2))


def _rows_aligned(t):
    """16-byte aligned rows with a contiguous head_dim: what the kernels' vector loads need."""
    st, el = t.stride(), t.element_size()
    if st[-1] != 1 or t.data_ptr() % 16:
        return False
    acc = 0
    for x in st[:-1]:
        acc |= x * el
    return acc % 16 == 0


def _check_index(name, t, dev, n=None, at_least=False):
    """int32 index tensor on `dev`, contiguous (the kernels read it through a raw pointer),
    with exactly (or at least) n entries."""
    _req(torch.is_tensor(t), f"{name}: tensor expected")
    _req(t.dtype == torch.int32, f"{name}: int32 expected, got {t.dtype}")
    _req(t.device == dev, f"{name}: must be on {dev}, got {t.device}")
    _req(t.is_contiguous(), f"{name}: must be contiguous")
    if n is not None:
        _req(t.numel() >= n if at_least else t.numel() == n,
             f"{name}: {'at least ' if at_least else ''}{n} entries expected, got {t.numel()}")


def _check_f32(name, t, dev, n=None):
    """float32 side input (alibi slopes, rotary tables) on `dev`, contiguous."""
    _req(torch.is_tensor(t), f"{name}: tensor expected")
    _req(t.dtype == torch.float32, f"{name}: float32 expected, got {t.dtype}")
    _req(t.device == dev, f"{name}: must be on {dev}, got {t.device}")
    _req(t.is_contiguous(), f"{name}: must be contiguous")
    if n is not None:
        _req(t.numel() == n, f"{name}: {n} entries expected, got {t.numel()}")


def _check_varlen_index(q, cu_q, cu_k, seqused_q, seqused_k):
    batch = cu_q.numel() - 1
    _req(batch >= 0, "cu_seqlens_q must have batch+1 entries")
    _check_index("cu_seqlens_q", cu_q, q.device)
    _check_index("cu_seqlens_k", cu_k, q.device, cu_q.numel())
    if seqused_q is not None:
        _check_index("seqused_q", seqused_q, q.device, batch)
    if seqused_k is not None:
        _check_index("seqused_k", seqused_k, q.device, batch)
    return batch


def _alibi(alibi, H, dev):
    """alibi slopes as float32 [H] on dev (converted, as the public API passes them)."""
    if alibi is None:
        return None
    _req(torch.is_tensor(alibi) and alibi.device == dev, f"alibi_slopes must be on {dev}")
    al = alibi.to(torch.float32).contiguous()
    _req(al.numel() == H, f"alibi_slopes: {H} entries (one per q head) expected, got {al.numel()}")
    return al


def _check_bhsd(name, t, dtype, dev):
    if t.dim() == 4 and t.dtype == dtype and t.is_cuda and t.device == dev and _rows_aligned(t):
        return  # (the common case, checked in one pass; the messages below name the failure)
    _req(t.is_cuda, f"{name}: GPU tensor required")
    _req(t.dim() == 4, f"{name}: expected [B,H,S,D]")
    _req(t.dtype == dtype, f"{name}: dtype {t.dtype} differs from q ({dtype})")
    _req(t.device == dev, f"{name}: device mismatch")
    _req(_rows_aligned(t), f"{name}: head_dim must be contiguous with 16-byte aligned rows")


def fwd(q, k, v, scale, causal, win_left, win_right, softcap, alibi, dropout_p, seed,
        attn_chunk=0, out=None):
    """q [B,Hq,SQ,D], k/v [B,Hk,SK,D] (strided views). Returns (out, lse [B,Hq,SQ] fp32).
    Reference: dispatch.cpp:35-80 (one launch here; the reference looped over the batch)."""
    B, Hq, SQ, D = q.shape
    Hk, SK = k.shape[1], k.shape[2]
    for n, t in (("q", q), ("k", k), ("v", v)):
        _check_bhsd(n, t, q.dtype, q.device)
    _req(k.shape[0] == B and v.shape == k.shape and k.shape[3] == D, "k/v shape mismatch")
    _req(Hq % Hk == 0, "Hq must be a multiple of Hk (GQA)")
    if out is None:
        out = torch.empty((B, SQ, Hq, D), dtype=q.dtype, device=q.device).transpose(1, 2)
    else:
        _req(tuple(out.shape) == tuple(q.shape), "out must have the shape of q [B,H,SQ,D]")
        _req(out.dtype == q.dtype, "out must have the dtype of q")
        _req(_rows_aligned(out), "out: head_dim must be contiguous with 16-byte aligned rows")
    lse = torch.empty((B, Hq, SQ), dtype=torch.float32, device=q.device)
    al = _alibi(alibi, Hq, q.device)
    # (one positional construction: a fraction of the host time of 30 field assignments)
    p = FableFwdParams(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                       _bhs(q), _bhs(k), _bhs(v), _bhs(out), SQ, SK, D, Hq, Hq // Hk,
                       float(scale), float(softcap), int(win_left), int(win_right),
                       al.data_ptr() if al is not None else None, 1 if causal else 0,
                       float(dropout_p), int(seed) & ((1 << 64) - 1), None, None, B, int(attn_chunk),
                       None, None, Hq * SQ, SQ)
    with _on(q.device):
        _launch_fwd(p, _dt(q), q.device, _stream(q))
    return out, lse


def _launch_fwd(p, dt, device, stream, ws_bytes=None):
    """fable_attn_fwd, or fable_attn_fwd_ws with a fresh workspace when the library splits this
    call's keys (a small grid); ws_bytes: the library's answer, when the caller has it cached."""
    if ws_bytes is None:
        ws_bytes = _L.fable_attn_fwd_ws_bytes(p, dt)
    if ws_bytes > 0:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
        _lib.check(_L.fable_attn_fwd_ws(p, dt, ws.data_ptr(), ws_bytes, stream), "fable_attn_fwd")
    else:
        _lib.check(_L.fable_attn_fwd(p, dt, stream), "fable_attn_fwd")


def fwd_varlen(q, k, v, cu_q, cu_k, max_sq, max_sk, scale, causal, win_left, win_right, softcap,
               alibi, dropout_p, seed, attn_chunk=0, seqused_q=None, seqused_k=None,
               return_lse=False):
    """q (total_q, Hq, D), k/v (total_k, Hk, D), cu_* int32 [batch+1]. One launch for all
    sequences; LSE [Hq, total_q] is produced on request (the reference wrote none,
    dispatch.cpp:116,139). Reference: dispatch.cpp:117-157."""
    _req(q.is_cuda and k.is_cuda and v.is_cuda, "GPU tensors required")
    _req(q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "varlen expects [total, H, D]")
    Hq, D, Hk = q.shape[1], q.shape[2], k.shape[1]
    _req(Hq % Hk == 0, "Hq must be a multiple of Hk (GQA)")
    for n, t in (("q", q), ("k", k), ("v", v)):
        _req(t.dtype == q.dtype, f"{n}: dtype mismatch")
        _req(_rows_aligned(t), f"{n}: head_dim must be contiguous with 16-byte aligned rows")
    _req(k.device == q.device and v.device == q.device, "q, k, v must be on one device")
    _req(k.shape[2] == D and v.shape[:2] == k.shape[:2], "k/v shape mismatch")
    batch = _check_varlen_index(q, cu_q, cu_k, seqused_q, seqused_k)
    out = torch.zeros_like(q) if seqused_q is not None else torch.empty_like(q)
    lse = torch.empty((Hq, q.shape[0]), dtype=torch.float32, device=q.device) if return_lse else None
    al = _alibi(alibi, Hq, q.device)
    p = FableFwdParams()
    p.Q, p.K, p.V, p.O = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    p.LSE = lse.data_ptr() if lse is not None else None
    p.sQ = Strides(0, q.stride(1), q.stride(0))
    p.sK = Strides(0, k.stride(1), k.stride(0))
    p.sV = Strides(0, v.stride(1), v.stride(0))
    p.sO = Strides(0, out.stride(1), out.stride(0))
    p.SQ, p.SK, p.HD, p.NH, p.gqa = int(max_sq), int(max_sk), D, Hq, Hq // Hk
    p.scale, p.softcap = float(scale), float(softcap)
    p.win_left, p.win_right = int(win_left), int(win_right)
    p.alibi_slopes = al.data_ptr() if al is not None else None
    p.causal = 1 if causal else 0
    p.dropout_p, p.philox_seed = float(dropout_p), int(seed) & ((1 << 64) - 1)
    p.cu_q, p.cu_k = cu_q.data_ptr(), cu_k.data_ptr()
    p.batch = batch
    p.attn_chunk = int(attn_chunk)
    p.seqused_q = seqused_q.data_ptr() if seqused_q is not None else None
    p.seqused_k = seqused_k.data_ptr() if seqused_k is not None else None
    p.lse_sb, p.lse_sh = 0, q.shape[0]
    with _on(q.device):
        _launch_fwd(p, _dt(q), q.device, _stream(q))
    return (out, lse) if return_lse else out


def fwd_paged(q, k_cache, v_cache, block_table, cu_q, cu_k, max_sq, scale, causal, win_left, win_right,
              softcap, alibi, attn_chunk=0, seqused_q=None, seqused_k=None):
    """Packed queries q (total_q, Hq, D) against caches [num_blocks, page, Hk, D] (strided pages,
    rows and heads) through block_table int32 [batch, max_blocks]; key counts from cu_k or
    seqused_k. Returns out, or None when the library has no paged kernel for the call (the
    caller gathers the pages). The reference gathers in Python (flash_attn_interface.py:455-470)."""
    Hq, D, page, Hk = q.shape[1], q.shape[2], k_cache.shape[1], k_cache.shape[2]
    batch = _check_varlen_index(q, cu_q, cu_k, seqused_q, seqused_k)
    _check_index("block_table", block_table, q.device, batch, at_least=True)
    _req(block_table.dim() == 2 and block_table.shape[0] == batch, "block_table must be [batch, max_blocks]")
    al = _alibi(alibi, Hq, q.device)
    p = FableFwdParams()
    p.Q, p.K, p.V = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    p.sQ = Strides(0, q.stride(1), q.stride(0))
    p.sK = Strides(0, k_cache.stride(2), k_cache.stride(1))
    p.sV = Strides(0, v_cache.stride(2), v_cache.stride(1))
    p.sO = Strides(0, D, Hq * D)
    p.SQ, p.SK, p.HD, p.NH, p.gqa = int(max_sq), block_table.shape[1] * page, D, Hq, Hq // Hk
    p.scale, p.softcap = float(scale), float(softcap)
    p.win_left, p.win_right = int(win_left), int(win_right)
    p.alibi_slopes = al.data_ptr() if al is not None else None
    p.causal = 1 if causal else 0
    p.cu_q, p.cu_k = cu_q.data_ptr(), cu_k.data_ptr()
    p.batch, p.attn_chunk = batch, int(attn_chunk)
    p.seqused_q = seqused_q.data_ptr() if seqused_q is not None else None
    p.seqused_k = seqused_k.data_ptr() if seqused_k is not None else None
    kv = _lib.FablePagedKV(block_table.data_ptr(), block_table.shape[1], page, k_cache.stride(0),
                           v_cache.stride(0))
    need = int(_L.fable_attn_fwd_paged_ws_bytes(p, kv, _dt(q)))
    if need == -2:
        return None
    make = torch.zeros if seqused_q is not None else torch.empty   # (rows past seqused_q stay 0)
    out = make(tuple(q.shape), dtype=q.dtype, device=q.device)
    p.O = out.data_ptr()
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    with _on(q.device):
        _lib.check(_L.fable_attn_fwd_paged(p, kv, _dt(q), _ptr(ws), max(need, 0), _stream(q)), "fable_attn_fwd_paged")
    return out


def bwd(dout, q, k, v, out, lse, scale, causal, win_left, win_right, softcap, alibi, dropout_p,
        seed, ds_max_bytes=None):
    """All tensors [B,H,S,D] views (D contiguous); lse [B,Hq,SQ] fp32. Returns (dq, dk, dv)
    with the (B,S,H,D)-dense memory of the public API, viewed as [B,H,S,D].
    Reference: dispatch.cpp:83-111 (no bf16 .item() host syncs here)."""
    B, Hq, SQ, D = q.shape
    Hk, SK = k.shape[1], k.shape[2]
    for n, t in (("dout", dout), ("q", q), ("k", k), ("v", v), ("out", out)):
        _check_bhsd(n, t, q.dtype, q.device)
    _req(lse.dtype == torch.float32 and lse.is_contiguous() and tuple(lse.shape) == (B, Hq, SQ)
         and lse.device == q.device, "lse must be contiguous fp32 [B,Hq,SQ] on q's device")
    dq = torch.empty((B, SQ, Hq, D), dtype=q.dtype, device=q.device).transpose(1, 2)
    dk = torch.empty((B, SK, Hk, D), dtype=k.dtype, device=q.device).transpose(1, 2)
    dv = torch.empty((B, SK, Hk, D), dtype=v.dtype, device=q.device).transpose(1, 2)
    dsum = torch.empty((B, Hq, SQ), dtype=torch.float32, device=q.device)
    al = _alibi(alibi, Hq, q.device)
    p = FableBwdParams()
    p.Q, p.K, p.V, p.O, p.dO = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr()
    p.dQ, p.dK, p.dV = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    p.lse, p.dsum = lse.data_ptr(), dsum.data_ptr()
    p.qs, p.ks, p.vs, p.os, p.dos = _bhs(q), _bhs(k), _bhs(v), _bhs(out), _bhs(dout)
    p.dqs, p.dks, p.dvs = _bhs(dq), _bhs(dk), _bhs(dv)
    p.B, p.Hq, p.Hk, p.SQ, p.SK, p.D, p.gqa = B, Hq, Hk, SQ, SK, D, Hq // Hk
    p.scale, p.softcap = float(scale), float(softcap)
    p.alibi = al.data_ptr() if al is not None else None
    p.causal, p.win_left, p.win_right = 1 if causal else 0, int(win_left), int(win_right)
    p.dropout = 1 if dropout_p > 0 else 0
    p.drop_seed, p.dropout_p = int(seed) & ((1 << 64) - 1), float(dropout_p)
    p.keep_scale = 1.0 / (1.0 - dropout_p) if dropout_p > 0 else 1.0
    p.lse_sb, p.lse_sh = Hq * SQ, SQ
    ws = _ds_workspace(p, _dt(q), q.device, ds_max_bytes)  # noqa: F841  (alive through the launch)
    with _on(q.device):
        _lib.check(_L.fable_attn_bwd(p, _dt(q), _stream(q)), "fable_attn_bwd")
    return dq, dk, dv


def bwd_varlen(dout, q, k, v, out, lse, cu_q, cu_k, max_sq, max_sk, scale, causal, win_left,
               win_right, softcap, alibi, dropout_p, seed, seqused_q=None, seqused_k=None,
               ds_max_bytes=None):
    """Packed variable-length backward: dout/q/out (total_q, Hq, D), k/v (total_k, Hk, D),
    cu_* int32 [batch+1], lse [Hq, total_q] fp32 (fwd_varlen(..., return_lse=True)). One launch
    of each backward kernel for all sequences; the reference has none and loops over the
    sequences in Python (flash_attn_interface.py:523-540). Returns (dq, dk, dv) packed; rows
    outside every sequence (and past seqused) get zero gradient."""
    _req(q.is_cuda and k.is_cuda and v.is_cuda, "GPU tensors required")
    for n, t in (("dout", dout), ("q", q), ("k", k), ("v", v), ("out", out)):
        _req(t.dim() == 3, f"{n}: varlen expects [total, H, D]")
        _req(t.dtype == q.dtype and t.device == q.device, f"{n}: dtype/device mismatch")
        _req(_rows_aligned(t), f"{n}: head_dim must be contiguous with 16-byte aligned rows")
    Hq, D, Hk = q.shape[1], q.shape[2], k.shape[1]
    _req(Hq % Hk == 0, "Hq must be a multiple of Hk (GQA)")
    _req(dout.shape == q.shape and out.shape == q.shape and v.shape == k.shape, "shape mismatch")
    _req(lse.dtype == torch.float32 and lse.is_contiguous() and tuple(lse.shape) == (Hq, q.shape[0])
         and lse.device == q.device, "lse must be contiguous fp32 [Hq, total_q] on q's device")
    batch = _check_varlen_index(q, cu_q, cu_k, seqused_q, seqused_k)
    # dense; the kernels write every row a sequence uses, one launch ahead of them zeroes the others
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    dsum = torch.empty((Hq, q.shape[0]), dtype=torch.float32, device=q.device)
    al = _alibi(alibi, Hq, q.device)
    row = lambda t: Strides(0, t.stride(1), t.stride(0))
    p = FableBwdParams()
    p.Q, p.K, p.V, p.O, p.dO = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr()
    p.dQ, p.dK, p.dV = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    p.lse, p.dsum = lse.data_ptr(), dsum.data_ptr()
    p.qs, p.ks, p.vs, p.os, p.dos = row(q), row(k), row(v), row(out), row(dout)
    p.dqs, p.dks, p.dvs = row(dq), row(dk), row(dv)
    p.B, p.Hq, p.Hk, p.SQ, p.SK, p.D, p.gqa = batch, Hq, Hk, int(max_sq), int(max_sk), D, Hq // Hk
    p.scale, p.softcap = float(scale), float(softcap)
    p.alibi = al.data_ptr() if al is not None else None
    p.causal, p.win_left, p.win_right = 1 if causal else 0, int(win_left), int(win_right)
    p.dropout = 1 if dropout_p > 0 else 0
    p.drop_seed, p.dropout_p = int(seed) & ((1 << 64) - 1), float(dropout_p)
    p.keep_scale = 1.0 / (1.0 - dropout_p) if dropout_p > 0 else 1.0
    p.cu_q, p.cu_k = cu_q.data_ptr(), cu_k.data_ptr()
    p.seqused_q = seqused_q.data_ptr() if seqused_q is not None else None
    p.seqused_k = seqused_k.data_ptr() if seqused_k is not None else None
    p.lse_sb, p.lse_sh = 0, q.shape[0]
    with _on(q.device):
        _lib.check(_L.fable_attn_bwd_zero_gaps(p, _dt(q), q.shape[0], k.shape[0], _stream(q)), "fable_attn_bwd (varlen)")
        ws = _ds_workspace(p, _dt(q), q.device, ds_max_bytes)  # noqa: F841  (alive through the launch)
        _lib.check(_L.fable_attn_bwd(p, _dt(q), _stream(q)), "fable_attn_bwd (varlen)")
    return dq, dk, dv


def num_splits(batch, nq, nheads, gqa, ctx_bound, hint):
    return int(_L.fa_decode_num_splits(batch, nq, nheads, gqa, int(ctx_bound), int(hint)))


def dec(q, k_cache, v_cache, block_table, cache_seqlens, new_k, new_v, rotary_cos, rotary_sin,
        rotary_interleaved, scale, window, num_splits=0, cache_leftpad=None, return_lse=False,
        softcap=0.0, alibi=None, rotary_dim=0, rotary_pos=None):
    """q [B,nq,Hq,D]; caches [num_blocks,page,Hk,D] contiguous; block_table [B,max_blocks]
    int32; cache_seqlens [B] int32 (length before append). Returns (out [B,nq,Hq,D],
    lse [B,nq,Hq] or an empty tensor). Reference: dispatch.cpp:162-231."""
    _req(q.is_cuda and k_cache.is_cuda and v_cache.is_cuda, "GPU tensors required")
    _req(q.dim() == 4, "decode expects q [B,nq,Hq,D]")
    _req(k_cache.dim() == 4, "k_cache expected [num_blocks, page, nheads_k, D]")
    B, NQ, Hq, D = q.shape
    page, Hk = k_cache.shape[1], k_cache.shape[2]
    _req(Hq % Hk == 0, "Hq must be a multiple of nheads_k (GQA)")
    _req(page > 0 and (page & (page - 1)) == 0, "page must be a power of two")
    dev = q.device
    for n, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)):
        _req(t.is_contiguous() and t.dtype == q.dtype and t.device == dev,
             f"{n}: contiguous, dtype and device of q")
        _req(t.data_ptr() % 16 == 0 and (D * t.element_size()) % 16 == 0,
             f"{n}: rows must be 16-byte aligned (base pointer and head_dim)")
    _req(v_cache.shape == k_cache.shape and k_cache.shape[3] == D,
         "k_cache/v_cache must both be [num_blocks, page, nheads_k, D] with q's D")
    _req(block_table.dim() == 2 and block_table.shape[0] == B, "block_table must be [B, max_blocks]")
    _check_index("block_table", block_table, dev)
    _check_index("cache_seqlens", cache_seqlens, dev, B)
    if cache_leftpad is not None:
        _check_index("cache_leftpad", cache_leftpad, dev, B)
    if rotary_pos is not None:
        _check_index("rotary_seqlens", rotary_pos, dev, B)
    if alibi is not None:
        _check_f32("alibi_slopes", alibi, dev, Hq)
    _req((rotary_cos is None) == (rotary_sin is None), "rotary_cos and rotary_sin go together")
    if rotary_cos is not None:
        _check_f32("rotary_cos", rotary_cos, dev)
        _check_f32("rotary_sin", rotary_sin, dev)
        _req(rotary_cos.dim() == 2 and rotary_sin.shape == rotary_cos.shape,
             "rotary_cos/rotary_sin must be [seqlen_ro, rotary_dim/2]")
        rd = int(rotary_dim) or D
        _req(rotary_cos.shape[1] * 2 == rd and rd <= D and rd % 2 == 0,
             f"rotary tables of width {rotary_cos.shape[1]} do not match rotary_dim {rd}")
    if new_k is not None:
        _req(new_v is not None, "new_k and new_v go together")
        for n, t in (("k", new_k), ("v", new_v)):
            _req(tuple(t.shape) == (B, NQ, Hk, D) and t.dtype == q.dtype and t.device == dev and
                 t.is_contiguous() and t.data_ptr() % 16 == 0,
                 f"{n}: contiguous, 16-byte aligned [B, seqlen_q, nheads_k, D] of q's dtype")
    else:
        _req(new_v is None, "new_k and new_v go together")
    out = torch.empty((B, NQ, Hq, D), dtype=q.dtype, device=q.device)
    lse = (torch.empty((B, NQ, Hq), dtype=torch.float32, device=q.device) if return_lse
           else torch.empty((0,), dtype=torch.float32, device=q.device))
    p = FableDecParams()
    p.q, p.Kc, p.Vc = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    p.block_table, p.o = block_table.data_ptr(), out.data_ptr()
    p.ctx_len = cache_seqlens.data_ptr()
    p.cos = rotary_cos.data_ptr() if rotary_cos is not None else None
    p.sin = rotary_sin.data_ptr() if rotary_sin is not None else None
    p.batch, p.NH, p.gqa, p.HD, p.page = B, Hq, Hq // Hk, D, page
    p.max_blocks, p.nsplit, p.window = block_table.shape[1], int(num_splits or 0), int(window)
    p.rotary = (2 if rotary_interleaved else 1) if rotary_cos is not None else 0
    p.scale = float(scale)
    p.leftpad = cache_leftpad.data_ptr() if cache_leftpad is not None else None
    p.lse_out = lse.data_ptr() if return_lse else None
    p.softcap = float(softcap)
    p.alibi = alibi.data_ptr() if alibi is not None else None
    p.nq, p.rotary_dim = NQ, int(rotary_dim)
    p.rotary_pos = rotary_pos.data_ptr() if rotary_pos is not None else None
    # (split partials, the parts of a rotated q: the library says what this call uses)
    ws_bytes = int(_L.fable_attn_dec_ws_bytes(p, _dt(q), 1 if new_k is not None else 0))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes > 0 else None
    with _on(q.device):
        _lib.check(_L.fable_attn_dec_ws(p, _dt(q), _ptr(ws), max(ws_bytes, 0), _stream(q), _ptr(new_k),
                                        _ptr(new_v)), "fable_attn_dec")
    return out, lse


# ----------------------------------------------------------------------------- caches in 8 bits, append, gather
FP8, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _cache_strides(name, t, dev):
    """(page, head, row) strides of a cache [num_blocks, page, nheads_k, D] that the kernels can address."""
    _req(t.is_cuda and t.device == dev, f"{name}: must be on {dev}, got {t.device}")
    _req(_rows_aligned(t), f"{name}: head_dim must be contiguous with 16-byte aligned rows")
    return Strides(t.stride(0), t.stride(2), t.stride(1))


def _check_cache(k_cache, v_cache, k_scale, v_scale, dtype, dev):
    """Shapes and types of a cache pair: of `dtype`, or e4m3 codes with e8m0 scales. Returns (k strides, v strides,
    tokens per scale; 0 without scales)."""
    _req(k_cache.dim() == 4 and v_cache.shape == k_cache.shape,
         "k_cache/v_cache must both be [num_blocks, page, nheads_k, D]")
    _req((k_scale is None) == (v_scale is None), "k_scale and v_scale go together")
    want = FP8 if k_scale is not None else dtype
    nb, page, Hk, D = k_cache.shape
    for n, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _req(t.dtype == want, f"{n}: dtype {want} expected, got {t.dtype}"
             + ("" if k_scale is not None else " (8-bit caches need k_scale and v_scale)"))
    _req(nb > 0, "the cache has no pages")
    _req(page > 0 and (page & (page - 1)) == 0, "page must be a power of two")
    ks, vs = _cache_strides("k_cache", k_cache, dev), _cache_strides("v_cache", v_cache, dev)
    if k_scale is None:
        return ks, vs, 0
    _req(D % 16 == 0 and D <= 256, f"8-bit caches need a head_dim that is a multiple of 16 up to 256, got {D}")
    _req(page >= 16, f"8-bit caches need pages of at least 16 rows, got {page}")
    for n, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        _req(torch.is_tensor(t) and t.dtype == E8M0, f"{n}: {E8M0} expected")
        _req(t.device == dev and t.is_contiguous(), f"{n}: must be contiguous on {dev}")
        subs = t.shape[2] if t.dim() == 3 else 0
        _req(t.dim() == 3 and t.shape[0] == nb and t.shape[1] == Hk and subs > 0 and page % subs == 0
             and (subs & (subs - 1)) == 0 and page // subs <= 256,
             f"{n}: must be [num_blocks, nheads_k, page / G] = [{nb}, {Hk}, {page} / G] with G a power of two up to "
             f"min(page, 256), got {tuple(t.shape)}")
    _req(v_scale.shape == k_scale.shape, "v_scale: must have the shape of k_scale")
    subs = k_scale.shape[2]
    return ks, vs, page // subs


def _cache8(k_cache, v_cache, k_scale, v_scale, dtype, dev, rotary_rows=0):
    ks, vs, group = _check_cache(k_cache, v_cache, k_scale, v_scale, dtype, dev)
    _req(k_cache.stride() == v_cache.stride(), "8-bit k_cache and v_cache must have the same strides")
    return _lib.FableCache8(k_scale.data_ptr(), v_scale.data_ptr(), ks, group, k_cache.shape[0], rotary_rows, None)


def _check_table(block_table, batch, dev):
    _check_index("block_table", block_table, dev)
    _req(block_table.dim() == 2 and block_table.shape[0] == batch and block_table.shape[1] > 0,
         f"block_table must be [batch, max_blocks], got {tuple(block_table.shape)} for batch={batch}")


def _check_rotary(cos, sin, rotary_dim, D, dev):
    _req((cos is None) == (sin is None), "rotary_cos and rotary_sin go together")
    if cos is None:
        return
    _check_f32("rotary_cos", cos, dev)
    _check_f32("rotary_sin", sin, dev)
    _req(cos.dim() == 2 and sin.shape == cos.shape and cos.shape[0] > 0,
         "rotary_cos/rotary_sin must be [seqlen_ro, rotary_dim/2]")
    _req(cos.shape[1] * 2 == rotary_dim and 0 < rotary_dim <= D,
         f"rotary tables of width {cos.shape[1]} do not fit a head_dim of {D}")


def dec8(q, k_cache, v_cache, k_scale, v_scale, block_table, cache_seqlens, new_k, new_v, cos, sin, interleaved, scale,
         window, num_splits, leftpad, return_lse, softcap, alibi, rotary_pos, held=None):
    """dec over a cache in 8 bits: codes [num_blocks, page, Hk, D] (strided pages, rows and heads), scales
    [num_blocks, Hk, page / G]. block_table None: a dense cache, sequence b in page b. leftpad: the first row a sequence's
    queries see; held: the first one it has (an append keeps those of its block under its scale)."""
    _req(q.is_cuda, "GPU tensors required")
    _req(q.dim() == 4 and q.is_contiguous() and q.data_ptr() % 16 == 0, "decode expects contiguous q [B,nq,Hq,D], 16-byte aligned")
    _req(q.dtype in (torch.float16, torch.bfloat16), f"8-bit caches take fp16 or bf16 queries, got {q.dtype}")
    B, NQ, Hq, D = q.shape
    dev = q.device
    _req(k_cache.dim() == 4 and k_cache.shape[3] == D, "k_cache/v_cache must both be [num_blocks, page, nheads_k, D] with q's D")
    nb, page, Hk = k_cache.shape[:3]
    _req(Hk > 0 and Hq % Hk == 0, "Hq must be a multiple of nheads_k (GQA)")
    c = _cache8(k_cache, v_cache, k_scale, v_scale, q.dtype, dev, cos.shape[0] if cos is not None else 0)
    if block_table is not None:
        _check_table(block_table, B, dev)
    else:
        _req(nb >= B, f"a dense cache of {nb} rows for a batch of {B}")
    _check_index("cache_seqlens", cache_seqlens, dev, B)
    for n, t in (("cache_leftpad", leftpad), ("cache_leftpad", held), ("rotary_seqlens", rotary_pos)):
        if t is not None:
            _check_index(n, t, dev, B)
    c.held = held.data_ptr() if held is not None else None
    if alibi is not None:
        _check_f32("alibi_slopes", alibi, dev, Hq)
    rd = int(cos.shape[-1] * 2) if cos is not None else 0
    _check_rotary(cos, sin, rd, D, dev)
    _req((new_k is None) == (new_v is None), "new_k and new_v go together")
    if new_k is not None:
        for n, t in (("k", new_k), ("v", new_v)):
            _req(tuple(t.shape) == (B, NQ, Hk, D) and t.dtype == q.dtype and t.device == dev and
                 t.is_contiguous() and t.data_ptr() % 16 == 0,
                 f"{n}: contiguous, 16-byte aligned [B, seqlen_q, nheads_k, D] of q's dtype")
    out = torch.empty((B, NQ, Hq, D), dtype=q.dtype, device=dev)
    lse = torch.empty((B, NQ, Hq) if return_lse else (0,), dtype=torch.float32, device=dev)
    p = FableDecParams()
    p.q, p.Kc, p.Vc, p.o = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
    p.block_table = block_table.data_ptr() if block_table is not None else None
    p.ctx_len = cache_seqlens.data_ptr()
    p.cos = cos.data_ptr() if cos is not None else None
    p.sin = sin.data_ptr() if sin is not None else None
    p.batch, p.NH, p.gqa, p.HD, p.page = B, Hq, Hq // Hk, D, page
    p.max_blocks, p.nsplit, p.window = block_table.shape[1] if block_table is not None else 1, int(num_splits or 0), int(window)
    p.rotary, p.rotary_dim = ((2 if interleaved else 1) if cos is not None else 0), rd
    p.scale, p.softcap, p.nq = float(scale), float(softcap), NQ
    p.leftpad = leftpad.data_ptr() if leftpad is not None else None
    p.lse_out = lse.data_ptr() if return_lse else None
    p.alibi = alibi.data_ptr() if alibi is not None else None
    p.rotary_pos = rotary_pos.data_ptr() if rotary_pos is not None else None
    need = int(_L.fable_attn_dec8_ws_bytes(p, c, _dt(q), 1 if new_k is not None else 0))
    if need < 0:
        _lib.check(1, "fable_attn_dec8")
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    with _on(dev):
        _lib.check(_L.fable_attn_dec8(p, c, _dt(q), _ptr(ws), need, _stream(q), _ptr(new_k), _ptr(new_v)), "fable_attn_dec8")
    return out, lse


def fwd_paged8(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_q, cu_k, max_sq, scale, causal, win_left, win_right,
               softcap, alibi, attn_chunk=0, seqused_q=None, seqused_k=None):
    """fwd_paged over a cache in 8 bits (as dec8's). Returns (out, the launch's parameters)."""
    _req(q.is_cuda, "GPU tensors required")
    _req(q.dtype in (torch.float16, torch.bfloat16), f"8-bit caches take fp16 or bf16 queries, got {q.dtype}")
    _req(q.dim() == 3 and _rows_aligned(q), "q: [total, H, D] with a contiguous head_dim and 16-byte aligned rows expected")
    _req(k_cache.dim() == 4 and k_cache.shape[3] == q.shape[2], "k/v must be paged [num_blocks, page, nheads_k, D] with q's D")
    Hq, D, page, Hk = q.shape[1], q.shape[2], k_cache.shape[1], k_cache.shape[2]
    _req(Hk > 0 and Hq % Hk == 0, "Hq must be a multiple of nheads_k (GQA)")
    c = _cache8(k_cache, v_cache, k_scale, v_scale, q.dtype, q.device)
    batch = _check_varlen_index(q, cu_q, cu_k, seqused_q, seqused_k)
    _check_table(block_table, batch, q.device)
    al = _alibi(alibi, Hq, q.device)
    p = FableFwdParams()
    p.Q, p.K, p.V = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    p.sQ, p.sO = Strides(0, q.stride(1), q.stride(0)), Strides(0, D, Hq * D)
    p.SQ, p.HD, p.NH, p.gqa = int(max_sq), D, Hq, Hq // Hk
    p.scale, p.softcap = float(scale), float(softcap)
    p.win_left, p.win_right, p.causal = int(win_left), int(win_right), 1 if causal else 0
    p.alibi_slopes = al.data_ptr() if al is not None else None
    p.cu_q, p.cu_k = cu_q.data_ptr(), cu_k.data_ptr()
    p.batch, p.attn_chunk = batch, int(attn_chunk)
    p.seqused_q = seqused_q.data_ptr() if seqused_q is not None else None
    p.seqused_k = seqused_k.data_ptr() if seqused_k is not None else None
    kv = _lib.FablePagedKV(block_table.data_ptr(), block_table.shape[1], page, 0, 0)
    need = int(_L.fable_attn_fwd_paged8_ws_bytes(p, kv, c, _dt(q)))
    if need < 0:
        _lib.check(1, "fable_attn_fwd_paged8")
    make = torch.zeros if seqused_q is not None else torch.empty   # (rows past seqused_q stay 0)
    out = make(tuple(q.shape), dtype=q.dtype, device=q.device)
    p.O = out.data_ptr()
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    with _on(q.device):
        _lib.check(_L.fable_attn_fwd_paged8(p, kv, c, _dt(q), _ptr(ws), need, _stream(q)), "fable_attn_fwd_paged8")
    return out, (p, kv, c, _dt(q))


def append(k, v, k_cache, v_cache, cache_seqlens, q=None, cu=None, max_seqlen=0, block_table=None, leftpad=None, cos=None,
           sin=None, interleaved=False, rotary_pos=None, k_scale=None, v_scale=None):
    """New tokens k, v (and q, which comes back rotated) [B,N,H,D], or [total,H,D] with cu int32 [batch+1], into the
    caches at positions cache_seqlens[b] + t. block_table None: a dense cache, sequence b in page b. Returns (the
    launch's parameters and dtype, q rotated or None)."""
    dev = k.device
    packed = cu is not None
    _req(k.is_cuda, "GPU tensors required")
    _req(k.dim() == (3 if packed else 4) and v.shape == k.shape, "k/v: [B,N,nheads_k,D], or [total,nheads_k,D] with cu_seqlens")
    D, Hk = k.shape[-1], k.shape[-2]
    for n, t in (("k", k), ("v", v)) + ((("q", q),) if q is not None else ()):
        _req(t.dtype == k.dtype and t.device == dev, f"{n}: dtype and device of k")
        _req(_rows_aligned(t), f"{n}: head_dim must be contiguous with 16-byte aligned rows")
    if q is not None:
        _req(q.dim() == k.dim() and q.shape[:-2] == k.shape[:-2] and q.shape[-1] == D, "q: the tokens and head_dim of k")
    dt = _dt(k)
    _req(k_cache.dim() == 4 and tuple(k_cache.shape[2:]) == (Hk, D),
         f"k_cache/v_cache must be [num_blocks, page, {Hk}, {D}], got {tuple(k_cache.shape)}")
    kc, vc, group = _check_cache(k_cache, v_cache, k_scale, v_scale, k.dtype, dev)
    _req(group == 0 or k.dtype != torch.float32, "8-bit caches take fp16 or bf16 tokens")
    _req(D % 8 == 0 and D <= 256, f"head_dim must be a multiple of 8 up to 256, got {D}")
    batch = cu.numel() - 1 if packed else k.shape[0]
    _req(batch >= 0, "cu_seqlens must have batch+1 entries")
    if packed:
        _check_index("cu_seqlens", cu, dev)
    _check_index("cache_seqlens", cache_seqlens, dev, batch)
    for n, t in (("cache_leftpad", leftpad), ("rotary_seqlens", rotary_pos)):
        if t is not None:
            _check_index(n, t, dev, batch)
    if block_table is not None:
        _check_table(block_table, batch, dev)
    else:
        _req(k_cache.shape[0] >= batch, f"a dense cache of {k_cache.shape[0]} rows for a batch of {batch}")
    rd = int(cos.shape[-1] * 2) if cos is not None else 0
    _check_rotary(cos, sin, rd, D, dev)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=dev) if q is not None else None
    st = lambda t: Strides(0 if packed else t.stride(0), t.stride(-2), t.stride(-3))
    p = _lib.FableAppendParams()
    p.k, p.v, p.Kc, p.Vc = k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    p.sk, p.sv, p.kc, p.vc = st(k), st(v), kc, vc
    if q is not None:
        p.q, p.q_out, p.sq, p.NH = q.data_ptr(), q_out.data_ptr(), st(q), q.shape[-2]
    if group:
        p.k_scale, p.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    p.block_table = block_table.data_ptr() if block_table is not None else None
    p.ctx_len = cache_seqlens.data_ptr()
    p.cu = cu.data_ptr() if packed else None
    p.leftpad = leftpad.data_ptr() if leftpad is not None else None
    p.rotary_pos = rotary_pos.data_ptr() if rotary_pos is not None else None
    p.batch, p.n, p.NKV, p.HD = batch, int(max_seqlen) if packed else k.shape[1], Hk, D
    p.page, p.num_blocks, p.group = k_cache.shape[1], k_cache.shape[0], group
    p.max_blocks = block_table.shape[1] if block_table is not None else 1
    if cos is not None:
        p.cos, p.sin, p.rotary, p.rotary_dim, p.rotary_rows = cos.data_ptr(), sin.data_ptr(), 2 if interleaved else 1, rd, cos.shape[0]
    if k.numel():
        with _on(dev):
            _lib.check(_L.fable_attn_append(p, dt, _stream(k)), "fable_attn_append")
    return p, dt, q_out


def gather(k_cache, v_cache, cu, total, dtype, block_table=None, k_scale=None, v_scale=None, used=None):
    """The first cu[b+1] - cu[b] cached rows of every sequence as packed k, v [total, Hk, D] in dtype; with used
    int32 [batch] only that many of them, the others of the result left as they were allocated.
    Returns (the launch's parameters and dtype, (k, v))."""
    dev = k_cache.device
    kc, vc, group = _check_cache(k_cache, v_cache, k_scale, v_scale, dtype, dev)
    nb, page, Hk, D = k_cache.shape
    _req(D % 8 == 0 and D <= 256, f"head_dim must be a multiple of 8 up to 256, got {D}")
    _check_index("cu_seqlens_k", cu, dev)
    batch = cu.numel() - 1
    _req(batch >= 0, "cu_seqlens_k must have batch+1 entries")
    if block_table is not None:
        _check_table(block_table, batch, dev)
    else:
        _req(nb >= batch, f"a dense cache of {nb} rows for a batch of {batch}")
    k, v = (torch.empty((int(total), Hk, D), dtype=dtype, device=dev) for _ in range(2))
    p = _lib.FableGatherParams()
    p.Kc, p.Vc, p.k_out, p.v_out, p.kc, p.vc = k_cache.data_ptr(), v_cache.data_ptr(), k.data_ptr(), v.data_ptr(), kc, vc
    if group:
        p.k_scale, p.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    p.block_table = block_table.data_ptr() if block_table is not None else None
    p.cu, p.total, p.batch, p.NKV, p.HD, p.page = cu.data_ptr(), int(total), batch, Hk, D, page
    if used is not None:
        _check_index("used", used, dev, batch)
        p.used = used.data_ptr()
    p.max_blocks = block_table.shape[1] if block_table is not None else 1
    p.num_blocks, p.group = nb, group
    if k.numel():
        with _on(dev):
            _lib.check(_L.fable_attn_gather(p, _dt(k), _stream(k)), "fable_attn_gather")
    return p, _dt(k), (k, v)


def combine(out_partial, lse_partial, out_dtype):
    """out_partial [nsplit,B,S,H,D] (D contiguous), lse_partial [nsplit,B,H,S] fp32 ->
    dense [B,S,H,D] in out_dtype. Reference math: flash_attn_interface.py:567-580."""
    _req(out_partial.is_cuda and lse_partial.is_cuda, "GPU tensors required")
    _req(out_partial.dim() == 5 and lse_partial.dim() == 4, "shapes [nsplit,B,S,H,D] / [nsplit,B,H,S]")
    _req(out_partial.stride(-1) == 1, "out_partial: head_dim must be contiguous")
    ns, B, S, H, D = out_partial.shape
    _req(tuple(lse_partial.shape) == (ns, B, H, S),
         f"lse_partial must be [nsplit, B, H, S] = {(ns, B, H, S)}, got {tuple(lse_partial.shape)}")
    _req(lse_partial.device == out_partial.device, "out_partial and lse_partial on one device")
    lp = lse_partial.float()
    out = torch.empty((B, S, H, D), dtype=out_dtype, device=out_partial.device)
    c = CombineParams()
    c.out_partial, c.lse_partial, c.out = out_partial.data_ptr(), lp.data_ptr(), out.data_ptr()
    c.nsplit, c.B, c.S, c.H, c.D = ns, B, S, H, D
    c.op_split, c.op_b, c.op_seq, c.op_h = (out_partial.stride(0), out_partial.stride(1),
                                            out_partial.stride(2), out_partial.stride(3))
    c.lp_split, c.lp_b, c.lp_h, c.lp_seq = lp.stride(0), lp.stride(1), lp.stride(2), lp.stride(3)
    c.in_dtype, c.out_dtype = _dt(out_partial), _dt(out)
    with _on(out_partial.device):
        _lib.check(_L.fa_combine_launch(c, _stream(out_partial)), "fa_combine_launch")
    return out


# ----------------------------------------------------------------------------- linear attention
def _rows_strides(t, packed):
    """(b, h, s) strides of a (B,S,H,D) tensor, or of a packed (total,H,D) one."""
    return Strides(0, t.stride(1), t.stride(0)) if packed else Strides(t.stride(0), t.stride(2), t.stride(1))


def _linear_params(q, k, v, decay, scale, cu, max_seqlen, state_in=None, slots=None):
    """FableLinearParams of q [B,S,H,DK], k [B,S,Hk,DK], v [B,S,Hk,DV] (packed [total,H,D] with cu int32 [batch+1]),
    decay f32 [H] or [batch,H] and states f32 [slots,H,DK,DV]."""
    packed, dev = cu is not None, q.device
    _req(q.is_cuda, "GPU tensors required")
    _req(q.dim() == (3 if packed else 4), "q: [B,S,H,D], or [total,H,D] with cu_seqlens")
    for n, t in (("q", q), ("k", k), ("v", v)):
        _req(t.dim() == q.dim() and t.dtype == q.dtype and t.device == dev, f"{n}: dims, dtype and device of q")
        _req(_rows_aligned(t), f"{n}: head_dim must be contiguous with 16-byte aligned rows")
    H, Hk, DK, DV = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
    _req(k.shape[:-2] == q.shape[:-2] and k.shape[-1] == DK and v.shape[:-1] == k.shape[:-1],
         f"q, k, v of one batch expected, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    _req(Hk > 0 and H > 0 and H % Hk == 0, "nheads must be a multiple of nheads_k (GQA)")
    p = _lib.FableLinearParams()
    if packed:
        _check_index("cu_seqlens", cu, dev)
        _req(max_seqlen >= 0, f"max_seqlen={max_seqlen}")
        p.batch, p.n, p.total, p.cu = cu.numel() - 1, min(int(max_seqlen), q.shape[0]), q.shape[0], cu.data_ptr()
        _req(p.batch >= 0, "cu_seqlens must have batch+1 entries")
    else:
        p.batch, p.n = q.shape[0], q.shape[1]
    _check_f32("decay", decay, dev)
    _req(tuple(decay.shape) in ((H,), (p.batch, H)), f"decay must be [{H}] or [{p.batch}, {H}], got {tuple(decay.shape)}")
    p.decay, p.decay_b = decay.data_ptr(), H if decay.dim() == 2 else 0
    p.q, p.k, p.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    p.sq, p.sk, p.sv = _rows_strides(q, packed), _rows_strides(k, packed), _rows_strides(v, packed)
    p.NH, p.gqa, p.DK, p.DV, p.scale = H, H // Hk, DK, DV, float(scale)
    if state_in is not None:
        _check_f32("state", state_in, dev)
        _req(state_in.dim() == 4 and tuple(state_in.shape[1:]) == (H, DK, DV) and state_in.data_ptr() % 16 == 0,
             f"states must be [slots, {H}, {DK}, {DV}], 16-byte aligned, got {tuple(state_in.shape)}")
        p.state_in = state_in.data_ptr()
        if slots is None:
            _req(state_in.shape[0] >= p.batch, f"{state_in.shape[0]} states for a batch of {p.batch}")
    if slots is not None:
        _check_index("state_idx", slots, dev, p.batch)
        p.slots, p.num_slots = slots.data_ptr(), state_in.shape[0]
    return p


def _linear_ws(p, dt, backward, dev):
    need = int(_L.fable_linear_attn_ws_bytes(p, dt, backward))
    if need < 0:
        _lib.check(1, "linear attention")
    return (torch.empty(need, dtype=torch.uint8, device=dev) if need else None), need


def linear_fwd(q, k, v, decay, scale, cu=None, max_seqlen=0, state_in=None, state_out=None, slots=None):
    """Linear attention by chunks -> (out, dense of q's rows and v's width; the states before the segments of long sequences for
    linear_bwd, or None; the launch's parameters, dtype and workspace size). state_out: where the states behind the last rows go
    (as state_in; may be it)."""
    p = _linear_params(q, k, v, decay, scale, cu, max_seqlen, state_in, slots)
    out = torch.empty((*q.shape[:-1], v.shape[-1]), dtype=q.dtype, device=q.device)
    p.o, p.so = out.data_ptr(), _rows_strides(out, cu is not None)
    if state_out is not None:
        p.state_out = state_out.data_ptr()
    if p.batch == 0:
        return out.zero_(), None, p, _dt(q), 0
    dt = _dt(q)
    ws, need = _linear_ws(p, dt, 0, q.device)
    with _on(q.device):
        _lib.check(_L.fable_linear_attn_fwd(p, dt, _ptr(ws), need, _stream(q)), "fable_linear_attn_fwd")
    return out, ws, p, dt, need


def linear_bwd(dout, q, k, v, decay, scale, cu=None, max_seqlen=0, state_in=None, dstate_out=None, want_dstate=False, seg_states=None):
    """-> (dq, dk, dv, dstate_in or None, the launch's parameters, dtype and workspace size)"""
    p = _linear_params(q, k, v, decay, scale, cu, max_seqlen, state_in)
    _req(dout.dtype == q.dtype and tuple(dout.shape) == (*q.shape[:-1], v.shape[-1]) and _rows_aligned(dout),
         "dout: out's shape and dtype, 16-byte aligned rows")
    packed = cu is not None
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    p.dout, p.dq, p.dk, p.dv = dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    p.sdo, p.sdq, p.sdk, p.sdv = (_rows_strides(t, packed) for t in (dout, dq, dk, dv))
    dstate = None
    if want_dstate:
        dstate = torch.empty((p.batch, p.NH, p.DK, p.DV), dtype=torch.float32, device=q.device)
        p.dstate_in = dstate.data_ptr()
    if dstate_out is not None:
        _check_f32("dstate_out", dstate_out, q.device, p.batch * p.NH * p.DK * p.DV)
        p.dstate_out = dstate_out.data_ptr()
    if seg_states is not None:
        p.seg_states = seg_states.data_ptr()
    if p.batch == 0:
        return dq.zero_(), dk.zero_(), dv.zero_(), dstate, p, _dt(q), 0
    dt = _dt(q)
    ws, need = _linear_ws(p, dt, 1, q.device)
    with _on(q.device):
        _lib.check(_L.fable_linear_attn_bwd(p, dt, _ptr(ws), need, _stream(q)), "fable_linear_attn_bwd")
    return dq, dk, dv, dstate, p, dt, need


def linear_step(q, k, v, state, decay, scale, cu=None, max_seqlen=0, slots=None):
    """A few rows per sequence, token by token; the states of the pool [slots,H,DK,DV] updated in place. Returns (out,
    the launch's parameters and dtype)."""
    p = _linear_params(q, k, v, decay, scale, cu, max_seqlen, state, slots)
    out = torch.empty((*q.shape[:-1], v.shape[-1]), dtype=q.dtype, device=q.device)
    p.o, p.so, p.state_out = out.data_ptr(), _rows_strides(out, cu is not None), state.data_ptr()
    dt = _dt(q)
    if p.batch == 0:
        out.zero_()
    else:
        with _on(q.device):
            _lib.check(_L.fable_linear_attn_step(p, dt, _stream(q)), "fable_linear_attn_step")
    return out, p, dt


# ----------------------------------------------------------------------------- rotation
def rotary(q, k, cos, sin, interleaved, cu=None, start=None, conj=False):
    """q [B,S,H,D] (or [total,H,D] with cu) and k (may be None) turned by the tables' rows at their positions.
    Returns (q, k, the launch's parameters and dtype), dense."""
    packed, dev = cu is not None, q.device
    _req(q.is_cuda, "GPU tensors required")
    _req(q.dim() == (3 if packed else 4), "q: [B,S,H,D], or [total,H,D] with cu_seqlens")
    for n, t in (("q", q),) + ((("k", k),) if k is not None else ()):
        _req(t.dim() == q.dim() and t.dtype == q.dtype and t.device == dev and t.shape[:-2] == q.shape[:-2] and t.shape[-1] == q.shape[-1],
             f"{n}: the tokens, head_dim, dtype and device of q")
        _req(t.stride(-1) == 1 or t.shape[-1] == 1, f"{n}: head_dim must be contiguous")
        _req(t.shape[-2] > 0, f"{n}: no heads")
    dt, D = _dt(q), q.shape[-1]
    rd = int(cos.shape[-1] * 2)
    _check_rotary(cos, sin, rd, D, dev)
    p = _lib.FableRotaryParams()
    if packed:
        _check_index("cu_seqlens", cu, dev)
        p.batch, p.total, p.cu = cu.numel() - 1, q.shape[0], cu.data_ptr()
        _req(p.batch >= 0, "cu_seqlens must have batch+1 entries")
    else:
        p.batch, p.n = q.shape[0], q.shape[1]
    if start is not None:
        _check_index("rotary_seqlens", start, dev, p.batch)
        p.start = start.data_ptr()
    qo = torch.empty(q.shape, dtype=q.dtype, device=dev)
    ko = torch.empty(k.shape, dtype=k.dtype, device=dev) if k is not None else None
    p.q, p.q_out, p.sq, p.sqo, p.NH = q.data_ptr(), qo.data_ptr(), _rows_strides(q, packed), _rows_strides(qo, packed), q.shape[-2]
    if k is not None:
        p.k, p.k_out, p.sk, p.sko, p.NKV = k.data_ptr(), ko.data_ptr(), _rows_strides(k, packed), _rows_strides(ko, packed), k.shape[-2]
    p.cos, p.sin, p.rotary, p.rotary_dim, p.rotary_rows = cos.data_ptr(), sin.data_ptr(), 2 if interleaved else 1, rd, cos.shape[0]
    p.HD, p.conj = D, 1 if conj else 0
    if q.numel():
        with _on(dev):
            _lib.check(_L.fable_attn_rotary(p, dt, _stream(q)), "fable_attn_rotary")
    return qo, ko, p, dt


def rotary_tables(rows, first, pairs, base, factor, original, low, high, amplitude, dev):
    """cos and sin [rows, pairs] in fp32 of positions first, first + 1, ..."""
    cos = torch.empty((rows, pairs), dtype=torch.float32, device=dev)
    sin = torch.empty_like(cos)
    p = _lib.FableRotaryTableParams(cos.data_ptr(), sin.data_ptr(), rows, first, pairs, base, factor, original, low, high, amplitude)
    with _on(cos.device):
        _lib.check(_L.fable_attn_rotary_tables(p, _stream(cos)), "fable_attn_rotary_tables")
    return cos, sin
