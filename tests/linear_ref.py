"""Linear attention with a decay per head and the rotation of queries and keys, in 64 bits on the CPU, and the bounds that the kernels' results
are held to."""
import math

import torch

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def unit(dtype):
    """Half a step of a type, relative to the value: what one rounding is off by at most."""
    return torch.finfo(dtype).eps / 2


def shared(x, heads):
    """(n, heads_k, d) with each head repeated for the heads of queries that read it."""
    return x.repeat_interleave(heads // x.shape[-2], dim=-2)


def one(q, k, v, decay, scale, state=None):
    """One sequence: q (n, H, dk), k (n, Hk, dk), v (n, Hk, dv), decay (H), state (H, dk, dv) -> out (n, H, dv) and the state behind
    the last row. By the definition: all pairs of rows, weights exp(-decay (t - s))."""
    n, H = q.shape[0], q.shape[1]
    k, v = shared(k, H), shared(v, H)
    t = torch.arange(n, dtype=torch.float64)
    far = (t[:, None] - t).clamp_min(0)
    w = torch.where(far * decay[:, None, None] == far * decay[:, None, None], torch.exp(-far * decay[:, None, None]), torch.ones(()).double())
    w = torch.where((t[:, None] >= t)[None], w, torch.zeros(()).double())
    p = torch.einsum("thd,shd->hts", q, k) * w
    out = torch.einsum("hts,she->the", p, v) * scale
    left = torch.where(((n - 1 - t) * decay[:, None]) == ((n - 1 - t) * decay[:, None]), torch.exp(-(n - 1 - t) * decay[:, None]), torch.ones(()).double())
    final = torch.einsum("hs,shd,she->hde", left, k, v)
    if state is not None:
        gone = torch.exp(-(t + 1)[:, None] * decay)                                # (n, H)
        out = out + scale * torch.einsum("thd,th,hde->the", q, gone, state)
        final = final + (torch.exp(-n * decay)[:, None, None] * state if n else state)
    return out, final


def batch(q, k, v, decay, scale, cu=None, state=None):
    """Dense (cu None) or packed; all in float64. Rows of no sequence are zeros."""
    if decay.dim() == 1:
        n = q.shape[0] if cu is None else len(cu) - 1
        decay = decay.expand(n, -1)
    if cu is None:
        got = [one(q[b], k[b], v[b], decay[b], scale, None if state is None else state[b]) for b in range(q.shape[0])]
        return torch.stack([g[0] for g in got]), torch.stack([g[1] for g in got])
    got = [one(q[cu[b]:cu[b + 1]], k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]], decay[b], scale, None if state is None else state[b])
           for b in range(len(cu) - 1)]
    zeros = lambda n: torch.zeros(n, q.shape[1], v.shape[2], dtype=torch.float64)
    return torch.cat([zeros(cu[0])] + [g[0] for g in got] + [zeros(q.shape[0] - cu[-1])]), torch.stack([g[1] for g in got])


def sums(q, k, v, decay, scale, cu=None, state=None):
    """The same of absolute values: what the roundings of operands are relative to."""
    a = lambda x: None if x is None else x.abs()
    return batch(a(q), a(k), a(v), decay, abs(scale), cu, a(state))


def bound(want, size, dtype, rows, dk):
    """How far an output of `dtype` may be from `want`. size: the same sum of absolute values. One rounding of the output
    (unit |want|); in 16 bits one of each weighted score or of each state value as an operand (unit size, each term passes one of
    them); sums in 32 bits: a score has dk terms, an output 64 and dk, a state a chunk's 64 terms and one multiply-add per
    chunk of 32 rows or more, weights and their exponents 16 roundings, each 2^-24 of the terms' size."""
    u = unit(dtype)
    f32 = 2.0 ** -24 * (2 * dk + 128 + rows / 16 + 16)
    return u * want.abs() + ((u if dtype != torch.float32 else 0.0) + f32) * size * (1 + u) + torch.finfo(dtype).smallest_normal * u * 2


def state_bound(size, dtype, rows, dk):
    """A state: its operands are split without loss (bf16, fp32) or to two parts of 11 bits (fp16: 2^-22 of each term), sums as above."""
    return (2.0 ** -24 * (128 + rows / 16 + 16) + (2.0 ** -22 if dtype == torch.float16 else 0.0)) * size + 1e-37


def check(got, want, tol, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - tol
    worst = float(((got - want).abs() / tol.clamp_min(1e-300)).max()) if got.numel() else 0.0
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} of {over.numel()} values off, the worst {worst:.2f} times its bound"
    return worst


def rotated(x, cos, sin, pos, interleaved, conj=False):
    """x (tokens, heads, d) at table rows pos, float64: pairs of columns as complex numbers."""
    rd = 2 * cos.shape[1]
    turn = torch.complex(cos[pos], -sin[pos] if conj else sin[pos])[:, None]
    x = x.clone()
    i, j = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    z = torch.complex(x[..., i].contiguous(), x[..., j].contiguous()) * turn
    x[..., i], x[..., j] = z.real, z.imag
    return x


def frequencies(rotary_dim, base=10000.0, factor=1.0, original=None, low=1.0, high=32.0):
    out = []
    for i in range(rotary_dim // 2):
        f = base ** (-2 * i / rotary_dim)
        if factor != 1.0:
            keep = min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low))) if original else 0.0
            f = f * (keep + (1 - keep) / factor)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64)
