"""Plain implementations in 64 bits (torch on the CPU) of the operators over a cache held in 8 bits, and the
bounds that the kernels' roundings allow.

Codes are e4m3 (torch.float8_e4m3fn), scales e8m0 bytes; a cache is (blocks, page, heads, d) codes and (blocks,
heads, page / G) scales. Every pool starts as NaN codes under scale byte 255 (itself no number), so a row that
a call has no business with poisons whatever reads it."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative

_V = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
CODES = torch.tensor(_V + [-v for v in _V], dtype=torch.float64)
CODES[127] = CODES[255] = math.nan
_MID = (CODES[1:127] + CODES[:126]) / 2


def quantize(x):
    """Codes of x (float64, at most 448 in size or not finite): nearest, ties to even; not finite: NaN."""
    a = x.abs()
    i = torch.searchsorted(_MID, torch.nan_to_num(a, nan=0.0, posinf=0.0).contiguous())
    tie = _MID[i.clamp_max(125)] == a
    i = torch.where(tie & (i % 2 == 1), i + 1, i)
    i = torch.where(torch.isfinite(x), i, torch.full_like(i, 127))
    return (i + 128 * torch.signbit(x)).to(torch.uint8)


def least_exponent(amax):
    """The least e in [-126, 119] with amax <= 448 * 2^e."""
    if amax == 0:
        return -126
    e = -126
    while e < 119 and amax > 448 * 2.0 ** e:
        e += 1
    return e


class Pool:
    """A cache on the CPU: codes and scale bytes of K and V, a block table, and how many rows each sequence holds."""

    def __init__(self, batch, max_blocks, page, heads, d, group, seed, spare=2, dense=False):
        g = torch.Generator().manual_seed(seed)
        self.page, self.group, self.dense = page, group, dense
        nb = batch * max_blocks + (0 if dense else spare)
        shape = (nb, page, heads, d)
        self.codes = [torch.full(shape, 0x7F, dtype=torch.uint8) for _ in range(2)]
        self.scales = [torch.full((nb, heads, page // group), 255, dtype=torch.uint8) for _ in range(2)]
        if dense:
            self.table = torch.arange(batch, dtype=torch.int32).view(batch, 1)
        else:
            self.table = torch.randperm(nb, generator=g)[:batch * max_blocks].to(torch.int32).view(batch, max_blocks)

    def at(self, b, pos):
        return int(self.table[b, pos // self.page]), pos % self.page

    def append(self, b, start, k, v, leftpad=0, clamp=None):
        """Rows k, v (n, heads, d; float64, rotated) of sequence b at positions start.."""
        for codes, scales, x in zip(self.codes, self.scales, (k, v)):
            n, heads = x.shape[:2]
            if clamp is not None:
                x = torch.where(torch.isfinite(x), x.clamp(-clamp, clamp), x)
            pos = start
            while pos < start + n:
                s = pos // self.group * self.group
                stop = min(s + self.group, start + n)
                blk, row = self.at(b, s)
                old = max(s, leftpad)
                for h in range(heads):
                    new = x[pos - start:stop - start, h]
                    a = new[torch.isfinite(new)].abs()
                    e = least_exponent(float(a.max()) if a.numel() else 0.0)
                    if pos > old:
                        was = int(scales[blk, h, row // self.group]) - 127
                        if was < e:
                            r = slice(row + old - s, row + pos - s)
                            codes[blk, r, h] = quantize(CODES[codes[blk, r, h].long()] * 2.0 ** (was - e))
                        e = max(e, was)
                    codes[blk, row + pos - s:row + stop - s, h] = quantize(new * 2.0 ** -e)
                    scales[blk, h, row // self.group] = e + 127
                pos = stop

    def values(self, b, start, stop):
        """(K, V) of positions start..stop of sequence b, float64 (n, heads, d)."""
        out = []
        for codes, scales in zip(self.codes, self.scales):
            rows = []
            for pos in range(start, stop):
                blk, row = self.at(b, pos)
                rows.append(CODES[codes[blk, row].long()] * 2.0 ** (scales[blk, :, row // self.group].double() - 127)[:, None])
            out.append(torch.stack(rows) if rows else torch.zeros((0,) + codes.shape[2:], dtype=torch.float64))
        return out

    def cuda(self, cu=None):
        """(k_cache, v_cache, k_scale, v_scale, block_table) on the GPU."""
        c = [x.cuda().view(torch.float8_e4m3fn) for x in self.codes]
        s = [x.cuda().view(torch.float8_e8m0fnu) for x in self.scales]
        return c[0], c[1], s[0], s[1], None if self.dense else self.table.cuda()


def rotate(x, cos, sin, pos, interleaved):
    """x (n, heads, d; float64) rotated at rows pos (a list) of the tables (fp32), over their width."""
    half = cos.shape[1]
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * c - b * s, b * c + a * s
    return out


def rotated_size(x, cos, sin, pos, interleaved):
    """|x c| + |y s| of every rotated value: two products and their sum in fp32 are off by 3 * 2^-24 of it at most."""
    a = rotate(x.abs(), cos.abs(), 0 * sin, pos, interleaved)        # |x c|, both halves of a pair
    flip = rotate(x.abs(), 0 * cos, sin.abs(), pos, interleaved)     # -|y s| and |x s|
    return a.abs() + flip.abs()


def tables(rows, half, seed=3):
    ang = torch.randn(rows, half, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 3
    return torch.cos(ang).float(), torch.sin(ang).float()


def attend(q, k, v, lo, hi, pos, scale, softcap=0.0, slopes=None, two_part_q=False):
    """q (n, hq, d), k and v (m, hk, d), float64: row t sees keys lo[t] .. hi[t] - 1 and stands at pos[t]. Returns
    (out, lse, allowed error of out before its own rounding and without that of P, P's weight sum p|v|, allowed
    error of lse). A row that sees nothing: 0, -inf."""
    n, hq, d = q.shape
    m, hk = k.shape[:2]
    g = hq // hk
    out, lse = torch.zeros(n, hq, d, dtype=torch.float64), torch.full((n, hq), -math.inf, dtype=torch.float64)
    err, weight, lerr = torch.zeros_like(out), torch.zeros_like(out), torch.zeros(n, hq, dtype=torch.float64)
    for t in range(n):
        a, b = max(lo[t], 0), min(hi[t], m)
        if a >= b:
            continue
        j = torch.arange(a, b, dtype=torch.float64)
        for h in range(hq):
            kk, vv = k[a:b, h // g], v[a:b, h // g]
            s = kk @ q[t, h] * scale
            # scores: products in fp32 (d additions, the scale, the slope), a rotated q in two 16-bit parts
            size = (kk.abs() @ q[t, h].abs()).max() * scale
            delta = float(size) * ((d + 8) * 2.0 ** -24 + (2.0 ** -16 if two_part_q else 0.0)) + 2.0 ** -20
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                delta += softcap * 2.0 ** -20
            if slopes is not None:
                s = s + float(slopes[h]) * (j - pos[t])
                delta += float((abs(float(slopes[h])) * (j - pos[t]).abs()).max()) * 2.0 ** -22
            mx = s.max()
            delta += float(abs(mx)) * 2.0 ** -22
            p = torch.exp(s - mx)
            l = p.sum()
            out[t, h], lse[t, h] = (p / l) @ vv, mx + torch.log(l)
            weight[t, h] = (p / l) @ vv.abs()
            # exp within 2 ulp and sums of (b - a) terms, both relative
            err[t, h] = weight[t, h] * (2 * delta + (b - a + 16) * 2.0 ** -23)
            lerr[t, h] = 2 * delta + (b - a + 16) * 2.0 ** -23 + float(abs(lse[t, h])) * 2.0 ** -22
    return out, lse, err, weight, lerr


def close(got, want, err, weight, dtype, p_half, name=""):
    """got (of `dtype`) within its own rounding, P's (p_half relative to every p|v|) and err of want."""
    got = got.detach().cpu().double()
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    tol = HALF[dtype] * (want.abs() + err) + p_half * weight + err + tiny
    bad = (got - want).abs() > tol
    assert not bad.any() and not torch.isnan(got).any(), (
        name, int(bad.sum()), float(((got - want).abs() / tol.clamp_min(1e-300)).max()))
