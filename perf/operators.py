"""The operators of a serving cache held in 8 bits, measured through the public API.

A cache row of D values is D e4m3 codes; every G consecutive tokens of a head share one e8m0 scale
(a power of two in one byte): value = code * 2^(byte - 127). Codes are (num_blocks, page, heads, D),
scales (num_blocks, heads, page / G); a dense cache is one page per sequence. Four operators:

  append  flash_attn_append_kvcache: new keys and values (padded or packed) into the cache, keys and
          queries rotated on the way; caches in 8 or 16 bits
  cache   flash_attn_with_kvcache over an 8-bit cache: one new token, several, a chunk of a prompt,
          with or without appending them
  prompt  flash_attn_varlen_func over 8-bit pages: packed prompts, part of whose keys are cached
  gather  flash_attn_gather_kvcache: the cached rows back as packed 16-bit keys and values

Where a call changes an 8-bit cache, the rows that its sequences hold come back as the values they
stand for (read through the gather, both ways). Keys and values are N(0, 1) with a size of their own
per head and larger tokens in between, as projections have them.
"""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(ROOT, "flash-attention-rdna2_amd")

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
_FP8, _E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _case(name, op, dtype, **kw):
    """A case with every field present. page 0: a dense cache of `cap` rows; group 0: a 16-bit cache;
    new tokens per sequence nlo..nhi (packed) or nhi (padded); cached keys lo..hi."""
    c = {"op": op, "dtype": dtype, "packed": False, "group": 16, "rotary": True, "interleaved": False,
         "with_q": False, "append": False, "window": -1, "softcap": 0.0}
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # One decoding step's new token of 48 requests, early in their answers: keys and queries rotated,
        # written to pages of 16 rows. Latency counts, and scales that grow inside a block.
        _case("append_step", "append", "bf16", batch=48, nlo=1, nhi=1, lo=64, hi=512, page=16, hq=64, hk=8, d=128,
              with_q=True),
        # The prompt phase of a batch of requests: some thousand tokens, packed, behind cached prefixes.
        _case("append_prompts", "append", "bf16", batch=8, nlo=16, nhi=2048, lo=0, hi=512, page=256, hq=32, hk=8,
              d=128, group=64, packed=True, with_q=True),
        # The same kind of call on a cache that stays in 16 bits.
        _case("append_16bit", "append", "fp16", batch=24, nlo=64, nhi=2048, lo=0, hi=1000, page=16, hq=32, hk=8,
              d=128, group=0, packed=True),
        # One request being answered: its new key goes into a dense cache, then one query reads 2000 keys.
        _case("decode_step", "cache", "bf16", batch=1, nlo=1, nhi=1, lo=2000, hi=2000, cap=4096, page=0, hq=32, hk=8,
              d=128, append=True),
        # A serving batch in flight: 48 requests with contexts of very different lengths.
        _case("decode_ragged", "cache", "bf16", batch=48, nlo=1, nhi=1, lo=64, hi=8192, page=16, hq=64, hk=8, d=128,
              rotary=False),
        # Long contexts: the benchmark's paged decode, its cache in half the bytes (HBM bound).
        _case("decode_long", "cache", "fp16", batch=16, nlo=1, nhi=1, lo=32768, hi=32768, page=256, hq=32, hk=8, d=128,
              group=64, rotary=False),
        # Four drafted tokens of 8 requests to verify: wide heads, windowed layers with capped logits, a scale
        # for every token.
        _case("decode_draft", "cache", "bf16", batch=8, nlo=4, nhi=4, lo=500, hi=4000, page=64, hq=16, hk=4, d=256,
              group=1, append=True, window=512, softcap=30.0),
        # A prompt taken in chunks: 512 new tokens of two requests behind up to 7000 cached keys.
        _case("prompt_chunk", "cache", "bf16", batch=2, nlo=512, nhi=512, lo=1000, hi=7000, page=256, hq=32, hk=8,
              d=128, group=64, append=True),
        # The prompt phase of a batch of requests over the paged cache (matrix-core bound).
        _case("prompt_paged", "prompt", "bf16", batch=8, nlo=16, nhi=2048, lo=0, hi=4096, page=16, hq=32, hk=8, d=128,
              packed=True, rotary=False),
        # Windowed layers with capped logits and wide heads over packed prompts.
        _case("prompt_window", "prompt", "fp16", batch=6, nlo=500, nhi=4000, lo=0, hi=1000, page=64, hq=16, hk=4, d=256,
              group=64, packed=True, rotary=False, window=512, softcap=30.0),
        # A finished request's prefix, read back to be kept elsewhere: the smallest work.
        _case("gather_one", "gather", "bf16", batch=1, nlo=0, nhi=0, lo=300, hi=300, cap=512, page=0, hq=8, hk=8, d=64,
              rotary=False),
        # A batch of requests moved to another machine.
        _case("gather_batch", "gather", "fp16", batch=16, nlo=0, nhi=0, lo=500, hi=8000, page=16, hq=32, hk=8, d=128,
              rotary=False),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above, the operators in the proportion in which they are listed."""
    op = rng.choice(["append"] * 3 + ["cache"] * 5 + ["prompt"] * 2 + ["gather"] * 2)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 4, 8])
    d = rng.choice([64, 80, 96, 128, 128, 192, 256])
    page = rng.choice([16, 16, 64, 256])
    kw = {"hq": hq, "hk": hk, "d": d, "interleaved": rng.random() < 0.3}
    if op in ("cache", "gather") and rng.random() < 0.25:
        page = 0
    if op == "append":
        nhi = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 17, 2048)])
        hi = _log_int(rng, 16, 2048)
        batch = _log_int(rng, 1, max(1, min(64, (1 << 25) // ((nhi + hi) * hk * d))))
        kw.update(packed=rng.random() < 0.6, with_q=rng.random() < 0.6, rotary=rng.random() < 0.85)
        kw.update(nlo=max(1, nhi // 8) if kw["packed"] else nhi, nhi=nhi, lo=rng.choice([0, hi // 4]), hi=hi)
        kw["with_q"] = kw["with_q"] and kw["rotary"]
    elif op == "gather":
        hi = _log_int(rng, 16, 32768)
        batch = _log_int(rng, 1, max(1, min(64, (1 << 27) // (hi * hk * d))))
        kw.update(nlo=0, nhi=0, lo=rng.choice([hi, hi // 8]), hi=hi, rotary=False)
    elif op == "prompt":
        nhi, hi = _log_int(rng, 64, 4096), rng.choice([1, _log_int(rng, 64, 8192)])
        nhi = min(nhi, max(64, int(1e11 / ((nhi + hi) * hq * d))))
        batch = _log_int(rng, 1, max(1, min(16, int(1e11 / (nhi * (nhi + hi) * hq * d)))))
        kw.update(packed=True, nlo=rng.randint(1, 64), nhi=nhi, lo=0, hi=hi, rotary=False)
    else:
        nhi = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 17, 1024)])
        hi = _log_int(rng, 128, 32768)
        nhi = min(nhi, max(1, int(1e11 / (hi * hq * d))))
        batch = _log_int(rng, 1, max(1, min(64, (1 << 29) // (hi * hk * d), int(1e11 / (nhi * hi * hq * d)))))
        kw.update(nlo=nhi, nhi=nhi, lo=rng.choice([hi, max(1, hi // 16)]), hi=hi, append=batch * (hi + nhi) * hk * d <= (1 << 26))
        kw["rotary"] = kw["append"] and rng.random() < 0.8
    if op in ("cache", "prompt"):
        opt = rng.choice(["", "", "", "window", "softcap"])
        kw.update(window=_log_int(rng, 64, 4096) if opt == "window" else -1, softcap=30.0 if opt == "softcap" else 0.0)
    if page == 0:
        kw["cap"] = 1 << max(6, (kw["hi"] + kw["nhi"]).bit_length())
    group = min(rng.choice([1, 16, 16, 64, 256]), page or kw["cap"])
    if op == "append" and rng.random() < 0.3:
        group = 0
    return _case(None, op, dtype, batch=batch, page=page, group=group, **kw)


# ----------------------------------------------------------------------------- sizes of a case
def _spread(seed, n, lo, hi):
    """n lengths of [lo, hi], even over their range; the longest is hi."""
    r = random.Random(seed)
    v = [r.randint(min(lo, hi), hi) for _ in range(n)]
    v[r.randrange(n)] = hi
    return v


def _lengths(case):
    """(new tokens, keys held before them) of the sequences of a case, the same for every seed."""
    return _spread(11, case["batch"], case["nlo"], case["nhi"]), _spread(13, case["batch"], case["lo"], case["hi"])


def _pairs(case, n, c):
    """Visible (query, key) pairs of one head of a sequence of n new tokens behind c cached keys."""
    if case["op"] == "cache" and not case["append"]:
        spans = [(i + c, c) for i in range(n)]
    else:
        spans = [(i + c, c + i + 1) for i in range(n)]
    w = case["window"]
    return sum(max(0, hi - (max(0, pos - w) if w >= 0 else 0)) for pos, hi in spans)


def work(case):
    """Operations: two products per visible pair (4 d). Bytes: each input read and each output written once."""
    ns, cs = _lengths(case)
    hq, hk, d, g = case["hq"], case["hk"], case["d"], case["group"]
    row = 2 * hk * (d + 1.0 / g) if g else 4 * hk * d            # keys and values of a token, cached
    op, n, c = case["op"], sum(ns), sum(cs)
    if op == "append":
        return {"bytes": n * (4 * hk * d + row + (4 * hq * d if case["with_q"] else 0)), "flops": 0}
    if op == "gather":
        return {"bytes": c * (row + 4 * hk * d), "flops": 0}
    flops = sum(4 * d * hq * _pairs(case, a, b) for a, b in zip(ns, cs))
    w = case["window"]
    seen = sum(min(b + (a if case["append"] or op == "prompt" else 0), a + w if w >= 0 else 1 << 60) for a, b in zip(ns, cs))
    return {"bytes": seen * row + 4 * n * hq * d + (n * (4 * hk * d + row) if case["append"] else 0), "flops": flops}


# ----------------------------------------------------------------------------- inputs
def _exponent(amax):
    """The least e with amax <= 448 * 2^e (448 = 0.875 * 2^9, the largest e4m3), in [-126, 119]."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(-126, 119)


def _pow2(e):
    """2^e for e in [-126, 127], 0 below (pow and ldexp are an ulp off on the GPU, which moves a power of two)."""
    return ((e.int() + 127).clamp_min(0) << 23).view(torch.float32)


def _tokens(gen, shape, dtype):
    """Keys or values (..., heads, d): every head has its size, one token in 61 is three times larger."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    size = torch.rand(shape[-2], 1, generator=gen, device="cuda") * 2 - 1
    x *= torch.exp2(size).to(dtype)
    x.view(-1, *shape[-2:])[::61] *= 3
    return x


def _cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    """What a serving program holds before the call: the cache with its pages, scales and tables, the lengths,
    the rotary tables, and the new tokens."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    b, hq, hk, d, g = case["batch"], case["hq"], case["hk"], case["d"], case["group"]
    ns, cs = _lengths(case)
    s = {"case": case, "max_n": max(ns), "max_k": max(x + y for x, y in zip(ns, cs)), "total_k": 0}
    if case["page"]:
        page, per = case["page"], -(-s["max_k"] // case["page"])
        blocks = sum(-(-(x + y) // page) for x, y in zip(ns, cs))
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        table, at = torch.full((b, per), -1, dtype=torch.int32), 0   # entries past a sequence's pages name none
        for z, (x, y) in enumerate(zip(ns, cs)):
            m = -(-(x + y) // page)
            table[z, :m] = order[at:at + m]
            at += m
        s["table"] = table.cuda()
    else:
        page, blocks, s["table"] = case["cap"], b, None
    s["page"] = page
    for name in ("k", "v"):
        x = _tokens(gen, (blocks, page, hk, d), dt)
        if g:
            x = x.view(blocks, page // g, g, hk, d)
            e = _exponent(x.abs().amax(dim=(2, 4)).float())                       # (blocks, page / g, hk)
            codes = (x * _pow2(-e).to(torch.bfloat16)[:, :, None, :, None].to(dt) if dt == torch.bfloat16
                     else x.float() * _pow2(-e)[:, :, None, :, None]).to(_FP8)
            s[name + "c"] = codes.view(blocks, page, hk, d)
            s[name + "s"] = (e + 127).to(torch.uint8).transpose(1, 2).contiguous().view(_E8)
            del codes
        else:
            s[name + "c"], s[name + "s"] = x, None
        del x
    s["lens"] = torch.tensor(cs, dtype=torch.int32, device="cuda")
    held = [y + (x if case["append"] or case["op"] in ("append", "prompt") else 0) for x, y in zip(ns, cs)]
    s["cu_k"], s["total_k"] = _cu(held), sum(held)
    if case["packed"]:
        s["cu_q"] = _cu(ns)
        new = (sum(ns),)
    else:
        new = (b, max(ns))
    if case["op"] != "gather" and (case["op"] != "append" or case["with_q"]):
        s["q"] = torch.randn(new + (hq, d), generator=gen, device="cuda", dtype=dt)
    if case["op"] == "append" or case["append"]:
        s["k"], s["v"] = _tokens(gen, new + (hk, d), dt), _tokens(gen, new + (hk, d), dt)
    if case["rotary"]:
        pos = torch.arange(s["max_k"] + 1, device="cuda", dtype=torch.float64)[:, None]
        freq = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        s["cos"], s["sin"] = torch.cos(pos * freq).float(), torch.sin(pos * freq).float()
    return s


# ----------------------------------------------------------------------------- one pass
def run(state):
    """One call of an operator, and what it leaves."""
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import fable_attn as fa
    case = s["case"]
    cache = {"block_table": s["table"], "k_scale": s["ks"], "v_scale": s["vs"]}
    window = (case["window"], 0) if case["window"] >= 0 else (-1, -1)

    def held():
        return fa.flash_attn_gather_kvcache(s["kc"], s["vc"], s["cu_k"], s["total_k"], dtype=_DT[case["dtype"]], **cache)

    if case["op"] == "gather":
        return held()
    if case["op"] == "prompt":
        return fa.flash_attn_varlen_func(s["q"], s["kc"], s["vc"], s["cu_q"], s["cu_k"], s["max_n"], s["max_k"], causal=True,
                                         window_size=window, softcap=case["softcap"], **cache)
    rotary = {"rotary_cos": s["cos"], "rotary_sin": s["sin"], "rotary_interleaved": case["interleaved"]} if case["rotary"] else {}
    if case["op"] == "append":
        packed = {"cu_seqlens": s["cu_q"], "max_seqlen": s["max_n"]} if case["packed"] else {}
        q = fa.flash_attn_append_kvcache(s["k"], s["v"], s["kc"], s["vc"], s["lens"], q=s.get("q"), **packed, **cache, **rotary)
        kept = (s["kc"], s["vc"]) if not case["group"] else held()
        return {"kept": kept} if q is None else {"q": q, "kept": kept}
    out = fa.flash_attn_with_kvcache(s["q"], s["kc"], s["vc"], k=s.get("k"), v=s.get("v"), cache_seqlens=s["lens"], causal=True,
                                     window_size=window, softcap=case["softcap"], **cache, **rotary)
    return {"out": out, "kept": held()} if case["append"] else out


# -- the plain form
def _rotated(s, x, pos):
    """x (rows, heads, d) at positions pos, rotated in 32 bits."""
    x = x.float()
    if not s["case"]["rotary"]:
        return x
    c, w = s["cos"][pos][:, None], s["sin"][pos][:, None]
    if s["case"]["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * w, b * c + a * w), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * w, b * c + a * w), -1)


def _new_rows(s):
    """(sequence, position) of every new token, packed or padded."""
    case = s["case"]
    if case["packed"]:
        row = torch.arange(s["k" if "k" in s else "q"].shape[0], device="cuda")
        seq = torch.searchsorted(s["cu_q"][1:].long(), row, right=True)
        return seq, s["lens"].long()[seq] + row - s["cu_q"].long()[seq]
    row = torch.arange(case["batch"] * s["max_n"], device="cuda")
    seq = row // s["max_n"]
    return seq, s["lens"].long()[seq] + row % s["max_n"]


def _append(s, x, seq, pos, name):
    """x (rows, heads, d), in 32 bits, into the cache `name` at positions pos of sequences seq."""
    codes, scale, page, g = s[name + "c"], s[name + "s"], s["page"], s["case"]["group"]
    blk = s["table"].long()[seq, pos // page] if s["table"] is not None else seq
    if scale is None:
        codes[blk, pos % page] = x.to(codes.dtype)
        return
    nb, hk = scale.shape[0], scale.shape[1]
    subs = page // g
    at = blk * subs + pos % page // g                                     # the row's block of g tokens
    old = scale.view(torch.uint8).transpose(1, 2).reshape(nb * subs, hk).int() - 127
    amax = torch.zeros(nb * subs, hk, device="cuda").index_reduce_(0, at, x.abs().amax(-1), "amax")
    first = torch.full((nb * subs,), g, device="cuda").index_reduce_(0, at, pos % g, "amin")   # its first new row
    e = torch.where((first == 0)[:, None], _exponent(amax), torch.maximum(old, _exponent(amax)))
    e = torch.where((first == g)[:, None], old, e)
    # rows before the first new one keep their values under a scale that grew
    down = _pow2(old - e).view(nb, subs, 1, hk, 1)
    rows = codes.view(nb, subs, g, hk, -1)
    before = (torch.arange(g, device="cuda") < first[:, None]).view(nb, subs, g, 1, 1) & (down < 1)
    kept = torch.where(before, (rows.float() * down).to(_FP8).view(torch.uint8), rows.view(torch.uint8))
    rows.view(torch.uint8).copy_(kept)
    codes.view(torch.uint8)[blk, pos % page] = (x * _pow2(-e)[at][..., None]).to(_FP8).view(torch.uint8)
    scale.view(torch.uint8).copy_((e + 127).to(torch.uint8).view(nb, subs, hk).transpose(1, 2))


def _values(s, name, rows):
    """The cached values (batch, rows, heads, d) of the first `rows` positions of every sequence, in 32 bits."""
    codes, scale, page = s[name + "c"], s[name + "s"], s["page"]
    j = torch.arange(rows, device="cuda")
    if s["table"] is None:
        blk = torch.arange(s["case"]["batch"], device="cuda")[:, None]
    else:
        blk = s["table"].long()[:, j // page].clamp_min(0)
    x = codes.view(torch.uint8)[blk, j % page].view(_FP8).float()
    e = scale.view(torch.uint8).transpose(1, 2)[blk, j % page // s["case"]["group"]].int() - 127
    return x.mul_(_pow2(e)[..., None])


def _attend(s, q, delta, held):
    """Attention of q (batch, n, heads, d; 32 bits), row t at position delta + t of its sequence, over the keys
    below held (batch, n)."""
    case = s["case"]
    b, n, hq, d = q.shape
    hk, rows = case["hk"], s["max_k"]
    k = _values(s, "k", rows).permute(0, 2, 3, 1).contiguous()            # (b, hk, d, rows)
    q = q.view(b, n, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, n * (hq // hk), d).contiguous()
    p = torch.matmul(q, k).mul_(d ** -0.5).view(b, hk, n, hq // hk, rows)
    del k
    if case["softcap"]:
        p.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    j = torch.arange(rows, device="cuda")
    seen = j < held[:, :, None]
    if case["window"] >= 0:
        pos = delta[:, None] + torch.arange(n, device="cuda")
        seen &= j >= pos[:, :, None] - case["window"]
    p.masked_fill_(~seen[:, None, :, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    v = _values(s, "v", rows).transpose(1, 2).contiguous()
    out = torch.matmul(p.view(b, hk, n * (hq // hk), rows), v)
    return out.view(b, hk, n, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, n, hq, d)


def _held(s):
    """The rows that the sequences hold, packed, in the model's type."""
    dt = _DT[s["case"]["dtype"]]
    row = torch.arange(s["total_k"], device="cuda")
    seq = torch.searchsorted(s["cu_k"][1:].long(), row, right=True)
    pos = row - s["cu_k"].long()[seq]
    return tuple(_values(s, x, s["max_k"])[seq, pos].to(dt) for x in ("k", "v"))


def _run_plain(s):
    case = s["case"]
    dt, b = _DT[case["dtype"]], case["batch"]
    if case["op"] == "gather":
        return _held(s)
    if case["op"] == "prompt":
        n = s["cu_q"][1:].long() - s["cu_q"][:-1].long()
        t = torch.arange(s["max_n"], device="cuda")
        row = torch.minimum(s["cu_q"][:-1].long()[:, None] + t, s["cu_q"][-1].long() - 1)
        delta = (s["cu_k"][1:] - s["cu_k"][:-1]).long() - n
        out = _attend(s, s["q"].float()[row], delta, (delta[:, None] + t + 1).minimum((delta + n)[:, None]))
        seq, pos = _new_rows(s)
        return out[seq, pos - s["lens"].long()[seq]].to(dt)
    seq, pos = _new_rows(s)
    q = _rotated(s, s["q"].reshape(-1, case["hq"], case["d"]), pos) if "q" in s else None
    if "k" in s:
        _append(s, _rotated(s, s["k"].reshape(-1, case["hk"], case["d"]), pos), seq, pos, "k")
        _append(s, s["v"].reshape(-1, case["hk"], case["d"]).float(), seq, pos, "v")
    if case["op"] == "append":
        kept = (s["kc"], s["vc"]) if not case["group"] else _held(s)
        return {"kept": kept} if q is None else {"q": q.to(dt).view(s["q"].shape), "kept": kept}
    q = q.view(b, s["max_n"], case["hq"], case["d"])
    delta, t = s["lens"].long(), torch.arange(s["max_n"], device="cuda")
    held = (delta[:, None] + t + 1) if case["append"] else delta[:, None].expand(b, s["max_n"])
    out = _attend(s, q, delta, held).to(dt)
    return {"out": out, "kept": _held(s)} if case["append"] else out


# ----------------------------------------------------------------------------- the same in 64 bits
def _power(e):
    """2^e in float64, e whole and in a double's range."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _code_values():
    """The 128 codes without sign: eight steps per power of two, the last is no number."""
    v = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    v[127] = math.nan
    return torch.tensor(v, dtype=torch.float64, device="cuda")


def _nearest(x):
    """x (float64, at most 448 in size) at the nearest value of a code, ties to the even code."""
    v = _code_values()[:127]
    mid = (v[1:] + v[:-1]) / 2
    a = x.abs().contiguous()
    i = torch.searchsorted(mid, a)
    tie = mid[i.clamp_max(125)] == a
    i = torch.where(tie & (i % 2 == 1), i + 1, i)
    return torch.copysign(v[i], x)


def _turn(s, x, pos):
    """x (n, heads, d; float64) turned by the angles of its positions."""
    if not s["case"]["rotary"]:
        return x
    z = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    d = x.shape[-1]
    pair = x.unflatten(-1, (d // 2, 2)) if s["case"]["interleaved"] else x.unflatten(-1, (2, d // 2)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
    return y.flatten(-2) if s["case"]["interleaved"] else y.transpose(-1, -2).flatten(-2)


def _cached(s, name, z, rows):
    """The first `rows` cached rows of sequence z in float64, with their scales' exponents (rows, heads)."""
    page, g = s["page"], s["case"]["group"]
    pages = torch.tensor([z], device="cuda") if s["table"] is None else s["table"][z, :-(-rows // page)].long()
    codes = s[name + "c"].view(torch.uint8)[pages].flatten(0, 1)[:rows].long()
    table = _code_values()
    x = torch.where(codes >= 128, -table[codes % 128], table[codes % 128])
    e = s[name + "s"].view(torch.uint8)[pages].repeat_interleave(g, -1).transpose(1, 2).flatten(0, 1)[:rows].long() - 127
    return x * _power(e)[..., None], e


def _written(s, name, z, old, x):
    """The values that sequence z holds after x (n, heads, d) is appended to its `old` cached rows."""
    g, n = s["case"]["group"], x.shape[0]
    val, e = _cached(s, name, z, old)
    first = old // g * g                                                   # the block that the first new row is in
    rows = torch.cat((val[first:], x))
    blocks = -(-rows.shape[0] // g)
    rows = torch.nn.functional.pad(rows, (0, 0, 0, 0, 0, blocks * g - rows.shape[0])).unflatten(0, (blocks, g))
    new = (torch.arange(blocks * g, device="cuda") >= old - first).view(blocks, g, 1, 1)
    top = (rows.abs() * new).amax(dim=(1, 3))                              # (blocks, heads)
    need = torch.ceil(torch.log2(top.clamp_min(1e-60) / 448))
    need = torch.where(448 * _power(need - 1) >= top, need - 1, need)      # (log2 rounds)
    need = torch.where(448 * _power(need) < top, need + 1, need).clamp(-126, 119)
    if old % g:
        need[0] = torch.maximum(need[0], e[first].double())
    step = _power(need)[:, None, :, None]
    return torch.cat((val[:first], (_nearest(rows / step) * step).flatten(0, 1)[:old + n - first]))


def exact(case, seed):
    """What run() returns for these inputs, in float64, a sequence and a head at a time."""
    s = prepare(case, seed)
    ns, cs = _lengths(case)
    hq, hk, d = case["hq"], case["hk"], case["d"]
    outs, qs, ks, vs = [], [], [], []
    pools = [s["kc"].double(), s["vc"].double()] if not case["group"] else None
    at = 0
    for z, (n, c) in enumerate(zip(ns, cs)):
        take = (lambda t: t[at:at + n]) if case["packed"] else (lambda t: t[z])
        pos = torch.arange(c, c + n, device="cuda")
        q = _turn(s, take(s["q"]).double(), pos) if "q" in s else None
        if q is not None:
            qs.append(q)
        new = [_turn(s, take(s["k"]).double(), pos), take(s["v"]).double()] if "k" in s else None
        at += n
        if pools:
            pages = s["table"][z, pos // s["page"]].long() if s["table"] is not None else torch.full_like(pos, z)
            for pool, x in zip(pools, new):
                pool[pages, pos % s["page"]] = x
            continue
        if new:
            k, v = (_written(s, name, z, c, x) for name, x in zip("kv", new))
        else:
            rows = c + (n if case["op"] == "prompt" else 0)
            k, v = _cached(s, "k", z, rows)[0], _cached(s, "v", z, rows)[0]
        ks.append(k)
        vs.append(v)
        if case["op"] in ("append", "gather"):
            continue
        rows = k.shape[0]
        last = pos[:, None] if new or case["op"] == "prompt" else torch.full((n, 1), rows - 1, device="cuda")
        j = torch.arange(rows, device="cuda")[None]
        hidden = j > last
        if case["window"] >= 0:
            hidden |= j < pos[:, None] - case["window"]
        out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
        for h in range(hq):
            w = (q[:, h] @ k[:, h // (hq // hk)].t()) / math.sqrt(d)
            if case["softcap"]:
                w = torch.tanh(w / case["softcap"]) * case["softcap"]
            w = w.masked_fill_(hidden, -math.inf)
            w = w.sub_(torch.logsumexp(w, 1, keepdim=True).clamp_min(-1e300)).exp_()
            out[:, h] = w @ v[:, h // (hq // hk)]
        outs.append(out)
    joined = (lambda x: torch.cat(x)) if case["packed"] else (lambda x: torch.stack(x))
    kept = tuple(pools) if pools else (torch.cat(ks), torch.cat(vs))
    if case["op"] == "gather":
        return kept
    if case["op"] == "append":
        return {"q": joined(qs), "kept": kept} if qs else {"kept": kept}
    return {"out": joined(outs), "kept": kept} if case["append"] else joined(outs)
