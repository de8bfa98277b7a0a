"""The operators over a cache held in 8 bits against plain 64-bit implementations (tests/cache8_ref.py): append,
gather, decode and packed prompts, alone and as they are used together. Pools start as NaN codes under a scale byte
that is no number, so whatever a call reads or writes beside its rows shows."""
import math
import random

import pytest
import torch

from tests import cache8_ref as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _fa():
    import fable_attn
    return fable_attn


def _rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale).to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(lens):
    return _i32([sum(lens[:i]) for i in range(len(lens) + 1)])


def _filled(lens, max_blocks, page, heads, d, group, dtype, seed, scale=2.0, dense=False, leftpad=None):
    """A pool that holds lens[b] rows of every sequence (from leftpad[b] on), written in one go."""
    pool = ref.Pool(len(lens), max_blocks, page, heads, d, group, seed, dense=dense)
    for b, n in enumerate(lens):
        lo = leftpad[b] if leftpad else 0
        if n > lo:
            k, v = (_rand((n - lo, heads, d), dtype, 1000 * seed + 2 * b + i, scale).double() for i in range(2))
            pool.append(b, lo, k, v, leftpad=lo)
    return pool


def _same_pool(pool, got, exact, moved=0.0):
    """The pool on the GPU against the plain one: scales equal, codes equal (or, of rotated keys, up to a share
    `moved` of them one step away: the rotation's fp32 rounding may cross a border between two codes)."""
    for name, want_c, want_s, c, s in zip("kv", pool.codes, pool.scales, got[:2], got[2:4]):
        c, s = c.view(torch.uint8).cpu(), s.view(torch.uint8).cpu()
        assert torch.equal(s, want_s), (name, int((s != want_s).sum()))
        no = lambda x: torch.where((x & 127) == 127, torch.full_like(x, 127), x)   # (a NaN code may have either sign)
        diff = no(c) != no(want_c)
        if name == "k" and not exact:
            assert diff.double().mean() <= moved, float(diff.double().mean())
            assert ((c.int() - want_c.int()).abs()[diff] <= 1).all()
        else:
            assert not diff.any(), (name, int(diff.sum()))


# ----------------------------------------------------------------------------- append
APPENDS = [
    # d, page, group, new tokens per sequence, cached rows per sequence
    (64, 16, 16, [1, 1, 1], [0, 5, 31]),
    (128, 16, 16, [3, 0, 40], [15, 7, 1]),
    (128, 16, 1, [1, 9, 33], [0, 16, 30]),
    (128, 64, 64, [70, 1, 64], [3, 64, 0]),
    (128, 256, 256, [300, 5], [250, 0]),
    (256, 16, 4, [5, 20], [2, 61]),
    (256, 64, 32, [33, 1], [31, 32]),
    (80, 32, 8, [1, 17, 50], [7, 8, 9]),
    (192, 16, 2, [2, 19], [13, 14]),
    (16, 32, 32, [40, 3], [1, 30]),
    (96, 128, 128, [130, 2], [127, 100]),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"d{c[0]}p{c[1]}g{c[2]}")
def test_append_packed(case, dtype):
    d, page, group, new, held = case
    dt, heads = DT[dtype], 3
    blocks = max(-(-(n + c) // page) for n, c in zip(new, held))
    pool = _filled(held, blocks, page, heads, d, group, dt, 5, scale=0.5)
    k, v = (_rand((sum(new) + 2, heads, d), dt, 11 + i, 2.0) for i in range(2))   # two rows behind the last sequence
    dev = pool.cuda()
    _fa().flash_attn_append_kvcache(k.cuda(), v.cuda(), *dev[:2], _i32(held), cu_seqlens=_cu(new), max_seqlen=max(new),
                                    block_table=dev[4], k_scale=dev[2], v_scale=dev[3])
    at = 0
    for b, (n, c) in enumerate(zip(new, held)):
        pool.append(b, c, k[at:at + n].double(), v[at:at + n].double())
        at += n
    _same_pool(pool, dev, exact=True)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rdim", [(128, 128), (128, 64), (64, 20), (80, 80), (256, 128), (96, 36), (192, 192)])
def test_append_rotated(d, rdim, interleaved):
    """Keys and queries rotated, padded batch, strided tokens (slices of one projection), a dense cache."""
    dt, heads, hq, group, page, n = torch.bfloat16, 2, 4, 16, 64, 5
    held = [0, 14, 50]
    pool = _filled(held, 1, page, heads, d, group, dt, 2, dense=True)
    cos, sin = ref.tables(page, rdim // 2)
    qkv = _rand((3, n, hq + 2 * heads, d), dt, 9)
    q, k, v = qkv.cuda().split((hq, heads, heads), 2)
    dev = pool.cuda()
    got = _fa().flash_attn_append_kvcache(k, v, *dev[:2], _i32(held), q=q, rotary_cos=cos.cuda(), rotary_sin=sin.cuda(),
                                          rotary_interleaved=interleaved, k_scale=dev[2], v_scale=dev[3])
    assert got.shape == q.shape and got.is_contiguous()
    for b, c in enumerate(held):
        pos = list(range(c, c + n))
        rk = ref.rotate(k[b].cpu().double(), cos, sin, pos, interleaved)
        pool.append(b, c, rk, v[b].cpu().double())
        want = ref.rotate(q[b].cpu().double(), cos, sin, pos, interleaved)
        size = ref.rotated_size(q[b].cpu().double(), cos, sin, pos, interleaved)
        assert ((got[b].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * 2.0 ** -24 * size).all()
    _same_pool(pool, dev, exact=False, moved=1e-3)


def test_append_growing_scales_token_by_token():
    """A block whose tokens get larger: older rows follow the scale, in any order of sizes."""
    dt, heads, d, group, page = torch.bfloat16, 2, 128, 16, 32
    pool = ref.Pool(2, 2, page, heads, d, group, 1)
    dev = pool.cuda()
    r = random.Random(4)
    for t in range(40):
        k, v = (_rand((2, 1, heads, d), dt, 50 + 2 * t + i, 2.0 ** r.randint(-6, 6)) for i in range(2))
        _fa().flash_attn_append_kvcache(k.cuda(), v.cuda(), *dev[:2], t, block_table=dev[4], k_scale=dev[2], v_scale=dev[3])
        for b in range(2):
            pool.append(b, t, k[b].double(), v[b].double())
    _same_pool(pool, dev, exact=True)


def test_append_values_that_are_not_finite_or_extreme():
    """NaN and infinities become NaN codes and set no scale; zeros, the least and the largest values hold."""
    heads, d, group, page = 1, 64, 4, 16
    for dt in DT.values():
        big = float(torch.finfo(dt).max)
        x = _rand((12, heads, d), dt, 3)
        x[0, 0, 5], x[1, 0, 0], x[2, 0, 1] = math.nan, math.inf, -math.inf
        x[4:8] = 0
        x[8, 0, :3] = torch.tensor([big, -big, big / 2], dtype=dt)
        x[9, 0, 0] = float(torch.finfo(dt).tiny)
        pool = ref.Pool(1, 1, page, heads, d, group, 0)
        dev = pool.cuda()
        _fa().flash_attn_append_kvcache(x[None].cuda(), x[None].cuda(), *dev[:2], 0, block_table=dev[4], k_scale=dev[2], v_scale=dev[3])
        pool.append(0, 0, x.double(), x.double(), clamp=61440.0 if dt == torch.float16 else 448 * 2.0 ** 119)
        _same_pool(pool, dev, exact=True)
        back, _ = _fa().flash_attn_gather_kvcache(*dev[:2], _cu([12]), 12, block_table=dev[4], k_scale=dev[2], v_scale=dev[3], dtype=dt)
        assert torch.equal(torch.isfinite(back).cpu(), torch.isfinite(x))


def test_append_leftpad_starts_a_block_afresh():
    """The rows ahead of a left pad are no rows of the sequence: their scale does not count."""
    dt, heads, d, group, page = torch.bfloat16, 2, 64, 16, 32
    pool = ref.Pool(2, 1, page, heads, d, group, 0)
    dev = pool.cuda()
    k, v = (_rand((2, 3, heads, d), dt, i) for i in range(2))
    pads = [5, 21]
    _fa().flash_attn_append_kvcache(k.cuda(), v.cuda(), *dev[:2], _i32(pads), block_table=dev[4], cache_leftpad=_i32(pads),
                                    k_scale=dev[2], v_scale=dev[3])
    for b in range(2):
        pool.append(b, pads[b], k[b].double(), v[b].double(), leftpad=pads[b])
    _same_pool(pool, dev, exact=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 72, 128, 256])
def test_append_and_gather_of_a_16_bit_cache(d, dtype):
    """Caches without scales: strided pages (keys and values side by side), rotated keys, the rest as it was."""
    heads, page, new, held = 2, 16, [1, 0, 70], [15, 3, 20]
    blocks = 6
    table = torch.randperm(3 * blocks, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(3, blocks)
    pool = torch.full((3 * blocks, 2, page, heads, d), 7.0, dtype=dtype, device="cuda")
    kc, vc = pool[:, 0], pool[:, 1]
    k, v = (_rand((sum(new), heads, d), dtype, i) for i in range(2))
    cos, sin = ref.tables(128, d // 2)
    _fa().flash_attn_append_kvcache(k.cuda(), v.cuda(), kc, vc, _i32(held), cu_seqlens=_cu(new), max_seqlen=70,
                                    block_table=table.cuda(), rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), rotary_interleaved=False)
    want = torch.full(pool.shape, 7.0, dtype=torch.float64)
    at = 0
    for b, (n, c) in enumerate(zip(new, held)):
        rk = ref.rotate(k[at:at + n].double(), cos, sin, list(range(c, c + n)), False)
        for t in range(n):
            blk, row = int(table[b, (c + t) // page]), (c + t) % page
            want[blk, 0, row], want[blk, 1, row] = rk[t], v[at + t].double()
        at += n
    got = pool.cpu().double()
    assert torch.equal(got[:, 1], want[:, 1])
    assert ((got[:, 0] - want[:, 0]).abs() <= ref.HALF[dtype] * want[:, 0].abs() + 2.0 ** -21).all()
    lens = [n + c for n, c in zip(new, held)]
    gk, gv = _fa().flash_attn_gather_kvcache(kc, vc, _cu(lens), sum(lens) + 3, block_table=table.cuda())
    at = 0
    for b, n in enumerate(lens):
        for t in range(n):
            assert torch.equal(gk[at + t], kc[int(table[b, t // page]), t % page])
            assert torch.equal(gv[at + t], vc[int(table[b, t // page]), t % page])
        at += n
    assert (gk[at:] == 0).all() and (gv[at:] == 0).all()


def test_append_drops_what_has_no_place():
    """Positions past the table, entries that name no page, lengths below zero: nothing is written for them."""
    dt, heads, d, group, page = torch.bfloat16, 2, 64, 16, 16
    pool = ref.Pool(3, 2, page, heads, d, group, 0)
    pool.table[1, 1] = -1
    keep = pool.table.clone()
    dev = pool.cuda()
    bad = dev[4].clone()
    bad[2, 0] = 10 ** 6
    k, v = (_rand((3, 4, heads, d), dt, i) for i in range(2))
    _fa().flash_attn_append_kvcache(k.cuda(), v.cuda(), *dev[:2], _i32([30, 14, 2]), block_table=bad, k_scale=dev[2], v_scale=dev[3])
    pool.table = keep
    before = [x.clone() for x in pool.codes]
    for name, x, c in (("k", k, 0), ("v", v, 1)):
        got = dev[c].view(torch.uint8).cpu()
        changed = (got != before[c]).any(dim=(2, 3))
        want = torch.zeros_like(changed)
        want[int(keep[0, 1]), 14:16] = True     # positions 30 and 31; 32 and 33 are past the table
        want[int(keep[1, 0]), 14:16] = True     # 14 and 15; 16 and 17 are in a page that is not there
        assert torch.equal(changed, want), name
    _fa().flash_attn_append_kvcache(k.cuda(), v.cuda(), *dev[:2], _i32([-2, 50, 32]), block_table=dev[4], k_scale=dev[2], v_scale=dev[3])
    again = (dev[1].view(torch.uint8).cpu() != before[1]).any(dim=(2, 3))
    assert bool(again[int(keep[0, 0]), :2].all())    # tokens 2 and 3 of sequence 0 are at positions 0 and 1
    assert not again[int(keep[2, 0])].any() and not again[int(keep[2, 1])].any()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 8, 16, 32, 64, 128, 256])
def test_append_turns_every_query(group, d):
    """Queries ride along whatever the block's length: every token comes back, packed, the sequences of any length."""
    dt, heads, hq, page = torch.bfloat16, 2, 6, 256
    new, held = [1, 300, 0, 70], [5, 250, 9, 256]
    pool = ref.Pool(4, 3, page, heads, d, group, 1)
    c = pool.cuda()
    cos, sin = ref.tables(600, d // 2)
    q, k, v = (_rand((sum(new), h, d), dt, i) for i, h in enumerate((hq, heads, heads)))
    got = _fa().flash_attn_append_kvcache(k.cuda(), v.cuda(), *c[:2], _i32(held), q=q.cuda(), cu_seqlens=_cu(new), max_seqlen=max(new),
                                          block_table=c[4], rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), rotary_interleaved=False,
                                          k_scale=c[2], v_scale=c[3]).cpu().double()
    pos = [c0 + t for n, c0 in zip(new, held) for t in range(n)]
    want = ref.rotate(q.double(), cos, sin, pos, False)
    size = ref.rotated_size(q.double(), cos, sin, pos, False)
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 4 * 2.0 ** -24 * size).all()


# ----------------------------------------------------------------------------- gather
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,page,group", [(64, 16, 16), (128, 64, 1), (256, 32, 8), (80, 256, 256), (16, 16, 2)])
def test_gather(d, page, group, dtype):
    lens = [0, 1, 37, page, 2 * page + 1]
    pool = _filled(lens, 3, page, 3, d, group, DT[dtype], 7)
    c = pool.cuda()
    k, v = _fa().flash_attn_gather_kvcache(*c[:2], _cu(lens), sum(lens) + 5, block_table=c[4], k_scale=c[2], v_scale=c[3], dtype=DT[dtype])
    assert k.dtype == DT[dtype] and k.shape == (sum(lens) + 5, 3, d)
    at = 0
    for b, n in enumerate(lens):
        for got, want in zip((k, v), pool.values(b, 0, n)):
            assert torch.equal(got[at:at + n].cpu().double(), want.to(DT[dtype]).double())   # (exact in bf16)
        at += n
    assert (k[at:] == 0).all() and (v[at:] == 0).all()


def test_gather_of_missing_pages_and_dense_rows():
    pool = _filled([40, 20], 2, 32, 2, 64, 16, torch.bfloat16, 3)
    c = pool.cuda()
    table = c[4].clone()
    table[0, 1] = -5
    k, _ = _fa().flash_attn_gather_kvcache(*c[:2], _cu([40, 70]), 110, block_table=table, k_scale=c[2], v_scale=c[3])
    assert (k[32:40] == 0).all() and (k[40 + 64:] == 0).all() and torch.isfinite(k[:32].float()).all()
    dense = _filled([9, 33, 64], 1, 64, 2, 64, 16, torch.bfloat16, 3, dense=True)
    c = dense.cuda()
    k, v = _fa().flash_attn_gather_kvcache(*c[:2], _cu([33, 9]), 42, cache_batch_idx=_i32([1, 0]), k_scale=c[2], v_scale=c[3])
    assert torch.equal(v.cpu().double(), torch.cat((dense.values(1, 0, 33)[1], dense.values(0, 0, 9)[1])))
    none, _ = _fa().flash_attn_gather_kvcache(*c[:2], _cu([0]), 0, k_scale=c[2], v_scale=c[3])
    assert none.shape == (0, 2, 64)


@pytest.mark.parametrize("batch", [2, 63, 64, 65, 200, 4100])
def test_gather_finds_the_sequence_among_many(batch):
    """Rows of many sequences, empty ones among them, all over the same few pages."""
    r = random.Random(batch)
    pool = _filled([16] * 4, 1, 16, 2, 64, 16, torch.bfloat16, 13)
    c = pool.cuda()
    lens = [r.choice([0, 0, 1, 2, 5]) for _ in range(batch)]
    which = [r.randrange(4) for _ in range(batch)]
    table = c[4][_i32(which).long()].contiguous()
    k, v = _fa().flash_attn_gather_kvcache(*c[:2], _cu(lens), sum(lens) + 3, block_table=table, k_scale=c[2], v_scale=c[3])
    want = [torch.cat([pool.values(w, 0, n)[i] for w, n in zip(which, lens)] + [torch.zeros(3, 2, 64, dtype=torch.float64)]) for i in range(2)]
    assert torch.equal(k.cpu().double(), want[0]) and torch.equal(v.cpu().double(), want[1])


# ----------------------------------------------------------------------------- decode
def _check_decode(dtype, lens, hq, hk, d, page, group, nq=1, append=False, window=-1, softcap=0.0, alibi=False, leftpad=None,
                  rotary=0, interleaved=False, dense=False, max_blocks=None, num_splits=0, lse=True, hide=True, seed=0, scale=None,
                  wide=None):
    """flash_attn_with_kvcache against the plain form, its cache too where the call appends."""
    dt, B = DT[dtype], len(lens)
    new = nq if append else 0
    blocks = 1 if dense else max_blocks or max(-(-max(n + new, 1) // page) for n in lens)
    pool = _filled(lens, blocks, page, hk, d, group, dt, 20 + seed, dense=dense, leftpad=leftpad)
    if window >= 0 and hide:   # rows that left every token's window: nothing may read them
        for b, n in enumerate(lens):
            for pos in range(0, min(max(n - window, 0), n)):
                blk, row = pool.at(b, pos)
                for c in pool.codes:
                    c[blk, row] = 0x7F
    q = _rand((B, nq, hq, d), dt, 31 + seed)
    k, v = (_rand((B, nq, hk, d), dt, 41 + seed + i) for i in range(2))
    c = pool.cuda()
    if wide:   # a wider table, as a server keeps one: its further entries are never read for a key
        c = c[:4] + type(c)([torch.cat((c[4], c[4][:, :1].expand(B, wide - c[4].shape[1])), 1).contiguous()])
    kw = {}
    cos = sin = None
    if rotary:
        cos, sin = ref.tables(max(lens) + nq + 1, rotary // 2)
        kw.update(rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), rotary_interleaved=interleaved)
    slopes = torch.tensor([2.0 ** -(1 + h % 8) for h in range(hq)]) if alibi else None
    if append:
        kw.update(k=k.cuda(), v=v.cuda())
    if leftpad:
        kw.update(cache_leftpad=_i32(leftpad))
    res = _fa().flash_attn_with_kvcache(q.cuda(), *c[:2], cache_seqlens=_i32(lens), block_table=c[4], causal=True,
                                        window_size=(window, 0) if window >= 0 else (-1, -1), softcap=softcap, softmax_scale=scale,
                                        alibi_slopes=slopes.cuda() if alibi else None, num_splits=num_splits,
                                        return_softmax_lse=lse, k_scale=c[2], v_scale=c[3], **kw)
    out, got_lse = res if lse else (res, None)
    tiles = B * hk * -(-nq * (hq // hk) // 16) > 16 and nq * (hq // hk) >= 64   # (the many-token path keeps P in q's type)
    half = ref.HALF[dt] if tiles or dt == torch.bfloat16 else 2.0 ** -16
    for b, n in enumerate(lens):
        pos = list(range(n, n + nq))
        turn = (lambda x: ref.rotate(x, cos, sin, pos, interleaved)) if rotary else (lambda x: x)
        if append:
            # (the kernel's own codes from here on: what it wrote is compared below)
            pool.append(b, n, turn(k[b].double()), v[b].double(), leftpad=leftpad[b] if leftpad else 0)
    if append:
        _same_pool(pool, c, exact=not rotary, moved=1e-3)
        pool.codes = [x.view(torch.uint8).cpu() for x in c[:2]]
    for b, n in enumerate(lens):
        pos = list(range(n, n + nq))
        qb = ref.rotate(q[b].double(), cos, sin, pos, interleaved) if rotary else q[b].double()
        kk, vv = pool.values(b, 0, n + new)
        lo = [max(leftpad[b] if leftpad else 0, p - window if window >= 0 else 0) for p in pos]
        hi = [p + 1 if append else n for p in pos]
        want, wl, err, weight, lerr = ref.attend(qb, kk, vv, lo, hi, pos, scale or d ** -0.5, softcap, slopes, bool(rotary))
        if tiles and dt == torch.float16:   # (small P, in fp16's subnormals)
            err = err + (n + new) * 2.0 ** -25 * float(vv.nan_to_num().abs().max() if vv.numel() else 0)
        ref.close(out[b], want, err, weight, dt, half, f"sequence {b}")
        if lse:
            g = got_lse[b].transpose(0, 1).cpu().double()
            assert torch.equal(torch.isinf(g), torch.isinf(wl))
            fin = torch.isfinite(wl)
            assert ((g - wl).abs()[fin] <= lerr[fin] + 2.0 ** -21).all(), float((g - wl).abs()[fin].max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,hq,hk,page,group", [
    (64, 4, 4, 16, 16), (128, 8, 2, 16, 1), (128, 16, 1, 64, 64), (256, 8, 2, 32, 8), (192, 6, 2, 256, 256), (80, 3, 1, 16, 4),
    (96, 40, 2, 16, 2), (16, 2, 2, 16, 16), (160, 4, 2, 128, 32), (224, 2, 1, 16, 16)])
def test_decode(d, hq, hk, page, group, dtype):
    _check_decode(dtype, [0, 1, 15, 16, 33, 200], hq, hk, d, page, group)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,rotary,interleaved,nq", [(128, 128, False, 1), (128, 64, True, 3), (64, 64, False, 5), (256, 256, True, 2), (80, 40, False, 1)])
def test_decode_append(d, rotary, interleaved, nq, dtype):
    _check_decode(dtype, [0, 5, 15, 31, 100], 8, 2, d, 16, 16, nq=nq, append=True, rotary=rotary, interleaved=interleaved)


@pytest.mark.parametrize("kw", [
    {"window": 10}, {"window": 40, "nq": 4, "append": True}, {"softcap": 5.0}, {"alibi": True},
    {"window": 33, "softcap": 20.0, "alibi": True, "nq": 3, "append": True}, {"leftpad": [0, 3, 64, 90]},
    {"leftpad": [0, 17, 70, 150], "nq": 2, "append": True}, {"window": 0}, {"window": 0, "append": True}, {"nq": 7},
    {"num_splits": 3}, {"num_splits": 1}, {"scale": 0.3, "softcap": 2.0},
], ids=str)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_options(kw, dtype):
    _check_decode(dtype, [0, 17, 70, 150], 8, 2, 128, 16, 8, **kw)


def test_decode_dense_cache():
    _check_decode("bf16", [0, 64, 100], 4, 2, 64, 128, 32, append=True, dense=True)
    _check_decode("fp16", [5, 127], 4, 4, 128, 128, 1, dense=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_long_splits_and_shares(dtype):
    """Splits of a long cache, and batches whose keys are shared out on the device (a large table)."""
    _check_decode(dtype, [3000], 4, 1, 64, 64, 16)
    _check_decode(dtype, [1, 2000, 17, 700, 129], 2, 1, 64, 64, 16, max_blocks=4096)
    _check_decode(dtype, [500, 0, 900], 2, 1, 64, 64, 64, max_blocks=8192, append=True, window=300, hide=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,hq,hk,d,page,wide,kw", [
    # tables of so many keys that a workgroup takes four heads, or two; shares worked out on the device (6
    # sequences) and splits (8, and one)
    ([0, 1, 300, 129, 64, 2000], 16, 8, 128, 16, 1024, {}),
    ([0, 1, 300, 129, 64, 700, 31, 33], 8, 8, 128, 64, 256, {"append": True, "rotary": 64}),
    ([0, 1, 300, 129, 64, 2000], 8, 8, 64, 64, 512, {"append": True, "window": 100, "hide": False}),
    ([5, 1, 300, 129, 64, 700, 31, 33], 32, 4, 80, 16, 2048, {"nq": 3, "append": True, "alibi": True, "softcap": 20.0}),
    ([0, 1, 300, 129, 64, 1000], 6, 6, 128, 16, 2048, {"leftpad": [0, 0, 40, 100, 63, 500], "append": True}),
    ([0, 1, 300, 129, 64, 700, 31, 33], 12, 6, 64, 32, 1024, {"alibi": True}),
    ([0, 1, 300, 129, 64, 1000], 4, 2, 192, 16, 3000, {}),
    ([700, 1, 300, 129, 64, 0, 31, 33], 4, 4, 160, 64, 512, {"append": True, "rotary": 160, "interleaved": True}),
    ([1500], 64, 32, 128, 64, 512, {}),
    ([900], 16, 16, 128, 128, 512, {"window": 500}),
], ids=str)
def test_decode_heads_of_a_workgroup(lens, hq, hk, d, page, wide, kw, dtype):
    _check_decode(dtype, lens, hq, hk, d, page, 16, wide=wide, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,kw", [
    (64, {"append": True, "rotary": 64}), (128, {"append": True, "rotary": 128, "interleaved": True}), (128, {}),
    (256, {"append": True}), (128, {"append": True, "window": 40}), (64, {"softcap": 10.0, "append": True}), (96, {"append": True}),
    (192, {"append": True}), (128, {"leftpad": [0, 10, 33], "append": True}), (128, {"rotary": 64}), (256, {"alibi": True, "append": True})])
def test_many_new_tokens(d, kw, dtype):
    """Enough rows per K/V head for the tile kernel."""
    _check_decode(dtype, [0, 40, 130], 8, 2, d, 16, 16, nq=17, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d,nq,kw", [(128, 70, {"rotary": 128}), (128, 33, {}), (64, 70, {"rotary": 64, "interleaved": True}), (96, 40, {"rotary": 32}),
                                     (64, 33, {})])
def test_many_rows_of_a_head(d, nq, kw, page, dtype):
    """Rows of a K/V head on both sides of the tall tile's half (128 rows), and past one tile."""
    _check_decode(dtype, [0, 40, 130, 7, 65], 8, 2, d, page, 16, nq=nq, append=True, **kw)


def test_decode_reads_strided_caches_and_packed_queries():
    dt, lens, hq, hk, d, page = torch.bfloat16, [40, 7], 4, 2, 64, 16
    pool = _filled(lens, 3, page, hk, d, 16, dt, 1)
    c = pool.cuda()
    both = torch.stack((c[0].view(torch.uint8), c[1].view(torch.uint8)), 1).view(torch.float8_e4m3fn)   # pages of K and V
    q = _rand((2, 2, hq, d), dt, 5).cuda()
    kw = dict(cache_seqlens=_i32(lens), block_table=c[4], k_scale=c[2], v_scale=c[3])
    want = _fa().flash_attn_with_kvcache(q, c[0], c[1], **kw)
    assert torch.equal(want, _fa().flash_attn_with_kvcache(q, both[:, 0], both[:, 1], **kw))
    packed = _fa().flash_attn_with_kvcache(q.reshape(4, hq, d), c[0], c[1], cu_seqlens_q=_cu([2, 2]), max_seqlen_q=2, **kw)
    assert torch.equal(want.reshape(4, hq, d), packed)


def test_decode_offsets_past_32_bits():
    """A cache of more than 2^32 bytes, its last pages in use; and pages far apart."""
    dt, hk, d, page, nb = torch.bfloat16, 8, 256, 256, 8200        # 4.3e9 bytes of keys
    pool = ref.Pool(1, 2, page, hk, d, 16, 1, spare=0)
    k, v = (_rand((300, hk, d), dt, i).double() for i in range(2))
    pool.append(0, 0, k, v)
    kc = torch.full((nb, page, hk, d), 0x7F, dtype=torch.uint8, device="cuda")
    ks = torch.full((nb, hk, page // 16), 255, dtype=torch.uint8, device="cuda")
    vs = ks.clone()
    vc = kc.clone()
    at = [nb - 1, nb - 2]
    for i, blk in enumerate(pool.table[0].tolist()):
        kc[at[i]], vc[at[i]], ks[at[i]], vs[at[i]] = (x[blk].cuda() for x in pool.codes + pool.scales)
    q = _rand((1, 1, hk, d), dt, 9)
    e4, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    out = _fa().flash_attn_with_kvcache(q.cuda(), kc.view(e4), vc.view(e4), cache_seqlens=_i32([300]), block_table=_i32([at]),
                                        k_scale=ks.view(e8), v_scale=vs.view(e8))
    kk, vv = pool.values(0, 0, 300)
    want, _, err, weight, _ = ref.attend(q[0].double(), kk, vv, [0], [300], [300], d ** -0.5)
    ref.close(out[0], want, err, weight, dt, 2.0 ** -8)


# ----------------------------------------------------------------------------- packed prompts
def _check_prompts(dtype, new, cached, hq, hk, d, page, group, window=(-1, -1), softcap=0.0, alibi=False, causal=True, chunk=0,
                   seqused=False, seed=0):
    dt = DT[dtype]
    total = [n + c for n, c in zip(new, cached)]
    pool = _filled(total, max(-(-max(t, 1) // page) for t in total), page, hk, d, group, dt, 60 + seed)
    c = pool.cuda()
    q = _rand((sum(new), hq, d), dt, 71 + seed)
    slopes = torch.tensor([2.0 ** -(1 + h % 8) for h in range(hq)]) if alibi else None
    used = [max(n - 2, 0) for n in new] if seqused else new
    kw = dict(seqused_q=_i32(used), seqused_k=_i32(total)) if seqused else {}
    out = _fa().flash_attn_varlen_func(q.cuda(), *c[:2], _cu(new), _cu(total), max(new), max(total), causal=causal, window_size=window,
                                       softcap=softcap, alibi_slopes=slopes.cuda() if alibi else None, attention_chunk=chunk,
                                       block_table=c[4], k_scale=c[2], v_scale=c[3], **kw)
    at = 0
    for b, (n, t, u) in enumerate(zip(new, total, used)):
        kk, vv = pool.values(b, 0, t)
        pos = [i + t - u for i in range(u)]
        lo = [max(0, p - window[0]) if window[0] >= 0 else 0 for p in pos]
        hi = [min(t, p + 1 if causal else (p + window[1] + 1 if window[1] >= 0 else t)) for p in pos]
        if chunk:
            lo = [max(a, max(p, 0) // chunk * chunk) for a, p in zip(lo, pos)]
            hi = [min(a, max(p, 0) // chunk * chunk + chunk) for a, p in zip(hi, pos)]
        rows = pos if slopes is None else list(range(u))     # (slopes count from the query's row)
        want, _, err, weight, _ = ref.attend(q[at:at + u].double(), kk, vv, lo, hi, rows, d ** -0.5, softcap, slopes)
        if dt == torch.float16:
            err = err + t * 2.0 ** -25 * float(vv.abs().max() if vv.numel() else 0)
        ref.close(out[at:at + u], want, err, weight, dt, ref.HALF[dt], f"sequence {b}")
        assert (out[at + u:at + n] == 0).all()
        at += n


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,hq,hk,page,group", [(64, 4, 2, 16, 16), (128, 4, 4, 16, 1), (128, 8, 2, 64, 64), (256, 4, 1, 32, 8),
                                                (192, 2, 1, 16, 2), (80, 3, 3, 256, 256), (16, 2, 1, 16, 4)])
def test_prompts(d, hq, hk, page, group, dtype):
    _check_prompts(dtype, [1, 70, 0, 33], [0, 0, 20, 90], hq, hk, d, page, group)


@pytest.mark.parametrize("kw", [{"window": (20, 0)}, {"softcap": 8.0}, {"alibi": True, "causal": False}, {"causal": False},
                                {"causal": False, "window": (10, 5)}, {"chunk": 32}, {"seqused": True}], ids=str)
@pytest.mark.parametrize("d", [128, 256])
def test_prompt_options(kw, d):
    _check_prompts("bf16", [5, 70, 33], [0, 50, 90], 4, 2, d, 16, 16, **kw)


def test_prompts_split_and_long():
    _check_prompts("fp16", [3], [1500], 2, 1, 64, 64, 16)
    _check_prompts("bf16", [300, 2], [0, 700], 2, 2, 128, 16, 16)


# ----------------------------------------------------------------------------- together
def test_a_serving_run():
    """Prompts appended (rotated keys and queries) and attended, then tokens one by one, then the cache read back: each
    step against the plain forms on the cache it was given."""
    fa = _fa()
    dt, hq, hk, d, page, group = torch.bfloat16, 8, 2, 128, 16, 16
    new = [37, 5, 20]
    pool = ref.Pool(3, 4, page, hk, d, group, 1)
    c = pool.cuda()
    cos, sin = ref.tables(64, d // 2)
    rot = dict(rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), rotary_interleaved=False)
    scales = dict(k_scale=c[2], v_scale=c[3])
    q, k, v = (_rand((sum(new), h, d), dt, i) for i, h in enumerate((hq, hk, hk)))
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    rq = fa.flash_attn_append_kvcache(k.cuda(), v.cuda(), *c[:2], lens, q=q.cuda(), cu_seqlens=_cu(new), max_seqlen=max(new),
                                      block_table=c[4], **rot, **scales)
    out = fa.flash_attn_varlen_func(rq, *c[:2], _cu(new), _cu(new), max(new), max(new), causal=True, block_table=c[4], **scales)
    lens += _i32(new)
    at = 0
    for b, n in enumerate(new):
        pool.append(b, 0, ref.rotate(k[at:at + n].double(), cos, sin, list(range(n)), False), v[at:at + n].double())
        at += n
    _same_pool(pool, c, exact=False, moved=1e-3)
    pool.codes = [x.view(torch.uint8).cpu() for x in c[:2]]
    at = 0
    for b, n in enumerate(new):
        kk, vv = pool.values(b, 0, n)
        want, _, err, weight, _ = ref.attend(rq[at:at + n].cpu().double(), kk, vv, [0] * n, range(1, n + 1), range(n), d ** -0.5)
        ref.close(out[at:at + n], want, err, weight, dt, 2.0 ** -8)
        at += n
    for step in range(18):
        tq, tk, tv = (_rand((3, 1, h, d), dt, 100 + 3 * step + i) for i, h in enumerate((hq, hk, hk)))
        res = fa.flash_attn_with_kvcache(tq.cuda(), *c[:2], k=tk.cuda(), v=tv.cuda(), cache_seqlens=lens, block_table=c[4],
                                         causal=True, **rot, **scales)
        at = lens.tolist()
        lens += 1
        for b in range(3):
            pool.append(b, at[b], ref.rotate(tk[b].double(), cos, sin, [at[b]], False), tv[b].double())
        _same_pool(pool, c, exact=False, moved=1e-3)
        pool.codes = [x.view(torch.uint8).cpu() for x in c[:2]]
        for b in range(3):
            kk, vv = pool.values(b, 0, at[b] + 1)
            qb = ref.rotate(tq[b].double(), cos, sin, [at[b]], False)
            want, _, err, weight, _ = ref.attend(qb, kk, vv, [0], [at[b] + 1], [at[b]], d ** -0.5, two_part_q=True)
            ref.close(res[b], want, err, weight, dt, 2.0 ** -8, f"step {step}")
    n = lens.tolist()
    gk, gv = fa.flash_attn_gather_kvcache(*c[:2], _cu(n), sum(n), block_table=c[4], **scales)
    assert torch.equal(gv.cpu().double(), torch.cat([pool.values(b, 0, n[b])[1] for b in range(3)]))
    dense = fa.flash_attn_varlen_func(rq[:3].contiguous(), gk, gv, _cu([1, 1, 1]), _cu(n), 1, max(n), causal=True)
    paged = fa.flash_attn_varlen_func(rq[:3].contiguous(), *c[:2], _cu([1, 1, 1]), _cu(n), 1, max(n), causal=True, block_table=c[4], **scales)
    assert (dense.float() - paged.float()).abs().max() <= 2.0 ** -6 * paged.float().abs().max()


def test_another_stream_and_a_graph():
    """A step captured into a graph and replayed, its workspaces from the graph's pool, beside eager calls on another
    stream; every replay is bitwise the eager call."""
    fa = _fa()
    dt, hq, hk, d, page, group = torch.bfloat16, 8, 2, 128, 16, 16
    pool = _filled([900, 40], 64, page, hk, d, group, dt, 1)
    c, e = pool.cuda(), pool.cuda()
    cos, sin = ref.tables(1024, d // 2)
    rot = dict(rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), rotary_interleaved=False)
    q, k, v = (_rand((2, 1, h, d), dt, i).cuda() for i, h in enumerate((hq, hk, hk)))
    lens = _i32([900, 40])

    def step(x):
        out = fa.flash_attn_with_kvcache(q, *x[:2], k=k, v=v, cache_seqlens=lens, block_table=x[4], causal=True, k_scale=x[2],
                                         v_scale=x[3], **rot)
        more = fa.flash_attn_with_kvcache(q, *x[:2], cache_seqlens=lens + 1, block_table=x[4], k_scale=x[2], v_scale=x[3])
        return out, more, *fa.flash_attn_gather_kvcache(*x[:2], cu, 942, block_table=x[4], k_scale=x[2], v_scale=x[3])

    cu = _cu([901, 41])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(c)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(c)
    for i in range(3):
        for t in (q, k, v):
            t.copy_(_rand(t.shape, dt, 10 * i + t.shape[2]).cuda())
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(s):
            s.wait_stream(torch.cuda.current_stream())
            wants = step(e)
        torch.cuda.synchronize()
        for a, b in zip(outs, wants):
            assert torch.equal(a, b)
        assert torch.equal(c[0].view(torch.uint8), e[0].view(torch.uint8)) and torch.equal(c[2].view(torch.uint8), e[2].view(torch.uint8))


def test_python_refusals():
    fa = _fa()
    dt = torch.bfloat16
    pool = _filled([20], 2, 16, 2, 64, 16, dt, 1)
    kc, vc, ks, vs, table = pool.cuda()
    q = torch.zeros(1, 1, 2, 64, dtype=dt, device="cuda")
    one = _i32([20])

    def step(**kw):
        a = dict(q=q, k_cache=kc, v_cache=vc, cache_seqlens=one, block_table=table, k_scale=ks, v_scale=vs)
        a.update(kw)
        return fa.flash_attn_with_kvcache(**a)

    step()
    for kw, exc, word in [
        (dict(q=q.float()), ValueError, "fp16 or bf16"), (dict(k_scale=ks.view(torch.uint8)), RuntimeError, "k_scale"),
        (dict(k_scale=ks[:, :, :0]), RuntimeError, "k_scale"), (dict(v_scale=vs[:1]), RuntimeError, "v_scale"),
        (dict(k_cache=kc.view(torch.uint8)), RuntimeError, "k_cache"), (dict(k_cache=q.new_zeros(kc.shape)), RuntimeError, "k_cache"),
        (dict(k=q), ValueError, "together"), (dict(q_descale=1.0), NotImplementedError, "FP8"),
        (dict(q=q[..., :48].contiguous()), NotImplementedError, "head_dim"), (dict(block_table=table.new_zeros(2, 2)), RuntimeError, "block_table"),
        (dict(k_scale=None, v_scale=None), RuntimeError, "k_cache"), (dict(cache_seqlens=_i32([1, 2])), RuntimeError, "cache_seqlens"),
        (dict(k=q.half(), v=q.half()), RuntimeError, "dtype"),
    ]:
        with pytest.raises(exc, match=word):
            step(**kw)
    with pytest.raises(RuntimeError, match="cu_seqlens_q"):
        fa.flash_attn_interface._C.fwd_paged8(q[0], kc, vc, ks, vs, table, one.float(), one, 1, 1.0, True, -1, -1, 0.0, None)
    with pytest.raises(ValueError, match="rotated"):
        fa.flash_attn_append_kvcache(q, q, kc, vc, one, q=q, block_table=table, k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="k_cache"):
        fa.flash_attn_append_kvcache(q, q, kc, vc, one, block_table=table)
    with pytest.raises(RuntimeError, match="8-bit"):
        fa.flash_attn_append_kvcache(q.float(), q.float(), kc, vc, one, block_table=table, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="cu_seqlens"):
        fa.flash_attn_append_kvcache(q[0], q[0], kc, vc, one, block_table=table, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="fp16 or bf16"):
        fa.flash_attn_gather_kvcache(kc, vc, _cu([20]), 20, block_table=table, k_scale=ks, v_scale=vs, dtype=torch.float32)
    with pytest.raises(ValueError, match="without scales"):
        fa.flash_attn_gather_kvcache(kc, vc, _cu([20]), 20, block_table=table)


@pytest.mark.parametrize("page,seqused", [(16, False), (64, True)])
def test_wide_prompts_gathered_first(page, seqused, monkeypatch):
    """Head dims past 128 with enough work go through the gather; the results are those of the other path."""
    from fable_attn import flash_attn_interface as fai
    monkeypatch.setattr(fai, "_GATHER8_PAIRS", 0)
    calls = []
    gather = fai._C.gather
    monkeypatch.setattr(fai._C, "gather", lambda *a: calls.append(1) or gather(*a))
    _check_prompts("bf16", [5, 70, 33], [0, 50, 90], 4, 2, 256, page, 16, seqused=seqused)
    _check_prompts("fp16", [40], [3], 4, 4, 192, page, 8, softcap=10.0)
    assert len(calls) == 2


@pytest.mark.parametrize("leftpad", [None, [0, 18]])
def test_a_chunk_of_attention_leaves_the_rows_before_it_their_scale(leftpad):
    """attention_chunk ends inside a block of tokens: the new token's block keeps the older rows under its scale, though
    the query does not see them."""
    dt, hq, hk, d, page, group, lens, chunk = torch.bfloat16, 4, 2, 128, 32, 16, [30, 29], 24
    pool = _filled(lens, 1, page, hk, d, group, dt, 77, scale=20.0, leftpad=leftpad)
    q, k, v = (_rand((2, 1, h, d), dt, 3 + i, 0.01) for i, h in enumerate((hq, hk, hk)))
    c = pool.cuda()
    out = _fa().flash_attn_with_kvcache(q.cuda(), c[0], c[1], k=k.cuda(), v=v.cuda(), cache_seqlens=_i32(lens), block_table=c[4],
                                        k_scale=c[2], v_scale=c[3], attention_chunk=chunk, causal=True,
                                        cache_leftpad=_i32(leftpad) if leftpad else None)
    for b, n in enumerate(lens):
        pool.append(b, n, k[b].double(), v[b].double(), leftpad=leftpad[b] if leftpad else 0)
    _same_pool(pool, c, exact=True)
    for b, n in enumerate(lens):
        kk, vv = pool.values(b, 0, n + 1)
        want, _, err, weight, _ = ref.attend(q[b].double(), kk, vv, [n // chunk * chunk], [n + 1], [n], d ** -0.5)
        ref.close(out[b], want, err, weight, dt, ref.HALF[dt], f"sequence {b}")


def test_wide_prompts_gather_into_memory_that_held_no_numbers(monkeypatch):
    from fable_attn import flash_attn_interface as fai
    monkeypatch.setattr(fai, "_GATHER8_PAIRS", 0)
    torch.cuda.empty_cache()
    # (the gathered rows: 3 sequences of the longest length, 140)
    stale = [torch.full((3 * 140, 2, 256), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    del stale
    _check_prompts("bf16", [5, 70, 33], [0, 70, 90], 4, 2, 256, 16, 16)


def test_a_call_of_a_known_signature_still_checks_its_hints():
    pool = _filled([20], 2, 16, 2, 64, 16, torch.bfloat16, 9)
    c = pool.cuda()
    q = _rand((20, 4, 64), torch.bfloat16, 1).cuda()
    call = lambda **kw: _fa().flash_attn_varlen_func(q, *c[:2], _cu([20]), _cu([20]), 20, 20, causal=True, block_table=c[4],
                                                     k_scale=c[2], v_scale=c[3], **kw)
    want = call(pack_gqa=True)
    assert torch.equal(call(pack_gqa=True), want)
    with pytest.raises(TypeError, match="pack_gqa"):
        call(pack_gqa=1)
    with pytest.raises(TypeError, match="num_splits"):
        call(pack_gqa=True, num_splits=1.0)
    with pytest.raises(ValueError, match="attention_chunk"):
        call(pack_gqa=True, attention_chunk=0.0)


def test_two_graphs_over_one_pool(monkeypatch):
    """A prompt step (packed append, prompts in place and gathered, many new tokens) and a decode step (shared out on the
    device, four heads to a workgroup) in two graphs over one memory pool, replayed in turn with eager work between."""
    fa = _fa()
    from fable_attn import flash_attn_interface as fai
    monkeypatch.setattr(fai, "_GATHER8_PAIRS", 0)
    dt, hq, hk, page, new, held = torch.bfloat16, 16, 8, 16, [33, 5, 20, 1, 64], [0, 300, 40, 900, 7]
    total = [a + b for a, b in zip(new, held)]
    pools = [(d, _filled(held, 64, page, hk, d, 16, dt, 5)) for d in (128, 256)]
    mine, eager = ([p.cuda() for _, p in pools] for _ in range(2))
    wide = [torch.cat((c[4], c[4][:, :1].expand(5, 2048 - 64)), 1).contiguous() for c in mine]
    cu, cuk, hold, full = _cu(new), _cu(total), _i32(held), _i32(total)
    cos, sin = (x.cuda() for x in ref.tables(1024, 64))
    toks = [[_rand((sum(new), h, d), dt, d + i).cuda() for i, h in enumerate((hq, hk, hk))] for d in (128, 256)]
    qd = [_rand((5, n, hq, 128), dt, n).cuda() for n in (1, 40)]

    def prompts(caches):
        outs = []
        for c, (q, k, v) in zip(caches, toks):
            s = dict(block_table=c[4], k_scale=c[2], v_scale=c[3])
            rq = fa.flash_attn_append_kvcache(k, v, *c[:2], hold, q=q, cu_seqlens=cu, max_seqlen=64, rotary_cos=cos, rotary_sin=sin, **s)
            outs += [rq, fa.flash_attn_varlen_func(rq, *c[:2], cu, cuk, 64, 964 if c[0].shape[3] > 128 else 0, causal=True, **s)]
        return outs

    def decode(caches):
        c = caches[0]
        s = dict(k_scale=c[2], v_scale=c[3], cache_seqlens=full)
        return [fa.flash_attn_with_kvcache(qd[0], *c[:2], block_table=wide[0], **s),
                fa.flash_attn_with_kvcache(qd[1], *c[:2], block_table=c[4], rotary_cos=cos, rotary_sin=sin, **s)]

    for f in (prompts, decode):   # (warm: the first call of a signature also checks it)
        f(mine)
        f(eager)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, f in zip(graphs, (prompts, decode)):
        with torch.cuda.graph(g, pool=graphs[0].pool() if outs else None):
            outs.append(f(mine))
    for i in range(3):
        for t in [x for ts in toks for x in ts] + qd:
            t.copy_(_rand(t.shape, dt, 100 * i + t.shape[-1] + t.shape[-2]).cuda())
        torch.cuda.synchronize()
        for g, f, got in zip(graphs, (prompts, decode), outs):
            g.replay()
            torch.cuda.synchronize()
            got = [x.clone() for x in got]   # (the pool's memory is shared: the next graph may write there)
            for a, b in zip(got, f(eager)):
                assert torch.equal(a, b), i
        for a, b in zip(mine, eager):
            for x, y in zip(a[:4], b[:4]):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("d", [128, 256])
def test_append_prompts_and_gather_past_32_bits(d):
    """A cache of more than 2^32 bytes, its last pages in use: the same bits as in a small one."""
    fa = _fa()
    dt, hq, hk, page, n = torch.bfloat16, 16, 8, 256, 300
    nb = (1 << 32) // (page * hk * d) + 5
    e4, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    q, k, v = (_rand((n, h, d), dt, 5 + i).cuda() for i, h in enumerate((hq, hk, hk)))
    got = []
    for blocks, table in ((2, [1, 0]), (nb, [nb - 1, nb - 2])):
        kc, vc = (torch.full((blocks, page, hk, d), 0x7F, dtype=torch.uint8, device="cuda").view(e4) for _ in range(2))
        ks, vs = (torch.full((blocks, hk, page // 16), 255, dtype=torch.uint8, device="cuda").view(e8) for _ in range(2))
        s = dict(block_table=_i32([table]), k_scale=ks, v_scale=vs)
        fa.flash_attn_append_kvcache(k, v, kc, vc, _i32([0]), cu_seqlens=_cu([n]), max_seqlen=n, **s)
        out = fa.flash_attn_varlen_func(q, kc, vc, _cu([n]), _cu([n]), n, n, causal=True, **s)
        many = fa.flash_attn_with_kvcache(q[None, :100].contiguous(), kc, vc, cache_seqlens=_i32([n]), **s)
        got.append((*fa.flash_attn_gather_kvcache(kc, vc, _cu([n]), n, **s), out, many))
    for a, b in zip(*got):
        assert torch.isfinite(a.float()).all() and torch.equal(a, b)
