"""Seeded random sweeps of the operators over a cache in 8 bits, at the bounds of the fixed cases: head dims, group sizes,
pages, lengths, masks, splits and rotations in combinations that those do not list. A case is its seed."""
import random

import pytest
import torch

from tests import cache8_ref as ref
from tests.test_cache8_gpu import DT, _check_decode, _check_prompts, _cu, _fa, _i32, _rand, _same_pool

pytestmark = pytest.mark.gpu

GROUPS = (1, 2, 4, 8, 16, 32, 64, 128, 256)


def _shape(r):
    """(dtype, q heads, K/V heads, head dim, page, tokens per scale)"""
    hk = r.choice([1, 2, 3, 4, 8])
    hq = hk * (r.choice([1, 2, 5, 8, 17]) if hk < 4 else r.choice([1, 2, 4]))
    page = r.choice([16, 16, 32, 64, 256])
    return r.choice(["bf16", "fp16"]), hq, hk, 16 * r.randint(1, 16), page, r.choice([g for g in GROUPS if g <= page])


@pytest.mark.parametrize("seed", range(40))
def test_decode(seed):
    r = random.Random(seed)
    dtype, hq, hk, d, page, group = _shape(r)
    lens = [r.choice([0, 1, 15, 16, 31, 32, 33, 100, r.randint(0, 900)]) for _ in range(r.choice([1, 2, 3, 5, 6]))]
    kw = {"nq": r.choice([1, 1, 1, 2, 3, 4, 7, 17, 33]), "append": r.random() < 0.5}
    if kw["nq"] * hq * sum(lens) > 2_500_000:
        kw["nq"] = 1
    if r.random() < 0.3:
        kw.update(window=r.choice([0, 1, 5, 33, 200]), hide=kw["nq"] == 1)
    if r.random() < 0.3:
        kw["softcap"] = r.choice([3.0, 30.0])
    if r.random() < 0.25:
        kw["alibi"] = True
    if r.random() < 0.25:
        kw["leftpad"] = [r.randint(0, max(n, 1)) for n in lens]
    if r.random() < 0.3:
        kw.update(rotary=2 * r.randint(1, d // 2), interleaved=r.random() < 0.5)
    if r.random() < 0.3:
        kw["num_splits"] = r.choice([1, 2, 3, 9, 32])
    if "leftpad" not in kw:
        form = r.random()
        if form < 0.3:
            kw["wide"] = r.choice([64, 512, 2048])
        elif form < 0.4:
            kw["dense"], page = True, 1 << max(6, (max(lens) + kw["nq"]).bit_length())
    _check_decode(dtype, lens, hq, hk, d, page, min(group, page), seed=seed, **kw)


@pytest.mark.parametrize("seed", range(20))
def test_prompts(seed):
    r = random.Random(1000 + seed)
    dtype, hq, hk, d, page, group = _shape(r)
    batch = r.choice([1, 2, 3])
    new = [r.choice([0, 1, 5, 33, r.randint(1, 150)]) for _ in range(batch - 1)] + [r.randint(1, 100)]
    cached = [r.choice([0, 1, 16, 90, r.randint(0, 300)]) for _ in range(batch)]
    kw = {"causal": r.random() < 0.7, "seqused": r.random() < 0.25, "alibi": r.random() < 0.25}
    if r.random() < 0.35:
        kw["window"] = (r.choice([0, 3, 20, 100]), 0 if kw["causal"] else r.choice([0, 5, 40]))
    if r.random() < 0.3:
        kw["softcap"] = r.choice([3.0, 30.0])
    _check_prompts(dtype, new, cached, hq if hq <= 8 else hk, hk, d, page, group, seed=seed, **kw)


@pytest.mark.parametrize("seed", range(40))
def test_append(seed):
    """Packed and padded, rotated over any even width, queries too, tokens in rows of their own or sliced from one
    projection, started blocks and left pads; the same call twice gives the same bytes."""
    r = random.Random(2000 + seed)
    dtype, hq, hk, d, page, group = _shape(r)
    dt, batch, packed = DT[dtype], r.choice([1, 2, 3, 5]), r.random() < 0.6
    new = [r.choice([0, 1, 1, 5, r.randint(0, 60), r.randint(0, 300)]) for _ in range(batch - 1)] + [r.randint(1, 100)]
    if not packed:
        new = [new[-1]] * batch
    held = [r.choice([0, 1, 15, 16, 17, r.randint(0, 300)]) for _ in range(batch)]
    pad = [r.randint(0, h + 3) for h in held] if r.random() < 0.3 else [0] * batch
    half = r.choice([0, d // 2, r.randint(1, d // 2), max(d // 16 * 4, 1)])
    interleaved, with_q, sliced, size = r.random() < 0.5, half > 0 and r.random() < 0.6, r.random() < 0.4, r.choice([0.01, 1.0, 50.0])
    pool = ref.Pool(batch, max(-(-(a + b) // page) for a, b in zip(new, held)), page, hk, d, group, seed)
    for b in range(batch):
        if held[b] > pad[b]:
            pool.append(b, pad[b], *(_rand((held[b] - pad[b], hk, d), dt, 10 * seed + 2 * b + i, 2.0).double() for i in range(2)), leftpad=pad[b])
    shape = (sum(new),) if packed else (batch, new[0])
    q, k, v = (_rand(shape + (h, d), dt, 5 * seed + i, s) for i, (h, s) in enumerate(((hq, 1.0), (hk, size), (hk, size))))
    gq, gk, gv = (torch.cat((q, k, v), -2).cuda().split((hq, hk, hk), -2) if sliced else (x.cuda() for x in (q, k, v)))
    kw = {"cache_leftpad": _i32(pad)} if any(pad) else {}
    cos = sin = None
    if half:
        cos, sin = ref.tables(max(held) + max(new) + 1, half)
        kw.update(rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), rotary_interleaved=interleaved)
    if with_q:
        kw["q"] = gq
    if packed:
        kw.update(cu_seqlens=_cu(new), max_seqlen=r.choice([max(new), max(new) + 7, None]))
    runs = []
    for _ in range(2):
        c = pool.cuda()
        got = _fa().flash_attn_append_kvcache(gk, gv, *c[:2], _i32(held), block_table=c[4], k_scale=c[2], v_scale=c[3], **kw)
        runs.append([x.view(torch.uint8) for x in c[:4]] + ([got] if with_q else []))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    at = 0
    for b, n in enumerate(new):
        take = (lambda x: x[at:at + n]) if packed else (lambda x: x[b])
        pos, kb = list(range(held[b], held[b] + n)), take(k).double()
        if half:
            kb = ref.rotate(kb, cos, sin, pos, interleaved)
        if with_q:
            qb = take(q).double()
            want = ref.rotate(qb, cos, sin, pos, interleaved)
            # (its own rounding, and the rotation's three in 32 bits; fp16's smallest step)
            tol = ref.HALF[dt] * want.abs() * (1 + 2.0 ** -8) + ref.rotated_size(qb, cos, sin, pos, interleaved) * 2.0 ** -22 + 2.0 ** -24
            assert ((take(got).cpu().double() - want).abs() <= tol).all()
        pool.append(b, held[b], kb, take(v).double(), leftpad=pad[b])
        at += n
    # (a rotated key within 2^-22 of a border between codes may fall on its other side: some 2^-17 of them, and one is 2^-8
    # of the smallest pool, 16 rows of one head of 16)
    _same_pool(pool, c, exact=not half, moved=2.0 ** -8)
