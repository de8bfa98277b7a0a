"""Scores that are not numbers: a query row (or a key that it sees) with a NaN gives NaN in its output row and in its LSE,
in every form of the attention over caches: one split, several, shares worked out on the device, many new tokens; caches
in 8, 16 and 32 bits. Other rows keep their values, and a row that sees no key stays 0 with an LSE of -inf."""
import math

import pytest
import torch

from tests.test_cache8_gpu import _cu, _fa, _filled, _i32, _rand

pytestmark = pytest.mark.gpu

KINDS = ["8 bits bf16", "8 bits fp16", "bf16", "fp16", "fp32"]
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _caches(kind, lens, hk, d, page, wide=None):
    """(k, v cache, the call's cache arguments, dtype); every page past the sequences' own is garbage."""
    dt = DTYPES[kind.split()[-1]]
    pool = _filled(lens, max(-(-max(n, 1) // page) for n in lens), page, hk, d, 16, torch.bfloat16 if dt == torch.float32 else dt, 3)
    kc, vc, ks, vs, table = pool.cuda()
    if wide:
        table = torch.cat((table, table[:, :1].expand(len(lens), wide - table.shape[1])), 1).contiguous()
    kw = {"cache_seqlens": _i32(lens), "block_table": table}
    if kind.startswith("8"):
        return kc, vc, dict(kw, k_scale=ks, v_scale=vs), dt
    shape = (kc.shape[0], page, hk, d)
    return _rand(shape, dt, 4).cuda(), _rand(shape, dt, 5).cuda(), kw, dt


def _check(clean, poisoned, bad, blind, dt, vmax):
    """bad, blind (B, nq, hq): the rows that must not be numbers, and those that see no key."""
    (a, al), (b, bl) = [(o.float().cpu(), lse.transpose(1, 2).cpu()) for o, lse in (clean, poisoned)]
    assert torch.isfinite(a).all() and (a[blind] == 0).all() and (al[blind] == -math.inf).all()
    bad = bad & ~blind
    assert torch.isnan(b[bad]).all() and torch.isnan(bl[bad]).all(), (b[bad].isnan().double().mean(), bl[bad])
    rest = ~bad
    # (both within P's rounding and their own of the same value; a maximum may be kept with other rows)
    tol = 4 * torch.finfo(dt).eps / 2 * vmax
    assert ((a - b).abs()[rest] <= tol).all() and torch.equal(bl[rest & blind], al[rest & blind])
    seen = rest & ~blind
    assert ((al - bl).abs()[seen] <= 2.0 ** -18 * (1 + al.abs()[seen])).all()


FORMS = [
    # lens, hq, hk, d, page, nq, width of the table, options
    ([0, 40, 130], 8, 2, 128, 16, 1, None, {"num_splits": 1}),
    ([0, 40, 700], 8, 2, 128, 16, 1, None, {"num_splits": 3}),
    ([1, 1000], 4, 4, 64, 16, 2, None, {"num_splits": 7, "softcap": 10.0}),
    ([0, 700, 300, 129, 64, 1000], 8, 8, 128, 16, 1, 2048, {}),           # shares; heads together in 8 bits
    ([0, 700, 300, 129, 64, 1000], 8, 1, 128, 16, 3, 8192, {"window_size": (900, 0)}),
    ([0, 40, 130], 8, 2, 128, 16, 17, None, {}),                           # the tile kernel
    ([0, 40, 130], 8, 2, 64, 16, 33, 512, {}),                             # the tile kernel, split
    ([0, 40, 130], 8, 2, 256, 64, 40, 256, {"softcap": 10.0}),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_query_that_is_no_number(form, kind):
    lens, hq, hk, d, page, nq, wide, opts = form
    kc, vc, kw, dt = _caches(kind, lens, hk, d, page, wide)
    q = _rand((len(lens), nq, hq, d), dt, 6)
    bad = torch.zeros(len(lens), nq, hq, dtype=torch.bool)
    for b in range(len(lens)):
        bad[b, b % nq, (3 * b + 1) % hq] = True
        bad[b, nq - 1, 0] = True
    worse = q.clone()
    worse[..., 5][bad] = math.nan
    call = lambda x: _fa().flash_attn_with_kvcache(x.cuda(), kc, vc, return_softmax_lse=True, **kw, **opts)
    blind = torch.tensor([n == 0 for n in lens])[:, None, None].expand_as(bad)
    _check(call(q), call(worse), bad, blind, dt, 20.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_key_that_is_no_number(form, kind):
    """One key of one head in the last sequence: in the middle, so in one split of several; and a sequence's only key."""
    lens, hq, hk, d, page, nq, wide, opts = form
    lens = lens[:-1] + [lens[-1]] if lens[0] else [1] + lens[1:]
    kc, vc, kw, dt = _caches(kind, lens, hk, d, page, wide)
    q = _rand((len(lens), nq, hq, d), dt, 6).cuda()
    call = lambda: _fa().flash_attn_with_kvcache(q, kc, vc, return_softmax_lse=True, **kw, **opts)
    clean = call()
    bad = torch.zeros(len(lens), nq, hq, dtype=torch.bool)
    table = kw["block_table"]
    for b, pos in ((len(lens) - 1, lens[-1] // 2), (0, 0)):
        row = (int(table[b, pos // page]), pos % page, hk - 1)
        if kind.startswith("8"):
            kc.view(torch.uint8)[row][3] = 0x7F
        else:
            kc[row][3] = math.nan
        bad[b, :, (hk - 1) * (hq // hk):] = True
    _check(clean, call(), bad, torch.zeros_like(bad), dt, 20.0)


@pytest.mark.parametrize("kind", KINDS[:4])
@pytest.mark.parametrize("d,new,cached,opts", [(128, [5, 70], [0, 50], {}), (64, [3], [3000], {}), (256, [2, 9], [2000, 1500], {"softcap": 20.0})], ids=str)
def test_a_prompt_row_that_is_no_number(d, new, cached, opts, kind):
    """Packed prompts, in one piece and with their keys split over workgroups."""
    hq, hk, page = 4, 2, 16
    total = [a + b for a, b in zip(new, cached)]
    kc, vc, kw, dt = _caches(kind, total, hk, d, page)
    scales = {n: kw[n] for n in ("k_scale", "v_scale") if n in kw}
    q = _rand((sum(new), hq, d), dt, 7)
    worse = q.clone()
    worse[-1, 2, 0] = math.nan
    worse[1, 1, 1] = math.nan
    call = lambda x: _fa().flash_attn_varlen_func(x.cuda(), kc, vc, _cu(new), _cu(total), max(new), max(total), causal=True,
                                                  block_table=kw["block_table"], **scales, **opts).float().cpu()
    a, b = call(q), call(worse)
    bad = torch.zeros(sum(new), hq, dtype=torch.bool)
    bad[-1, 2] = bad[1, 1] = True
    assert torch.isnan(b[bad]).all() and torch.isfinite(a).all()
    assert ((a - b).abs()[~bad] <= 4 * torch.finfo(dt).eps / 2 * 20.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("packed", [False, True])
def test_a_row_of_contiguous_keys_split_over_workgroups(packed, dtype):
    """The forward of few rows over many keys: its keys are split too."""
    dt, d, h, n, m = DTYPES[dtype], 128, 2, 40, 4000
    q = _rand((1, n, h, d), dt, 1)
    k, v = (_rand((1, m, h, d), dt, 2 + i).cuda() for i in range(2))
    worse = q.clone()
    worse[0, 7, 1, 9] = math.nan

    def call(x):
        if packed:
            return _fa().flash_attn_varlen_func(x[0].cuda(), k[0], v[0], _cu([n]), _cu([m]), n, m)[None].float().cpu()
        return _fa().flash_attn_func(x.cuda(), k, v).float().cpu()

    a, b = call(q), call(worse)
    bad = torch.zeros(1, n, h, dtype=torch.bool)
    bad[0, 7, 1] = True
    assert torch.isnan(b[bad]).all()
    assert ((a - b).abs()[~bad] <= 4 * torch.finfo(dt).eps / 2 * 5.0).all()
