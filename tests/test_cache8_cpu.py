"""Caches held in 8 bits, on the CPU: the plain implementation against torch's own conversions, and every refusal
of the C entry points, which come before any device work."""
import math

import pytest
import torch

from tests import cache8_ref as ref


def test_codes_are_torch_e4m3():
    all_codes = torch.arange(256, dtype=torch.uint8)
    want = all_codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.nan_to_num(ref.CODES, nan=1e9), torch.nan_to_num(want, nan=1e9))
    x = torch.cat((torch.randn(4000) * 30, torch.linspace(-448, 448, 4001), ref.CODES[:127].float(), torch.tensor([448.0, -448.0])))
    x = x.clamp(-448, 448)
    assert torch.equal(ref.quantize(x.double()), x.to(torch.float8_e4m3fn).view(torch.uint8))
    mid = ref._MID.float()     # ties
    assert torch.equal(ref.quantize(mid.double()), mid.to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("amax", [0.0, 448.0, 448.0001, 449.0, 1.0, 0.875, 0.876, 1e-30, 448 * 2.0 ** 119, 2.0 ** -126])
def test_least_exponent(amax):
    e = ref.least_exponent(amax)
    assert amax <= 448 * 2.0 ** e
    assert e == -126 or amax > 448 * 2.0 ** (e - 1)


def test_a_grown_scale_keeps_old_rows():
    """Powers of two: older rows under a larger scale are what they were, but for e4m3's subnormals."""
    p = ref.Pool(1, 1, 16, 1, 16, 16, 0)
    g = torch.Generator().manual_seed(1)
    a, b = torch.randn(5, 1, 16, generator=g, dtype=torch.float64), 9 * torch.randn(3, 1, 16, generator=g, dtype=torch.float64)
    p.append(0, 0, a, a)
    before = p.values(0, 0, 5)[0]
    p.append(0, 5, b, b)
    after = p.values(0, 0, 5)[0]
    step = 2.0 ** -9 * 2.0 ** (float(p.scales[0][p.table[0, 0], 0, 0]) - 127)   # the smallest code's value
    assert ((after - before).abs() <= step / 2).all()
    assert torch.equal(after[before.abs() >= 2.0 ** -6 / 2.0 ** -9 * step], before[before.abs() >= 2.0 ** -6 / 2.0 ** -9 * step])


# ----------------------------------------------------------------------------- refusals of the C entry points
def _lib():
    from fable_attn import _lib
    return _lib, _lib.load()


def _cache(**kw):
    L, _ = _lib()
    c = L.FableCache8(16, 16, L.Strides(16 * 128, 64, 128), 16, 4, 0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _dec(**kw):
    L, _ = _lib()
    p = L.FableDecParams()
    p.q = p.Kc = p.Vc = p.o = p.ctx_len = p.block_table = 16    # never dereferenced
    p.batch, p.NH, p.gqa, p.HD, p.page, p.max_blocks, p.nq, p.window, p.scale = 1, 2, 1, 64, 16, 4, 1, -1, 0.125
    for k, v in kw.items():
        setattr(p, k, v)
    return p


ARG, DTYPE, HEADDIM = 3, 1, 2


@pytest.mark.parametrize("dec,cache,dtype,code,word", [
    ({}, {}, 2, DTYPE, "dtype"), ({}, {}, 9, DTYPE, "dtype"),
    ({"HD": 72}, {}, 1, HEADDIM, "head_dim=72"), ({"HD": 272}, {}, 1, HEADDIM, "head_dim"), ({"HD": 0}, {}, 1, HEADDIM, "head_dim"),
    ({"page": 24}, {}, 1, ARG, "page"), ({"page": 8}, {}, 1, ARG, "page"), ({"page": 0}, {}, 1, ARG, "page"),
    ({"NH": 3, "gqa": 2}, {}, 1, ARG, "gqa"), ({"gqa": 0}, {}, 1, ARG, "gqa"),
    ({"max_blocks": 0}, {}, 1, ARG, "max_blocks"), ({"max_blocks": 1 << 30}, {}, 1, ARG, "max_blocks"),
    ({"nsplit": 513}, {}, 1, ARG, "nsplit"), ({"batch": 70000}, {}, 1, ARG, "batch"),
    ({"rotary": 1}, {}, 1, ARG, "cos"), ({"rotary": 1, "cos": 16, "sin": 16}, {}, 1, ARG, "rotary_rows"),
    ({"rotary": 1, "cos": 16, "sin": 16, "rotary_dim": 7}, {"rotary_rows": 9}, 1, ARG, "rotary_dim"),
    ({}, {"group": 0}, 1, ARG, "group"), ({}, {"group": 12}, 1, ARG, "group"), ({}, {"group": 32}, 1, ARG, "group"),
    ({"page": 512}, {"group": 512}, 1, ARG, "group"),
    ({}, {"num_blocks": 0}, 1, ARG, "num_blocks"), ({}, {"k_scale": None}, 1, ARG, "null"), ({"q": None}, {}, 1, ARG, "null"),
])
def test_decode_refuses(dec, cache, dtype, code, word):
    _, lib = _lib()
    rc = lib.fable_attn_dec8(_dec(**dec), _cache(**cache), dtype, None, 0, None, None, None)
    assert rc == code, lib.fable_attn_last_error()
    assert word.encode() in lib.fable_attn_last_error()


def test_decode_refuses_strides_lone_keys_and_small_workspaces():
    L, lib = _lib()
    for s in (L.Strides(16, 8, 128), L.Strides(16, 64, 48), L.Strides(-16, 64, 128), L.Strides(16, 64, 1 << 26)):
        assert lib.fable_attn_dec8(_dec(), _cache(s=s), 1, None, 0, None, None, None) == ARG
        assert b"strides" in lib.fable_attn_last_error()
    assert lib.fable_attn_dec8(_dec(), _cache(), 1, None, 0, None, 16, None) == ARG
    need = lib.fable_attn_dec8_ws_bytes(_dec(max_blocks=4096), _cache(), 1, 0)
    assert need > 0
    assert lib.fable_attn_dec8(_dec(max_blocks=4096), _cache(), 1, 16, need - 1, None, None, None) == ARG
    assert b"workspace" in lib.fable_attn_last_error()
    assert lib.fable_attn_dec8(_dec(batch=0), _cache(), 1, None, 0, None, None, None) == 0   # nothing to do
    assert lib.fable_attn_dec8_ws_bytes(_dec(HD=72), _cache(), 1, 0) == -1


@pytest.mark.parametrize("kw,dtype,code,word", [
    ({}, 4, DTYPE, "dtype"), ({}, 2, DTYPE, "8-bit"), ({"HD": 72}, 1, HEADDIM, "head_dim"),
    ({"HD": 72, "k_scale": None, "v_scale": None}, 1, 0, ""), ({"HD": 60, "k_scale": None, "v_scale": None}, 1, HEADDIM, "head_dim"),
    ({"v_scale": None}, 1, ARG, "go together"), ({"k": None}, 1, ARG, "null"), ({"Kc": None}, 1, ARG, "null"),
    ({"page": 20}, 1, ARG, "page"), ({"page": 8}, 1, ARG, "page"), ({"group": 3}, 1, ARG, "group"), ({"group": 32}, 1, ARG, "group"),
    ({"NKV": 0}, 1, ARG, "NKV"), ({"n": -1}, 1, ARG, "n=-1"), ({"num_blocks": 0}, 1, ARG, "num_blocks"),
    ({"q": 16}, 1, ARG, "q_out"), ({"q": 16, "q_out": 16}, 1, ARG, "NH"),
    ({"rotary": 1}, 1, ARG, "cos"), ({"rotary": 3, "cos": 16, "sin": 16, "rotary_rows": 4}, 1, ARG, "rotary"),
    ({"rotary": 1, "cos": 16, "sin": 16}, 1, ARG, "rotary_rows"),
    ({"rotary": 2, "cos": 16, "sin": 16, "rotary_rows": 4, "rotary_dim": 66}, 1, ARG, "rotary_dim"),
])
def test_append_refuses(kw, dtype, code, word):
    L, lib = _lib()
    p = L.FableAppendParams()
    p.k = p.v = p.Kc = p.Vc = p.k_scale = p.v_scale = p.ctx_len = p.block_table = 16
    p.sk = p.sv = L.Strides(0, 64, 64)
    p.kc = p.vc = L.Strides(16 * 64, 64, 64)
    p.batch, p.n, p.NKV, p.HD, p.page, p.max_blocks, p.num_blocks, p.group = 1, 0, 1, 64, 16, 1, 1, 16   # (no tokens: no launch)
    for k, v in kw.items():
        setattr(p, k, v)
    assert lib.fable_attn_append(p, dtype, None) == code, lib.fable_attn_last_error()
    assert word.encode() in lib.fable_attn_last_error() or not code


def test_append_refuses_misaligned_rows():
    L, lib = _lib()
    p = L.FableAppendParams()
    p.k = p.v = p.Kc = p.Vc = p.ctx_len = 16
    p.batch, p.n, p.NKV, p.HD, p.page, p.max_blocks, p.num_blocks = 1, 0, 1, 64, 16, 1, 1
    p.kc = p.vc = p.sv = L.Strides(64, 64, 64)
    p.sk = L.Strides(0, 64, 68)
    assert lib.fable_attn_append(p, 1, None) == ARG and b"aligned" in lib.fable_attn_last_error()
    p.sk, p.kc = p.sv, L.Strides(64, 4, 64)
    assert lib.fable_attn_append(p, 1, None) == ARG and b"aligned" in lib.fable_attn_last_error()


@pytest.mark.parametrize("kw,dtype,code", [
    ({}, 5, DTYPE), ({}, 2, DTYPE), ({"HD": 40}, 1, HEADDIM), ({"v_scale": None}, 1, ARG), ({"cu": None}, 1, ARG),
    ({"page": 12}, 1, ARG), ({"group": 64}, 1, ARG), ({"total": -1}, 1, ARG), ({"num_blocks": 0}, 1, ARG), ({}, 1, 0),
])
def test_gather_refuses(kw, dtype, code):
    L, lib = _lib()
    p = L.FableGatherParams()
    p.Kc = p.Vc = p.k_scale = p.v_scale = p.k_out = p.v_out = p.cu = p.block_table = 16
    p.kc = p.vc = L.Strides(16 * 64, 64, 64)
    p.total, p.batch, p.NKV, p.HD, p.page, p.max_blocks, p.num_blocks, p.group = 0, 1, 1, 64, 16, 1, 1, 16
    for k, v in kw.items():
        setattr(p, k, v)
    assert lib.fable_attn_gather(p, dtype, None) == code, lib.fable_attn_last_error()


def test_prompts_refuse():
    L, lib = _lib()

    def call(c=None, dtype=1, kv=None, **kw):
        p = L.FableFwdParams()
        p.Q = p.K = p.V = p.O = p.cu_q = p.cu_k = 16
        p.sQ = p.sO = L.Strides(0, 64, 128)
        p.SQ, p.HD, p.NH, p.gqa, p.batch, p.win_left, p.win_right = 8, 64, 2, 1, 1, -1, -1
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.fable_attn_fwd_paged8(p, kv or L.FablePagedKV(16, 4, 16, 0, 0), c or _cache(), dtype, None, 0, None)

    assert call(dtype=2) == DTYPE
    assert call(HD=24) == HEADDIM and call(HD=264) == HEADDIM
    assert call(cu_k=None) == ARG and call(dropout_p=0.5) == ARG and call(Q=None) == ARG
    assert call(c=_cache(k_scale=None)) == ARG and call(c=_cache(group=5)) == ARG
    assert call(kv=L.FablePagedKV(None, 4, 16, 0, 0)) == ARG and call(kv=L.FablePagedKV(16, 0, 16, 0, 0)) == ARG
    assert call(kv=L.FablePagedKV(16, 4, 8, 0, 0)) == ARG
    assert call(c=_cache(s=L.Strides(1 << 31, 64, 128))) == ARG


# ----------------------------------------------------------------------------- refusals of the Python entry points
def test_python_refuses_on_the_cpu():
    import fable_attn as fa
    k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    kc = torch.zeros(4, 16, 2, 64, dtype=torch.float8_e4m3fn)
    ks = torch.zeros(4, 2, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        fa.flash_attn_append_kvcache(k, k, kc, kc, one, k_scale=ks, v_scale=ks)
    with pytest.raises(ValueError, match="GPU"):
        fa.flash_attn_gather_kvcache(kc, kc, one, 0, k_scale=ks, v_scale=ks)
    with pytest.raises(ValueError, match="GPU"):
        fa.flash_attn_with_kvcache(k, kc, kc, cache_seqlens=one, k_scale=ks, v_scale=ks)
    with pytest.raises(ValueError, match="go together"):
        fa.flash_attn_with_kvcache(k, kc, kc, cache_seqlens=one, k_scale=ks)
    with pytest.raises(NotImplementedError, match="qv"):
        fa.flash_attn_with_kvcache(k, kc, kc, qv=k, cache_seqlens=one, k_scale=ks, v_scale=ks)
    with pytest.raises(ValueError, match="block_table"):
        fa.flash_attn_varlen_func(k[0], kc, kc, one, one, 1, 1, k_scale=ks, v_scale=ks)
    with pytest.raises(NotImplementedError, match="gradient"):
        fa.flash_attn_varlen_func(k[0].clone().requires_grad_(), kc, kc, one, one, 1, 1, k_scale=ks, v_scale=ks, block_table=one.view(1, 1))
    with pytest.raises(NotImplementedError, match="dropout"):
        fa.flash_attn_varlen_func(k[0], kc, kc, one, one, 1, 1, 0.1, k_scale=ks, v_scale=ks, block_table=one.view(1, 1))


def test_plain_attention_is_softmax():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(3, 2, 16, generator=g, dtype=torch.float64) for _ in range(3))
    out, lse, *_ = ref.attend(q, k, v, [0, 0, 3], [1, 3, 3], [0, 1, 2], 0.25)
    assert torch.allclose(out[0], v[0]) and math.isinf(float(lse[2, 0])) and (out[2] == 0).all()
    w = torch.softmax(torch.einsum("hd,mhd->hm", q[1], k) * 0.25, -1)
    assert torch.allclose(out[1], torch.einsum("hm,mhd->hd", w, v))


def test_pages_whose_rows_pass_32_bits_are_refused():
    """A lone page's stride may be any number: its rows are what the kernels address."""
    L, lib = _lib()
    wide = L.Strides(0, 64, 1 << 20)
    assert lib.fable_attn_dec8(_dec(page=4096), _cache(s=wide, num_blocks=1), 1, None, 0, None, None, None) == ARG
    assert b"4 GiB" in lib.fable_attn_last_error()
    p = L.FableFwdParams()
    p.Q = p.K = p.V = p.O = p.cu_q = p.cu_k = 16
    p.sQ = p.sO = L.Strides(0, 64, 128)
    p.SQ, p.HD, p.NH, p.gqa, p.batch, p.win_left, p.win_right = 8, 64, 2, 1, 1, -1, -1
    assert lib.fable_attn_fwd_paged8(p, L.FablePagedKV(16, 1, 2048, 0, 0), _cache(s=wide, num_blocks=1), 1, None, 0, None) == ARG
    assert b"2 GiB" in lib.fable_attn_last_error()
