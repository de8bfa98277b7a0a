"""The rotation of queries and keys and its tables against their definitions in 64 bits."""
import pytest
import torch

from tests import linear_ref as ref
from tests.linear_ref import DT

pytestmark = pytest.mark.gpu


def _fa():
    import fable_attn
    return fable_attn


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables(rows, rd, g):
    angle = torch.rand(rows, rd // 2, generator=g) * 100
    return angle.cos(), angle.sin()


def _bound(x, want, cos, sin, pos, interleaved, dtype):
    """One rounding of the result, and in fp32 the two products and their sum (3 roundings of 2^-24 of their size)."""
    size = ref.rotated(x.abs(), cos.abs(), -sin.abs(), pos, interleaved).abs().maximum(ref.rotated(x.abs(), cos.abs(), sin.abs(), pos, interleaved).abs())
    return ref.unit(dtype) * want.abs() * (1 + 2.0 ** -8) + 3 * 2.0 ** -24 * size + torch.finfo(dtype).smallest_normal * ref.unit(dtype) * 2


def _run(dtype, lens, hq, hk, d, rd, interleaved, *, packed=True, start=None, rows=300, front=0, tail=0, seed=0):
    print(f"[rotary] {dtype} lens={lens} {hq}/{hk} d={d} rd={rd} il={interleaved} packed={packed} start={start}", flush=True)
    fa = _fa()
    g = torch.Generator().manual_seed(seed)
    cos, sin = _tables(rows, rd, g)
    B = len(lens)
    shape = (front + sum(lens) + tail,) if packed else (B, lens[0])
    q = torch.randn(*shape, hq, d, generator=g).to(DT[dtype])
    k = torch.randn(*shape, hk, d, generator=g).to(DT[dtype]) if hk else None
    cu = [front]
    for n in lens:
        cu.append(cu[-1] + n)
    pos = torch.cat([torch.arange(n) + (start[b] if start else 0) for b, n in enumerate(lens)]).clamp(0, rows - 1).long()
    dq, dk = torch.randn(q.shape, generator=g).to(DT[dtype]), torch.randn(k.shape, generator=g).to(DT[dtype]) if hk else None
    args = [x.cuda().requires_grad_() if x is not None else None for x in (q, k)]
    got = fa.flash_attn_rotary_func(*args, cos.cuda(), sin.cuda(), rotary_interleaved=interleaved, rotary_seqlens=_i32(start) if start else None,
                                    cu_seqlens=_i32(cu) if packed else None)
    got = got if hk else (got,)
    grads = torch.autograd.grad(got, [x for x in args if x is not None], [x.cuda() for x in (dq, dk) if x is not None])
    for x, y, gx, gy in zip((q, k), got, (dq, dk), grads):
        for a, b, conj in ((x, y, False), (gx, gy, True)):
            assert b.is_contiguous() and b.dtype == DT[dtype] and b.shape == a.shape
            b = b.detach().cpu().view(-1, *b.shape[-2:])
            a = a.reshape(-1, *a.shape[-2:])
            if packed:
                assert not b[:front].any() and not b[cu[-1]:].any()
                a, b = a[front:cu[-1]], b[front:cu[-1]]
            want = ref.rotated(a.double(), cos.double(), sin.double(), pos, interleaved, conj)
            ref.check(b, want, _bound(a.double(), want, cos.double(), sin.double(), pos, interleaved, DT[dtype]), "turned")
            assert torch.equal(b[..., rd:], a[..., rd:])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rd", [(128, 128), (128, 32), (64, 64), (80, 80), (80, 48), (256, 256), (256, 16), (96, 20), (40, 2), (7, 6), (8, 8), (520, 512)])
def test_head_dims(dtype, interleaved, d, rd):
    _run(dtype, [5, 1, 0, 33], 6, 2, d, rd, interleaved, start=[0, 100, 4, 280], seed=d + rd)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("hq,hk", [(1, 1), (64, 8), (3, 0), (40, 40)])
def test_heads(packed, hq, hk):
    _run("bf16", [17, 17, 17], hq, hk, 64, 64, False, packed=packed, start=[0, 7, 250])
    _run("fp16", [1, 1], hq, hk, 128, 64, True, packed=packed)


@pytest.mark.parametrize("front,tail", [(0, 0), (3, 5)])
def test_rows_of_no_sequence(front, tail):
    for d, rd in ((64, 64), (64, 20)):
        _run("bf16", [0, 4, 0, 0, 9, 0], 4, 2, d, rd, False, front=front, tail=tail)


def test_positions_past_the_tables():
    """The last row serves them, the first one those below 0."""
    _run("fp32", [6, 6], 2, 1, 32, 32, True, start=[296, -3], rows=300)


def test_strided_inputs_and_one_gradient():
    fa = _fa()
    g = torch.Generator().manual_seed(1)
    cos, sin = (t.cuda() for t in _tables(64, 64, g))
    x = torch.randn(2, 50, 12, 64, device="cuda", dtype=torch.bfloat16)
    q, k = x[:, :, :8], x[:, :, 8:10]
    want = fa.flash_attn_rotary_func(q.contiguous(), k.contiguous(), cos, sin)
    for a, b in ((q, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k), (x[..., ::1][:, :, :8], k)):
        got = fa.flash_attn_rotary_func(a, b, cos, sin)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    off = torch.empty(q.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view(q.shape).copy_(q)
    assert torch.equal(fa.flash_attn_rotary_func(off, k, cos, sin)[0], want[0])
    assert torch.equal(fa.flash_attn_rotary_func(q, None, cos, sin, rotary_seqlens=0), want[0])
    a, b = q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_()
    y = fa.flash_attn_rotary_func(a, b, cos, sin)
    (gb,) = torch.autograd.grad(y[1].sum(), b)             # (an expanded scalar; no gradient of q)
    assert torch.equal(gb, fa._C.rotary(torch.ones_like(k), None, cos, sin, True, conj=True)[0])


def test_same_as_the_decode_path():
    """Keys turned here and appended as they are give the cache that an append with rotation gives."""
    fa = _fa()
    g = torch.Generator().manual_seed(1)
    for interleaved in (False, True):
        cos, sin = (t.cuda() for t in _tables(256, 64, g))
        k = torch.randn(3, 5, 2, 64, device="cuda", dtype=torch.bfloat16)
        lens = _i32([0, 7, 100])
        caches = [torch.zeros(3, 128, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
        fa.flash_attn_append_kvcache(k, k, caches[0], caches[1], lens, rotary_cos=cos, rotary_sin=sin, rotary_interleaved=interleaved)
        turned = fa.flash_attn_rotary_func(k, None, cos, sin, rotary_interleaved=interleaved, rotary_seqlens=lens)
        fa.flash_attn_append_kvcache(turned, k, caches[2], caches[3], lens)
        step = 2.0 ** -7 * caches[0].float().abs() + 1e-6   # (one step of bf16: a product fused or not moves a tie)
        assert ((caches[0].float() - caches[2].float()).abs() <= step).all()


@pytest.mark.parametrize("rows,rd,kw", [(2048, 64, {}), (5, 2, {}), (1000, 128, dict(factor=4.0)), (3001, 90, dict(factor=8.0, original_seqlen=4096)),
                                        (131072, 32, dict(base=5e5, factor=2.5, original_seqlen=8192, low_turns=2, high_turns=16, amplitude=1.2)),
                                        (64, 4096, {}), (100, 64, dict(start=10 ** 8))])
def test_tables(rows, rd, kw):
    fa = _fa()
    cos, sin = fa.flash_attn_rotary_tables(rows, rd, **kw)
    assert cos.shape == sin.shape == (rows, rd // 2) and cos.dtype == torch.float32
    f = ref.frequencies(rd, kw.get("base", 10000.0), kw.get("factor", 1.0), kw.get("original_seqlen"), kw.get("low_turns", 1.0), kw.get("high_turns", 32.0))
    pos = torch.arange(rows, dtype=torch.float64) + kw.get("start", 0)
    angle = pos[:, None] * f
    amp = kw.get("amplitude", 1.0)
    # the fp32 function (4 ulp), the products with amplitude and first order (3 roundings); angles: a frequency is off by some 2^-50, twice
    tol = amp * (7 * 2.0 ** -24 + 2.0 ** -48 * angle)
    for got, want in ((cos, angle.cos() * amp), (sin, angle.sin() * amp)):
        ref.check(got, want, tol, "table")


def test_refusals():
    fa = _fa()
    q = torch.randn(2, 4, 2, 64, device="cuda")
    cos = torch.zeros(8, 32, device="cuda")
    with pytest.raises(ValueError):
        fa.flash_attn_rotary_func(q[0], None, cos, cos)
    with pytest.raises(ValueError):
        fa.flash_attn_rotary_func(q.double(), None, cos, cos)
    with pytest.raises(RuntimeError):
        fa.flash_attn_rotary_func(q, q[:, :2], cos, cos)
    with pytest.raises(RuntimeError):
        fa.flash_attn_rotary_func(q, q.half(), cos, cos)
    with pytest.raises(RuntimeError):
        fa.flash_attn_rotary_func(q, None, torch.zeros(8, 40, device="cuda"), torch.zeros(8, 40, device="cuda"))
    with pytest.raises(RuntimeError):
        fa.flash_attn_rotary_func(q, None, cos, cos[:4])
    with pytest.raises(RuntimeError):
        fa.flash_attn_rotary_func(q, None, cos, cos, rotary_seqlens=_i32([0]))
    with pytest.raises(NotImplementedError):
        fa.flash_attn_rotary_func(q, None, cos.clone().requires_grad_(), cos)
    with pytest.raises(ValueError):
        fa.flash_attn_rotary_tables(10, 7)
    with pytest.raises(ValueError):
        fa.flash_attn_rotary_tables(10, 8, factor=0)
    with pytest.raises(ValueError):
        fa.flash_attn_rotary_tables(-1, 8)
    with pytest.raises(ValueError):
        fa.flash_attn_rotary_tables(10, 8, factor=2, original_seqlen=100, low_turns=5, high_turns=5)
    with pytest.raises(ValueError):
        fa.flash_attn_rotary_tables(10, 8, device="cpu")
