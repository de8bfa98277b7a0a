"""Linear attention and rotation without a GPU: the plain implementation against the recurrence and against differences, and the refusals of
the C entry points, which come before any device work."""
import pytest
import torch

from tests import linear_ref as ref


def _recurrence(q, k, v, decay, scale, state):
    lam = torch.exp(-decay)[:, None, None]
    out = []
    for t in range(q.shape[0]):
        state = lam * state + k[t][:, :, None] * v[t][:, None, :]
        out.append(scale * (q[t][:, None, :] @ state)[:, 0])
    return torch.stack(out), state


def test_plain_form_is_the_recurrence():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    q, k, v, s = r(30, 4, 8), r(30, 2, 8), r(30, 2, 6), r(4, 8, 6)
    decay = torch.tensor([0.0, 0.01, 1.0, 50.0], dtype=torch.float64)
    a, b = ref.one(q, k, v, decay, 0.3, s)
    c, d = _recurrence(q, ref.shared(k, 4), ref.shared(v, 4), decay, 0.3, s)
    assert torch.allclose(a, c, rtol=1e-12, atol=1e-12) and torch.allclose(b, d, rtol=1e-12, atol=1e-12)


def test_plain_gradients_are_differences():
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
    q, k, v, s = r(7, 4, 3), r(7, 2, 3), r(7, 2, 5), r(4, 3, 5)
    decay = torch.tensor([0.0, 0.1, 1.0, 0.5], dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda q, k, v, s: ref.one(q, k, v, decay, 0.7, s), (q, k, v, s))


def test_gradient_formulas():
    """dq, dk and dv as the same sums with the roles changed, over rows in order or reversed, which the kernels use."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
    q, k, v = r(9, 2, 3), r(9, 2, 3), r(9, 2, 5)
    decay, dout = torch.tensor([0.05, 0.7], dtype=torch.float64), torch.randn(9, 2, 5, generator=g, dtype=torch.float64)
    want = torch.autograd.grad(ref.one(q, k, v, decay, 0.7)[0], (q, k, v), dout)
    q, k, v = q.detach(), k.detach(), v.detach()
    back = lambda *x: [y.flip(0) for y in x]
    dq = ref.one(dout, v, k, decay, 0.7)[0]
    dv = ref.one(*back(k, q, dout), decay, 0.7)[0].flip(0)
    dk = ref.one(*back(v, dout, q), decay, 0.7)[0].flip(0)
    for a, b in zip((dq, dk, dv), want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def _params(**kw):
    from fable_attn import _lib
    p = _lib.FableLinearParams()
    p.q = p.k = p.v = p.o = p.dout = p.dq = p.dk = p.dv = p.decay = p.state_in = p.state_out = 4096    # never read
    for s in ("sq", "sk", "sv", "so", "sdo", "sdq", "sdk", "sdv"):
        setattr(p, s, _lib.Strides(100 * 4 * 64, 64, 4 * 64))
    p.batch, p.n, p.NH, p.gqa, p.DK, p.DV, p.scale = 2, 100, 4, 2, 64, 64, 1.0
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [(dict(DK=60), 2), (dict(DV=264), 2), (dict(DK=0), 2), (dict(NH=0), 3), (dict(gqa=3), 3), (dict(batch=-1), 3), (dict(n=-1), 3),
                                     (dict(decay=None), 3), (dict(q=None), 3), (dict(k=4097), 3), (dict(v=4098), 3)])
def test_refusals(kw, code):
    from fable_attn import _lib
    L = _lib.load()
    p = _params(**kw)
    assert L.fable_linear_attn_fwd(p, _lib.FA_BF16, None, 0, None) == code
    assert L.fable_linear_attn_bwd(p, _lib.FA_BF16, None, 0, None) == code
    assert L.fable_linear_attn_step(p, _lib.FA_BF16, None) == code


def test_more_refusals():
    from fable_attn import _lib
    L = _lib.load()
    assert L.fable_linear_attn_fwd(_params(), 9, None, 0, None) == 1
    wide = _lib.Strides(0, 64, 1 << 25)              # 64 rows pass 2^31 bytes
    assert L.fable_linear_attn_fwd(_params(sk=wide), _lib.FA_BF16, None, 0, None) == 3
    assert L.fable_linear_attn_fwd(_params(sk=_lib.Strides(0, 60, 256)), _lib.FA_BF16, None, 0, None) == 3
    assert L.fable_linear_attn_step(_params(state_in=None), _lib.FA_BF16, None) == 3
    assert L.fable_linear_attn_step(_params(state_out=4100), _lib.FA_BF16, None) == 3
    assert L.fable_linear_attn_bwd(_params(slots=4096), _lib.FA_BF16, None, 0, None) == 3
    long = _params(batch=1, n=100000)
    need = L.fable_linear_attn_ws_bytes(long, _lib.FA_BF16, 0)
    assert need > 0 and need % (4 * 64 * 64 * 4) == 0           # a state for each segment and head
    assert L.fable_linear_attn_fwd(long, _lib.FA_BF16, None, 0, None) == 3 and b"workspace" in L.fable_attn_last_error()
    assert L.fable_linear_attn_fwd(long, _lib.FA_BF16, 4096, need - 1, None) == 3
    assert L.fable_linear_attn_ws_bytes(_params(batch=64, NH=64, gqa=1, n=100000), _lib.FA_BF16, 0) == 0    # enough heads
    assert L.fable_linear_attn_ws_bytes(_params(DK=60), _lib.FA_BF16, 0) == -1
    assert L.fable_linear_attn_fwd(_params(batch=0), _lib.FA_BF16, None, 0, None) == 0


def test_rotary_refusals():
    from fable_attn import _lib
    L = _lib.load()

    def params(**kw):
        p = _lib.FableRotaryParams()
        p.q = p.q_out = p.cos = p.sin = 4096
        for s in ("sq", "sk", "sqo", "sko"):
            setattr(p, s, _lib.Strides(100 * 4 * 64, 64, 4 * 64))
        p.batch, p.n, p.NH, p.HD, p.rotary, p.rotary_dim, p.rotary_rows = 2, 100, 4, 64, 1, 64, 10
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for kw in (dict(rotary=0), dict(rotary=3), dict(rotary_dim=66), dict(rotary_dim=7), dict(rotary_rows=0), dict(NH=0), dict(q=None),
               dict(cos=None), dict(k=4096), dict(batch=-1), dict(batch=1 << 20, n=1 << 10)):
        assert L.fable_attn_rotary(params(**kw), _lib.FA_BF16, None) == 3, kw
    assert L.fable_attn_rotary(params(), 7, None) == 1
    assert L.fable_attn_rotary(params(n=0), _lib.FA_BF16, None) == 0
    t = lambda **kw: _lib.FableRotaryTableParams(**{**dict(cos=4096, sin=4096, rows=8, pairs=4, base=1e4, factor=1.0, low=1.0, high=32.0, amplitude=1.0), **kw})
    for kw in (dict(rows=-1), dict(pairs=0), dict(pairs=5000), dict(base=0.0), dict(factor=0.0), dict(factor=float("nan")), dict(cos=None),
               dict(original=100.0, low=2.0, high=2.0), dict(original=-1.0)):
        assert L.fable_attn_rotary_tables(t(**kw), None) == 3, kw
    assert L.fable_attn_rotary_tables(t(rows=0), None) == 0
