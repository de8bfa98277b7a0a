"""Linear attention where values differ in size by more than a 16-bit type's range holds: small scores against large values, fast decays over rows
that add nothing, columns and rows far apart in size.

Bounds are those of linear_ref, whose terms are relative to each product's own size, and for fp16 2^-15 of that size: a weighted score
and a weighted row of the state's update are taken as two parts of 8 bits each (2^-16 left over), and the product of both second parts
(2^-8 of each factor) is left out. A weight l^n is off by its exponent's two roundings, 2^-23 of n d, relatively."""
import pytest
import torch

from tests import linear_ref as ref
from tests.linear_ref import DT

pytestmark = pytest.mark.gpu
ALL = ["bf16", "fp16", "fp32"]


def _fa():
    import fable_attn
    return fable_attn


def _bound(want, size, dtype, rows, dk, far=0.0):
    more = (2.0 ** -15 if dtype == "fp16" else 0.0) + 2.0 ** -22 * far
    return ref.bound(want, size, DT[dtype], rows, dk) + more * size


def _against(dtype, q, k, v, dec, scale, state=None, dout=None, far=0.0, hk=None):
    """(rows, heads, d) of one sequence, forward and with dout backward, against the definition."""
    fa = _fa()
    n, dk, dv = q.shape[0], q.shape[2], v.shape[2]
    grad = dout is not None
    wide = [x.double()[None].requires_grad_(grad) for x in (q, k, v)]
    first = None if state is None else state.double()[None]
    eo, es = ref.batch(*wide, dec.double(), scale, None, first)
    mag = [x.detach().abs().requires_grad_(grad) for x in wide]
    mo, ms = ref.batch(*mag, dec.double(), abs(scale), None, None if first is None else first.abs())
    dev = [x.cuda()[None].requires_grad_(grad) for x in (q, k, v)]
    out = fa.linear_attn_func(*dev, dec.cuda(), scale=scale, initial_state=None if state is None else state.cuda()[None])
    worst = ref.check(out, eo.detach(), _bound(eo.detach(), mo.detach(), dtype, n, dk, far), "out")
    if grad:
        want = torch.autograd.grad(eo, wide, dout.double()[None])
        size = torch.autograd.grad(mo, mag, dout.double().abs()[None])
        got = torch.autograd.grad(out, dev, dout.cuda()[None])
        for name, x, e, m in zip(("dq", "dk", "dv"), got, want, size):
            worst = max(worst, ref.check(x, e, _bound(e, m, dtype, n, max(dk, dv), far), name))
    else:
        out, last = fa.linear_attn_func(*dev, dec.cuda(), scale=scale, initial_state=None if state is None else state.cuda()[None], return_final_state=True)
        worst = max(worst, ref.check(out, eo, _bound(eo, mo, dtype, n, dk, far), "out with a state"))
        worst = max(worst, ref.check(last, es, ref.state_bound(ms, DT[dtype], n, dk) + 2.0 ** -22 * far * ms, "state"))
    print(f"[ranges]   worst {worst:.3f} of its bound", flush=True)


def _of(g, rows, heads, d, size, dtype, plus=True):
    x = torch.randn(rows, heads, d, generator=g)
    return ((x.abs() + 2.0 ** -6 if plus else x) * size).to(DT[dtype])


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("scale,sv", [(2.0 ** -28, 2.0 ** 14), (2.0 ** -34, 2.0 ** 13), (2.0 ** -18, 1.0)])
@pytest.mark.parametrize("n", [5, 80])
def test_small_scores_against_large_values(dtype, scale, sv, n):
    g = torch.Generator().manual_seed(1)
    q, k, v = _of(g, n, 2, 64, 2.0, dtype), _of(g, n, 1, 64, 4.0, dtype), _of(g, n, 1, 64, sv, dtype)
    _against(dtype, q, k, v, torch.tensor([0.0, 0.05]), scale, far=n * 0.05)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("sd,sv,sk,sq", [(1e-5, 1.0, 8.0, 1.0), (1e-6, 1.0, 8.0, 1.0), (1e-3, 1e-2, 10.0, 1.0), (1e-3, 1e-3, 30.0, 5.0)])
@pytest.mark.parametrize("hk,plus", [(2, True), (2, False), (1, True)])
def test_gradients_of_small_dout(dtype, sd, sv, sk, sq, hk, plus):
    """The gradients' scores are products of dout and v."""
    g = torch.Generator().manual_seed(2)
    q, k, v = _of(g, 70, 2, 64, sq, dtype, plus), _of(g, 70, hk, 64, sk, dtype, plus), _of(g, 70, hk, 64, sv, dtype, plus)
    _against(dtype, q, k, v, torch.tensor([0.003, 0.05]), 0.125, dout=_of(g, 70, 2, 64, sd, dtype, plus), far=70 * 0.05)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", [32, 72])
@pytest.mark.parametrize("zero", ["keys", "values"])
def test_old_rows_of_fast_heads(dtype, n, zero):
    """Rows 0, 32 and 64 alone add something; what the rows behind them leave of it is exact to its own size, however little."""
    for decays in ([0.2, 0.35], [0.5, 0.7], [0.84, 2.0]):
        g = torch.Generator().manual_seed(3)
        q, k, v = _of(g, n, 2, 64, 4.0, dtype), _of(g, n, 2, 64, 4.0, dtype), _of(g, n, 2, 64, 100.0, dtype)
        for row in range(n):
            if row % 32:
                (k if zero == "keys" else v)[row] = 0
        _against(dtype, q, k, v, torch.tensor(decays), 0.125, far=n * max(decays))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("d", [0.0, 0.5])
def test_columns_and_rows_far_apart_in_size(dtype, d):
    """Columns of v 2^24 apart in one state; elements of q, k and v from 2^-6 to 2^6 each, and whole rows from 2^-4 to 2^4."""
    g = torch.Generator().manual_seed(4)
    dec = torch.tensor([d, d])
    q, k, v = _of(g, 100, 2, 64, 1.0, dtype), _of(g, 100, 2, 64, 1.0, dtype), _of(g, 100, 2, 64, 1.0, dtype)
    wide = v * torch.exp2(12.0 - 2.0 * (torch.arange(64) % 13)).to(v.dtype)
    _against(dtype, q, k, wide, dec, 2.0 ** -10, far=100 * d)
    mixed = [x * torch.exp2(torch.randint(-6, 7, x.shape, generator=g).float() + torch.randint(-4, 5, x.shape[:1], generator=g).float()[:, None, None]).to(x.dtype)
             for x in (q, k, v)]
    _against(dtype, *mixed, dec, 2.0 ** -22, far=100 * d)


@pytest.mark.parametrize("dtype", ALL)
def test_states_columns_far_apart(dtype):
    """An initial state whose columns are 2^31 apart, read one element at a time."""
    g = torch.Generator().manual_seed(5)
    state = (1 + 0.9 * torch.rand(2, 64, 64, generator=g)) * torch.where(torch.arange(64) % 2 == 0, 2.0 ** 23, 2.0 ** -8)
    q = torch.eye(64)[:, None].repeat(1, 2, 1).to(DT[dtype])
    zero = torch.zeros(64, 2, 64, dtype=DT[dtype])
    _against(dtype, q, zero, zero, torch.zeros(2), 2.0 ** -8, state=state)


@pytest.mark.parametrize("dtype", ALL)
def test_an_infinite_column_of_a_state(dtype):
    """It makes its own column of the outputs infinite, or no number; the others, past fp16's range as they are, stay what they were."""
    fa = _fa()
    g = torch.Generator().manual_seed(6)
    q, k, v = (_of(g, 40, 2, 64, 1.0, dtype) for _ in range(3))
    state = torch.rand(1, 2, 64, 64, generator=g) * 2.0 ** 18
    dec = torch.tensor([0.0, 0.1], device="cuda")
    run = lambda s: fa.linear_attn_func(q.cuda()[None], k.cuda()[None], v.cuda()[None], dec, scale=2.0 ** -12, initial_state=s.cuda())
    want = run(state)
    state[:, 1, 5, 9] = float("inf")
    got = run(state)
    keep = torch.ones(64, dtype=torch.bool)
    keep[9] = False
    assert torch.isfinite(want).all() and not torch.isfinite(got[:, :, 1, 9]).any()
    assert torch.equal(got[:, :, 0], want[:, :, 0]) and torch.equal(got[:, :, 1, keep], want[:, :, 1, keep])
