"""Calls of linear attention and the rotation that are refused because a derivative would be lost, and outputs that ask for none."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def _fa():
    import fable_attn
    return fable_attn


def _x(*shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", dtype=dtype)


def test_tangents_are_refused():
    """There is no forward-mode derivative: a dual tensor raises, whichever input it is and whatever else asks for a gradient."""
    fa = _fa()
    q, k, v, dec = _x(2, 20, 2, 32), _x(2, 20, 2, 32), _x(2, 20, 2, 32), torch.tensor([0.1, 0.2], device="cuda")
    state, cu = _x(2, 2, 32, 32), torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda")
    cos, sin = fa.flash_attn_rotary_tables(20, 32)
    flat = lambda t: t.flatten(0, 1) if t.dim() == 4 and t.shape[1] == 20 else t
    for _ in range(2):                                             # (also calls whose signature is known)
        fa.linear_attn_func(q, k, v, dec, initial_state=state)
        fa.linear_attn_with_state(q[:, :1], k[:, :1], v[:, :1], state, dec)
        fa.flash_attn_rotary_func(q, k, cos, sin)
    with fwAD.dual_level():
        for grad in (False, True):
            for i in range(5):
                x = [t.clone() for t in (q, k, v, dec, state)]
                x[1].requires_grad_(grad)
                x[i] = fwAD.make_dual(x[i], torch.ones_like(x[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fa.linear_attn_func(*x[:4], initial_state=x[4])
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fa.linear_attn_varlen_func(*(flat(t) for t in x[:3]), cu, 20, x[3], initial_state=x[4])
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fa.linear_attn_with_state(x[0][:, :1], x[1].detach()[:, :1] if i != 1 else x[1][:, :1], x[2][:, :1], x[4], x[3])
            for i in range(4):
                x = [t.clone() for t in (q, k, cos, sin)]
                x[1].requires_grad_(grad)
                x[i] = fwAD.make_dual(x[i], torch.ones_like(x[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fa.flash_attn_rotary_func(*x)
        # other tensors of a dual level are served
        want = fa.linear_attn_func(q, k, v, dec)
        turned = fa.flash_attn_rotary_func(q, k, cos, sin)
    assert torch.equal(fa.linear_attn_func(q, k, v, dec), want) and torch.equal(fa.flash_attn_rotary_func(q, k, cos, sin)[1], turned[1])


@pytest.mark.parametrize("n", [1, 17])
def test_steps_refuse_what_asks_for_a_gradient(n):
    """They give none: a q, k, v, pool or decay that requires one raises, but for torch.no_grad(), where results are the same."""
    fa = _fa()
    x = [_x(2, n, 2, 32) for _ in range(3)] + [_x(2, 2, 32, 32), torch.tensor([0.1, 0.2], device="cuda")]
    pool = x[3].clone()
    want = fa.linear_attn_with_state(*x[:3], pool, x[4])
    for _ in range(2):
        for i in range(5):
            y = [t.clone() for t in x]
            y[i].requires_grad_()
            with pytest.raises(NotImplementedError, match="no_grad"):
                fa.linear_attn_with_state(*y)
            assert torch.equal(y[3], x[3])
            with torch.no_grad():
                assert torch.equal(fa.linear_attn_with_state(*y), want) and torch.equal(y[3], pool)


def test_rotation_asks_for_no_more_gradients_than_its_inputs():
    fa = _fa()
    q, k = _x(2, 20, 4, 32), _x(2, 20, 2, 32)
    cos, sin = fa.flash_attn_rotary_tables(20, 32)
    turn = lambda t: fa._C.rotary(t, None, cos, sin, True, conj=True)[0]
    for need in ((True, False), (False, True), (True, True), (False, False)):
        a, b = q.clone().requires_grad_(need[0]), k.clone().requires_grad_(need[1])
        out = fa.flash_attn_rotary_func(a, b, cos, sin)
        assert (out[0].requires_grad, out[1].requires_grad) == need
        wants = [x for x, n in zip((a, b), need) if n]
        outs = [x for x, n in zip(out, need) if n]
        if wants:
            douts = [torch.randn_like(x) for x in outs]
            for got, d in zip(torch.autograd.grad(outs, wants, douts), douts):
                assert torch.equal(got, turn(d))


@pytest.mark.parametrize("dq,dk", [(60, 64), (64, 60), (60, 40), (64, 128), (5, 8), (64, 32)])
def test_keys_of_another_width_are_refused(dq, dk):
    """Also where the width that is zero-padded to would fit both."""
    fa = _fa()
    dec, cu = torch.tensor([0.1, 0.2], device="cuda"), torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda")
    q, k, v = _x(2, 20, 2, dq), _x(2, 20, 2, dk), _x(2, 20, 2, 32)
    with pytest.raises((ValueError, RuntimeError)):
        fa.linear_attn_func(q, k, v, dec)
    with pytest.raises((ValueError, RuntimeError)):
        fa.linear_attn_varlen_func(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), cu, 20, dec)
    pool = torch.zeros(2, 2, dq, 32, device="cuda")
    with pytest.raises((ValueError, RuntimeError)):
        fa.linear_attn_with_state(q, k, v, pool, dec)
    assert not pool.any()


def test_max_seqlen_of_any_size():
    """It only sizes the launch, also past what 32 bits count; below 0 it is refused."""
    fa = _fa()
    dec, cu = torch.tensor([0.1, 0.2], device="cuda"), torch.tensor([0, 20, 400], dtype=torch.int32, device="cuda")
    q, k, v = (_x(400, 2, 32) for _ in range(3))
    want = fa.linear_attn_varlen_func(q, k, v, cu, 400, dec)
    pools = [torch.zeros(2, 2, 32, 32, device="cuda") for _ in range(2)]
    steps = fa.linear_attn_with_state(q, k, v, pools[0], dec, cu_seqlens=cu, max_seqlen=400)
    for most in (401, 2 ** 30 + 1, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 40):
        assert torch.equal(fa.linear_attn_varlen_func(q, k, v, cu, most, dec), want)
        pools[1].zero_()
        assert torch.equal(fa.linear_attn_with_state(q, k, v, pools[1], dec, cu_seqlens=cu, max_seqlen=most), steps) and torch.equal(*pools)
    for most in (-1, -2 ** 32 + 5):
        with pytest.raises(RuntimeError, match="max_seqlen"):
            fa.linear_attn_varlen_func(q, k, v, cu, most, dec)
        with pytest.raises(RuntimeError, match="max_seqlen"):
            fa.linear_attn_with_state(q, k, v, pools[1], dec, cu_seqlens=cu, max_seqlen=most)
