"""Linear attention and rotation beside torch's autograd: states changed in place, tangents, what requires a gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _fa():
    import fable_attn
    return fable_attn


def _qkv(rows, heads=2, d=32, dtype=torch.float32, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*rows, heads, d, generator=g).to("cuda", dtype) for _ in range(3)]


@pytest.mark.parametrize("n", [1, 17])
@pytest.mark.parametrize("idx", [None, [1, 0]])
def test_a_pool_stepped_before_backward(n, idx):
    """A pool that a graph holds as its initial state and that is stepped afterwards (the first call of a signature, a later one, by chunks) is
    seen by that graph's backward pass, which raises as for any tensor changed in place."""
    fa = _fa()
    dec = torch.tensor([0.1, 0.01], device="cuda")
    q, k, v = _qkv((2, 40))
    new = _qkv((2, n), seed=2)
    idx = None if idx is None else torch.tensor(idx, dtype=torch.int32, device="cuda")
    for call in range(3):
        pool = torch.randn(2, 2, 32, 32, device="cuda")
        leaf = q.clone().requires_grad_()
        out = fa.linear_attn_func(leaf, k, v, dec, initial_state=pool)
        before = pool._version
        fa.linear_attn_with_state(*new, pool, dec, state_idx=idx)
        assert pool._version > before, call
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
    # a clone keeps what the graph needs
    leaf = q.clone().requires_grad_()
    out = fa.linear_attn_func(leaf, k, v, dec, initial_state=pool.clone())
    fa.linear_attn_with_state(*new, pool, dec, state_idx=idx)
    out.sum().backward()
    assert torch.isfinite(leaf.grad).all()


def test_a_packed_pool_stepped_before_backward():
    fa = _fa()
    dec, cu = torch.tensor([0.1, 0.01], device="cuda"), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    q, k, v = _qkv((2,))
    pool = torch.randn(2, 2, 32, 32, device="cuda")
    leaf = q.clone().requires_grad_()
    out = fa.linear_attn_varlen_func(leaf, k, v, cu, 1, dec, initial_state=pool)
    fa.linear_attn_with_state(q, k, v, pool, dec, cu_seqlens=cu, max_seqlen=1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_pools_of_inference_mode():
    """Tensors of inference mode have no version to raise; they are stepped all the same."""
    fa = _fa()
    with torch.inference_mode():
        dec = torch.tensor([0.1, 0.01], device="cuda")
        for n in (1, 17):
            new = _qkv((2, n))
            one, two = (torch.zeros(2, 2, 32, 32, device="cuda") for _ in range(2))
            for _ in range(3):
                assert torch.equal(fa.linear_attn_with_state(*new, one, dec), fa.linear_attn_with_state(*new, two, dec))
            assert torch.equal(one, two) and one.any()
