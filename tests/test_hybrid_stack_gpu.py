"""Exact and linear attention layers over the same rotated queries and keys: a training step's gradients against 64 bits, and serving (a
prompt, then tokens one by one, caches and states side by side) against the training path."""
import pytest
import torch

from tests import linear_ref as ref

pytestmark = pytest.mark.gpu

H, HK, D, ROWS = 4, 2, 64, 64


def _fa():
    import fable_attn
    return fable_attn


def _weights(g, width=H * D):
    """Two layers' projections (q, k, v, out), N(0, 1 / width)."""
    w = lambda rows, cols: torch.randn(rows, cols, generator=g, dtype=torch.float64) * rows ** -0.5
    return [[w(width, H * D), w(width, HK * D), w(width, HK * D), w(H * D, width)] for _ in range(2)]


DECAY = torch.tensor([0.5, 0.1, 0.02, 0.004], dtype=torch.float64)


def _plain(x, weights, cos, sin):
    """One sequence (n, width) in float64: an exact causal layer, then a linear one, residuals around both."""
    n = x.shape[0]
    pos = torch.arange(n)
    for i, (wq, wk, wv, wo) in enumerate(weights):
        q, k, v = (x @ wq).view(n, H, D), (x @ wk).view(n, HK, D), (x @ wv).view(n, HK, D)
        q, k = ref.rotated(q, cos, sin, pos, False), ref.rotated(k, cos, sin, pos, False)
        if i == 0:
            s = torch.einsum("thd,shd->hts", q, ref.shared(k, H)) * D ** -0.5
            s = s.masked_fill(torch.ones(n, n).triu(1).bool(), float("-inf"))
            y = torch.einsum("hts,shd->thd", s.softmax(-1), ref.shared(v, H))
        else:
            y = ref.one(q, k, v, DECAY, D ** -0.5)[0]
        x = x + y.reshape(n, -1) @ wo
    return x


def _layers(fa, x, weights, cos, sin, cu, most):
    """The same over a packed batch (total, width) through the library."""
    for i, (wq, wk, wv, wo) in enumerate(weights):
        n = x.shape[0]
        q, k, v = (x @ wq).view(n, H, D), (x @ wk).view(n, HK, D), (x @ wv).view(n, HK, D)
        q, k = fa.flash_attn_rotary_func(q, k, cos, sin, rotary_interleaved=False, cu_seqlens=cu)
        if i == 0:
            y = fa.flash_attn_varlen_func(q, k, v, cu, cu, most, most, causal=True)
        else:
            y = fa.linear_attn_varlen_func(q, k, v, cu, most, DECAY.float().cuda())
        x = x + y.reshape(n, -1) @ wo
    return x


def test_training_step_fp32():
    """Gradients of the input and of all projections. Sums in 32 bits over up to 256 and 60 terms a step, some ten steps: 1e-4 of
    the largest is ample, and a wrong sign, head or position is of the order of 1."""
    fa = _fa()
    g = torch.Generator().manual_seed(1)
    lens = [37, 1, 60]
    cu = [0, 37, 38, 98]
    weights = _weights(g)
    x, dy = torch.randn(98, H * D, generator=g, dtype=torch.float64), torch.randn(98, H * D, generator=g, dtype=torch.float64)
    cos, sin = (t.double().cpu() for t in fa.flash_attn_rotary_tables(ROWS, D))
    leaves = [x.clone().requires_grad_()] + [w.clone().requires_grad_() for layer in weights for w in layer]
    pair = lambda ls: [ls[1:5], ls[5:9]]
    want = torch.cat([_plain(leaves[0][cu[b]:cu[b + 1]], pair(leaves), cos, sin) for b in range(3)])
    wg = torch.autograd.grad(want, leaves, dy)
    dev = [t.detach().float().cuda().requires_grad_() for t in leaves]
    got = _layers(fa, dev[0], pair(dev), cos.float().cuda(), sin.float().cuda(), torch.tensor(cu, dtype=torch.int32, device="cuda"), max(lens))
    gg = torch.autograd.grad(got, dev, dy.float().cuda())
    assert (got.detach().cpu().double() - want.detach()).abs().max() <= 1e-4 * want.abs().max()
    for a, b in zip(gg, wg):
        assert (a.cpu().double() - b).abs().max() <= 1e-4 * b.abs().max()


def test_serving_goes_on_from_a_prompt():
    """fp32: prompts of two requests, then ten tokens each: keys appended with rotation, states in a pool."""
    fa = _fa()
    g = torch.Generator().manual_seed(2)
    weights = [[w.float().cuda() for w in layer] for layer in _weights(g)]
    cos, sin = fa.flash_attn_rotary_tables(ROWS, D)
    lens, extra = [21, 40], 10
    full = [torch.randn(n + extra, H * D, generator=g).cuda() for n in lens]
    cu = torch.tensor([0, lens[0] + extra, sum(lens) + 2 * extra], dtype=torch.int32, device="cuda")
    want = _layers(fa, torch.cat(full), weights, cos, sin, cu, 50)
    want = [want[:lens[0] + extra], want[lens[0] + extra:]]
    kc, vc = (torch.zeros(2, 64, HK, D, device="cuda") for _ in range(2))
    pool, slots = torch.zeros(5, H, D, D, device="cuda"), torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    held = torch.zeros(2, dtype=torch.int32, device="cuda")
    decay = DECAY.float().cuda()

    def run(x, count):
        """New tokens (total, width), `count` of each request: packed prompts, or one each."""
        nonlocal held
        cu = torch.tensor([0, count[0], sum(count)], dtype=torch.int32, device="cuda")
        for i, (wq, wk, wv, wo) in enumerate(weights):
            n = x.shape[0]
            q, k, v = (x @ wq).view(n, H, D), (x @ wk).view(n, HK, D), (x @ wv).view(n, HK, D)
            if i == 0 and count == [1, 1]:
                y = fa.flash_attn_with_kvcache(q.unsqueeze(1), kc, vc, k.unsqueeze(1), v.unsqueeze(1), rotary_cos=cos, rotary_sin=sin,
                                               rotary_interleaved=False, cache_seqlens=held, causal=True)
            elif i == 0:
                q = fa.flash_attn_append_kvcache(k, v, kc, vc, held, q=q, cu_seqlens=cu, max_seqlen=max(count), rotary_cos=cos, rotary_sin=sin,
                                                 rotary_interleaved=False)
                kk, vv = fa.flash_attn_gather_kvcache(kc, vc, cu, sum(count))
                y = fa.flash_attn_varlen_func(q, kk, vv, cu, cu, max(count), max(count), causal=True)
            else:
                q, k = fa.flash_attn_rotary_func(q, k, cos, sin, rotary_interleaved=False, rotary_seqlens=held, cu_seqlens=cu)
                y = fa.linear_attn_with_state(q, k, v, pool, decay, state_idx=slots, cu_seqlens=cu, max_seqlen=max(count))
            x = x + y.reshape(n, -1) @ wo
        held = held + torch.tensor(count, dtype=torch.int32, device="cuda")
        return x

    outs = [run(torch.cat([full[b][:lens[b]] for b in range(2)]), lens)]
    near = lambda a, b: (a - b).abs().max() <= 1e-4 * b.abs().max()
    assert near(outs[0][:lens[0]], want[0][:lens[0]]) and near(outs[0][lens[0]:], want[1][:lens[1]])
    for t in range(extra):
        y = run(torch.stack([full[b][lens[b] + t] for b in range(2)]), [1, 1])
        assert near(y[0], want[0][lens[0] + t]) and near(y[1], want[1][lens[1] + t]), t
    assert not pool[[0, 2, 4]].any()


def test_captured_training_pass():
    """Rotation, linear attention of packed sequences and the gradients of both in one graph, on leaves that no other graph holds:
    replays on new inputs give an eager pass's bits."""
    fa = _fa()
    g = torch.Generator().manual_seed(3)
    n = 1500
    make = lambda heads: torch.randn(n, heads, D, generator=g).to(torch.bfloat16)
    new = lambda: [make(H), make(HK), make(HK), make(H)]
    cos, sin = fa.flash_attn_rotary_tables(n, D)
    cu, decay = torch.tensor([0, 1100, 1101, 1400], dtype=torch.int32, device="cuda"), DECAY.float().cuda()
    *leaves, dout = (t.cuda() for t in new())
    for t in leaves:
        t.requires_grad_()

    def step(leaves, dout):
        q, k = fa.flash_attn_rotary_func(leaves[0], leaves[1], cos, sin, cu_seqlens=cu)
        out = fa.linear_attn_varlen_func(q, k, leaves[2], cu, 1100, decay)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(leaves, dout)
    for _ in range(4):
        fresh = [t.cuda() for t in new()]
        with torch.no_grad():
            for x, y in zip((*leaves, dout), fresh):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in kept]
        want = step([t.requires_grad_() for t in fresh[:3]], fresh[3])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_threads():
    """Two threads, each on a stream of its own, train and step at once: plans are a thread's own."""
    import threading
    fa = _fa()
    g = torch.Generator().manual_seed(4)
    cos, sin = fa.flash_attn_rotary_tables(ROWS, D)
    decay = DECAY.float().cuda()
    data = [[torch.randn(2, 50, heads, D, generator=g).half().cuda() for heads in (H, HK, HK, H)] for _ in range(2)]

    def work(t):
        *leaves, dout = (x.clone() for x in data[t])
        for x in leaves:
            x.requires_grad_()
        pool = torch.zeros(2, H, D, D, device="cuda")
        res = []
        for i in range(8):
            q, k = fa.flash_attn_rotary_func(leaves[0], leaves[1], cos, sin, rotary_seqlens=i)
            out = fa.linear_attn_func(q, k, leaves[2], decay)
            res += [out.detach(), *torch.autograd.grad(out, leaves, dout)]
            q, k, v = (x.detach()[:, :1] for x in (q, k, leaves[2]))
            res.append(fa.linear_attn_with_state(q, k, v, pool, decay))
        return [*res, pool]

    want = [work(t) for t in range(2)]
    torch.cuda.synchronize()
    got = [None, None]

    def run(t):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[t] = work(t)
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
