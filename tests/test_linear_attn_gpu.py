"""Linear attention against its definition in 64 bits: forward, gradients, states, steps."""
import pytest
import torch

from tests import linear_ref as ref
from tests.linear_ref import DT

pytestmark = pytest.mark.gpu


def _fa():
    import fable_attn
    return fable_attn


def _cu(lens, front=0):
    cu = [front]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _rand(gen, shape, dtype, kind):
    x = torch.randn(shape, generator=gen, dtype=torch.float32)
    if kind == "plus":               # no cancellation: the bounds are as tight as they get
        x = x.abs()
    elif kind == "whole":
        x = x.round().clamp(-1, 1)
    return x.to(DT[dtype])


def _inputs(dtype, rows, hq, hk, dk, dv, seed, kind="any"):
    g = torch.Generator().manual_seed(seed)
    return _rand(g, (*rows, hq, dk), dtype, kind), _rand(g, (*rows, hk, dk), dtype, kind), _rand(g, (*rows, hk, dv), dtype, kind), g


def _decay(H, name):
    i = torch.arange(1, H + 1, dtype=torch.float32)
    return {"slopes": torch.exp2(-8 * i / H), "slow": torch.exp2(-8 * i / H) / 64, "none": torch.zeros(H),
            "mixed": torch.tensor([0.0, 1e-6, 0.01, 0.3, 3.0, 200.0, 1e30, float("inf")]).repeat(-(-H // 8))[:H]}[name]


def _run(dtype, lens, hq, hk, dk, dv, *, packed=True, decay="slopes", carry=False, want=True, grad=False, seed=0, kind="any", front=0, tail=0,
         scale=None, most=None, per_batch=False):
    """One call, forward and (grad) backward, against the definition."""
    print(f"[linear] {dtype} lens={lens} hq={hq} hk={hk} dk={dk} dv={dv} packed={packed} decay={decay} carry={carry} grad={grad} {kind} seed={seed}", flush=True)
    fa = _fa()
    B = len(lens)
    cu = _cu(lens, front) if packed else None
    rows = (cu[-1] + tail,) if packed else (B, lens[0])
    q, k, v, g = _inputs(dtype, rows, hq, hk, dk, dv, seed, kind)
    dec = _decay(hq, decay)
    if per_batch:
        dec = dec[None] * torch.linspace(0.5, 2, B)[:, None]
    state = _rand(g, (B, hq, dk, dv), "fp32", kind) if carry else None
    dout, dlast = _rand(g, (*rows, hq, dv), dtype, kind), _rand(g, (B, hq, dk, dv), "fp32", kind)
    sc = dk ** -0.5 if scale is None else scale
    wide = [x.double().requires_grad_(grad) for x in (q, k, v)] + [state.double().requires_grad_(grad) if carry else None]
    eo, es = ref.batch(*wide[:3], dec.double(), sc, cu, wide[3])
    dev = [x.cuda().requires_grad_(grad) for x in (q, k, v)] + [state.cuda().requires_grad_(grad) if carry else None]
    kw = dict(scale=scale, initial_state=dev[3], return_final_state=want)
    if packed:
        got = fa.linear_attn_varlen_func(*dev[:3], _i32(cu), max(lens) if most is None else most, dec.cuda(), **kw)
    else:
        got = fa.linear_attn_func(*dev[:3], dec.cuda(), **kw)
    out, last = got if want else (got, None)
    assert out.dtype == DT[dtype] and out.is_contiguous()
    with torch.no_grad():
        plain = [x.detach() for x in wide[:3]] + [wide[3].detach() if carry else None]
        mo, ms = ref.sums(*plain[:3], dec.double(), sc, cu, plain[3])
        n = max(lens + [1])
        worst = ref.check(out, eo.detach(), ref.bound(eo.detach(), mo, DT[dtype], n, dk), "out")
        if want:
            assert last.dtype == torch.float32
            worst = max(worst, ref.check(last, es.detach(), ref.state_bound(ms, DT[dtype], n, dk), "state"))
    if cu is not None:
        assert not out[:front].any() and not out[cu[-1]:].any()
    if grad:
        dl = dlast if want else None
        eg = torch.autograd.grad([eo] + ([es] if want else []), [x for x in wide if x is not None], [dout.double()] + ([dl.double()] if want else []))
        gg = torch.autograd.grad([out] + ([last] if want else []), [x for x in dev if x is not None], [dout.cuda()] + ([dl.cuda()] if want else []))
        # what the gradients' terms sum to in size: the same products of absolute values
        mag = [x.detach().abs().requires_grad_() for x in wide if x is not None]
        ao, as_ = ref.batch(mag[0], mag[1], mag[2], dec.double(), abs(sc), cu, mag[3] if carry else None)
        am = torch.autograd.grad([ao] + ([as_] if want else []), mag, [dout.double().abs()] + ([dl.double().abs()] if want else []))
        for name, x, e, m in zip(("dq", "dk", "dv", "dstate"), gg, eg, am):
            assert x.is_contiguous()
            if name == "dstate":
                tol = ref.state_bound(m, DT[dtype], n, dk)
            else:
                tol = ref.bound(e, m, DT[dtype], n, max(dk, dv))
            worst = max(worst, ref.check(x, e, tol, name))
        if cu is not None:
            for x in gg[:3]:
                assert not x[:front].any() and not x[cu[-1]:].any()
    print(f"[linear]   worst {worst:.3f} of its bound", flush=True)


ALL = ["bf16", "fp16", "fp32"]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 100, 129])
def test_lengths(dtype, n):
    _run(dtype, [n, n], 2, 2, 64, 64, packed=False, seed=n, carry=n % 2 == 1)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("dk,dv", [(8, 8), (16, 40), (32, 64), (64, 128), (80, 80), (96, 32), (128, 128), (128, 200), (136, 72), (192, 192), (256, 64), (64, 256), (256, 256)])
def test_head_dims(dtype, dk, dv):
    _run(dtype, [70, 150], 2, 1, dk, dv, seed=dk + dv, carry=True)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("dk,dv", [(5, 12), (100, 70)])
def test_head_dims_padded(dtype, dk, dv):
    _run(dtype, [40, 70], 2, 2, dk, dv, seed=7, carry=True, grad=True)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("decay", ["slopes", "slow", "none", "mixed"])
@pytest.mark.parametrize("kind", ["any", "plus"])
def test_decays(dtype, decay, kind):
    _run(dtype, [200, 333], 8, 4, 64, 64, decay=decay, kind=kind, seed=3)


@pytest.mark.parametrize("dtype", ALL)
def test_whole_numbers_are_exact(dtype):
    """Without decay and with values in {-1, 0, 1} every product, score, state and sum is exact in every type."""
    fa = _fa()
    for packed, lens, dk, dv in ((False, [200, 200], 64, 64), (True, [1, 0, 63, 190], 128, 96), (True, [65, 130], 32, 256)):
        cu = _cu(lens) if packed else None
        rows = (cu[-1],) if packed else (len(lens), lens[0])
        q, k, v, _ = _inputs(dtype, rows, 4, 2, dk, dv, 5, "whole")
        want, last = ref.batch(q.double(), k.double(), v.double(), torch.zeros(4).double(), 1.0, cu)
        args = [x.cuda() for x in (q, k, v)]
        kw = dict(scale=1.0, return_final_state=True)
        got = (fa.linear_attn_varlen_func(*args, _i32(cu), max(lens), torch.zeros(4).cuda(), **kw) if packed
               else fa.linear_attn_func(*args, torch.zeros(4).cuda(), **kw))
        assert torch.equal(got[0].cpu(), want.to(DT[dtype])) and torch.equal(got[1].cpu().double(), last)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("lens,front,tail", [([0], 0, 0), ([0, 0, 5], 0, 3), ([5, 0, 70, 1], 4, 9), ([300, 1, 64, 0], 0, 0), ([0], 3, 2)])
def test_packed(dtype, lens, front, tail):
    _run(dtype, lens, 4, 2, 64, 64, front=front, tail=tail, carry=True, grad=True, seed=11)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (8, 2), (5, 5)])
@pytest.mark.parametrize("carry", [False, True])
def test_gradients(dtype, hq, hk, carry):
    _run(dtype, [97, 97], hq, hk, 64, 96, packed=False, grad=True, want=carry, carry=carry, seed=hq)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("decay", ["slow", "none", "mixed"])
def test_gradients_of_decays(dtype, decay):
    _run(dtype, [150, 70], 8, 8, 32, 32, decay=decay, grad=True, carry=True, seed=2, kind="plus")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("dk,dv", [(128, 128), (256, 80), (80, 256)])
def test_gradients_of_wide_heads(dtype, dk, dv):
    _run(dtype, [130, 33], 2, 1, dk, dv, grad=True, carry=True, seed=4)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("packed", [False, True])
def test_segments(dtype, packed):
    """Few heads and long sequences: cut into segments, whose states are chained."""
    _run(dtype, [1500, 1500] if not packed else [2000, 3, 900, 0], 2, 2, 64, 64, packed=packed, grad=True, carry=True, decay="slow", seed=6)


@pytest.mark.parametrize("most", [1, 100, 5000, 10 ** 9])
def test_max_seqlen_only_sizes_the_launch(most):
    _run("bf16", [700, 90], 2, 1, 64, 64, grad=True, carry=True, seed=8, most=most)


def test_decay_per_sequence():
    _run("bf16", [100, 160, 3], 4, 4, 64, 64, per_batch=True, grad=True, seed=9)


def test_scale():
    for scale in (0.0, -0.3, 2.5):
        _run("fp32", [90], 2, 2, 32, 32, packed=False, scale=scale, grad=True, carry=True, seed=10)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 16, 17, 70])
@pytest.mark.parametrize("idx", [None, "some"])
def test_state_steps(dtype, n, idx):
    """A pool's states move by the new tokens, padded entries change nothing, other states stay."""
    fa = _fa()
    for hq, hk, dk, dv in ((4, 2, 64, 64), (2, 2, 128, 136), (1, 1, 256, 8), (3, 1, 8, 40)):
        print(f"[step] {dtype} n={n} {hq}/{hk} {dk}x{dv} idx={idx}", flush=True)
        slots = [4, 0, 2] if idx is None else [3, -1, 0, 99]
        B = 3 if idx is None else 4
        order = [0, 1, 2] if idx is None else slots
        q, k, v, g = _inputs(dtype, (B, n), hq, hk, dk, dv, n + dk)
        pool = torch.randn(5, hq, dk, dv, generator=g)
        dec = _decay(hq, "slopes")
        got_pool = pool.cuda()
        out = fa.linear_attn_with_state(q.cuda(), k.cuda(), v.cuda(), got_pool, dec.cuda(), state_idx=None if idx is None else _i32(slots))
        want_pool, tol = pool.double().clone(), torch.zeros_like(pool, dtype=torch.float64)
        for b, s in enumerate(order):
            if not 0 <= s < 5:
                assert not out[b].any()
                continue
            args = (q[b].double(), k[b].double(), v[b].double(), dec.double(), dk ** -0.5)
            eo, es = ref.one(*args, pool[s].double())
            mo, ms = ref.one(*(x.abs() for x in args[:3]), *args[3:], pool[s].double().abs())
            ref.check(out[b], eo, ref.bound(eo, mo, DT[dtype], n, dk), "out")
            want_pool[s], tol[s] = es, ref.state_bound(ms, DT[dtype], n, dk)
        ref.check(got_pool, want_pool, tol + 1e-300, "pool")
        untouched = [s for s in range(5) if s not in order]
        assert torch.equal(got_pool.cpu()[untouched], pool[untouched])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens", [[1, 3, 0, 2], [40, 1, 0, 300], [700, 2, 900, 1]])
def test_state_ragged(dtype, lens):
    """Prompts and single tokens in one packed call, with rows behind the last sequence."""
    fa = _fa()
    cu = _cu(lens)
    q, k, v, g = _inputs(dtype, (cu[-1] + 5,), 4, 2, 64, 64, 1)
    pool, dec, slots = torch.randn(6, 4, 64, 64, generator=g), _decay(4, "slow"), [5, 1, 0, 2]
    got = pool.cuda()
    out = fa.linear_attn_with_state(q.cuda(), k.cuda(), v.cuda(), got, dec.cuda(), state_idx=_i32(slots), cu_seqlens=_i32(cu), max_seqlen=max(lens))
    assert not out[cu[-1]:].any()
    wide = [x.double() for x in (q, k, v)]
    eo, es = ref.batch(*wide, dec.double(), 0.125, cu, pool[slots].double())
    mo, ms = ref.sums(*wide, dec.double(), 0.125, cu, pool[slots].double())
    ref.check(out, eo, ref.bound(eo, mo, DT[dtype], max(lens), 64), "out")
    ref.check(got[slots], es, ref.state_bound(ms, DT[dtype], max(lens), 64), "states")
    rest = [s for s in range(6) if s not in slots]
    assert torch.equal(got.cpu()[rest], pool[rest])


def test_steps_go_on_from_a_prompt():
    """A prompt and then single tokens give what one call over all of them gives."""
    fa = _fa()
    q, k, v, _ = _inputs("fp32", (2, 140), 4, 4, 64, 64, 3)
    q, k, v, dec = q.cuda(), k.cuda(), v.cuda(), _decay(4, "slow").cuda()
    whole, last = fa.linear_attn_func(q, k, v, dec, return_final_state=True)
    part, state = fa.linear_attn_func(q[:, :120], k[:, :120], v[:, :120], dec, return_final_state=True)
    outs = [part] + [fa.linear_attn_with_state(q[:, i:i + 1], k[:, i:i + 1], v[:, i:i + 1], state, dec) for i in range(120, 140)]
    assert torch.allclose(torch.cat(outs, 1), whole, rtol=1e-4, atol=1e-4) and torch.allclose(state, last, rtol=1e-4, atol=1e-4)


def test_strided_inputs():
    """Columns of one projection, a transposed layout, an expanded batch and a misaligned base give what dense copies give."""
    fa = _fa()
    dec = _decay(4, "slopes").cuda()
    x = torch.randn(2, 90, 12, 64, device="cuda", dtype=torch.bfloat16)
    q, k, v = x[:, :, :4], x[:, :, 4:8], x[:, :, 8:]
    want = fa.linear_attn_func(q.contiguous(), k.contiguous(), v.contiguous(), dec)
    assert torch.equal(fa.linear_attn_func(q, k, v, dec), want)
    t = lambda y: y.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(fa.linear_attn_func(t(q), t(k), t(v), dec), want)
    off = torch.empty(q.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view(q.shape).copy_(q)
    assert torch.equal(fa.linear_attn_func(off, k, v, dec), want)
    one = k[:1].expand(2, -1, -1, -1)
    assert torch.equal(fa.linear_attn_func(q, one, v, dec), fa.linear_attn_func(q, one.contiguous(), v, dec))
    row = k[:, :1].expand(-1, 90, -1, -1)
    assert torch.equal(fa.linear_attn_func(q, row, v, dec), fa.linear_attn_func(q, row.contiguous(), v, dec))
    # a gradient that is an expanded scalar
    a, b = q.detach().clone().requires_grad_(), q.detach().clone().requires_grad_()
    fa.linear_attn_func(a, k, v, dec).sum().backward()
    o = fa.linear_attn_func(b, k, v, dec)
    o.backward(torch.ones_like(o))
    assert torch.equal(a.grad, b.grad)


def test_values_of_every_size():
    """fp16 scores and states past its range, and values near its smallest, in the forward pass and the gradients."""
    fa = _fa()
    for sq, sk, sv in ((1.0, 200.0, 200.0), (100.0, 100.0, 0.01), (1e-3, 1.0, 1e-4), (1.0, 1e-4, 1e-4)):
        q, k, v, g = _inputs("fp16", (1, 300), 2, 2, 64, 64, 1, "plus")
        q, k, v = (q.float() * sq).half(), (k.float() * sk).half(), (v.float() * sv).half()
        dec = _decay(2, "slow")
        # outputs within fp16's own range
        wide = [x.double() for x in (q, k, v)]
        scale = 1.0 / float(ref.batch(*wide, dec.double(), 1.0)[0].abs().max())
        eo, es = ref.batch(*wide, dec.double(), scale)
        mo, ms = ref.sums(*wide, dec.double(), scale)
        out, last = fa.linear_attn_func(q.cuda(), k.cuda(), v.cuda(), dec.cuda(), scale=scale, return_final_state=True)
        # (subnormal scores and products of them round by half of fp16's smallest step, 2^-25, of the values they meet)
        ref.check(out, eo, ref.bound(eo, mo, torch.float16, 300, 64) + 64 * 2.0 ** -25 * v.double().abs().max(), "out")
        ref.check(last, es, ref.state_bound(ms, torch.float16, 300, 64), "state")


def test_two_streams_and_bits():
    """Calls on two streams at once, and repeated ones, give the same bits."""
    fa = _fa()
    q, k, v, _ = _inputs("bf16", (1, 3000), 2, 2, 64, 64, 1)
    q, k, v, dec = q.cuda(), k.cuda(), v.cuda(), _decay(2, "slow").cuda()
    want = fa.linear_attn_func(q, k, v, dec)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(fa.linear_attn_func(q, k, v, dec))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_graph_replays():
    """A prompt cut into segments, a step and a backward pass, captured and replayed with new inputs."""
    fa = _fa()
    q, k, v, _ = _inputs("bf16", (1, 1200), 2, 2, 64, 64, 1)
    q, k, v, dec = q.cuda(), k.cuda(), v.cuda(), _decay(2, "slow").cuda()
    state = torch.zeros(2, 2, 64, 64, device="cuda")
    idx = _i32([1])

    def work():
        out, last = fa.linear_attn_func(q, k, v, dec, return_final_state=True)
        state[1:].copy_(last)
        step = fa.linear_attn_with_state(q[:, :1], k[:, :1], v[:, :1], state, dec, state_idx=idx)
        grads = fa._C.linear_bwd(out, q, k, v, dec, 0.125)[:3]
        return out, step, state.clone(), *grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = work()
    for seed in range(4):
        new = _inputs("bf16", (1, 1200), 2, 2, 64, 64, 50 + seed)
        for x, y in zip((q, k, v), new):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in kept]
        want = work()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_refusals():
    fa = _fa()
    q, k, v, _ = _inputs("bf16", (2, 10), 4, 2, 64, 64, 1)
    q, k, v, dec = q.cuda(), k.cuda(), v.cuda(), torch.zeros(4, device="cuda")
    with pytest.raises(ValueError):
        fa.linear_attn_func(q, k, v[0], dec)
    with pytest.raises(ValueError):
        fa.linear_attn_func(q[:, :, :3], k, v, dec)
    with pytest.raises(RuntimeError):
        fa.linear_attn_func(q, k[:, :5], v, dec)
    with pytest.raises(RuntimeError):
        fa.linear_attn_func(q, k, v, dec[:3])
    with pytest.raises(RuntimeError):
        fa.linear_attn_func(q, k.half(), v, dec)
    with pytest.raises(TypeError):
        fa.linear_attn_func(q, k, v, 0.5)
    with pytest.raises(NotImplementedError):
        fa.linear_attn_func(q, k, v, torch.zeros(4, device="cuda", requires_grad=True))
    with pytest.raises(ValueError):
        fa.linear_attn_func(q, k, v, dec, initial_state=torch.zeros(2, 4, 64, 32, device="cuda"))
    with pytest.raises(ValueError):
        fa.linear_attn_func(q.double(), k.double(), v.double(), dec)
    with pytest.raises(ValueError):
        fa.linear_attn_with_state(q, k, v, torch.zeros(2, 4, 64, 64, device="cuda", dtype=torch.bfloat16), dec)
    with pytest.raises(RuntimeError):
        fa.linear_attn_with_state(q, k, v, torch.zeros(1, 4, 64, 64, device="cuda"), dec)
    with pytest.raises(RuntimeError):
        fa.linear_attn_with_state(q, k, v, torch.zeros(2, 4, 64, 64, device="cuda"), dec, state_idx=_i32([0]))
    a = q.float().requires_grad_()
    (g,) = torch.autograd.grad(fa.linear_attn_func(a, k.float(), v.float(), dec).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_many_short_sequences_and_a_long_one(dtype):
    """More sequences than a workgroup has threads, most of one or two rows, a few of several segments, rows in front and behind."""
    lens = [1] * 281 + [700] + [0, 2] * 20 + [513, 256, 257] + [1] * 30
    _run(dtype, lens, 2, 1, 64, 64, front=3, tail=2, grad=True, carry=True, decay="slow", seed=12)


def test_mixed_batch_of_a_pool():
    """The same kind of batch over a pool in place, some of its entries naming no state."""
    fa = _fa()
    lens = [1] * 260 + [900, 0, 1, 600]
    cu = _cu(lens)
    q, k, v, g = _inputs("bf16", (cu[-1],), 2, 2, 64, 64, 1)
    slots = torch.randperm(300, generator=g)[:len(lens)].tolist()
    slots[5], slots[262] = -1, 300
    pool, dec = torch.randn(300, 2, 64, 64, generator=g), _decay(2, "slow")
    got = pool.cuda()
    out = fa.linear_attn_with_state(q.cuda(), k.cuda(), v.cuda(), got, dec.cuda(), state_idx=_i32(slots), cu_seqlens=_i32(cu), max_seqlen=900).cpu()
    want, tol = pool.double().clone(), torch.zeros(pool.shape, dtype=torch.float64)
    for b, s in enumerate(slots):
        rows = slice(cu[b], cu[b + 1])
        if not 0 <= s < 300:
            assert not out[rows].any()
            continue
        args = (q[rows].double(), k[rows].double(), v[rows].double(), dec.double(), 0.125)
        eo, es = ref.one(*args, pool[s].double())
        mo, ms = ref.one(*(x.abs() for x in args[:3]), *args[3:], pool[s].double().abs())
        ref.check(out[rows], eo, ref.bound(eo, mo, torch.bfloat16, lens[b], 64), "out")
        want[s], tol[s] = es, ref.state_bound(ms, torch.bfloat16, lens[b], 64)
    ref.check(got, want, tol + 1e-300, "pool")


@pytest.mark.parametrize("dtype", ALL)
def test_nothing_new_behind_old_rows(dtype):
    """Padding by rows whose keys are zeros: the state is only what is left of the earlier rows, exact to its own size. An
    exponent k d is off by two roundings, so is what it weighs, relatively."""
    fa = _fa()
    q, k, v, _ = _inputs(dtype, (1, 700), 4, 4, 64, 64, 5, "plus")
    k[:, 400:] = 0
    dec = torch.tensor([0.0, 0.003, 0.05, 0.2])
    out, last = fa.linear_attn_func(q.cuda(), k.cuda(), v.cuda(), dec.cuda(), return_final_state=True)
    wide = [x.double() for x in (q, k, v)]
    eo, es = ref.batch(*wide, dec.double(), 0.125)
    tol = ref.state_bound(es, DT[dtype], 700, 64) + 2.0 ** -22 * 700 * dec.double()[None, :, None, None] * es
    ref.check(last, es, tol, "state")
    more = ref.bound(eo, eo, DT[dtype], 700, 64) + 2.0 ** -22 * 700 * dec.double()[None, None, :, None] * eo
    ref.check(out, eo, more, "out")
    # and one by one
    state = last.clone()
    zero = torch.zeros(1, 8, 4, 64, device="cuda", dtype=DT[dtype])
    fa.linear_attn_with_state(zero, zero, zero, state, dec.cuda())
    assert torch.allclose(state.cpu().double(), last.cpu().double() * torch.exp(-8 * dec.double())[None, :, None, None], rtol=16 * 2.0 ** -24, atol=0)


def test_rows_far_apart():
    """Rows 8 MiB apart: offsets past 32 bits over the sequence, buffer descriptors of 64 rows, in both directions."""
    fa = _fa()
    big = torch.empty(600, 1 << 22, device="cuda", dtype=torch.bfloat16)
    dense = [torch.randn(600, 1, 64, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    far = []
    for i, x in enumerate(dense):
        view = big[:, 64 * i:64 * i + 64].unsqueeze(1)
        view.copy_(x)
        far.append(view)
    dec = torch.tensor([0.01], device="cuda")
    cu = _i32([0, 600])
    assert torch.equal(fa.linear_attn_varlen_func(*far[:3], cu, 600, dec), fa.linear_attn_varlen_func(*dense[:3], cu, 600, dec))
    for x, y in zip(fa._C.linear_bwd(far[3], *far[:3], dec, 0.125, cu, 600)[:3], fa._C.linear_bwd(dense[3], *dense[:3], dec, 0.125, cu, 600)[:3]):
        assert torch.equal(x, y)
    del big, far


def test_empty_batches():
    fa = _fa()
    dec = torch.zeros(2, device="cuda")
    mk = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)
    out, last = fa.linear_attn_func(mk(0, 5, 2, 64), mk(0, 5, 2, 64), mk(0, 5, 2, 64), dec, return_final_state=True)
    assert out.shape == (0, 5, 2, 64) and last.shape == (0, 2, 64, 64)
    first = torch.randn(3, 2, 64, 64, device="cuda")
    out, last = fa.linear_attn_func(mk(3, 0, 2, 64), mk(3, 0, 2, 64), mk(3, 0, 2, 64), dec, initial_state=first, return_final_state=True)
    assert out.shape == (3, 0, 2, 64) and torch.equal(last, first)
    out = fa.linear_attn_varlen_func(mk(4, 2, 64) + 1, mk(4, 2, 64) + 1, mk(4, 2, 64) + 1, _i32([0]), 0, dec)
    assert out.shape == (4, 2, 64) and not out.any()
    assert fa.linear_attn_with_state(mk(0, 1, 2, 64), mk(0, 1, 2, 64), mk(0, 1, 2, 64), first, dec).shape == (0, 1, 2, 64)


def test_bad_lengths_stay_in_bounds():
    """Offsets past the rows, or not in order, are not refused (they are on the GPU), but nothing outside the tensors is touched."""
    fa = _fa()
    big = torch.full((64, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    q, k, v = big[16:48].clone(), big[16:48].clone(), big[16:48].clone()
    dec = torch.zeros(2, device="cuda")
    for cu in ([0, 100], [-5, 10, 32], [20, 10, 32], [0, 40, 20, 90]):
        for most in (4, 32):
            assert fa.linear_attn_varlen_func(q, k, v, _i32(cu), most, dec).shape == q.shape
            pool = torch.zeros(len(cu) - 1, 2, 64, 64, device="cuda")
            fa.linear_attn_with_state(q, k, v, pool, dec, cu_seqlens=_i32(cu), max_seqlen=most)
            fa.flash_attn_rotary_func(q, k, torch.ones(8, 32, device="cuda"), torch.zeros(8, 32, device="cuda"), cu_seqlens=_i32(cu))
    torch.cuda.synchronize()


def test_calls_of_a_known_signature():
    """Later calls of a signature fill in addresses only: other tensors, tables and lengths, the same results as first calls."""
    fa = _fa()
    dec = _decay(4, "slopes").cuda()
    for seed in range(3):
        q, k, v, g = (x.cuda() if torch.is_tensor(x) else x for x in _inputs("bf16", (2, 300), 4, 2, 64, 64, seed))
        first = torch.randn(2, 4, 64, 64, generator=g).cuda()
        q.requires_grad_()
        got = fa.linear_attn_func(q, k, v, dec, initial_state=first, return_final_state=True)
        (dq,) = torch.autograd.grad(got[0], q, got[0].detach())
        fresh, seg = fa._C.linear_fwd(q.detach(), k, v, dec, 0.125, None, 0, first, torch.empty_like(first))[:2]
        assert torch.equal(got[0], fresh)
        # (over the forward pass's states: with a final state wanted they have a part more than those the backward pass would form)
        assert torch.equal(dq, fa._C.linear_bwd(got[0].detach(), q.detach(), k, v, dec, 0.125, None, 0, first, seg_states=seg)[0])
        step, pool = [x[:, :1].detach().contiguous() for x in (q, k, v)], first.clone()
        idx = _i32([seed % 2, 1 - seed % 2])
        out = fa.linear_attn_with_state(*step, pool, dec, state_idx=idx)
        other = first.clone()
        assert torch.equal(out, fa._C.linear_step(*step, other, dec, 0.125, None, 1, idx)[0]) and torch.equal(pool, other)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_keys_and_queries_that_are_no_numbers(dtype, bad):
    """A query reaches its own row only, a key its row and later ones, in another sequence nothing."""
    fa = _fa()
    q, k, v, _ = (x.cuda() if torch.is_tensor(x) else x for x in _inputs(dtype, (120,), 2, 2, 64, 64, 1))
    dec, cu = torch.tensor([0.0, 0.01], device="cuda"), _i32([0, 70, 120])
    want = fa.linear_attn_varlen_func(q, k, v, cu, 70, dec)
    q2, k2 = q.clone(), k.clone()
    q2[20, 0, 3] = bad
    k2[40, 1, 5] = bad
    out = fa.linear_attn_varlen_func(q2, k2, v, cu, 70, dec)
    keep = torch.ones(120, 2, dtype=torch.bool, device="cuda")
    keep[20, 0] = False
    keep[40:70, 1] = False
    assert torch.equal(out[keep], want[keep])
    assert not torch.isfinite(out[20, 0]).any() and not torch.isfinite(out[40:70, 1]).any()


@pytest.mark.parametrize("packed", [False, True])
def test_more_states_than_sixteen_bits_count(packed):
    """2100 sequences x 32 heads: steps, and packed prompts with gradients, against the same in two halves."""
    fa = _fa()
    B, H, D = 2100, 32, 8
    q, k, v, _ = _inputs("bf16", (3 * B,) if packed else (B, 1), H, H, D, D, 3)
    q, k, v = (x.cuda() for x in (q, k, v))
    dec = torch.linspace(0.0, 1.0, H, device="cuda")
    if not packed:
        pool = torch.randn(B, H, D, D, device="cuda")
        halves = [pool[i:i + B // 2].clone() for i in (0, B // 2)]
        out = fa.linear_attn_with_state(q, k, v, pool, dec)
        parts = [fa.linear_attn_with_state(q[i:i + B // 2], k[i:i + B // 2], v[i:i + B // 2], s, dec) for i, s in zip((0, B // 2), halves)]
        assert torch.equal(out, torch.cat(parts)) and torch.equal(pool, torch.cat(halves))
        return
    cu = torch.arange(0, 3 * B + 1, 3, dtype=torch.int32, device="cuda")
    def run(a, b):
        x = [t[3 * a:3 * b].detach().requires_grad_() for t in (q, k, v)]
        out = fa.linear_attn_varlen_func(*x, cu[a:b + 1] - 3 * a, 3, dec)
        out.float().square().sum().backward()
        return [out] + [t.grad for t in x]
    for whole, one, two in zip(run(0, B), run(0, B // 2), run(B // 2, B)):
        assert torch.equal(whole, torch.cat([one, two]))


def test_a_single_row_has_any_stride():
    """A token per sequence out of a layout whose row stride is past what several rows may have."""
    fa = _fa()
    D = 64
    base = torch.randn(2, 4, D, device="cuda", dtype=torch.bfloat16)
    q = torch.as_strided(base, (2, 1, 4, D), (4 * D, 1 << 25, D, 1))
    pool = torch.zeros(2, 4, D, D, device="cuda")
    dec = torch.zeros(4, device="cuda")
    out = fa.linear_attn_with_state(q, q, q, pool, dec)
    want = fa.linear_attn_func(base[:, None], base[:, None], base[:, None], dec)
    assert torch.equal(fa.linear_attn_func(q, q, q, dec), want)
    # (two roundings on the way of the chunks, one on the steps')
    ref = (base.double() * base.double()).sum(-1, keepdim=True) * D ** -0.5 * base.double()
    assert torch.allclose(out[:, 0].double(), ref, rtol=2.0 ** -7, atol=0)


def test_scale_and_lengths_given_as_tensors():
    """A plan is known by their values, not by the objects."""
    fa = _fa()
    x = torch.randn(2, 1, 2, 32, device="cuda", dtype=torch.float32)
    dec, scale = torch.zeros(2, device="cuda"), torch.tensor(0.5)
    run = lambda s: fa.linear_attn_with_state(x, x, x, torch.zeros(2, 2, 32, 32, device="cuda"), dec, scale=s)
    first = run(scale)
    assert torch.equal(run(scale), first)
    scale.fill_(0.25)
    assert torch.equal(run(scale), run(0.25)) and torch.equal(2 * run(scale), first)
    p = x[:, 0]
    cu, most = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), torch.tensor(1)
    assert torch.equal(fa.linear_attn_varlen_func(p, p, p, cu, most, dec, scale=0.5), fa.linear_attn_varlen_func(p, p, p, cu, 1, dec, scale=0.5))


def test_long_gaps_are_zeroed():
    fa = _fa()
    q, k, v, _ = _inputs("fp16", (20011,), 2, 1, 40, 72, 5)
    q, k, v = (x.cuda() for x in (q, k, v))
    cu, dec = _i32([9000, 9010]), torch.zeros(2, device="cuda")
    torch.full((20011, 2, 72), 7.0, device="cuda", dtype=torch.float16)   # (freed: what the outputs may be laid over)
    for out in (fa.linear_attn_varlen_func(q, k, v, cu, 10, dec),
                fa.linear_attn_with_state(q, k, v, torch.zeros(1, 2, 40, 72, device="cuda"), dec, cu_seqlens=cu, max_seqlen=10),
                fa.linear_attn_with_state(q, k, v, torch.zeros(1, 2, 40, 72, device="cuda"), dec, cu_seqlens=cu, max_seqlen=100),
                fa.linear_attn_with_state(q, k, v, torch.zeros(1, 2, 40, 72, device="cuda"), dec, _i32([-1]), cu_seqlens=cu, max_seqlen=10)):
        assert not out[:9000].any() and not out[9010:].any()


@pytest.mark.parametrize("seed", range(32))
def test_sweep(seed):
    """Seeded calls over the whole range of what the fixed cases above list one by one."""
    import random
    r = random.Random(1000 + seed)
    packed = r.random() < 0.6
    B = r.choice([1, 2, 3, 7])
    lens = [r.choice([0, 1, 2, 31, 32, 33, 64, 65, 127, 300, 700]) for _ in range(B)] if packed else [r.choice([1, 5, 32, 100, 257, 640])] * B
    hk = r.choice([1, 2, 3])
    hq = hk * r.choice([1, 1, 2, 4])
    dk, dv = r.choice([8, 24, 64, 72, 128, 136, 256]), r.choice([8, 32, 40, 64, 96, 128, 200, 256])
    _run(r.choice(ALL), lens, hq, hk, dk, dv, packed=packed, decay=r.choice(["slopes", "slow", "none", "mixed"]), carry=r.random() < 0.5,
         want=r.random() < 0.5, grad=r.random() < 0.7, seed=seed, front=r.choice([0, 0, 3, 40]) if packed else 0,
         tail=r.choice([0, 0, 5, 70]) if packed else 0, scale=r.choice([None, 1.0, -0.3]), most=r.choice([None, 1, 4096]) if packed else None,
         per_batch=r.random() < 0.3)


def test_gradients_of_some_inputs_only():
    """One of q, k, v and the state asking for a gradient, a gradient of the final state alone, of broadcast heads and states: the
    bits (or, summed by torch, the sums) of the call that asks for all."""
    fa = _fa()
    q, k, v, g = _inputs("bf16", (2, 90), 4, 2, 32, 64, 9)
    dec = _decay(4, "slopes").cuda()
    data = [q.cuda(), k.cuda(), v.cuda(), _rand(g, (2, 4, 32, 64), "fp32", "any").cuda()]
    dout, dlast = _rand(g, (2, 90, 4, 64), "bf16", "any").cuda(), _rand(g, (2, 4, 32, 64), "fp32", "any").cuda()

    def grads(which, outs):
        x = [t.clone().requires_grad_(i in which) for i, t in enumerate(data)]
        out, last = fa.linear_attn_func(*x[:3], dec, initial_state=x[3], return_final_state=True)
        given = [(out, dout), (last, dlast)]
        return torch.autograd.grad([given[i][0] for i in outs], [x[i] for i in which], [given[i][1] for i in outs], allow_unused=True)

    for outs in ((0, 1), (0,), (1,)):
        every = grads(range(4), outs)
        # (v's is formed on the way to the state's, which keeps more bits where it is asked for)
        for which in ([0], [1], [3], [2, 3], [0, 2, 3], [1, 3]):
            for i, x in zip(which, grads(which, outs)):
                assert torch.equal(x, every[i]), (outs, which, i)
    # q does not reach the final state
    assert not grads([0], (1,))[0].any()
    # one state for all sequences, one head of k repeated by an expand
    one = data[3][:1].clone().requires_grad_()
    kk = data[1][:, :, :1].clone().requires_grad_()
    out = fa.linear_attn_func(data[0], kk.expand(-1, -1, 2, -1), data[2], dec, initial_state=one.expand(2, -1, -1, -1))
    dk, ds = torch.autograd.grad(out, [kk, one], dout)
    x = [data[0], kk.detach().repeat(1, 1, 2, 1).requires_grad_(), data[2], one.detach().repeat(2, 1, 1, 1).requires_grad_()]
    dk2, ds2 = torch.autograd.grad(fa.linear_attn_func(*x[:3], dec, initial_state=x[3]), [x[1], x[3]], dout)
    # (torch sums the parts in the type: two terms, one rounding each side)
    assert torch.equal(dk, dk2.sum(2, keepdim=True)) and torch.equal(ds, ds2.sum(0, keepdim=True))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dk,dv,n", [(64, 64, 70), (128, 128, 70), (32, 256, 1500)])
def test_values_that_are_no_numbers(dtype, bad, dk, dv, n):
    """A value makes its column so from its row on; rows before it, other columns, heads and sequences keep their bits. In reverse
    too: the gradient of v where dout has one. (The column is small, so that it sets no power of two for the others.)"""
    fa = _fa()
    q, k, v, g = _inputs(dtype, (n + 50,), 2, 2, dk, dv, 1)
    dout = _rand(g, (n + 50, 2, dv), dtype, "any")
    c, row = dv - 11, n - 27
    v[..., c] *= 2.0 ** -6
    dout[..., c] *= 2.0 ** -6
    q, k, v, dout = (x.cuda() for x in (q, k, v, dout))
    dec, cu = torch.tensor([0.0, 0.01], device="cuda"), _i32([0, n, n + 50])

    def run(v, dout):
        x = v.clone().requires_grad_()
        out = fa.linear_attn_varlen_func(q, k, x, cu, n, dec)
        return out.detach(), torch.autograd.grad(out, x, dout)[0]

    want, wgrad = run(v, dout)
    v2, d2 = v.clone(), dout.clone()
    v2[row, 1, c] = d2[row, 1, c] = bad
    out, grad = run(v2, d2)
    hit = torch.zeros(n + 50, 2, dv, dtype=torch.bool, device="cuda")
    hit[row:n, 1, c] = True
    assert not torch.isfinite(out[hit]).any() and torch.equal(out[~hit], want[~hit])
    hit = torch.zeros_like(hit)
    hit[:row + 1, 1, c] = True
    assert not torch.isfinite(grad[hit]).any() and torch.equal(grad[~hit], wgrad[~hit])
