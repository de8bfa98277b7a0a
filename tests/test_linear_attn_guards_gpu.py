"""What the C entry points of linear attention and the rotation write and read, between guard bands: outputs, states and workspaces lie in larger buffers of a
pattern that has to stay, inputs between bands that are no numbers. Lengths in order, and out of order or past the rows, which the kernels
keep within the rows that there are; one segment a sequence, and several."""
import pytest
import torch

from tests.linear_ref import DT

pytestmark = pytest.mark.gpu
BAND = 1 << 18


class _Banded:
    """A tensor of `shape` inside a buffer of bytes 0xA5 (or 0xFF: no number in any of the types)."""

    def __init__(self, shape, dtype, data=None):
        count = 1
        for n in shape:
            count *= n
        size = count * torch.empty((), dtype=dtype).element_size()
        self.fill = 0xA5 if data is None else 0xFF
        self.bytes = torch.full((BAND + size + BAND,), self.fill, dtype=torch.uint8, device="cuda")
        self.size = size
        self.t = self.bytes[BAND:BAND + size].view(dtype).view(shape)
        if data is not None:
            self.t.copy_(data)

    def whole(self):
        return bool((self.bytes[:BAND] == self.fill).all()) and bool((self.bytes[BAND + self.size:] == self.fill).all())


def _call(dtype, rows, batch, cu, most, hq, hk, dk, dv, seed):
    from fable_attn import _C, _lib
    L = _lib.load()
    g = torch.Generator().manual_seed(seed)
    packed = cu is not None
    shape = (rows,) if packed else (batch, rows)
    t = DT[dtype]
    x = lambda h, d: _Banded((*shape, h, d), t, torch.randn(*shape, h, d, generator=g).to(t))
    y = lambda h, d: _Banded((*shape, h, d), t)
    q, k, v, dout = x(hq, dk), x(hk, dk), x(hk, dv), x(hq, dv)
    o, dq, dk_, dv_ = y(hq, dv), y(hq, dk), y(hk, dk), y(hk, dv)
    states = (batch, hq, dk, dv)
    first = _Banded(states, torch.float32, torch.randn(states, generator=g))
    dlast = _Banded(states, torch.float32, torch.randn(states, generator=g))
    last, dfirst, pool = (_Banded(states, torch.float32) for _ in range(3))
    decay = _Banded((hq,), torch.float32, torch.linspace(0.0, 0.1, hq))
    index = _Banded((batch + 1,), torch.int32, torch.tensor(cu, dtype=torch.int32)) if packed else None
    kept = [q, k, v, dout, o, dq, dk_, dv_, first, dlast, last, dfirst, pool, decay] + ([index] if packed else [])

    p = _C._linear_params(q.t, k.t, v.t, decay.t, 0.125, index.t if packed else None, most, first.t)
    strides = lambda b: _C._rows_strides(b.t, packed)
    p.o, p.so = o.t.data_ptr(), strides(o)
    p.dout, p.sdo, p.dq, p.sdq = dout.t.data_ptr(), strides(dout), dq.t.data_ptr(), strides(dq)
    p.dk, p.sdk, p.dv, p.sdv = dk_.t.data_ptr(), strides(dk_), dv_.t.data_ptr(), strides(dv_)
    p.state_out = last.t.data_ptr()
    code, stream = _C._dt(q.t), torch.cuda.current_stream().cuda_stream
    need = L.fable_linear_attn_ws_bytes(p, code, 0)
    ws = _Banded((need,), torch.uint8)
    _lib.check(L.fable_linear_attn_fwd(p, code, ws.t.data_ptr() if need else None, need, stream), "fwd")
    p.dstate_out, p.dstate_in = dlast.t.data_ptr(), dfirst.t.data_ptr()
    spaces = [ws]
    for given in ([True, False] if need else [False]):
        p.seg_states = ws.t.data_ptr() if given else None
        more = L.fable_linear_attn_ws_bytes(p, code, 1)
        spaces.append(_Banded((more,), torch.uint8))
        _lib.check(L.fable_linear_attn_bwd(p, code, spaces[-1].t.data_ptr() if more else None, more, stream), "bwd")
    pool.t.copy_(first.t)
    p.state_in = p.state_out = pool.t.data_ptr()
    _lib.check(L.fable_linear_attn_step(p, code, stream), "step")
    torch.cuda.synchronize()
    for i, b in enumerate(kept + spaces):
        assert b.whole(), i
    for b in (o, dq, dk_, dv_):
        assert torch.isfinite(b.t).all()
    return need


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hq,hk,dk,dv", [(2, 1, 64, 64), (2, 2, 72, 40), (1, 1, 128, 200)])
def test_rows_in_order(dtype, hq, hk, dk, dv):
    """Dense and packed, rows in front and behind, one segment and several."""
    print(f"[guards] {dtype} {hq}/{hk} {dk}x{dv}", flush=True)
    assert not _call(dtype, 45, 2, None, 0, hq, hk, dk, dv, 1)
    assert _call(dtype, 1500, 2, None, 0, hq, hk, dk, dv, 2)
    assert not _call(dtype, 50, 3, [3, 3, 40, 45], 37, hq, hk, dk, dv, 3)
    assert _call(dtype, 2000, 4, [5, 6, 1000, 1000, 1990], 994, hq, hk, dk, dv, 4)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hq,hk,dk,dv", [(2, 1, 64, 64), (2, 2, 72, 40)])
def test_lengths_out_of_order(dtype, hq, hk, dk, dv):
    """Past the rows, below 0, not in order, under a max_seqlen that is too small, right, or too large."""
    for rows, lists in ((40, [[0, 100], [-5, 10, 40], [20, 10, 40], [0, 40, 20, 90], [50, 60, 70]]),
                        (1500, [[0, 4000], [-500, 700, 1500], [900, 300, 1500], [0, 1500, 700, 2000], [1400, 0, 1500, 2, 1500], [1600, 1700, 1800]])):
        for cu in lists:
            for most in (4, rows, 10 * rows):
                print(f"[guards] {dtype} {hq}/{hk} {dk}x{dv} rows={rows} cu={cu} most={most}", flush=True)
                _call(dtype, rows, len(cu) - 1, cu, most, hq, hk, dk, dv, rows + most)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,rd", [(64, 64), (72, 20)])
@pytest.mark.parametrize("cu", [[0, 10, 40], [3, 3, 37], [0, 100, 200], [-5, 10, 40], [20, 10, 40], [50, 60, 70]])
def test_rotation(dtype, d, rd, cu):
    """Lengths as above, positions in front of the tables and behind them, by 16-byte units and one value at a time."""
    from fable_attn import _C, _lib
    print(f"[guards] rotation {dtype} {d} {rd} {cu}", flush=True)
    g, t = torch.Generator().manual_seed(1), DT[dtype]
    q, k = (_Banded((40, h, d), t, torch.randn(40, h, d, generator=g).to(t)) for h in (4, 2))
    qo, ko = (_Banded((40, h, d), t) for h in (4, 2))
    cos, sin = (_Banded((9, rd // 2), torch.float32, torch.randn(9, rd // 2, generator=g)) for _ in range(2))
    index = _Banded((len(cu),), torch.int32, torch.tensor(cu, dtype=torch.int32))
    start = _Banded((len(cu) - 1,), torch.int32, torch.tensor([-7, 2 ** 31 - 1], dtype=torch.int32))
    s = lambda b: _C._rows_strides(b.t, True)
    for rotary in (1, 2):
        p = _lib.FableRotaryParams()
        p.q, p.k, p.q_out, p.k_out = q.t.data_ptr(), k.t.data_ptr(), qo.t.data_ptr(), ko.t.data_ptr()
        p.sq, p.sk, p.sqo, p.sko = s(q), s(k), s(qo), s(ko)
        p.cos, p.sin, p.cu, p.start = cos.t.data_ptr(), sin.t.data_ptr(), index.t.data_ptr(), start.t.data_ptr()
        p.total, p.batch, p.NH, p.NKV, p.HD, p.rotary, p.rotary_dim, p.rotary_rows = 40, len(cu) - 1, 4, 2, d, rotary, rd, 9
        _lib.check(_lib.load().fable_attn_rotary(p, _C._dt(q.t), torch.cuda.current_stream().cuda_stream), "rotary")
        torch.cuda.synchronize()
        for i, b in enumerate((q, k, qo, ko, cos, sin, index, start)):
            assert b.whole(), i
        assert torch.isfinite(qo.t).all() and torch.isfinite(ko.t).all()
