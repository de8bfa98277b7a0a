"""The launch parameters that flash_attn_with_kvcache keeps of a signature (flash_attn_interface._decode_plan), on the
CPU: tensors without memory stand for a call's, and the plan's workspace has to be the one that the library asks for
when it is given the call itself, its optional tensors included."""
import itertools

import pytest
import torch

from fable_attn import _lib
from fable_attn import flash_attn_interface as fai


class OnGpu(torch.Tensor):
    """A tensor of cuda:0 without memory: what host code may ask of one."""

    @staticmethod
    def __new__(cls, shape, dtype):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} needs memory")

    def data_ptr(self):
        return 256


BF, I32, F32 = torch.bfloat16, torch.int32, torch.float32


def _call(q8, batch, hk, gqa, nq, d, page, blocks, leftpad, alibi, append=True, rotary=False, dense=False):
    """(arguments of _decode_plan but the options, the library's answer for that call)"""
    hq, nb = hk * gqa, batch * blocks
    cache = (nb, page, hk, d)
    kc, vc = (OnGpu(cache, torch.float8_e4m3fn if q8 else BF) for _ in range(2))
    ks, vs = (OnGpu((nb, hk, 1), torch.float8_e8m0fnu) if q8 else None for _ in range(2))
    q = OnGpu((batch, nq, hq, d), BF)
    k, v = (OnGpu((batch, nq, hk, d), BF) if append else None for _ in range(2))
    cos, sin = (OnGpu((64, d // 2), F32) if rotary else None for _ in range(2))
    args = (q, kc, vc, k, v, cos, sin, OnGpu((batch,), I32), OnGpu((batch,), I32) if leftpad else None,
            None if dense else OnGpu((batch, blocks), I32), OnGpu((hq,), F32) if alibi else None, ks, vs)
    p = _lib.FableDecParams()
    p.q = p.Kc = p.Vc = p.o = p.ctx_len = 256
    p.block_table = None if dense else 256
    p.leftpad, p.alibi = 256 if leftpad else None, 256 if alibi else None
    if rotary:
        p.cos = p.sin = 256
        p.rotary, p.rotary_dim = 2, d
    p.batch, p.NH, p.gqa, p.HD, p.page, p.max_blocks = batch, hq, gqa, d, page, blocks
    p.window, p.scale, p.nq = -1, d ** -0.5, nq
    lib = _lib.load()
    if q8:
        c = _lib.FableCache8(256, 256, _lib.Strides(page * hk * d, d, hk * d), page, nb, 64 if rotary else 0)
        return args, lib.fable_attn_dec8_ws_bytes(p, c, 1, int(append))
    return args, lib.fable_attn_dec_ws_bytes(p, 1, int(append))


@pytest.mark.parametrize("q8", [True, False], ids=["8 bits", "16 bits"])
def test_the_plan_holds_the_workspace_of_its_call(q8):
    """Masks by a left pad or slopes take another workgroup shape on the tile kernel, and with it another split: rows of
    a K/V head on both sides of the tile path (64) and of its tile heights, short and long tables."""
    seen = set()
    for leftpad, alibi, nq, batch, blocks, d in itertools.product(
            (False, True), (False, True), (1, 7, 8, 16, 32, 33, 40, 48, 64), (1, 3, 9), (4, 256, 2048), (64, 128, 256)):
        args, want = _call(q8, batch, 8, 8, nq, d, 16, blocks, leftpad, alibi)
        plan = fai._decode_plan(*args, None, (-1, -1), 0.0, True, 0)
        assert plan is not None and want >= 0
        assert plan[2] == want, (leftpad, alibi, nq, batch, blocks, d)
        seen.add((leftpad or alibi, nq, batch, blocks, d, want))
    plain, masked = ({s[1:] for s in seen if s[0] == m} for m in (False, True))
    assert plain != masked   # (the sizes do depend on it)


@pytest.mark.parametrize("q8", [True, False], ids=["8 bits", "16 bits"])
@pytest.mark.parametrize("kw", [{"rotary": True}, {"append": False}, {"dense": True, "blocks": 1, "page": 4096}], ids=str)
def test_the_plan_holds_no_address(q8, kw):
    a = dict(batch=9, hk=8, gqa=8, nq=40, d=128, page=16, blocks=256, leftpad=True, alibi=True)
    a.update(kw)
    if a["page"] > 256 and q8:
        a["page"] = 256
    args, want = _call(q8, **a)
    p, _, need, c = fai._decode_plan(*args, None, (-1, -1), 0.0, True, 0)
    assert need == want
    for name, kind in p._fields_:
        if kind is _lib.c_ptr:
            assert getattr(p, name) is None, name
    if c is not None:
        assert c.k_scale is None and c.v_scale is None and c.held is None


def test_prompts_are_gathered_within_bounds():
    """The route of packed prompts over an 8-bit cache: wide heads, enough pairs, no window, and a temporary copy that is
    small next to a cache, whatever the caller takes for the longest length."""
    pays = fai._gather8_pays
    many = dict(batch=4, heads=16, heads_k=4, max_sq=1000, max_sk=4000, rows=4000, wl=-1, d=256)
    assert pays(**many)
    for kw in ({"d": 128}, {"wl": 512}, {"max_sq": 100}, {"max_sk": 10}, {"rows": 0}, {"rows": 1 << 18}, {"batch": 1 << 12}):
        assert not pays(**dict(many, **kw)), kw
    assert pays(**dict(many, max_sk=1 << 20)) and not pays(**dict(many, max_sk=1 << 20, rows=16))


@pytest.mark.parametrize("batch,nq,heads,gqa,window", [
    (128, 1 << 24, 1, 1, 0), (65535, 32769, 1, 1, 0), (1, 1 << 24, 128, 1, -1), (1, 1 << 22, 512, 4, 64)])
def test_decode_refuses_more_rows_than_32_bits_count(batch, nq, heads, gqa, window):
    """Tokens of a call, and heads of a sequence's tokens: past 2^31 the kernels' row numbers would wrap around."""
    lib = _lib.load()
    p = _lib.FableDecParams()
    p.q = p.Kc = p.Vc = p.o = p.ctx_len = p.block_table = 16    # never dereferenced
    p.batch, p.NH, p.gqa, p.HD, p.page, p.max_blocks, p.nq, p.window, p.scale = batch, heads, gqa, 16, 16, 4, nq, window, 0.25
    c = _lib.FableCache8(16, 16, _lib.Strides(16 * 16 * heads, 16, 16 * heads), 16, 4, 0)
    assert lib.fable_attn_dec8_ws_bytes(p, c, 1, 0) == -1 and b"nq" in lib.fable_attn_last_error()
    assert lib.fable_attn_dec8(p, c, 1, None, 0, None, None, None) == 3
    p.nq = 1
    assert lib.fable_attn_dec8_ws_bytes(p, c, 1, 0) >= 0
