"""Calls over K/V caches that come again: the second call of a signature runs from the launch parameters that the first
one left, and gives bitwise what the first gave. Caches in 8 and in 16 bits."""
import pytest
import torch

from tests import cache8_ref as ref
from tests.test_cache8_gpu import _fa, _filled, _i32, _rand

pytestmark = pytest.mark.gpu


def _steps(q8, lens, hq, hk, d, page, nq, wide, append, **kw):
    """The same decode call three times, on equal caches: with an LSE (never planned), the first without, the second."""
    dt, B = torch.bfloat16, len(lens)
    pool = _filled(lens, -(-(max(lens) + nq) // page), page, hk, d, 16, dt, 5, leftpad=kw.get("cache_leftpad"))
    table = pool.table.cuda()
    table = torch.cat((table, table[:, :1].expand(B, wide - table.shape[1])), 1).contiguous()
    q = _rand((B, nq, hq, d), dt, 1).cuda()
    new = {"k": _rand((B, nq, hk, d), dt, 2).cuda(), "v": _rand((B, nq, hk, d), dt, 3).cuda()} if append else {}
    opts = dict(kw)
    if "cache_leftpad" in kw:
        opts["cache_leftpad"] = _i32(kw["cache_leftpad"])
    if kw.get("alibi_slopes"):
        opts["alibi_slopes"] = torch.tensor([2.0 ** -(1 + h % 8) for h in range(hq)]).cuda()
    if kw.get("rotary_cos"):
        cos, sin = ref.tables(max(lens) + nq + 1, d // 2)
        opts.update(rotary_cos=cos.cuda(), rotary_sin=sin.cuda())
    outs, caches = [], []
    for lse in (True, False, False):
        if q8:
            kc, vc, ks, vs, _ = pool.cuda()
            scales = dict(k_scale=ks, v_scale=vs)
        else:
            kc, vc = (_rand((pool.codes[0].shape[0], page, hk, d), dt, 9 + i).cuda() for i in range(2))
            scales = {}
        res = _fa().flash_attn_with_kvcache(q, kc, vc, cache_seqlens=_i32(lens), block_table=table, causal=True,
                                            return_softmax_lse=lse, **new, **opts, **scales)
        outs.append(res[0] if lse else res)
        caches.append([x.view(torch.uint8) for x in (kc, vc, *scales.values())])
    for out, cache in zip(outs[1:], caches[1:]):
        assert torch.equal(out, outs[0])
        for a, b in zip(cache, caches[0]):
            assert torch.equal(a, b)
    assert torch.isfinite(outs[0]).all()


OPTIONS = [{}, {"alibi_slopes": True}, {"cache_leftpad": [3, 40]}, {"cache_leftpad": [0, 33], "alibi_slopes": True},
           {"window_size": (50, 0)}, {"softcap": 20.0}, {"rotary_cos": True}, {"rotary_cos": True, "cache_leftpad": [1, 2]}]


@pytest.mark.parametrize("q8", [True, False], ids=["8 bits", "16 bits"])
@pytest.mark.parametrize("append", [True, False], ids=["append", "read"])
@pytest.mark.parametrize("kw", OPTIONS, ids=str)
@pytest.mark.parametrize("nq,wide", [(1, 20), (3, 256), (33, 20), (33, 256), (64, 256)])
def test_the_second_call_is_the_first(nq, wide, kw, append, q8):
    """Few new tokens (the decode kernels) and many (the tile kernel, whose workgroup shape, split and workspace follow
    from the masks), under short tables and long ones."""
    _steps(q8, [150, 200], 32, 8, 128, 16, nq, wide, append, **kw)


@pytest.mark.parametrize("kw", OPTIONS[1:4], ids=str)
@pytest.mark.parametrize("d", [64, 256])
def test_the_second_call_at_other_widths(d, kw):
    _steps(True, [150, 200], 32, 8, d, 16, 40, 512, True, **kw)
