"""A ragged append: flash_attn_with_kvcache refuses it and names the two calls that serve it, which agree with it where
both apply."""
import pytest
import torch

from tests import cache8_ref as ref


def test_the_refusals_name_the_way():
    import fable_attn as fa
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    kc = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    kv = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    cu, one = torch.tensor([0, 1], dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="cu_seqlens_k_new.*flash_attn_append_kvcache.*flash_attn_varlen_func"):
        fa.flash_attn_with_kvcache(q, kc, kc, k=kv, v=kv, cache_seqlens=one, cu_seqlens_k_new=cu)
    with pytest.raises(NotImplementedError, match="cu_seqlens_q.*flash_attn_append_kvcache.*flash_attn_varlen_func"):
        fa.flash_attn_with_kvcache(q[0], kc, kc, k=kv, v=kv, cache_seqlens=one, cu_seqlens_q=cu)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [True, False], ids=["8 bits", "16 bits"])
@pytest.mark.parametrize("nq", [1, 5, 40])
def test_the_two_calls_give_what_the_one_gives(nq, q8):
    from tests.test_cache8_gpu import _cu, _fa, _filled, _i32, _rand
    fa, dt, lens, hq, hk, d, page = _fa(), torch.bfloat16, [0, 17, 90], 8, 2, 128, 16
    pool = _filled(lens, 9, page, hk, d, 16, dt, 21)
    q, k, v = (_rand((3, nq, h, d), dt, 22 + i).cuda() for i, h in enumerate((hq, hk, hk)))
    cos, sin = (t.cuda() for t in ref.tables(200, d // 2))
    rot = dict(rotary_cos=cos, rotary_sin=sin, rotary_interleaved=False)

    def cache():
        kc, vc, ks, vs, table = pool.cuda()
        if q8:
            return kc, vc, table, dict(k_scale=ks, v_scale=vs)
        return (*(_rand(kc.shape, dt, 25 + i).cuda() for i in range(2)), table, {})

    kc, vc, table, scales = cache()
    want = fa.flash_attn_with_kvcache(q, kc, vc, k=k, v=v, cache_seqlens=_i32(lens), block_table=table, causal=True, **rot, **scales)
    kc2, vc2, table, scales2 = cache()
    flat = lambda x: x.reshape(3 * nq, *x.shape[2:])
    rq = fa.flash_attn_append_kvcache(flat(k), flat(v), kc2, vc2, _i32(lens), q=flat(q), cu_seqlens=_cu([nq] * 3), max_seqlen=nq,
                                      block_table=table, **rot, **scales2)
    got = fa.flash_attn_varlen_func(rq, kc2, vc2, _cu([nq] * 3), _cu([n + nq for n in lens]), nq, max(lens) + nq, causal=True,
                                    block_table=table, **scales2)
    for a, b in ((kc, kc2), (vc, vc2)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # (q is rounded to bf16 between the two calls: half a step of every product of a score, |s| <= 40 here, beside the
    # roundings of P and of the result on both sides)
    err = (got.view_as(want).float() - want.float()).abs()
    assert err.max() <= (2 * 40 * 2.0 ** -8 + 4 * 2.0 ** -8) * 8.0 and err.mean() <= 2.0 ** -7
