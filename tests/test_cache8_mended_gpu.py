"""Edges of the caches in 8 bits: a block under the largest scale, prompts whose max_seqlen_k says less than their lengths,
and gathers that find no memory."""
import pytest
import torch

from tests import cache8_ref as ref
from tests.test_cache8_gpu import _cu, _fa, _filled, _i32, _rand, _same_pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("byte", [254, 253, 1])
@pytest.mark.parametrize("d,group", [(128, 16), (64, 4), (256, 64)])
def test_a_block_filled_elsewhere_keeps_its_scale(d, group, byte):
    """Scale bytes at the ends of e8m0's range, which no append chooses: held rows keep their values (or, under a scale
    that grows, their share of them), and new ones go under the scale that the block has."""
    dt, hk, page, held = torch.bfloat16, 2, 64, [3, group + 1, 2 * group - 1]
    pool = _filled(held, 3, page, hk, d, group, dt, 11)
    for s in pool.scales:
        s[s != 255] = byte
    c = pool.cuda()
    # (under 2^127 a code stands for 2^118 at least: tokens of that size and far below)
    k, v = (_rand((3, 2, hk, d), dt, 12 + i, 2.0 ** 120 if byte > 100 else 2.0 ** -128) for i in range(2))
    _fa().flash_attn_append_kvcache(k.cuda(), v.cuda(), c[0], c[1], _i32(held), block_table=c[4], k_scale=c[2], v_scale=c[3])
    for b, n in enumerate(held):
        pool.append(b, n, k[b].double(), v[b].double())
    _same_pool(pool, c, exact=True)


def _prompts(max_sk, d=256, page=16):
    """Two causal prompts behind cached keys: (the result with this max_seqlen_k, with 0: none known)."""
    dt, hq, hk, new, cached = torch.bfloat16, 4, 2, [40, 33], [60, 90]
    total = [a + b for a, b in zip(new, cached)]
    pool = _filled(total, 8, page, hk, d, 16, dt, 13)
    c = pool.cuda()
    q = _rand((sum(new), hq, d), dt, 14).cuda()
    call = lambda m: _fa().flash_attn_varlen_func(q, c[0], c[1], _cu(new), _cu(total), max(new), m, causal=True, block_table=c[4],
                                                  k_scale=c[2], v_scale=c[3])
    return call(max_sk), call(0)


def _close(a, b):
    assert ((a.float() - b.float()).abs() <= 4 * 2.0 ** -8 * 20.0).all() and not torch.equal(b, torch.zeros_like(b))
    assert (a.float() - b.float()).abs().mean() <= 2.0 ** -8


@pytest.mark.parametrize("max_sk", [123, 70, 17, 1, 100000])
def test_the_longest_length_of_a_prompt_call_moves_no_key(max_sk, monkeypatch):
    """max_seqlen_k chooses between reading in place and gathering first, and nothing else."""
    from fable_attn import flash_attn_interface as fai
    monkeypatch.setattr(fai, "_GATHER8_PAIRS", 0)
    calls = []
    gather = fai._C.gather
    monkeypatch.setattr(fai._C, "gather", lambda *a: calls.append(1) or gather(*a))
    got, want = _prompts(max_sk)
    assert len(calls) == 1
    _close(got, want)


def test_prompts_that_find_no_memory_to_gather_in(monkeypatch):
    from fable_attn import flash_attn_interface as fai
    monkeypatch.setattr(fai, "_GATHER8_PAIRS", 0)

    def full(*a):
        raise torch.cuda.OutOfMemoryError("no memory")

    monkeypatch.setattr(fai._C, "gather", full)
    got, want = _prompts(123)
    assert torch.equal(got, want)   # read in place, both
