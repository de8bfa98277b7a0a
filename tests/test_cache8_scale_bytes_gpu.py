"""Caches in 8 bits that another program filled: blocks under scale bytes that no append chooses."""
import pytest
import torch

from tests.test_cache8_gpu import _fa, _filled, _i32, _rand, _same_pool

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
