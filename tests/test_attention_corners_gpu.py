"""Attention where its results are decided by something else than a sum: no keys, numbers that are not finite in one of several
shares of the keys, weights far below the largest, no room for shares while a stream is being captured."""
import math

import pytest
import torch

from tests.test_attention_gpu import TYPES, attend, bounds, check_paged, check_prompt, close, i32, paged_case, randn

pytestmark = pytest.mark.gpu


# ---- no keys, no pages -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,D", [((8, 2), 128), ((24, 1), 64)])
def test_paged_tables_of_no_width(hq, heads, D):
    """Lengths end with the table: nothing is seen, with and without groups, and the results are zeros."""
    q = randn(1, 5, heads[0], D).bfloat16()
    pages = randn(2, 3, heads[1], 16, D).bfloat16()
    table, lengths = torch.zeros((5, 0), dtype=torch.int32, device="cuda"), i32([7, 100, 0, 1, 2 ** 31 - 1])
    for groups in ((), (i32([0, 5]), i32([64])), (i32([0, 2, 4]), i32([0, 16]))):
        out = torch.full_like(q, 7.0)
        hq.paged_attention(q, pages, pages, table, lengths, *groups, out=out)
        assert (out == 0).all()


def test_keys_of_minus_infinity_in_one_share_and_in_all(hq):
    """Keys whose score is -inf have no weight, also where a share holds nothing else; where all have it the softmax is NaN."""
    dtype, u = TYPES["bf16"]
    D = 64
    q, k, v = torch.ones((4, 4, D), device="cuda").to(dtype), randn(2, 2500, 2, D).to(dtype), randn(3, 2500, 2, D).to(dtype)
    k[1500:2400, 1] = -math.inf
    out = hq.prompt_attention(q, k, v, i32([0, 4]), i32([0, 2500]), causal=False)
    keep = torch.cat([torch.arange(1500), torch.arange(2400, 2500)]).cuda()
    for h in (2, 3):
        want, a, big = attend(q[:, h].double(), k[keep, 1].double(), v[keep, 1].double(), torch.ones((4, 1600), dtype=torch.bool, device="cuda"), 0.125)
        close(out[:, h], want, a, big, u)
    k[:, 0] = -math.inf
    out = hq.prompt_attention(q, k, v, i32([0, 4]), i32([0, 2500]), causal=False)
    assert torch.isnan(out[:, :2]).all() and torch.isfinite(out[:, 2:]).all()
    for n, heads in ((129, (4, 2)), (700, (4, 2)), (9000, (4, 2)), (700, (40, 2))):
        q, k, v, table, lengths = paged_case(3, dtype, [n, n], heads, D, 16)
        q[:] = 1
        for t in range(n):
            k[table[0][t // 16], 1, t % 16] = -math.inf
        out = hq.paged_attention(q, k, v, i32(table), i32(lengths))
        r = heads[0] // 2
        assert torch.isnan(out[0, r:]).all() and torch.isfinite(out[0, :r]).all() and torch.isfinite(out[1]).all()
