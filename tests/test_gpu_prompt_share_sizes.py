"""Shares of keys whose size the kernel chooses from the lengths: odd sizes, and blocks of one row tile alone, which get half as much again."""
import pytest
import torch

from test_gpu_prompt import D, check, ops, randn  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n, own, step, heads, before", [
    (8, 7384, 129, (8, 2), 0),       # shares of 5 tiles, 7 for these blocks: an item for every CTA
    (8, 10779, 129, (16, 2), 0),     # 7 and 10
    (25, 3116, 37, (8, 2), 0),       # 9 and 13
    (25, 1000, 37, (8, 2), 2116),    # ... part of them a prefix
    (12, 4000, 300, (4, 1), 129),
])
@pytest.mark.parametrize("rows", [14, 32])
def test_odd_share_sizes(ops, n, own, step, heads, before, rows):  # noqa: F811
    q_len = [1 + (7 * i) % rows for i in range(n)]
    k_len = [m + own + step * i for i, m in enumerate(q_len)]
    nh, nkv = heads
    q, k, v = randn(1, sum(q_len), nh, D), randn(2, sum(k_len), nkv, D), randn(3, sum(k_len), nkv, D)
    prefix = (randn(4, before, nkv, D), randn(5, before, nkv, D)) if before else None
    first = check(ops, q, k, v, q_len, k_len, prefix)
    again = check(ops, q, k, v, q_len, k_len, prefix)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
