"""Rings seeded from packed prompts (prompt_importance, last_attn_weights.seed) against the ones that the probabilities themselves fill."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128
LENGTHS = [7, 300, 1, 20, 19, 21]


@pytest.fixture(scope="module")
def packed(cuda_device):
    from hqekv_b200.prompt import prompt_attention, prompt_importance
    gen = torch.Generator(device="cuda").manual_seed(1)
    T, nh, nkv = sum(LENGTHS), 8, 2
    q, k, v = (torch.randn(T, h, D, generator=gen, device="cuda").half() for h in (nh, nkv, nkv))
    at = [sum(LENGTHS[:i]) for i in range(len(LENGTHS) + 1)]
    starts = torch.tensor(at, dtype=torch.int32, device="cuda")
    _, lse = prompt_attention(q, k, v, starts)
    return q, k, at, prompt_importance(q, k, lse, starts, rows=20)


@pytest.mark.parametrize("i", range(len(LENGTHS)))
def test_seed_from_a_slice(packed, i):
    """As update does with the probabilities of the same prompt, and a decode step after it.  u = 2^-11: the probabilities are rounded one by
    one and their sum twice (3 u, 2^-25 for each of 8 heads that is subnormal), the rows once (u, 2^-25); fp32 arithmetic in a logit,
    2^-16 of the largest sum of its terms, in an exponential as much of its value."""
    from hqekv_b200.model.public_func import last_attn_weights
    q, k, at, rows = packed
    a, b, n = at[i], at[i + 1], LENGTHS[i]
    nh, rep = q.shape[1], q.shape[1] // k.shape[1]
    keys = k[a:b].double().repeat_interleave(rep, 1)
    s = torch.einsum("nhd,mhd->hnm", q[a:b].double(), keys) * D ** -0.5
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -torch.inf)
    top = float(torch.einsum("nhd,mhd->hnm", q[a:b].double().abs(), keys.abs()).max()) * D ** -0.5
    want, got = last_attn_weights(last_length=20), last_attn_weights(last_length=20)
    for ring in (want, got):
        ring.set_max_length(400)
    want.update(torch.softmax(s, -1).half()[None])
    got.seed(rows[:min(20, n), a:b])
    assert (got.next_line, got.kv_seq_len) == (want.next_line, want.kv_seq_len) == (min(20, n) % 20, n)
    err = (got.weights.double() - want.weights.double()).abs()
    assert bool((err <= (4.1 * 2.0 ** -11 + 2.0 ** -16 * top) * want.weights.double() + 9 * 2.0 ** -25).all())
    step = torch.rand(1, nh, 1, n + 1, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").half()
    for ring in (want, got):
        ring.update(step)
    assert (got.next_line, got.kv_seq_len) == (want.next_line, want.kv_seq_len)
    line = min(20, n) % 20
    assert torch.equal(got.weights[line], want.weights[line])
