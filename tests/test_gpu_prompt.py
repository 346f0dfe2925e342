"""GPU tests of the prompt operators (hqekv_b200/prompt.py) and of the decode behind a shared prefix against their formulas in 64 bits.

Tolerances, per element, with u = half a step of the type (2^-11 for fp16, 2^-8 for bf16):
* A logit is a sum of 128 products that are exact in fp32.  Every addition of it is off by at most 2^-23 (a unit of the last place: a matrix
  instruction may cut off instead of rounding) of a partial sum, which is at most t = scale sum |q_i k_i|: 2^-16 t in all.  As much
  relative to its value is an exponential off, and 2^-20 more for its own argument, value and sum.
* output: u sum_j p_j |v_j| for the probabilities rounded before the product with V, u |o| for the output's own rounding, and
  (2^-16 t + 2^-20) sum_j p_j |v_j| for fp32 arithmetic.  Probabilities below 2^-14 of the largest are subnormal halfs, off by up to 2^-25 of it:
  2^-25 p_max sum_j |v_j|.  An fp16 output below 2^-14 is off by 2^-25.
* lse: 2^-16 t + 2^-22 (1 + |lse|).
* rows of the importance: u of the value, 2^-16 t + 2^-20 of it for the exponentials, 2^-25.
"""
import math

import numpy as np
import pytest
import torch

from oracle import hqkv_oracle as O

pytestmark = pytest.mark.gpu

D = 128
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
NORMAL = "high_uniform_group_low_normal_group"


@pytest.fixture(scope="module")
def ops(cuda_device):
    import types
    from hqekv_b200 import prompt
    from hqekv_b200.quant import hqe_matmul
    return types.SimpleNamespace(attention=prompt.prompt_attention, importance=prompt.prompt_importance, decode=hqe_matmul.qkv_matmul_hqe_2,
                                 prefix=hqe_matmul.qkv_matmul_hqe_prefix)


def randn(seed, *shape, dtype=torch.float16, gain=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * gain).to(dtype)


def starts(lengths, first=0):
    return torch.tensor(np.cumsum([first] + list(lengths)), dtype=torch.int32, device="cuda")


def terms(q, k, scale):
    """The largest sum of a logit's terms without their signs."""
    return float(torch.einsum("nhd,mhd->hnm", q.abs(), k.abs()).amax()) * scale if k.numel() and q.numel() else 0.0


def reference(q, k, v, prefix, causal, scale):
    """One sequence in 64 bits: (out, lse, bound of the output's error, largest |s|)."""
    n, nh = q.shape[0], q.shape[1]
    own = k.shape[0]
    if prefix is not None:
        k, v = torch.cat((prefix[0], k)), torch.cat((prefix[1], v))
    rep, u = nh // k.shape[1], HALF[q.dtype]
    q, k, v = q.double(), k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    s = torch.einsum("nhd,mhd->hnm", q, k) * scale
    if causal:
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(k.shape[0], device="cuda") - (k.shape[0] - own)
        s = s.masked_fill((j >= 0) & (j > i + own - n), -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[..., None])
    out = torch.einsum("hnm,mhd->nhd", p, v)
    top = terms(q, k, scale)
    a = torch.einsum("hnm,mhd->nhd", p, v.abs())
    peak = p.amax(-1).T[..., None] if p.shape[-1] else torch.zeros(n, nh, 1, device="cuda", dtype=torch.float64)
    bound = u * (a + out.abs()) + (2.0 ** -16 * top + 2.0 ** -20) * a + 2.0 ** -25 * (1 + peak * v.abs().sum(0)) * (1 + 2.0 ** -8)
    return out, lse, bound, top


def check(ops, q, k, v, q_len, k_len, prefix=None, causal=True, scale=None, call=None):
    out, lse = (call or ops.attention)(q, k, v, starts(q_len), starts(k_len), prefix=prefix, causal=causal, scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (q.shape[1], q.shape[0]) and lse.dtype == torch.float32
    a = b = 0
    for n, m in zip(q_len, k_len):
        if n:
            o, l, bound, top = reference(q[a:a + n], k[b:b + m], v[b:b + m], prefix, causal, D ** -0.5 if scale is None else scale)
            over = (out[a:a + n].double() - o).abs() / bound
            assert float(over.max()) <= 1, f"output off by {float(over.max()):.3g} of what it may be (lengths {n}, {m})"
            got, none = lse[:, a:a + n].double(), l.isinf()
            assert torch.equal(got.isinf(), none) and bool((got[none] < 0).all())
            assert bool(((got - l).abs() <= 2.0 ** -16 * top + 2.0 ** -22 * (1 + l.abs()))[~none].all())
            assert bool((out[a:a + n].transpose(0, 1)[none] == 0).all())
        a, b = a + n, b + m
    return out, lse


LENGTHS = {
    "one": ([1], [1]),
    "few": ([17], [17]),
    "tile": ([128], [128]),
    "tile+1": ([129], [129]),
    "ragged": ([63, 1, 0, 257, 64, 2, 300], [63, 1, 0, 257, 64, 2, 300]),
    "chunks": ([5, 70, 1, 33], [130, 70, 513, 256]),
    "rows without keys": ([40, 7, 200], [10, 0, 129]),
    "long": ([700], [1500]),
    "many": ([3] * 70, [5] * 70),
}


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("heads", [(4, 1), (8, 2), (3, 3), (6, 2), (8, 1), (32, 8)])
def test_lengths_and_heads(ops, lengths, heads):
    q_len, k_len = LENGTHS[lengths]
    nh, nkv = heads
    q, k, v = randn(1, sum(q_len), nh, D), randn(2, sum(k_len), nkv, D), randn(3, sum(k_len), nkv, D)
    check(ops, q, k, v, q_len, k_len)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("before", [1, 100, 128, 129, 1000])
def test_prefix_types_and_masks(ops, dtype, causal, before):
    q_len, k_len = [1, 65, 0, 190], [1, 65, 3, 400]
    q, k, v = (randn(i, n, h, D, dtype=dtype) for i, n, h in ((1, 256, 8), (2, 469, 2), (3, 469, 2)))
    prefix = (randn(4, before, 2, D, dtype=dtype), randn(5, before, 2, D, dtype=dtype))
    check(ops, q, k, v, q_len, k_len, prefix, causal)
    check(ops, q, k, v, q_len, k_len, None, causal)


def test_prefix_without_own_keys(ops):
    q, none = randn(1, 9, 4, D), randn(2, 0, 2, D)
    prefix = (randn(3, 333, 2, D), randn(4, 333, 2, D))
    check(ops, q, none, none, [4, 5], [0, 0], prefix)


@pytest.mark.parametrize("gain, scale", [(10.0, None), (1.0, 3.0), (1.0, 1e-6), (0.01, 0.5)])
def test_peaked_and_flat_rows(ops, gain, scale):
    """Logits up to some hundreds (rows of one key in effect) and as good as none at all."""
    q, k, v = randn(1, 300, 8, D, gain=gain), randn(2, 300, 2, D), randn(3, 300, 2, D)
    check(ops, q, k, v, [260, 40], [260, 40], scale=scale)


def test_rising_logits(ops):
    """Every tile of keys brings a larger maximum than all before it, by a lot and by a little."""
    for step in (0.02, 0.3):
        k = randn(2, 1400, 2, D, gain=0.05)
        k[:, :, 0] = (torch.arange(1400, device="cuda") * step)[:, None].half()
        q, v = randn(1, 1400, 4, D, gain=0.05), randn(3, 1400, 2, D)
        q[:, :, 0] = 1.0
        check(ops, q, k, v, [1400], [1400], scale=1.0)


@pytest.mark.parametrize("q_len, k_len, heads, before, causal", [
    ([96, 37, 73, 14], [5096, 337, 9073, 14], (32, 8), 0, True),      # shares of sizes that follow from the lengths
    ([96, 37, 0, 73, 14, 60], [5096, 0, 40, 9073, 10, 50], (32, 8), 129, True),   # ... no queries, no keys, fewer keys than queries
    ([33, 64, 65, 31, 32, 1], [6000, 128, 6001, 129, 2000, 7000], (16, 4), 0, False),
    ([243 - 20 * i for i in range(12)], [9000 - 700 * i for i in range(12)], (8, 2), 0, True),
    ([5] * 32, [3000 + 10 * i for i in range(32)], (4, 2), 100, True),
    ([5] * 33, [3000 + 10 * i for i in range(33)], (4, 2), 100, True),   # more sequences than a warp counts at a time
    ([300, 290], [12000, 100], (8, 1), 0, True),                      # blocks of 32 tokens
    ([1, 1], [9000, 20000], (4, 1), 0, True),                         # more shares than a warp joins at a time
    ([1], [20000], (4, 1), 0, True),
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_shares(ops, q_len, k_len, heads, before, causal, dtype):
    """Few rows and many keys, which are shared out over the GPU and joined."""
    nh, nkv = heads
    q, k, v = randn(1, sum(q_len), nh, D, dtype=dtype), randn(2, sum(k_len), nkv, D, dtype=dtype), randn(3, sum(k_len), nkv, D, dtype=dtype)
    prefix = (randn(4, before, nkv, D, dtype=dtype), randn(5, before, nkv, D, dtype=dtype)) if before else None
    check(ops, q, k, v, q_len, k_len, prefix, causal)


@pytest.mark.parametrize("q_len, k_len, heads, before, causal", [
    ([64] * 20, [64] * 20, (32, 8), 300, True),                       # 160 blocks and head groups: twelve more than SMs
    ([17] * 21, [17] * 21, (32, 8), 400, True),                       # ... of which the second row tiles are empty
    ([100, 1, 0, 95, 129, 64, 65, 33, 128, 40, 97, 127, 31], [400, 30, 5, 95, 700, 0, 65, 600, 128, 333, 97, 900, 131], (32, 8), 0, True),
    ([2600], [2600], (32, 8), 0, False),
    ([150 + i % 10 for i in range(32)], [400 + 3 * i for i in range(32)], (8, 1), 129, True),
    ([150 + i % 10 for i in range(33)], [400 + 3 * i for i in range(33)], (8, 1), 129, True),   # more sequences than a warp counts at a time
    ([70] * 14, [70] * 14, (24, 24), 1000, False),                    # no groups of heads; second row tiles are empty
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_last_round_split(ops, q_len, k_len, heads, before, causal, dtype):
    """A few blocks more than fill the GPU a number of times: those of the last round are halved."""
    nh, nkv = heads
    q, k, v = randn(1, sum(q_len), nh, D, dtype=dtype), randn(2, sum(k_len), nkv, D, dtype=dtype), randn(3, sum(k_len), nkv, D, dtype=dtype)
    prefix = (randn(4, before, nkv, D, dtype=dtype), randn(5, before, nkv, D, dtype=dtype)) if before else None
    check(ops, q, k, v, q_len, k_len, prefix, causal)


def test_last_round_split_odd_values(ops):
    """Infinities in V at a key that only some rows of a halved block see reach those rows alone, and NaN that none of them sees nobody."""
    n, length = 20, 64
    q, k, v = randn(1, n * length, 32, D), randn(2, n * length, 8, D), randn(3, n * length, 8, D)
    prefix, at = (randn(4, 300, 8, D), randn(5, 300, 8, D)), starts([length] * n)
    want, want_lse = ops.attention(q, k, v, at, prefix=prefix)
    first = (n - 1) * length       # the last sequence, whose items are the last
    v[first + 20, :, 5], v[first + 50, :, 7], k[first + 63, :, 0], v[first + 63, :, 9] = math.inf, -math.inf, math.nan, math.nan
    out, lse = ops.attention(q, k, v, at, prefix=prefix)
    assert bool((out[first + 20:first + 63, :, 5] == math.inf).all()) and bool((out[first + 50:first + 63, :, 7] == -math.inf).all())
    out[first + 20:first + 63, :, 5], out[first + 50:first + 63, :, 7] = want[first + 20:first + 63, :, 5], want[first + 50:first + 63, :, 7]
    assert bool(out[first + 63].isnan().all()) and bool(lse[:, first + 63].isnan().all())
    assert torch.equal(out[:first + 63], want[:first + 63]) and torch.equal(lse[:, :first + 63], want_lse[:, :first + 63])


def test_strides_and_alignment(ops):
    """Heads before tokens, rows of a wider matrix, expanded heads, and bases on 2-byte boundaries."""
    q_len = [130, 70]
    T = sum(q_len)
    want = None
    qkv = randn(7, T, 12, D)
    q, k, v = qkv[:, :8].contiguous(), qkv[:, 8:10].contiguous(), qkv[:, 10:].contiguous()
    want = check(ops, q, k, v, q_len, q_len)
    views = {
        "fused": (qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]),
        "heads first": tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)),
        "odd base": tuple(torch.cat((x.new_zeros(1), x.flatten()))[1:].view(x.shape) for x in (q, k, v)),
        "odd rows": tuple(torch.nn.functional.pad(x, (0, 1))[..., :D] for x in (q, k, v)),
        "channels apart": tuple(x.repeat_interleave(2, -1)[..., ::2] for x in (q, k, v)),
    }
    for name, (a, b, c) in views.items():
        got = ops.attention(a, b, c, starts(q_len))
        assert all(torch.equal(x, y) for x, y in zip(got, want)), name
        rows = ops.importance(a, b, want[1], starts(q_len), rows=9)
        assert torch.equal(rows, ops.importance(q, k, want[1], starts(q_len), rows=9)), name
    one = randn(8, T, 1, D)
    got = ops.attention(q, one.expand(T, 2, D), one.expand(T, 2, D), starts(q_len).long())
    same = ops.attention(q, one.repeat(1, 2, 1), one.repeat(1, 2, 1), starts(q_len))
    assert all(torch.equal(x, y) for x, y in zip(got, same))


def test_what_is_not_seen_does_not_matter(ops):
    """NaN and infinities in keys and values behind a query, in the neighbours and outside of all sequences."""
    q_len = [150, 90]
    first, T = 5, 5 + 240 + 11
    q, k, v = randn(1, T, 8, D), randn(2, T, 2, D), randn(3, T, 2, D)
    at = starts(q_len, first)
    want, lse = ops.attention(q, k, v, at)
    for bad in (math.nan, math.inf, -math.inf):
        for where in (k, v):
            for lo, hi, same in ((0, first, (first, T - 11)), (T - 11, T, (first, T - 11)), (first + 100, first + 101, (first, first + 100)),
                                 (first + 149, first + 150, (first + 150, T - 11)), (first + 149, first + 150, (first, first + 149)),
                                 (first + 150, first + 190, (first, first + 150)), (first + 17, first + 40, (first, first + 17))):
                old = where[lo:hi].clone()
                where[lo:hi, :, 3::7] = bad
                got, l = ops.attention(q, k, v, at)
                assert torch.equal(got[same[0]:same[1]], want[same[0]:same[1]]), (bad, where is k, lo, same)
                assert torch.equal(l[:, same[0]:same[1]], lse[:, same[0]:same[1]])
                if where is v and lo >= first and hi <= T - 11:   # and who sees it, knows it: channel 3 of the last row of the sequence
                    last = first + 149 if lo < first + 150 else T - 12
                    assert bool((got[last, :, 3] == bad).all() if not math.isnan(bad) else got[last, :, 3].isnan().all())
                    assert bool(got[last, :, 2].isfinite().all())
                where[lo:hi] = old


def test_rows_outside_of_sequences_stay(ops):
    q, k, v = randn(1, 300, 8, D), randn(2, 300, 2, D), randn(3, 300, 2, D)
    out = torch.full_like(q, 7.0)
    got, lse = ops.attention(q, k, v, starts([100, 0, 90], 20), out=out)
    assert got.data_ptr() == out.data_ptr()
    assert bool((out[:20] == 7).all()) and bool((out[210:] == 7).all()) and bool((out[20:210] != 7).any(-1).all())
    rows = torch.full((20, 300), 7.0, dtype=torch.float16, device="cuda")
    ops.importance(q, k, lse, starts([100, 0, 90], 20), out=rows)
    assert bool((rows[:, :20] == 7).all()) and bool((rows[:, 210:] == 7).all()) and bool((rows[:, 20:210] <= 8).all())


def test_starts_out_of_range_are_clamped(ops):
    q, k, v = randn(1, 100, 4, D), randn(2, 100, 2, D), randn(3, 100, 2, D)
    want = ops.attention(q, k, v, starts([100]))
    got = ops.attention(q, k, v, torch.tensor([-50, 100000], dtype=torch.int32, device="cuda"))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rows = ops.importance(q, k, want[1], torch.tensor([-50, 100000], dtype=torch.int32, device="cuda"))
    assert torch.equal(rows, ops.importance(q, k, want[1], starts([100])))
    odd = torch.tensor([0, 70, 30, 100], dtype=torch.int32, device="cuda")   # decreasing: no result is promised, only that it ends
    ops.attention(q, k, v, odd)
    ops.importance(q, k, want[1], odd)
    torch.cuda.synchronize()


def test_nothing_to_do(ops):
    empty, k = randn(1, 0, 4, D), randn(2, 30, 2, D)
    out, lse = ops.attention(empty, k, k, starts([0]), starts([30]))
    assert out.shape == (0, 4, D) and lse.shape == (4, 0)
    out, lse = ops.attention(randn(1, 5, 4, D), k[:0], k[:0], starts([3, 2]), starts([0, 0]))
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    out, _ = ops.attention(randn(1, 5, 4, D), k, k, starts([]), starts([]), out=torch.full((5, 4, D), 3.0, device="cuda", dtype=torch.float16))
    assert bool((out == 3).all())
    assert bool((ops.importance(empty, k, torch.zeros(4, 0, device="cuda"), starts([0]), starts([30])) == 0).all())
    assert ops.importance(randn(1, 5, 4, D), k[:0], torch.zeros(4, 5, device="cuda"), starts([5]), starts([0])).shape == (20, 0)


def test_long_offsets(ops):
    """Keys behind 2^31 elements of K and V, and queries behind as many of q."""
    tokens, nkv = (1 << 21) + 5000, 8
    k, v = (torch.empty(tokens, nkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
    a, b = tokens - 400, tokens - 60
    k[a:], v[a:] = randn(2, 400, nkv, D), randn(3, 400, nkv, D)
    q = torch.empty(tokens, nkv, D, dtype=torch.float16, device="cuda")
    q[a:] = randn(1, 400, nkv, D)
    at = torch.tensor([a, b], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    _, lse = ops.attention(q, k, v, at, out=out)
    o, l, bound, _ = reference(q[a:b], k[a:b], v[a:b], None, True, D ** -0.5)
    assert float(((out[a:b].double() - o).abs() / bound).max()) <= 1
    rows = ops.importance(q, k, lse, at, rows=20)
    want = importance_reference(q[a:b], k[a:b], l, 20)
    assert float((rows[:, a:b].double() - want).abs().max()) <= 2.0 ** -11 * float(want.max()) * 1.1


@pytest.mark.parametrize("before", [0, 500])
def test_streams_and_graphs(ops, before):
    """Two calls at once on two streams, and a captured call replayed on other inputs and other starts."""
    def inputs(seed):
        return randn(seed, 400, 8, D), randn(seed + 1, 400, 2, D), randn(seed + 2, 400, 2, D)
    prefix = (randn(90, before, 2, D), randn(91, before, 2, D)) if before else None
    sets, at = [inputs(10), inputs(20)], [starts([300, 100]), starts([20, 380])]
    want = [ops.attention(*x, a, prefix=prefix) for x, a in zip(sets, at)]
    rows = [ops.importance(x[0], x[1], w[1], a) for x, a, w in zip(sets, at, want)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out, lse = ops.attention(*sets[i], at[i], prefix=prefix)
                got[i] = (out, lse, ops.importance(sets[i][0], sets[i][1], lse, at[i]))
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1]) and torch.equal(got[i][2], rows[i])
    bufs, a = [x.clone() for x in sets[0]], at[0].clone()
    ops.attention(*bufs, a, prefix=prefix)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.attention(*bufs, a, prefix=prefix)
        imp = ops.importance(bufs[0], bufs[1], lse, a)
    for i in (1, 0, 1):
        for x, y in zip(bufs, sets[i]):
            x.copy_(y)
        a.copy_(at[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1]) and torch.equal(imp, rows[i])


@pytest.mark.parametrize("q_len, k_len, other_q, other_k, before", [
    ([96, 37, 73, 14], [5096, 337, 9073, 14], [1, 160, 0, 59], [40, 200, 14000, 280], 0),      # shares by length
    ([64] * 20, [64] * 20, [1280] + [0] * 19, [1280] + [0] * 19, 300),                          # a last round that is halved, and none
])
def test_replay_with_other_lengths(ops, q_len, k_len, other_q, other_k, before):
    """A captured call, whose launches and workspace were chosen without the lengths, replayed with others."""
    assert sum(q_len) == sum(other_q) and sum(k_len) == sum(other_k)
    q, k, v = randn(1, sum(q_len), 32, D), randn(2, sum(k_len), 8, D), randn(3, sum(k_len), 8, D)
    prefix = (randn(4, before, 8, D), randn(5, before, 8, D)) if before else None
    lengths = [(q_len, k_len), (other_q, other_k)]
    want = [check(ops, q, k, v, *x, prefix) for x in lengths]
    at = [(starts(x), starts(y)) for x, y in lengths]
    a, b = at[0][0].clone(), at[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, lse = ops.attention(q, k, v, a, b, prefix=prefix)
    for i in (1, 0, 1):
        a.copy_(at[i][0])
        b.copy_(at[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


# ------------------------------------------------------------------------------------------------
# importance rows
# ------------------------------------------------------------------------------------------------
def importance_reference(q, k, lse, rows, causal=True):
    n, m, t = q.shape[0], k.shape[0], min(rows, q.shape[0])
    out = torch.zeros(rows, m, dtype=torch.float64, device="cuda")
    if t:
        rep = q.shape[1] // k.shape[1]
        s = torch.einsum("nhd,mhd->hnm", q[n - t:].double(), k.double().repeat_interleave(rep, 1)) * D ** -0.5
        if causal:
            i, j = torch.arange(n - t, n, device="cuda")[:, None], torch.arange(m, device="cuda")
            s = s.masked_fill(j > i + m - n, -math.inf)
        out[:t] = torch.exp(s - lse.double()[:, n - t:, None]).nan_to_num(0.0).sum(0)   # (no key, lse -inf: no share)
    return out


@pytest.mark.parametrize("heads", [(32, 8), (4, 4), (6, 2), (8, 1), (48, 3)])
@pytest.mark.parametrize("rows", [1, 7, 20, 33, 64])
def test_importance(ops, heads, rows):
    nh, nkv = heads
    q_len, k_len = [300, 1, 0, 13, 64, 5], [300, 1, 4, 13, 700, 3]
    for dtype in (torch.float16, torch.bfloat16):
        q, k, v = randn(1, sum(q_len), nh, D, dtype=dtype), randn(2, sum(k_len), nkv, D, dtype=dtype), randn(3, sum(k_len), nkv, D, dtype=dtype)
        for causal in (True, False):
            _, lse = ops.attention(q, k, v, starts(q_len), starts(k_len), causal=causal)
            got = ops.importance(q, k, lse, starts(q_len), starts(k_len), rows=rows, causal=causal)
            assert got.shape == (rows, sum(k_len)) and got.dtype == torch.float16
            a = b = 0
            for n, m in zip(q_len, k_len):
                want = importance_reference(q[a:a + n], k[b:b + m], lse[:, a:a + n], rows, causal)
                err = (got[:, b:b + m].double() - want).abs()
                top = terms(q[a:a + n].double(), k[b:b + m].double().repeat_interleave(nh // nkv, 1), D ** -0.5)
                assert bool((err <= (2.0 ** -11 + 2.0 ** -16 * top + 2.0 ** -20) * want + 2.0 ** -25).all())
                a, b = a + n, b + m


def test_importance_masks_and_prefix(ops):
    """NaN in keys that a row does not see; rows behind a prefix add up to what the prefix leaves."""
    q, k, v = randn(1, 200, 8, D), randn(2, 200, 2, D), randn(3, 200, 2, D)
    prefix = (randn(4, 150, 2, D), randn(5, 150, 2, D))
    _, lse = ops.attention(q, k, v, starts([120, 80]), prefix=prefix)
    got = ops.importance(q, k, lse, starts([120, 80]), rows=8)
    full = torch.cat((prefix[0], k[:120]))
    want = importance_reference(torch.cat((torch.zeros_like(q[:150]), q[:120])), full, torch.cat((torch.zeros(8, 150, device="cuda"), lse[:, :120]), 1), 8)
    assert bool(((got[:, :120].double() - want[:, 150:]).abs() <= 2.0 ** -11 * 1.1 * want[:, 150:] + 2.0 ** -25).all())
    k[116:120] = math.nan
    again = ops.importance(q, k, lse, starts([120, 80]), rows=8)
    assert torch.equal(again[:4], got[:4]) and torch.equal(again[:, 120:], got[:, 120:]) and bool(again[7, 116:120].isnan().all())
    assert torch.equal(again[:, :116], got[:, :116])


# ------------------------------------------------------------------------------------------------
# decode behind a shared prefix
# ------------------------------------------------------------------------------------------------
def build(cuda_device, strategy, batch, nh_q, nh_kv, group, tokens, residual, seed=11, shares=(0.25, 0.25, 0.25, 0.25)):
    from hqekv_b200 import synthetic
    cfg = synthetic.CacheConfig("prefix", batch, nh_q, nh_kv, D, tokens + residual, residual, shares, 0.125, group, False, 1, 64)
    return synthetic.build_cache(cfg, cuda_device, seed=seed, times_range=True, quant_strategy=strategy)


def check_prefix(ops, q, cache, prefix, group=32, strategy="uniform_group", call=None):
    """Against the formula in 64 bits on the dequantised cache; tolerances as above, p rounded relative to the cache's own sum in its part."""
    w, o = (call or ops.prefix)(q, cache, prefix, D, strategy, group, group)
    host = tuple(x.cpu().numpy() if torch.is_tensor(x) else x for x in cache)
    K, V = (torch.from_numpy(x).double().cuda() for x in O.reconstruct_fp32(host, group, group, strategy))
    B, nkv, L, _ = K.shape
    rep, P = q.shape[1] // nkv, prefix[0].shape[0]
    K = torch.cat((prefix[0].double().transpose(0, 1).expand(B, -1, -1, -1), K), 2).repeat_interleave(rep, 1)
    V = torch.cat((prefix[1].double().transpose(0, 1).expand(B, -1, -1, -1), V), 2).repeat_interleave(rep, 1)
    s = torch.matmul(q.double(), K.transpose(2, 3)) * D ** -0.5
    p = torch.softmax(s, -1)
    out, a, top = torch.matmul(p, V), torch.matmul(p, V.abs()), float(torch.matmul(q.double().abs(), K.abs().transpose(2, 3)).max()) * D ** -0.5
    own = p[..., P:].sum(-1, keepdim=True)
    lost = 2.0 ** -25 * (1 + own * V[:, :, P:].abs().sum(2, keepdim=True) + p.amax(-1, keepdim=True) * V.abs().sum(2, keepdim=True))
    over = (o.double() - out).abs() / (2.0 ** -11 * (a + out.abs()) + (2.0 ** -16 * top + 2.0 ** -20) * a + lost)
    assert w.shape == (B, q.shape[1], 1, L) and w.dtype == o.dtype == torch.float16 and o.shape == q.shape
    assert float(over.max()) <= 1, f"output off by {float(over.max()):.3g} of what it may be"
    err = (w.double() - p[..., P:]).abs()
    assert bool((err <= (2.0 ** -11 + 2.0 ** -16 * top + 2.0 ** -20) * p[..., P:] + 2.0 ** -25).all())
    return w, o


@pytest.mark.parametrize("before", [1, 127, 128, 129, 2000])
@pytest.mark.parametrize("batch, heads", [(1, (4, 1)), (3, (8, 2)), (2, (2, 2)), (5, (16, 2)), (33, (4, 2)), (70, (8, 1))])
def test_prefix_decode_residual_only(ops, cuda_device, batch, heads, before):
    nh, nkv = heads
    cache = (None,) * 39 + (randn(1, batch, nkv, 37, D), randn(2, batch, nkv, 37, D), 37)
    check_prefix(ops, randn(3, batch, nh, 1, D), cache, (randn(4, before, nkv, D), randn(5, before, nkv, D)))


@pytest.mark.parametrize("strategy", ["uniform_group", NORMAL])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_prefix_decode_tiers(ops, cuda_device, strategy, group):
    cache, q = build(cuda_device, strategy, 3, 8, 2, group, 1024, 40)
    prefix = (randn(4, 1500, 2, D), randn(5, 1500, 2, D))
    w, o = check_prefix(ops, q, cache, prefix, group, strategy)
    # the decode itself is as it was, before and after
    w2, o2 = ops.decode(q, cache, None, D, strategy, group, group)
    assert not torch.equal(o, o2)
    share = w.double().sum(-1) / w2.double().sum(-1)
    assert bool(((w.double() - share[..., None] * w2.double()).abs() <= 2.0 ** -10 * w.double() + 2.0 ** -23).all())


def test_prefix_decode_long_cache(ops, cuda_device):
    """More own tokens than one CTA of the join writes the weights of, an odd number of them."""
    cache, q = build(cuda_device, "uniform_group", 2, 8, 2, 32, 8192, 35)
    check_prefix(ops, q, cache, (randn(4, 300, 2, D), randn(5, 300, 2, D)))


def test_prefix_decode_strides_streams_graphs(ops, cuda_device):
    cache, q = build(cuda_device, "uniform_group", 4, 8, 2, 32, 512, 33)
    k, v = randn(4, 700, 2, D), randn(5, 700, 2, D)
    want = check_prefix(ops, q, cache, (k, v))
    heads_first = tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    odd = tuple(torch.cat((x.new_zeros(1), x.flatten()))[1:].view(x.shape) for x in (k, v))
    for prefix in (heads_first, odd, (heads_first[0], v)):
        assert all(torch.equal(x, y) for x, y in zip(ops.prefix(q, cache, prefix, D, "uniform_group"), want))
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(other):
            a = ops.prefix(q, cache, (k, v), D, "uniform_group")
        b = ops.prefix(q, cache, (k, v), D, "uniform_group")
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) and torch.equal(z, y) for x, y, z in zip(a, want, b))
    q2 = randn(9, 4, 8, 1, D)
    want2 = check_prefix(ops, q2, cache, (k, v))
    buf = q.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.prefix(buf, cache, (k, v), D, "uniform_group")
    for x, y in ((q2, want2), (q, want)):
        buf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(i, j) for i, j in zip(got, y))


def test_prompt_then_decode(ops, cuda_device):
    """The operators as they are used together: a prefix and the prompts behind it, the ring rows, then single tokens behind
    both - the same numbers as one prompt over everything."""
    nh, nkv, P, S = 8, 2, 200, 70
    B = 3
    prefix_q, pk, pv = randn(1, P, nh, D), randn(2, P, nkv, D), randn(3, P, nkv, D)
    q, k, v = randn(4, B * S, nh, D), randn(5, B * S, nkv, D), randn(6, B * S, nkv, D)
    check(ops, prefix_q, pk, pv, [P], [P])
    out, lse = check(ops, q, k, v, [S] * B, [S] * B, (pk, pv))
    rows = ops.importance(q, k, lse, starts([S] * B))
    heads_first = [x.view(B, S, nkv, D).transpose(1, 2).contiguous() for x in (k, v)]
    cache = (None,) * 39 + (heads_first[0], heads_first[1], S)
    last = q.view(B, S, nh, D)[:, -1:].transpose(1, 2)   # the last query again, as a decode step over the same keys
    w, o = check_prefix(ops, last, cache, (pk, pv))
    assert float((o[:, :, 0] - out.view(B, S, nh, D)[:, -1]).abs().max()) <= 2.0 ** -9
    got = w.double().sum(1)[:, 0]
    assert float((rows[-1].view(B, S).double() - got).abs().max()) <= 2.0 ** -11 * nh


def test_many_sequences(ops):
    """More sequences than a warp looks up at a time, empty ones among them, more blocks than CTAs."""
    rng = np.random.default_rng(5)
    q_len = [int(n) for n in rng.integers(0, 9, 500)]
    k_len = [n + int(m) for n, m in zip(q_len, rng.integers(0, 200, 500))]
    q, k, v = randn(1, sum(q_len), 8, D), randn(2, sum(k_len), 2, D), randn(3, sum(k_len), 2, D)
    check(ops, q, k, v, q_len, k_len)


def test_waits_did_not_run_out():
    import ctypes
    from hqekv_b200 import _lib
    count = ctypes.c_uint(7)
    assert _lib.lib.hqkv_prompt_waits_expired(1, ctypes.byref(count)) == 0 and count.value == 0
