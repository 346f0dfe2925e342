"""CPU-only: calls around the prompt operators that would have given a wrong result."""
import pytest
import torch


@pytest.mark.parametrize("queries", [1, 7, 19])
def test_rows_of_no_query_do_not_seed_a_ring(queries):
    """All rows for a prompt shorter than the ring, zeros behind its own: they would count as queries."""
    from hqekv_b200.model.public_func import last_attn_weights
    ring = last_attn_weights(last_length=20)
    ring.set_max_length(400)
    with pytest.raises(ValueError, match="positions"):
        ring.seed(torch.zeros(20, queries, dtype=torch.float16))
    assert ring.weights is None and (ring.next_line, ring.kv_seq_len) == (0, 0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ring.seed(torch.zeros(queries, queries, dtype=torch.float16))


def operands():
    from hqekv_b200.prompt import prompt_attention, prompt_importance
    from hqekv_b200.quant.hqe_matmul import qkv_matmul_hqe_prefix
    q, k, v, lse = torch.zeros(5, 4, 128).half(), torch.zeros(5, 2, 128).half(), torch.zeros(5, 2, 128).half(), torch.zeros(4, 5)
    pk, pv, q1 = torch.zeros(6, 2, 128).half(), torch.zeros(6, 2, 128).half(), torch.zeros(1, 4, 1, 128).half()
    at = torch.tensor([0, 5], dtype=torch.int32)
    cache = (None,) * 39 + (torch.zeros(1, 2, 3, 128).half(), torch.zeros(1, 2, 3, 128).half(), 3)
    x = dict(q=q, k=k, v=v, lse=lse, pk=pk, pv=pv, q1=q1, out=torch.zeros(5, 4, 128).half(), rows=torch.zeros(20, 5).half())
    calls = dict(
        attention=(lambda x: prompt_attention(x["q"], x["k"], x["v"], at, prefix=(x["pk"], x["pv"])), ("q", "k", "v", "pk", "pv")),
        attention_out=(lambda x: prompt_attention(x["q"], x["k"], x["v"], at, out=x["out"]), ("out",)),
        importance=(lambda x: prompt_importance(x["q"], x["k"], x["lse"], at), ("q", "k", "lse")),
        importance_out=(lambda x: prompt_importance(x["q"], x["k"], x["lse"], at, out=x["rows"]), ("rows",)),
        decode=(lambda x: qkv_matmul_hqe_prefix(x["q1"], cache, (x["pk"], x["pv"]), 128, "uniform_group"), ("q1", "pk", "pv")))
    return x, [(call, name) for call, names in calls.values() for name in names]


@pytest.mark.parametrize("i", range(13))
def test_no_derivatives_by_either_mode(i):
    """A tensor whose gradient is wanted, or that carries a tangent, is refused, not taken without it; under no_grad the former is
    taken (and refused only for not being on a GPU), the latter still refused."""
    from torch.autograd import forward_ad
    x, calls = operands()
    call, name = calls[i]
    plain = x[name]
    x[name] = plain.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        call(x)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors only"):
        call(x)
    with forward_ad.dual_level():
        x[name] = forward_ad.make_dual(plain, torch.ones_like(plain))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="no forward derivatives"):
                call(x)
    assert len(calls) == 13


@pytest.mark.parametrize("scale", [1e-46, 1e-300, 1e39, float("nan")])
def test_scales_outside_of_float32(scale):
    """What is 0 or infinite as the kernels take it is refused like a 0 or an infinity."""
    from hqekv_b200.prompt import prompt_attention, prompt_importance
    x, _ = operands()
    at = torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="scale"):
        prompt_attention(x["q"], x["k"], x["v"], at, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        prompt_importance(x["q"], x["k"], x["lse"], at, scale=scale)
    for small in (1e-40, 2.0 ** -149):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            prompt_attention(x["q"], x["k"], x["v"], at, scale=small)


def test_a_refused_prefill_leaves_the_layer_as_it_was():
    """No tokens are counted that were not taken: a mask, a prompt that needs a gradient, a type that is not served."""
    from hqekv_b200.model.attention_hqe import HqeAttention
    layer = HqeAttention(64, 2, 1, fused_prompt=True)
    layer.set_max_length(64)
    q, k = torch.zeros(1, 2, 40, 128).half(), torch.zeros(1, 1, 40, 128).half()
    for args, error in (((q, k, k, torch.zeros(1, 1, 40, 40)), ValueError), ((q.clone().requires_grad_(), k, k), RuntimeError),
                        ((q.float(), k.float(), k.float()), ValueError), ((q, k, k), RuntimeError)):
        with pytest.raises(error):
            layer.attend(*args)
        assert (layer.current_length, layer.history_reserve_length, layer.last_weights.next_line) == (0, 0, 0)
