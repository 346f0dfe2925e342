"""CPU-only: what the prompt operators and the decode behind a shared prefix refuse, in Python and at the C ABI."""
import ctypes as C

import pytest
import torch

from hqekv_b200 import _lib
from hqekv_b200.prompt import prompt_attention, prompt_importance
from hqekv_b200.quant.hqe_matmul import qkv_matmul_hqe_prefix

F16 = torch.float16


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


def starts(*at, dtype=torch.int32):
    return torch.tensor(at, dtype=dtype)


GOOD = dict(q=z(5, 4, 128), k=z(5, 2, 128), v=z(5, 2, 128), seq_starts=starts(0, 5))


@pytest.mark.parametrize("change, text", [
    (dict(q=z(5, 4, 128, dtype=torch.float32)), "float16 or bfloat16"),
    (dict(q=z(5, 4, 64)), "128"),
    (dict(q=z(5, 512)), "128"),
    (dict(q=z(5, 3, 128)), "multiple"),
    (dict(q=z(5, 0, 128)), "multiple"),
    (dict(k=z(5, 2, 128, dtype=torch.bfloat16)), "type and device"),
    (dict(k=z(6, 2, 128), v=z(6, 2, 128)), "kv_starts"),
    (dict(v=z(5, 1, 128)), "2 heads"),
    (dict(v=z(4, 2, 128)), "5 tokens"),
    (dict(seq_starts=[0, 5]), "seq_starts"),
    (dict(seq_starts=z(2)), "seq_starts"),
    (dict(seq_starts=torch.zeros(0, dtype=torch.int32)), "seq_starts"),
    (dict(kv_starts=starts(0, 2, 5)), "2 entries"),
    (dict(prefix=(z(7, 1, 128), z(7, 1, 128))), "2 heads"),
    (dict(prefix=(z(7, 2, 128), z(8, 2, 128))), "7 tokens"),
    (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(scale=2e38), "scale"),
])
def test_prompt_attention_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        prompt_attention(**{**GOOD, **change})


@pytest.mark.parametrize("rows", [0, 65, -1, 2.0, True])
def test_prompt_importance_refuses_rows(rows):
    with pytest.raises(ValueError, match="rows"):
        prompt_importance(z(5, 4, 128), z(5, 2, 128), torch.zeros(4, 5), starts(0, 5), rows=rows)


def test_no_gradients_and_no_cpu():
    q = z(5, 4, 128).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        prompt_attention(q, GOOD["k"], GOOD["v"], GOOD["seq_starts"])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        prompt_attention(**GOOD)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        prompt_importance(z(5, 4, 128), z(5, 2, 128), torch.zeros(4, 5), starts(0, 5))


def cache_of(batch=2, heads=2, tokens=3):
    return (None,) * 39 + (z(batch, heads, tokens, 128), z(batch, heads, tokens, 128), tokens)


def test_prefix_decode_refuses():
    q, pre = z(2, 4, 1, 128), (z(6, 2, 128), z(6, 2, 128))
    with pytest.raises(ValueError, match="invalid quant_strategy"):
        qkv_matmul_hqe_prefix(q, cache_of(), pre, 128, "other")
    with pytest.raises(ValueError, match="invalid past_key_value"):
        qkv_matmul_hqe_prefix(q, cache_of()[:41], pre, 128, "uniform_group")
    with pytest.raises(ValueError, match="invalid past_key_value"):
        qkv_matmul_hqe_prefix(q, (None,) * 41 + (0,), pre, 128, "uniform_group")
    for bad_q in (z(2, 4, 2, 128), z(2, 4, 1, 128, dtype=torch.bfloat16), z(2, 4, 128)):
        with pytest.raises(ValueError, match="q must be float16"):
            qkv_matmul_hqe_prefix(bad_q, cache_of(), pre, 128, "uniform_group")
    with pytest.raises(ValueError, match="does not match the cache"):
        qkv_matmul_hqe_prefix(z(3, 4, 1, 128), cache_of(), pre, 128, "uniform_group")
    for bad in ((z(6, 1, 128), z(6, 1, 128)), (z(6, 2, 64), z(6, 2, 64)), (z(1, 6, 2, 128), z(1, 6, 2, 128)),
                (z(6, 2, 128, dtype=torch.bfloat16), z(6, 2, 128))):
        with pytest.raises(ValueError, match="prefix must be float16"):
            qkv_matmul_hqe_prefix(q, cache_of(), bad, 128, "uniform_group")
    for bad in ((z(6, 2, 128), z(5, 2, 128)), (z(0, 2, 128), z(0, 2, 128))):
        with pytest.raises(ValueError, match="at least one"):
            qkv_matmul_hqe_prefix(q, cache_of(), bad, 128, "uniform_group")
    with pytest.raises(RuntimeError, match="no backward"):
        qkv_matmul_hqe_prefix(z(2, 4, 1, 128).requires_grad_(), cache_of(), pre, 128, "uniform_group")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        qkv_matmul_hqe_prefix(q, cache_of(), pre, 128, "uniform_group")


# ---- the C ABI: a status and a text before anything is enqueued.  Addresses are never read by these calls.
def good_prompt():
    p = _lib.Prompt()
    p.dtype, p.D, p.nh_q, p.nh_kv, p.n_seqs, p.causal, p.scale = 0, 128, 4, 2, 1, 1, 0.1
    p.total_q = p.total_k = 5
    p.q = p.k = p.v = 1 << 20
    p.q_token, p.q_head = 512, 128
    p.k_token, p.k_head, p.v_token, p.v_head = 256, 128, 256, 128
    p.q_starts = p.k_starts = 1 << 20
    return p


@pytest.mark.parametrize("field, value, text", [
    ("dtype", 2, "type"), ("D", 64, "128"), ("nh_q", 3, "multiple"), ("nh_q", 0, "multiple"), ("nh_kv", 0, "multiple"),
    ("nh_q", 1 << 17, "too many heads"), ("n_seqs", -1, "negative"), ("total_q", -1, "negative"), ("prefix_len", -1, "negative"),
    ("total_k", 1 << 30, "too many"), ("n_seqs", 1 << 24, "too many"), ("scale", 0.0, "scale"), ("scale", float("nan"), "scale"),
    ("q", None, "null"), ("k", None, "null"), ("v", None, "null"), ("prefix_len", 3, "null"), ("q_starts", None, "starts"),
    ("k_starts", 2, "starts"), ("q", 8 + (1 << 20), "16-byte"), ("k_token", 12, "multiples of 8"), ("v_head", -8, "multiples of 8"), ("k_head", 0, "multiples of 8"),
])
def test_c_abi_refuses_prompts(field, value, text):
    p = good_prompt()
    setattr(p, field, value)
    assert _lib.lib.hqkv_prompt_attention(C.byref(p), 1 << 20, 1 << 20, None, 0, None) == -1
    assert text in _lib.lib.hqkv_last_error().decode()


def test_c_abi_refuses_outputs_and_rows():
    p = good_prompt()
    assert _lib.lib.hqkv_prompt_attention(None, 1 << 20, 1 << 20, None, 0, None) == -1
    assert _lib.lib.hqkv_prompt_attention(C.byref(p), None, 1 << 20, None, 0, None) == -1
    assert _lib.lib.hqkv_prompt_attention(C.byref(p), 16 + (1 << 20), 1 << 20, None, 0, None) == -1
    assert _lib.lib.hqkv_prompt_attention(C.byref(p), 1 << 20, None, None, 0, None) == -1
    for rows in (0, 65):
        assert _lib.lib.hqkv_prompt_importance(C.byref(p), 1 << 20, rows, 1 << 20, None) == -1
    assert _lib.lib.hqkv_prompt_importance(C.byref(p), None, 20, 1 << 20, None) == -1
    assert _lib.lib.hqkv_prompt_importance(C.byref(p), 1 << 20, 20, None, None) == -1
    p.total_q = p.n_seqs = 0   # nothing to do: no pointer is looked at
    assert _lib.lib.hqkv_prompt_attention(C.byref(p), None, None, None, 0, None) == 0
    assert _lib.lib.hqkv_prompt_importance(C.byref(p), None, 20, None, None) == 0


def test_c_abi_refuses_prefix_decodes():
    d = _lib.CacheDesc()
    d.B, d.H, d.nh_q, d.D, d.group_k, d.group_v, d.n_new, d.softmax_scale = 2, 2, 4, 128, 32, 32, 3, 0.1
    d.new_k = d.new_v = 1 << 20
    lib, at = _lib.lib, 1 << 20

    def call(prefix_len=6, pw=at, pbytes=1 << 30, q=at, pk=at, stride=256):
        return lib.hqkv_decode_attention_prefix(C.byref(d), q, pk, at, prefix_len, stride, 128, 256, 128, at, at, at, 1 << 30, pw, pbytes, None)
    assert lib.hqkv_decode_prefix_workspace_bytes(C.byref(d), 6) > 0
    for bad in (0, -1, 1 << 30):
        assert lib.hqkv_decode_prefix_workspace_bytes(C.byref(d), bad) == 0
        assert call(prefix_len=bad) == -1
    for change in (dict(pw=None), dict(pw=at + 128), dict(q=None), dict(q=at + 8), dict(pk=None), dict(pk=at + 8), dict(stride=12)):
        assert call(**change) == -1, change
    assert call(pbytes=lib.hqkv_decode_prefix_workspace_bytes(C.byref(d), 6) - 1) == -3
    d.D = 64
    assert lib.hqkv_decode_prefix_workspace_bytes(C.byref(d), 6) == 0 and call() == -1


def test_a_prefix_that_fails_leaves_none(monkeypatch):
    """Every layer has the shared prefix or none has: a failure in the second of two layers leaves none."""
    from hqekv_b200.model import decoder
    calls = []

    def attention(q, k, v, starts, **kw):
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("out of memory")
        return torch.zeros_like(q), None

    monkeypatch.setattr(decoder, "prompt_attention", attention)
    model = decoder.HqeDecoder(decoder.DecoderConfig(hidden_size=64, num_layers=2, num_heads=2, num_kv_heads=1, intermediate_size=64))
    with pytest.raises(RuntimeError, match="out of memory"):
        model.share_prefix(torch.randn(1, 5, 64))
    assert model.prefix_length == 0 and all(layer.self_attn.prefix is None for layer in model.layers)
    model.share_prefix(torch.randn(1, 5, 64))
    assert model.prefix_length == 5 and all(layer.self_attn.prefix[0].shape == (5, 1, 128) for layer in model.layers)
