"""CPU-only: a shared prefix is part of the module that holds it."""
import copy

import torch


def test_a_prefix_goes_where_its_module_goes(monkeypatch):
    from hqekv_b200.model import decoder
    monkeypatch.setattr(decoder, "prompt_attention", lambda q, k, v, starts, **kw: (torch.zeros_like(q), None))
    model = decoder.HqeDecoder(decoder.DecoderConfig(hidden_size=64, num_layers=2, num_heads=2, num_kv_heads=1, intermediate_size=64))
    keys = set(model.state_dict())
    model.share_prefix(torch.randn(1, 5, 64))
    want = [tuple(x.half() for x in layer.self_attn.prefix) for layer in model.layers]
    model.half()
    for layer, pair in zip(model.layers, want):
        assert all(x.dtype == torch.float16 and torch.equal(x, y) for x, y in zip(layer.self_attn.prefix, pair))
    model.to("meta")
    assert all(x.is_meta for layer in model.layers for x in layer.self_attn.prefix)
    assert set(model.state_dict()) == keys       # (a checkpoint holds no prefix, and one without it loads)
    other = copy.deepcopy(model)
    model.share_prefix()
    assert all(layer.self_attn.prefix is None for layer in model.layers) and other.layers[0].self_attn.prefix is not None
