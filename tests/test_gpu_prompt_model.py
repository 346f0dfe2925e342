"""GPU tests of the model harness on the prompt kernels: the fused prefill against the library's, and a batch behind a shared prefix -
layer, decoder stack, graphed steps - against dense attention."""
import math

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

D = 128
U = 2.0 ** -11


@pytest.fixture(scope="module")
def mods(cuda_device):
    import types
    from hqekv_b200.model import attention_hqe, decoder
    return types.SimpleNamespace(a=attention_hqe, d=decoder)


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half()


def attention(mods, **kw):
    torch.manual_seed(0)
    layer = mods.a.HqeAttention(256, 8, 2, D, **kw).half().cuda().eval()
    layer.set_max_length(600)
    return layer


def by_token(x):
    """[B, heads, S, D] stored token by token, as the projections leave it."""
    return x.transpose(1, 2).contiguous().transpose(1, 2)


@pytest.mark.parametrize("S", [1, 7, 20, 31, 300])
@pytest.mark.parametrize("B", [1, 3])
def test_fused_prefill(mods, B, S):
    """Output: either path rounds the probabilities (u of sum p |v|, at most u max |v|) and the output (as much): 4 u max |v| between them,
    and a tenth for fp32 arithmetic.  Ring: the library's logits are halfs after the product, the scale and the mask (3 u |s| each, of an
    exponential and of the sum that divides it), its probabilities are rounded one by one, then their sums over batch and heads
    (3 u of the value, 2^-25 for each of B nh that is subnormal), the kernel's rows once per sequence and in their sum (2 u, 2^-25)."""
    q, k, v = by_token(randn(1, B, 8, S, D)), by_token(randn(2, B, 2, S, D)), by_token(randn(3, B, 2, S, D))
    plain, fused = attention(mods), attention(mods, fused_prompt=True)
    with torch.no_grad():
        want, _, cache, aux = plain.attend(q, k, v, mods.a.causal_mask(S, S, torch.float16, "cuda"))
        got, weights, cache2, aux2 = fused.attend(q, k, v)
    assert weights is None and got.shape == want.shape
    assert float((got.float() - want.float()).abs().max()) <= 4.4 * U * float(v.abs().max())
    assert (aux is None) == (aux2 is None) == (S < 32)
    assert fused.current_length == plain.current_length and fused.history_reserve_length == plain.history_reserve_length
    r, s = plain.last_weights, fused.last_weights
    assert (r.kv_seq_len, r.next_line) == (s.kv_seq_len, s.next_line)
    if S < 32:   # (a flush that evicts has moved the columns, in the order of two rankings)
        assert torch.equal(cache[39], cache2[39]) and torch.equal(cache[40], cache2[40])
        err = (r.weights.float() - s.weights.float()).abs()
        top = float(torch.matmul(q.float(), k.float().repeat_interleave(4, 1).transpose(2, 3)).abs().max()) * D ** -0.5
        assert bool((err <= (5.5 + 6 * top) * U * r.weights.float() + (8 * B + 2) * 2.0 ** -25).all())


def dense(q, k, v, pk, pv, causal):
    """softmax over [prefix | own] in 64 bits; q [B, nh, S, D], prefix [P, nkv, D] -> [B, S, nh, D] and the own tokens' weights."""
    B, nh, S, _ = q.shape
    rep, P, L = nh // k.shape[1], pk.shape[0], k.shape[2]
    K = torch.cat((pk.transpose(0, 1).expand(B, -1, -1, -1), k), 2).double().repeat_interleave(rep, 1)
    V = torch.cat((pv.transpose(0, 1).expand(B, -1, -1, -1), v), 2).double().repeat_interleave(rep, 1)
    s = torch.matmul(q.double(), K.transpose(2, 3)) * D ** -0.5
    if causal:
        j = torch.arange(P + L, device="cuda") - P
        s = s.masked_fill(j > torch.arange(L - S, L, device="cuda")[:, None], -math.inf)
    p = torch.softmax(s, -1)
    return torch.matmul(p, V).transpose(1, 2), p[..., P:]


@pytest.mark.parametrize("P", [1, 130, 1000])
def test_layer_behind_a_prefix(mods, P):
    """Prefill of a few tokens, then single ones: dense until the first flush, within 2.2 u max |v|; then through the tiers."""
    B, S = 3, 20
    layer = attention(mods)
    pk, pv = randn(4, P, 2, D), randn(5, P, 2, D)
    layer.set_prefix(pk, pv)
    ks, vs = randn(6, B, 2, 60, D), randn(7, B, 2, 60, D)
    qs = randn(8, B, 8, 60, D)
    bound = 2.2 * U * max(float(vs.abs().max()), float(pv.abs().max()))
    with torch.no_grad():
        ctx, _, cache, aux = layer.attend(by_token(qs[:, :, :S]), by_token(ks[:, :, :S]), by_token(vs[:, :, :S]))
        want, p = dense(qs[:, :, :S], ks[:, :, :S], vs[:, :, :S], pk, pv, True)
        assert float((ctx.view(B, S, 8, D).double() - want).abs().max()) <= bound
        rows = layer.last_weights.weights[:S, :S].double()
        assert bool(((rows - p.sum((0, 1))).abs() <= 3 * U * p.sum((0, 1)) + 2.0 ** -23).all())
        for t in range(S, 60):
            ctx, w, cache, aux = layer.attend(qs[:, :, t:t + 1], ks[:, :, t:t + 1], vs[:, :, t:t + 1], None, cache)
            assert bool(ctx.isfinite().all()) and bool((w.float().sum(-1) < 1.01).all())
            if t < 31:
                want, p = dense(qs[:, :, t:t + 1], ks[:, :, :t + 1], vs[:, :, :t + 1], pk, pv, False)
                assert float((ctx.view(B, 1, 8, D).double() - want).abs().max()) <= bound
                assert bool(((w.double() - p).abs() <= 1.2 * U * p + 2.0 ** -25).all())
    assert layer.history_reserve_length > 0 and layer.current_length == 28   # flushed at 32 of the sequence's own tokens
    layer.set_prefix()
    assert layer.prefix is None


def test_prefix_arguments(mods):
    layer = attention(mods)
    for bad in ((randn(1, 5, 2, D), None), (randn(1, 5, 3, D), randn(1, 5, 3, D)), (randn(1, 0, 2, D), randn(1, 0, 2, D)),
                (randn(1, 5, 2, D), randn(1, 6, 2, D)), (randn(1, 1, 5, 2, D), randn(1, 1, 5, 2, D))):
        with pytest.raises(ValueError):
            layer.set_prefix(*bad)
    layer.set_prefix(randn(1, 5, 2, D), randn(2, 5, 2, D))
    q, k = randn(1, 1, 8, 4, D), randn(2, 1, 2, 4, D)
    with pytest.raises(RuntimeError, match="no backward"):
        layer.attend(q.requires_grad_(), k, k)
    with torch.no_grad(), pytest.raises(ValueError, match="mask"):
        attention(mods, fused_prompt=True).attend(q, k, k, torch.zeros(1, 1, 4, 4, device="cuda"))


def dense_decoder(model, x):
    """All layers of the stack on whole sequences with the library's attention, in the model's type."""
    from hqekv_b200.model.attention_hqe import rotary_tables
    B, S, _ = x.shape
    rope = rotary_tables(torch.arange(S, device="cuda").unsqueeze(0).expand(B, S), D, model.cfg.rope_theta, x.dtype)
    for layer in model.layers:
        a = layer.self_attn
        q, k, v = a._project(layer.input_layernorm(x), rope)
        o = nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True, scale=a.scaling, enable_gqa=True)
        x = x + a.o_proj(o.transpose(1, 2).reshape(B, S, -1))
        x = x + layer.mlp(layer.post_attention_layernorm(x))
    return model.norm(x)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_decoder_behind_a_prefix(mods, qk_norm):
    """A stack whose batch shares a prefix against the same stack on whole sequences.  Both round alike, in another order: against the stack in fp32
    the one may be off by twice as much as the other.  Graphed steps behind the prefix as the plain ones."""
    cfg = mods.d.DecoderConfig(hidden_size=256, intermediate_size=384, num_layers=3, num_heads=8, num_kv_heads=2, qk_norm=qk_norm)
    model = mods.d.init_like_pretrained(mods.d.HqeDecoder(cfg).cuda(), 3).half().eval()
    exact = mods.d.HqeDecoder(cfg).cuda().eval()
    exact.load_state_dict(model.state_dict())
    B, P, S = 2, 150, 24
    pre, own = randn(1, 1, P, 256), randn(2, B, S + 6, 256)
    whole = torch.cat((pre.expand(B, -1, -1), own), 1)
    with torch.no_grad():
        want = dense_decoder(exact, whole.float())[:, P:]
        usual = float((dense_decoder(model, whole)[:, P:].float() - want).abs().max())
        model.share_prefix(pre)
        model.start_sequence(200)
        h, caches = model(own[:, :S])
        outs = [h]
        for t in range(S, S + 6):
            h, caches = model(own[:, t:t + 1], caches, t)
            outs.append(h)
        got = torch.cat(outs, 1)
        assert float((got.float() - want).abs().max()) <= 2 * usual
        model.start_sequence(200)
        h, caches = model(own[:, :S])
        step = mods.d.GraphedDecodeStep(model, B, fused=False)
        for t in range(S, S + 6):
            h, caches = step(own[:, t:t + 1], caches, t)
            assert float((h - outs[t - S + 1]).abs().max()) <= 2 * usual
        model.share_prefix()
        model.start_sequence(200)
        h, _ = model(own[:, :S])
        alone = dense_decoder(exact, own[:, :S].float())
        assert model.prefix_length == 0 and float((h.float() - alone).abs().max()) <= 2 * max(usual, float((dense_decoder(model, own[:, :S]).float() - alone).abs().max()))


def test_bench_model_with_prefix(mods):
    """The end-to-end benchmark runs on both paths (a small stack; what is asserted is that it ends and counts)."""
    from hqekv_b200.model import bench_model
    out = bench_model.main(["--layers", "1", "--ctx", "96", "--steps", "3", "--warmup", "1", "--batch", "2", "--fused-prompt", "--shared-prefix", "64"])
    assert out["steps"] == 3 and out["config"]["shared_prefix"] == 64 and out["value"] > 0
