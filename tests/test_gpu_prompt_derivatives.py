"""The native path refuses what derivatives are asked of, as the path in Python does (test_prompt_refusals.py)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_derivatives_by_either_mode(cuda_device):
    from torch.autograd import forward_ad
    from hqekv_b200.prompt import prompt_attention, prompt_importance
    from hqekv_b200.quant.hqe_matmul import qkv_matmul_hqe_prefix
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = {n: torch.randn(*shape, 128, generator=gen, device="cuda").half()
         for n, shape in dict(q=(5, 4), k=(5, 2), v=(5, 2), pk=(6, 2), pv=(6, 2), q1=(1, 4, 1), new=(1, 2, 3)).items()}
    at = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    cache = (None,) * 39 + (x["new"], x["new"], 3)
    x["lse"] = prompt_attention(x["q"], x["k"], x["v"], at)[1]
    calls = (
        (lambda x: prompt_attention(x["q"], x["k"], x["v"], at, prefix=(x["pk"], x["pv"])), ("q", "k", "v", "pk", "pv")),
        (lambda x: (prompt_importance(x["q"], x["k"], x["lse"], at),), ("q", "k", "lse")),
        (lambda x: qkv_matmul_hqe_prefix(x["q1"], cache, (x["pk"], x["pv"]), 128, "uniform_group"), ("q1", "pk", "pv")))
    for call, names in calls:
        want = call(x)
        for name in names:
            leaf = dict(x, **{name: x[name].clone().requires_grad_()})
            with pytest.raises(RuntimeError, match="no backward"):
                call(leaf)
            with torch.no_grad():
                assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(call(leaf), want))
            with forward_ad.dual_level():
                dual = dict(x, **{name: forward_ad.make_dual(x[name], torch.ones_like(x[name]))})
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(RuntimeError, match="no forward derivatives"):
                        call(dual)
                assert all(torch.equal(a, b) for a, b in zip(call(x), want))
