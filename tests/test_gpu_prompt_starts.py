"""Starts of packed sequences that int32 does not hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("starts", [[-2 ** 33, 2 ** 33 + 7], [-2 ** 63, 2 ** 63 - 1], [0, 2 ** 32], [-2 ** 31 - 1, 2 ** 31]])
def test_starts_beyond_int32_are_clamped(cuda_device, starts):
    from hqekv_b200.prompt import prompt_attention, prompt_importance
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(100, h, 128, generator=gen, device="cuda").half() for h in (4, 2, 2))
    whole = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    out, lse = prompt_attention(q, k, v, whole)
    far = torch.tensor(starts, dtype=torch.int64, device="cuda")
    for a, b in ((far, None), (whole, far), (far, whole)):
        got = prompt_attention(q, k, v, a, b)
        assert torch.equal(got[0], out) and torch.equal(got[1], lse)
        assert torch.equal(prompt_importance(q, k, lse, a, b), prompt_importance(q, k, lse, whole))
