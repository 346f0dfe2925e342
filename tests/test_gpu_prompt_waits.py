"""The prompt kernels where a wait runs out: the bounds-check build, told to give up after a few tries, ends every call with work under way in
all roles, counts what gave up, and calls without that limit are right again.  Nothing here is broken: the waits are for work
that comes, and a limit of microseconds is shorter than that."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import sys
import torch
sys.path.insert(0, {root!r})
from hqekv_b200 import _lib
from hqekv_b200.prompt import prompt_attention, prompt_importance, waits_expired
from hqekv_b200.quant.hqe_matmul import qkv_matmul_hqe_prefix
assert _lib.lib.hqkv_checks_enabled() == 1, "the checked library is not the one loaded"

def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half()

def starts(lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")

def prompt(q_len, k_len, nh, nkv, before=0):
    q, k, v = randn(1, sum(q_len), nh, 128), randn(2, sum(k_len), nkv, 128), randn(3, sum(k_len), nkv, 128)
    prefix = (randn(4, before, nkv, 128), randn(5, before, nkv, 128)) if before else None
    a, b = starts(q_len), starts(k_len)
    def call():
        out, lse = prompt_attention(q, k, v, a, b, prefix=prefix)
        return out, lse
    return call

def rows(q_len, k_len, nh, nkv):
    q, k = randn(1, sum(q_len), nh, 128), randn(2, sum(k_len), nkv, 128)
    a, b, lse = starts(q_len), starts(k_len), torch.full((nh, sum(q_len)), 9.0, device="cuda")
    return lambda: (prompt_importance(q, k, lse, a, b),)

def decode(batch, nh, nkv, before):
    cache = (None,) * 39 + (randn(1, batch, nkv, 37, 128), randn(2, batch, nkv, 37, 128), 37)
    q, prefix = randn(3, batch, nh, 1, 128), (randn(4, before, nkv, 128), randn(5, before, nkv, 128))
    return lambda: qkv_matmul_hqe_prefix(q, cache, prefix, 128, "uniform_group")

cases = [
    ("one prompt, several items per CTA", prompt([6000], [6000], 32, 8)),
    ("blocks of one row tile", prompt([300], [300], 32, 8)),
    ("tiles of V that few rows see", prompt([37] * 60, [150] * 60, 32, 8)),
    ("a prefix, a last round halved", prompt([64] * 20, [64] * 20, 32, 8, 300)),
    ("shares by length", prompt([96, 37, 73, 14], [5096, 337, 9073, 14], 32, 8)),
    ("shares of one sequence", prompt([1], [20000], 4, 1)),
    ("ring rows", rows([40000], [40000], 32, 8)),
    ("ring rows of many", rows([30] * 200, [90] * 200, 8, 1)),
    ("a decode behind a prefix", decode(33, 8, 2, 3000)),
]
want = [[x.clone() for x in call()] for _, call in cases]
assert waits_expired(reset=True) == 0
total = 0
for tries in (1, 2, 7):
    _lib.check(_lib.lib.hqkv_prompt_limit_waits(tries))
    for name, call in cases:
        for _ in range(3):
            call()
        torch.cuda.synchronize()
        n = waits_expired(reset=True)
        total += n
        print(tries, name, n)
    _lib.check(_lib.lib.hqkv_prompt_limit_waits(0))
    for (name, call), w in zip(cases, want):
        assert all(torch.equal(x, y) for x, y in zip(call(), w)), name
    assert waits_expired() == 0
assert total > 0, "no wait ran out"
print("gave up and went on:", total)
"""


def test_waits_that_run_out(cuda_device):
    from hqekv_b200 import build
    env = dict(os.environ, HQKV_LIB=build.build(checks=True))
    r = subprocess.run([sys.executable, "-c", CHILD.format(root=ROOT)], env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-4000:]
    assert "gave up and went on" in r.stdout


def test_the_regular_build_has_one_limit(cuda_device):
    from hqekv_b200 import _lib
    from hqekv_b200.prompt import waits_expired
    if _lib.lib.hqkv_checks_enabled():
        pytest.skip("the bounds-check build is loaded")
    assert _lib.lib.hqkv_prompt_limit_waits(1) == -2 and "bounds-check build" in _lib.lib.hqkv_last_error().decode()
    assert waits_expired() == 0


COUNT = r"""
import sys
import torch
sys.path.insert(0, {root!r})
from hqekv_b200 import _lib
from hqekv_b200.prompt import prompt_attention, waits_expired
q, k = (torch.randn(6000, h, 128, device="cuda").half() for h in (32, 8))
at = torch.tensor([0, 6000], dtype=torch.int32, device="cuda")
prompt_attention(q, k, k, at)
assert waits_expired(reset=True) == 0
_lib.check(_lib.lib.hqkv_prompt_limit_waits(1))
with torch.cuda.stream(torch.cuda.Stream()):
    torch.cuda._sleep(400_000_000)     # a fifth of a second
    prompt_attention(q, k, k, at)
n = waits_expired()
assert n > 0, "read before the call had ended"
torch.cuda.synchronize()
assert waits_expired(reset=True) == n
print("counted", n)
"""


def test_the_count_waits_for_every_stream(cuda_device):
    """torch's streams do not wait for the default one, nor it for them."""
    from hqekv_b200 import build
    env = dict(os.environ, HQKV_LIB=build.build(checks=True))
    r = subprocess.run([sys.executable, "-c", COUNT.format(root=ROOT)], env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "counted" in r.stdout, r.stdout[-3000:] + r.stderr[-4000:]
