"""Sizes that the token exchange refuses, and calls before the library may be initialised, still run through ``moe_forward`` over an expert MLP of torch functions."""
import os
import subprocess
import sys

import pytest
import torch
from torch._subclasses import FakeTensorMode

from tilelang_b200 import moe

DEV = "cuda"


def test_what_the_exchange_takes():
    def fits(rows, width, experts, top_k, num_experts, logit_rows=None, dtype=torch.bfloat16):
        with FakeTensorMode():                                       # sizes alone: nothing is allocated
            x = torch.empty(rows, width, dtype=dtype, device=DEV)
            return moe._fits_exchange(x, torch.empty(rows if logit_rows is None else logit_rows, experts, device=DEV), top_k, num_experts)

    assert fits(16, 128, 8, 2, 8) and fits(0, 128, 8, 2, 8) and fits(1, 1 << 28, 8, 2, 8)
    assert fits(1 << 28, 8, 8, 7, 8) and not fits(1 << 28, 8, 8, 8, 8)           # 2^31 pairs
    assert not fits(1, (1 << 28) + 8, 8, 2, 8) and not fits(4, 0, 8, 2, 8)
    assert not fits(16, 128, 9, 2, 8) and not fits(16, 128, 1025, 2, 1025)
    assert not fits(16, 128, 8, 2, 8, logit_rows=12)
    assert not fits(16, 128, 8, 2, 8, dtype=torch.float64)
    x = torch.empty(8, 16)
    assert moe._fits_exchange(x[::2], torch.empty(4, 4), 2, 4) and not moe._fits_exchange(x.t(), torch.empty(16, 4), 2, 4)
    assert not moe._fits_exchange(x[:1].expand(8, 16), torch.empty(8, 4), 2, 4)


def test_more_routes_than_tokens():
    mlp = moe.ExpertMLP(lambda rows, counts: rows, lambda rows, counts: rows, lambda h: h)
    with pytest.raises(ValueError, match="9 rows of logits for 8 tokens"):
        moe.moe_forward(torch.zeros(8, 16), torch.zeros(9, 4), 2, 4, mlp)


@pytest.mark.gpu
def test_wide_rows_and_tokens_without_a_route():
    mlp = moe.ExpertMLP(lambda rows, counts: rows, lambda rows, counts: rows, lambda h: h)
    logits = torch.randn(6, 4, device=DEV)
    wide = torch.ones(1, (1 << 28) + 8, device=DEV, dtype=torch.bfloat16)
    weights, _ = moe.route(logits, 1)
    out = moe.moe_forward(wide, logits[:1], 1, 4, mlp)
    assert out.shape == wide.shape and (out == weights[0, 0].to(torch.bfloat16)).all()
    x = torch.randn(8, 32, device=DEV)
    out = moe.moe_forward(x, logits, 2, 4, mlp)
    weights, _ = moe.route(logits, 2)
    # two products of one sign and their sum, a rounding each
    assert torch.allclose(out.double(), x[:6].double() * weights.double().sum(1, keepdim=True), rtol=2 ** -22, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("first", ["", "tb.check_status(); "])
def test_captured_before_anything_else_has_run(first):
    """A layer of torch functions as the first call of a process, inside a capture; and as the first after the library's
    own initialisation."""
    code = f"""
import torch
import tilelang_b200 as tb
from tilelang_b200 import moe
{first}
mlp = moe.ExpertMLP(lambda rows, counts: rows, lambda rows, counts: rows, lambda h: h)
x, logits = torch.randn(24, 16, device="cuda"), torch.randn(24, 4, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = moe.moe_forward(x, logits, 2, 4, mlp)
for _ in range(2):
    x.copy_(torch.randn(24, 16, device="cuda"))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, moe.moe_forward(x, logits, 2, 4, mlp))
print("CAPTURED")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=root), cwd=root, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "CAPTURED" in r.stdout, r.stdout[-2000:] + r.stderr[-3000:]
