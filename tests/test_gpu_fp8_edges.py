"""GPU: 8-bit floating point products, layers and quantisers at the edges of what they take: no rows, a single row
of any stride, many groups, skewed groups."""
import pytest
import torch

import tilelang_b200 as tb
from tilelang_b200 import moe, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("inner", [100, 128, 200])
def test_no_rows_whatever_the_contraction(inner):
    a, s = ops.quant_fp8(torch.empty(0, inner, device=DEV))
    w, g = ops.quant_fp8_weight(randn(72, inner)), ops.quant_fp8_weight(randn(2, 256, inner))
    assert ops.gemm_fp8(a, s, w).shape == (0, 72)
    assert ops.gemm_fp8(a, s, ops.quant_fp8_weight(randn(inner, 72)), trans_w=True).shape == (0, 72)
    for counts in ([0, 0], torch.zeros(2, dtype=torch.int64, device=DEV)):
        assert ops.gemm_fp8_grouped(a, s, g, counts).shape == (0, 256)
        codes, scales, h = ops.gemm_fp8_gated(a, s, g, counts, keep_h=True)
        assert codes.shape == (0, 128) and scales.shape == (0, 1) and h.shape == (0, 256)
    grouped = ops.quant_fp8_weight(randn(2, inner, 72))
    assert ops.gemm_fp8_grouped(a, s, grouped, [0, 0], trans_w=True).shape == (0, 72)
    tb.check_status()


@pytest.mark.parametrize("H,F", [(100, 72), (128, 128), (200, 80)])
def test_layers_without_tokens(H, F):
    linear = tb.Fp8Linear.from_float(randn(F, H), bias=randn(F))
    for lead in ((0,), (3, 0)):
        x = torch.empty(*lead, H, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        out = linear(x)
        assert out.shape == (*lead, F)
        assert torch.autograd.grad(out.sum(), x)[0].shape == x.shape
    mlp = moe.Fp8ExpertMLP(ops.quant_fp8_weight(randn(3, 2 * F, H)), ops.quant_fp8_weight(randn(3, H, F)))
    x = torch.empty(0, H, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    weights = torch.empty(0, 2, device=DEV, requires_grad=True)
    ids = torch.empty(0, 2, dtype=torch.int64, device=DEV)
    out = mlp.layer(x, ids, weights, 3)
    d_x, d_w = torch.autograd.grad(out.sum(), (x, weights))
    assert out.shape == (0, H) and d_x.shape == (0, H) and d_w.shape == (0, 2)
    assert torch.autograd.grad(mlp(x, [0, 0, 0]).sum(), x)[0].shape == (0, H)
    with torch.no_grad():
        assert mlp.layer(x, ids, weights, 3).shape == (0, H)
        assert mlp(x, torch.zeros(3, dtype=torch.int64, device=DEV)).shape == (0, H)
        assert moe.moe_forward(x, torch.empty(0, 3, device=DEV), 2, 3, mlp).shape == (0, H)
    tb.check_status()


def test_linear_of_one_strided_row():
    """One token is taken in every layout that two are taken in."""
    K, N = 200, 72
    layer = tb.Fp8Linear.from_float(randn(N, K, seed=1))
    base = randn(K, 5, seed=2, dtype=torch.bfloat16)
    vector = randn(2 * K, seed=3, dtype=torch.bfloat16)
    for x in (base.t()[:1], base.t()[2:3], base[:, 0], vector[::2], vector[::2].unsqueeze(0), base.t(), vector[:K].expand(3, K),
              vector[:1].expand(K), vector[1:K + 1]):
        want = layer(x.contiguous())
        assert torch.equal(layer(x), want)
        leaf = x.detach().requires_grad_()
        d = randn(*want.shape[:-1], 2 * N, seed=4, dtype=torch.bfloat16)[..., ::2]
        got, = torch.autograd.grad(layer(leaf), leaf, d)
        other = x.detach().contiguous().requires_grad_()
        assert torch.equal(got, torch.autograd.grad(layer(other), other, d.contiguous())[0])
    assert torch.equal(tb.Fp8Linear.from_float(randn(N, 1, seed=5))(base[:, :1]), tb.Fp8Linear.from_float(randn(N, 1, seed=5))(base[:, :1].contiguous()))
