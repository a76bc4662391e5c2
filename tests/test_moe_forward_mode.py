"""The 8-bit expert layer and the exchange have reverse-mode gradients only: forward-mode differentiation and functorch
transforms are refused, not answered with a tangent left out."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from tilelang_b200 import moe, ops

DEV = "cuda"
REFUSED = (NotImplementedError, RuntimeError)


def test_across_ranks():
    w1 = ops.Fp8Weight(torch.zeros(2, 256, 128).to(torch.float8_e4m3fn), torch.ones(2, 2, 1))
    w2 = ops.Fp8Weight(torch.zeros(2, 128, 128).to(torch.float8_e4m3fn), torch.ones(2, 1, 1))
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    with fwd.dual_level(), pytest.raises(ValueError, match="no gradient of the tokens"):
        moe.moe_forward_ep(fwd.make_dual(x, x), torch.zeros(4, 2), 1, 2, moe.Fp8ExpertMLP(w1, w2))


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_tangents(grad):
    T, E, k, H, F = 12, 4, 2, 128, 128
    x, weights = torch.randn(T, H, device=DEV).to(torch.bfloat16), torch.rand(T, k, device=DEV)
    ids = torch.randint(0, E, (T, k), device=DEV)
    mlp = moe.Fp8ExpertMLP(ops.quant_fp8_weight(torch.randn(E, 2 * F, H, device=DEV)), ops.quant_fp8_weight(torch.randn(E, H, F, device=DEV)))
    rows, plan = moe.dispatch(x, ids, E)
    calls = [(x, lambda t: moe.dispatch(t, ids, E)[0]), (rows, lambda t: moe.combine(t, plan, weights)),
             (weights, lambda t: moe.combine(rows, plan, t)), (weights, lambda t: moe.combine_rows(rows, plan.row_of, t)),
             (rows, lambda t: mlp(t, plan.counts)), (x, lambda t: mlp.layer(t, ids, weights, E)),
             (weights, lambda t: mlp.layer(x, ids, t, E))]
    with torch.set_grad_enabled(grad):
        for t, f in calls:
            with fwd.dual_level():
                f(t)                                                 # no tangent: an ordinary call
                with pytest.raises(REFUSED):
                    f(fwd.make_dual(t, torch.ones_like(t)))
            with pytest.raises(REFUSED):
                torch.func.jvp(f, (t,), (torch.ones_like(t),))
            with pytest.raises(REFUSED):
                torch.func.vmap(f)(torch.stack((t, t)))
    torch.cuda.synchronize()
