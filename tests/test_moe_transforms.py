"""The mixture-of-experts layer over an expert MLP of torch functions stays a torch function on a GPU: forward-mode
derivatives, vmap, gradients by torch.func, traces and compilation see all of it, not the values alone.

The MLP is x ** 3, so out = sum_s w_s x^3 with weights of one sign: a value and a derivative are off by a handful of
float32 roundings, 2^-20 of their size."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.utils._python_dispatch import TorchDispatchMode

from tilelang_b200 import moe, ops

DEV = "cuda"
E, K, T, H = 4, 2, 24, 16


def layer(x, logits):
    mlp = moe.ExpertMLP(lambda rows, counts: rows ** 3, lambda rows, counts: rows, lambda h: h)
    return moe.moe_forward(x, logits, K, E, mlp)


def inputs():
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    return [torch.randn(*shape, device=DEV, generator=g) for shape in ((T, H), (T, E), (T, H))]


def near(got, want):
    return torch.allclose(got.double(), want, rtol=2 ** -20, atol=0)


def plain(x, logits):
    weights, _ = moe.route(logits, K)
    return x.double() ** 3 * weights.double().sum(1, keepdim=True)


def slope(x, logits, v):
    weights, _ = moe.route(logits, K)
    return 3 * x.double() ** 2 * v.double() * weights.double().sum(1, keepdim=True)


def test_what_an_ordinary_call_is():
    x, p = torch.ones(3), torch.nn.Parameter(torch.ones(3))
    assert ops._ordinary(x, p)
    with torch.no_grad(), torch.device("cpu"):
        assert ops._ordinary(x)
    with fwd.dual_level():
        assert ops._ordinary(x) and not ops._ordinary(x, fwd.make_dual(x, x))
    seen = []
    look = lambda y: (seen.append(ops._ordinary(x)), y * 1)[1]                   # noqa: E731
    torch.func.jvp(look, (x,), (x,))
    torch.func.vmap(look)(x)
    torch.func.grad(lambda y: look(y).sum())(x)
    torch.jit.trace(look, (x,), check_trace=False)
    torch.compile(look, backend="eager")(x)

    class Looker(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Looker():
        look(x)
    assert len(seen) >= 6 and not any(seen)

    class Named(torch.Tensor):
        pass
    assert not ops._ordinary(x.as_subclass(Named))


@pytest.mark.gpu
def test_forward_mode():
    x, logits, v = inputs()
    with fwd.dual_level():
        out = fwd.unpack_dual(layer(fwd.make_dual(x, v), logits))
        assert near(out.primal, plain(x, logits)) and out.tangent is not None and near(out.tangent, slope(x, logits, v))
        w_only = fwd.unpack_dual(layer(x, fwd.make_dual(logits, torch.ones_like(logits)))).tangent
        assert w_only is not None and w_only.shape == x.shape
    out, tangent = torch.func.jvp(lambda x: layer(x, logits), (x,), (v,))
    assert near(out, plain(x, logits)) and near(tangent, slope(x, logits, v))


@pytest.mark.gpu
def test_batched():
    x, logits, v = inputs()
    out = torch.func.vmap(lambda x: layer(x, logits))(torch.stack((x, v)))
    assert near(out[0], plain(x, logits)) and near(out[1], plain(v, logits))
    out = torch.func.vmap(lambda l: layer(x, l))(torch.stack((logits, 2 * logits)))
    assert near(out[0], plain(x, logits)) and near(out[1], plain(x, 2 * logits))


@pytest.mark.gpu
def test_gradient_of_the_router():
    x, logits, _ = inputs()
    got = torch.func.grad(lambda l: layer(x, l).sum())(logits)
    leaf = logits.double().requires_grad_()
    weights, _ = torch.topk(torch.softmax(leaf, -1), K, -1, sorted=False)
    want, = torch.autograd.grad((x.double() ** 3 * weights.sum(1, keepdim=True)).sum(), leaf)
    # sums of H terms, then differences of products with weights below one: some 2 H roundings of the terms
    assert ((got.double() - want).abs() <= 2 * H * 2.0 ** -24 * 4 * (x.double().abs() ** 3).sum(1, keepdim=True)).all()


@pytest.mark.gpu
def test_recorded():
    x, logits, v = inputs()
    from torch.fx.experimental.proxy_tensor import make_fx
    f = lambda x: layer(x, logits)                                               # noqa: E731
    for recorded in (torch.jit.trace(f, (x,), check_trace=False), make_fx(f)(x), torch.compile(f, backend="eager", fullgraph=True)):
        assert near(recorded(x), plain(x, logits)) and near(recorded(v), plain(v, logits))
