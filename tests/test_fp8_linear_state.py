"""``Fp8Linear`` is a module like any other: its weight and bias are saved, loaded and moved with it."""
import copy
import io

import pytest
import torch

import tilelang_b200 as tb
from tilelang_b200 import ops

DEV = "cuda"


def weight(N, K, seed, dtype=torch.float8_e4m3fn):
    """Codes and scales as ``quant_fp8_weight`` lays them out, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.empty(N, (K + 15) // 16 * 16, dtype=dtype)[:, :K]
    codes.copy_(torch.randn(N, K, generator=g).to(dtype))
    return ops.Fp8Weight(codes, torch.rand(-(-N // 128), -(-K // 128), generator=g))


def same(a, b):
    return a.dtype == b.dtype and torch.equal(a.float().cpu(), b.float().cpu())


def through_a_file(state):
    f = io.BytesIO()
    torch.save(state, f)
    f.seek(0)
    return torch.load(f)


@pytest.mark.parametrize("K", [128, 200])
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_state(K, dtype):
    w = weight(150, K, 1, dtype)
    layer = tb.Fp8Linear(w, bias=torch.randn(150))
    assert layer.weight.codes is w.codes and layer.weight.scales is w.scales
    assert set(layer.state_dict()) == {"codes", "scales", "bias"} == dict(layer.named_buffers()).keys()
    for assign in (False, True):
        for packed in (False, True):                                 # as other programs write them: rows without gaps
            other = torch.nn.Sequential(tb.Fp8Linear(weight(150, K, 2, dtype), bias=torch.zeros(150)))
            state = {k: v.clone(memory_format=torch.contiguous_format) if packed else v for k, v in torch.nn.Sequential(layer).state_dict().items()}
            other.load_state_dict(through_a_file(state), assign=assign)
            assert same(other[0].codes, w.codes) and same(other[0].scales, w.scales) and same(other[0].bias, layer.bias)
            assert other[0].codes.stride(0) % 16 == 0


def test_bias():
    layer = tb.Fp8Linear(weight(8, 128, 1))
    assert layer.bias is None and set(layer.state_dict()) == {"codes", "scales"}
    bias = torch.nn.Parameter(torch.zeros(8))
    layer = tb.Fp8Linear(weight(8, 128, 1), bias)
    assert layer.bias is bias and [p for p in layer.parameters()] == [bias] and "bias" in layer.state_dict()
    leaf = torch.zeros(8, requires_grad=True)
    assert tb.Fp8Linear(weight(8, 128, 1), leaf).bias is leaf


def test_another_weight():
    layer, w = tb.Fp8Linear(weight(8, 128, 1)), weight(8, 128, 2)
    layer.weight = w
    assert layer.codes is w.codes and layer.state_dict()["scales"].equal(w.scales)
    with pytest.raises(ValueError):
        layer.weight = weight(9, 128, 2)


@pytest.mark.parametrize("K", [128, 200])
def test_moved_and_copied(K):
    w = weight(150, K, 1)
    layer = tb.Fp8Linear(w, bias=torch.randn(150))
    for change in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.float(), copy.deepcopy,
                   lambda m: m.to("cpu", torch.float16), lambda m: through_a_module_file(m)):
        moved = change(copy.deepcopy(layer))
        assert same(moved.codes, w.codes) and same(moved.scales, w.scales) and moved.codes.stride(0) % 16 == 0
    assert layer.half().bias.dtype == torch.float16
    empty = copy.deepcopy(layer).to("meta").to_empty(device="cpu")
    assert empty.codes.dtype == w.codes.dtype and empty.codes.shape == w.codes.shape and empty.codes.stride(0) % 16 == 0


def through_a_module_file(module):
    f = io.BytesIO()
    torch.save(module, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [128, 200])
def test_results_survive(K):
    w = torch.randn(150, K, device=DEV)
    layer = tb.Fp8Linear.from_float(w, bias=torch.randn(150, device=DEV))
    x = torch.randn(5, K, device=DEV).to(torch.bfloat16)
    want = layer(x)
    assert torch.equal(copy.deepcopy(layer).cpu().cuda()(x), want)
    assert torch.equal(copy.deepcopy(layer).bfloat16()(x), want)     # the bias is rounded to the output's type anyway
    for assign in (False, True):
        other = tb.Fp8Linear.from_float(torch.zeros_like(w), bias=torch.zeros(150, device=DEV))
        other.load_state_dict({k: v.cpu() if not assign else v.contiguous() for k, v in layer.state_dict().items()}, assign=assign)
        assert torch.equal(other(x), want)
