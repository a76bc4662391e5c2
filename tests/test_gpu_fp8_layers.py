"""GPU: layers in 8-bit floating point -- the linear layer, the expert MLP and the mixture-of-experts layer -- put
together from the operators, forward and backward, and refusals that need a device.

The layer has to be, bit for bit, the composition of the operators (each held to 64 bits in its own tests).
Against the unquantised layer in 64 bits: rounding to e4m3 moves a value by at most 2^-4, uniformly over a step
that is 2^-3 to 2^-4 of it, in the root mean square by at most 2^-4 / sqrt(3) = 0.036. Errors of n independent
roundings add up to sqrt(n) times that: forward 5 of them (x, w1, the gated value and w2; the gate counts twice)
0.081, backward 8 (those that reach the gate's slopes and four more) 0.102; 0.12 and 0.15 are asserted."""
import pytest
import torch

import tilelang_b200 as tb
from tilelang_b200 import moe, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=gen(seed)) * scale).to(dtype)


def far(got, want):
    got, want = got.detach().double(), want.detach().double()
    return float((got - want).norm() / want.norm())


def grid(*shape, seed, most):
    """Integers up to ``most`` with 448 in front of every 128 columns: up to 16 the quantiser takes them as they are."""
    v = torch.randint(-most, most + 1, shape, device=DEV, generator=gen(seed)).float()
    v[:, ::128] = 448.0
    return v


@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (20, 300, 200), (200, 128, 384)])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
def test_linear_is_the_composition(M, N, K, kind):
    w = randn(N, K, seed=1, scale=0.05)
    layer = tb.Fp8Linear.from_float(w, bias=randn(N, seed=2, dtype=kind))
    x = randn(2, M, K, seed=3, dtype=kind).requires_grad_()
    out = layer(x)
    x2 = x.detach().reshape(-1, K)
    want = ops.gemm_fp8(*ops.quant_fp8(x2), layer.weight, out_dtype=kind) + layer.bias
    assert out.shape == (2, M, N) and torch.equal(out.detach(), want.view(2, M, N))
    d = randn(2, M, N, seed=4, dtype=kind)
    d_x, = torch.autograd.grad(out, x, d)
    want = ops.gemm_fp8(*ops.quant_fp8(d.view(-1, N)), layer.weight, trans_w=True, out_dtype=kind)
    assert torch.equal(d_x, want.view(2, M, K))
    with torch.no_grad():
        assert torch.equal(layer(x), out)
    assert far(out.detach() - layer.bias, x2.double().view(2, M, K) @ w.double().t()) <= 0.12
    layer(x).sum().backward()                                        # a gradient of stride zero
    assert torch.equal(x.grad, torch.autograd.grad(layer(x), x, torch.ones_like(d))[0])


def test_linear_gradient_against_differences():
    """On the quantiser's own grid the layer is linear in x: a central difference is exact but for float32 sums."""
    M, N, K = 30, 256, 384
    layer = tb.Fp8Linear.from_float(randn(N, K, seed=1))
    x, v, d = grid(M, K, seed=2, most=8), grid(M, K, seed=3, most=8), grid(M, N, seed=4, most=15)
    v[:, ::128] = 0                                                  # x + v and x - v are integers up to 16: on the grid
    x.requires_grad_()
    d_x, = torch.autograd.grad(layer(x), x, d)
    with torch.no_grad():
        diff = ((layer(x + v) - layer(x - v)) / 2 * d).double().sum()
    one = (d_x.double() * v.double()).sum()
    size = (d_x.double() * v.double()).abs().sum()
    assert abs(one - diff) <= 2.0 ** -12 * size


def test_factory():
    M, N, K = 40, 200, 256
    a, a_scale = ops.quant_fp8(randn(M, K, seed=1), E5M2)
    w = ops.quant_fp8_weight(randn(N, K, seed=2))
    kernel = tb.matmul_fp8_block(M, N, K, "float8_e5m2", "float16", "float32", weight_dtype="float8_e4m3")
    assert torch.equal(kernel(a, a_scale, w.codes, w.scales), ops.gemm_fp8(a, a_scale, w, out_dtype=torch.float16))
    replay, out = kernel.capture(a, a_scale, w.codes, w.scales)
    replay()
    assert torch.equal(out, kernel(a, a_scale, w.codes, w.scales))


# ---- experts -------------------------------------------------------------------------------------

def experts(E, H, F, seed):
    w1, w2 = randn(E, 2 * F, H, seed=seed, scale=H ** -0.5), randn(E, H, F, seed=seed + 1, scale=F ** -0.5)
    return w1, w2, moe.Fp8ExpertMLP(ops.quant_fp8_weight(w1), ops.quant_fp8_weight(w2))


def plain_layer(x, ids, weights, w1, w2):
    """The layer in the inputs' (64-bit) arithmetic, a loop over the slots."""
    out = torch.zeros_like(x)
    for s in range(ids.shape[1]):
        kept = (ids[:, s] >= 0) & (ids[:, s] < w1.shape[0])
        e = ids[:, s].clamp(0, w1.shape[0] - 1)
        g, u = torch.einsum("th,tfh->tf", x, w1[e]).chunk(2, -1)
        y = torch.einsum("tf,thf->th", torch.sigmoid(g) * g * u, w2[e])
        out = out + torch.where(kept.unsqueeze(1), weights[:, s:s + 1] * y, 0.0)
    return out


SIZES = [(1, 4, 2, 128, 128), (5, 8, 3, 200, 80), (70, 3, 2, 256, 128), (900, 2, 2, 256, 256), (300, 64, 6, 128, 128)]


@pytest.mark.parametrize("T,E,k,H,F", SIZES)
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dropped", [False, True])
def test_layer_is_the_composition(T, E, k, H, F, kind, dropped):
    w1, w2, mlp = experts(E, H, F, T)
    x = randn(T, H, seed=1, dtype=kind).requires_grad_()
    ids = torch.rand(T, E, device=DEV, generator=gen(2)).topk(k).indices
    if dropped:
        ids[torch.rand(T, k, device=DEV, generator=gen(3)) < 0.3] = -1
        ids[0] = E + 5
    weights = torch.rand(T, k, device=DEV, generator=gen(4)).requires_grad_()
    d = randn(T, H, seed=5, dtype=kind)
    out = mlp.layer(x, ids, weights, E)
    d_x, d_w = torch.autograd.grad(out, (x, weights), d)
    tb.check_status()
    with torch.no_grad():
        assert torch.equal(mlp.layer(x, ids, weights, E), out)       # quantised on its way through the dispatch
        codes, scales, plan = moe.dispatch_fp8(x, ids, E)
        act, act_scales, h = ops.gemm_fp8_gated(codes, scales, mlp.w1, plan.counts, keep_h=True)
        y = ops.gemm_fp8_grouped(act, act_scales, mlp.w2, plan.counts, out_dtype=kind)
        assert torch.equal(moe.combine(y, plan, weights), out)
        kept = plan.row_of >= 0
        rows = plan.row_of[kept]
        d_y = torch.zeros(T * k, H, dtype=kind, device=DEV)
        d_y[rows] = (weights.unsqueeze(-1) * d.unsqueeze(1).float()).to(kind)[kept]
        d_act = ops.gemm_fp8_grouped(*ops.quant_fp8(d_y), mlp.w2, plan.counts, trans_w=True)
        d_h = ops.silu_mul_backward_quant_fp8(h, d_act)
        d_rows = ops.gemm_fp8_grouped(*d_h, mlp.w1, plan.counts, trans_w=True, out_dtype=kind)
        want = torch.where(kept.unsqueeze(-1), d_rows[plan.row_of.clamp(min=0)].float(), 0.0)
        half = torch.finfo(kind).eps / 2
        assert ((d_x.float() - want.sum(1)).abs() <= want.abs().sum(1) * (k * 2.0 ** -23) + want.sum(1).abs() * half + 2.0 ** -25).all()
        assert (d_w[~kept] == 0).all()
    if int(kept.sum()) * H < 2000:
        return                                                       # too few values for a root mean square
    leaves = x.detach().double().requires_grad_(), weights.detach().double().requires_grad_()
    ref = plain_layer(leaves[0], ids, leaves[1], w1.double(), w2.double())
    r_x, r_w = torch.autograd.grad(ref, leaves, d.double())
    assert far(out, ref) <= 0.12 and far(d_x, r_x) <= 0.15 and far(d_w, r_w) <= 0.15


def test_layer_behind_the_router():
    T, E, k, H, F = 200, 8, 2, 256, 128
    w1, w2, mlp = experts(E, H, F, 1)
    x = randn(T, H, seed=2, dtype=torch.bfloat16).requires_grad_()
    logits = randn(T, E, seed=3).requires_grad_()
    d = randn(T, H, seed=4, dtype=torch.bfloat16)
    out = moe.moe_forward(x, logits, k, E, mlp)
    d_x, d_l = torch.autograd.grad(out, (x, logits), d)
    with torch.no_grad():
        assert torch.equal(moe.moe_forward(x, logits, k, E, mlp), out)
    lx, ll = x.detach().double().requires_grad_(), logits.detach().double().requires_grad_()
    weights, ids = torch.topk(torch.softmax(ll, -1), k, -1)
    r_x, r_l = torch.autograd.grad(plain_layer(lx, ids, weights, w1.double(), w2.double()), (lx, ll), d.double())
    assert far(d_x, r_x) <= 0.15 and far(d_l, r_l) <= 0.15


def test_rows_behind_the_last_expert_have_no_gradient():
    _, _, mlp = experts(3, 128, 128, 1)
    x = randn(50, 128, seed=2, dtype=torch.bfloat16).requires_grad_()
    counts = torch.tensor([10, 0, 25], device=DEV)
    y = mlp(x, counts)
    d = torch.zeros_like(y)
    d[:35] = 1
    d_x, = torch.autograd.grad(y, x, d)
    assert (d_x[35:] == 0).all() and (d_x[:35] != 0).any(1).all()
    assert torch.equal(mlp(x.detach(), [10, 0, 25])[:35], y[:35])


def test_other_layers_keep_their_results():
    """The 4-bit layer through the new exchange is bit-equal to the rows gathered and combined by torch's order."""
    E, k, T, H, F, group = 8, 2, 96, 256, 128, 128
    g = gen(1)

    def pack(n, kk):
        return ops.stack_packed([ops.pack_w4a16(
            torch.randint(0, 256, (n, kk // 2), device=DEV, generator=g, dtype=torch.uint8),
            (torch.rand(n, kk // group, device=DEV, generator=g) * 0.015 + 0.005).to(torch.bfloat16), None, n, kk, group,
            torch.bfloat16) for _ in range(E)])

    mlp = moe.make_gpu_expert_mlp(pack(2 * F, H), pack(H, F), token_tile=32)
    x, logits = randn(T, H, seed=2, dtype=torch.bfloat16), randn(T, E, seed=3)
    weights, ids = moe.route(logits, k)
    order, token_of_row, counts = moe.sort_by_expert(ids, E)
    want = mlp.combine(mlp(x.index_select(0, token_of_row), counts), moe.rows_of_tokens(order, k), weights.contiguous())
    assert torch.equal(moe.moe_forward(x, logits, k, E, mlp), want)
    one = x[:1].expand(T, H)                                         # rows that overlap take the old way
    assert torch.equal(moe.moe_forward(one, logits, k, E, mlp), moe.moe_forward(one.contiguous(), logits, k, E, mlp))


def test_other_layers_with_a_router_wider_than_the_experts():
    """Tokens whose experts all exist come out as ever; their neighbours' row indices stay inside the rows."""
    E, k, T, H = 4, 2, 64, 128
    x, logits = randn(T, H, seed=2, dtype=torch.bfloat16), randn(T, 2 * E, seed=3)
    scale = torch.arange(1, E + 1, device=DEV, dtype=torch.bfloat16)
    seen = []

    def gemm(rows, counts):
        which = torch.repeat_interleave(torch.arange(E, device=DEV), counts)
        return rows * torch.cat((scale[which], scale.new_ones(rows.shape[0] - which.numel()))).unsqueeze(-1)

    def combine(y, row_of, weights):
        seen.append(((row_of >= 0) & (row_of < y.shape[0])).all())
        return ops.moe_combine(y, row_of.clamp(0, y.shape[0] - 1), weights)

    mlp = moe.ExpertMLP(gemm, lambda rows, counts: rows, lambda h: h, combine)
    out = moe.moe_forward(x, logits, k, E, mlp)
    assert len(seen) == 1 and seen[0]
    weights, ids = moe.route(logits, k)
    whole = (ids < E).all(1)
    assert 0 < int(whole.sum()) < T
    rows = x.unsqueeze(1) * scale[ids.clamp(max=E - 1)].unsqueeze(-1)            # rounded as the products round
    want = (rows.double() * weights.double().unsqueeze(-1)).sum(1)
    # one rounding of the sum, terms of one sign: 2^-8, and two fp32 ones
    assert torch.allclose(out[whole].double(), want[whole], rtol=2 ** -8 + 2 ** -20, atol=0)


def test_other_layers_can_be_differentiated_twice():
    """An expert MLP of torch functions on the GPU: gradients of gradients, as before."""
    E, k, T, H = 4, 2, 24, 16
    x, logits = randn(T, H, seed=2).requires_grad_(), randn(T, E, seed=3)
    mlp = moe.ExpertMLP(lambda rows, counts: rows ** 3, lambda rows, counts: rows, lambda h: h)
    d_x, = torch.autograd.grad(moe.moe_forward(x, logits, k, E, mlp).sum(), x, create_graph=True)
    dd_x, = torch.autograd.grad(d_x.sum(), x)
    weights, _ = moe.route(logits, k)
    want = 6 * x.detach().double() * weights.double().sum(1, keepdim=True)
    # a handful of roundings of 2^-24 each
    assert torch.allclose(dd_x.double(), want, rtol=2 ** -20, atol=0)


def test_layer_in_graphs_and_on_another_stream():
    T, E, k, H, F = 300, 8, 3, 256, 128
    _, _, mlp = experts(E, H, F, 1)
    x, d = randn(T, H, seed=2, dtype=torch.bfloat16), randn(T, H, seed=3, dtype=torch.bfloat16)
    ids = torch.randint(0, E, (T, k), device=DEV, generator=gen(4))
    weights = torch.rand(T, k, device=DEV, generator=gen(5))

    def train():
        leaves = x.detach().requires_grad_(), weights.detach().requires_grad_()
        out = mlp.layer(leaves[0], ids, leaves[1], E)
        return (out.detach(), *torch.autograd.grad(out, leaves, d))

    def serve():
        with torch.no_grad():
            return (mlp.layer(x, ids, weights, E),)

    for step in (serve, train):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = step()
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(first, step()):
            assert torch.equal(a, b)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                graphs.append((graph, step()))
        x.copy_(randn(T, H, seed=9, dtype=torch.bfloat16))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for _ in range(5):
            for (graph, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, got in graphs:
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    tb.check_status()


# ---- refusals ------------------------------------------------------------------------------------

def refused(error, f, *args, **kwargs):
    with pytest.raises(error):
        f(*args, **kwargs)


def test_refusals_of_the_operators():
    x = randn(8, 256, dtype=torch.bfloat16)
    a, s = ops.quant_fp8(x)
    w = ops.quant_fp8_weight(randn(256, 256))
    refused(TypeError, ops.quant_fp8, x, torch.float16)
    refused(TypeError, ops.quant_fp8, x.double())
    refused(ValueError, ops.quant_fp8, x[0])
    refused(ValueError, ops.quant_fp8, x.t())
    refused(ValueError, ops.quant_fp8, x[:1].expand(8, 256))
    refused(ValueError, ops.silu_mul_quant_fp8, x[:, :255])
    refused(ValueError, ops.silu_mul_backward_quant_fp8, x, x)
    refused(ValueError, ops.quant_fp8_weight, x.t())
    refused(TypeError, ops.gemm_fp8, x, s, w)
    refused(ValueError, ops.gemm_fp8, a, s[:, :1], w)
    refused(ValueError, ops.gemm_fp8, a, s.half(), w)
    refused(ValueError, ops.gemm_fp8, a[:, :128], s[:, :1], w)
    refused(ValueError, ops.gemm_fp8, a[:, 8:], s, ops.Fp8Weight(w.codes[:, 8:], w.scales))    # not on 16 bytes
    refused(ValueError, ops.gemm_fp8, a, s, ops.Fp8Weight(w.codes, w.scales[:1]))
    refused(ValueError, ops.gemm_fp8, a, s, ops.Fp8Weight(w.codes.unsqueeze(0), w.scales.unsqueeze(0)))
    refused(TypeError, ops.gemm_fp8, a, s, w, out_dtype=torch.int32)
    refused(ValueError, ops.gemm_fp8, a, s, w, out=torch.empty(8, 255, device=DEV))
    refused(ValueError, ops.gemm_fp8, a, s, w, out=torch.empty(256, 8, device=DEV).t())
    refused(RuntimeError, ops.gemm_fp8, a, s, w, token_tile=48)
    refused(RuntimeError, ops.gemm_fp8, a, s, w, split=9)
    g = ops.Fp8Weight(w.codes.unsqueeze(0), w.scales.unsqueeze(0))
    refused(ValueError, ops.gemm_fp8_grouped, a, s, w, [8])
    refused(ValueError, ops.gemm_fp8_grouped, a, s, g, [4, 4])
    refused(ValueError, ops.gemm_fp8_grouped, a, s, g, [9])
    refused(ValueError, ops.gemm_fp8_grouped, a, s, g, [-1])
    refused(ValueError, ops.gemm_fp8_grouped, a, s, g, torch.tensor([8.0], device=DEV))
    refused(ValueError, ops.gemm_fp8_grouped, a, s, g, torch.tensor([8]))
    refused(ValueError, ops.gemm_fp8_gated, a, s, ops.Fp8Weight(w.codes[:129], w.scales))


def test_refusals_of_the_exchange_and_the_layers():
    x = randn(8, 128, dtype=torch.bfloat16)
    ids = torch.zeros(8, 2, dtype=torch.int64, device=DEV)
    refused(TypeError, moe.dispatch, x, ids.float(), 4)
    refused(ValueError, moe.dispatch, x, ids.cpu(), 4)
    refused(ValueError, moe.dispatch, x, ids[:7], 4)
    refused(ValueError, moe.dispatch, x, ids[:, :0], 4)
    refused(ValueError, moe.dispatch, x, ids, 0)
    refused(ValueError, moe.dispatch, x, ids, 1025)
    refused(TypeError, moe.dispatch, x.double(), ids, 4)
    refused(TypeError, moe.dispatch_fp8, x, ids, 4, torch.int8)
    rows, plan = moe.dispatch(x, ids, 4)
    refused(ValueError, moe.combine, rows[:15], plan, torch.ones(8, 2, device=DEV))
    refused(ValueError, moe.combine, rows, plan, torch.ones(8, 3, device=DEV))
    refused(ValueError, moe.combine, rows, plan, torch.ones(8, 2, dtype=torch.int64, device=DEV))
    refused(ValueError, moe.combine, rows.t(), plan, torch.ones(8, 2, device=DEV))
    _, _, mlp = experts(4, 128, 128, 1)
    refused(ValueError, moe.Fp8ExpertMLP, mlp.w2, mlp.w1)
    refused(ValueError, mlp.layer, x, ids, torch.ones(8, 2, device=DEV), 5)
    refused(ValueError, mlp.layer, x.float(), ids, torch.ones(8, 2, device=DEV), 4)
    refused(ValueError, mlp, x[:, :64], [8, 0, 0, 0])
    refused(ValueError, tb.Fp8Linear, mlp.w1)
    refused(ValueError, tb.Fp8Linear.from_float(randn(64, 128)), x[:, :64])
