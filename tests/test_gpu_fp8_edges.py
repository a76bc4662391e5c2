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


# ---- many groups, skewed groups ------------------------------------------------------------------

def check_grouped(out, a, a_scale, w, counts, trans):
    """Rows against the definition in 64 bits. Bound: within a block of 128 at most 4 * 33 terms cut off at 2^-24 of the
    largest, < 2^-16.9 of the sum of magnitudes; a rounding of 2^-24 per block and 11 more (scales, fma, join)."""
    codes, scales = a.double(), a_scale.double()
    av = codes * scales[:, torch.arange(a.shape[1], device=DEV) // 128]
    blocks = -(-a.shape[1] // 128)
    at = 0
    for e, c in enumerate(counts):
        if c == 0:
            continue
        wv = w.codes[e].double() * w.scales[e].double()[torch.arange(w.N, device=DEV) // 128][:, torch.arange(w.K, device=DEV) // 128]
        wv = wv if trans else wv.t()
        rows = av[at:at + c]
        size = rows.abs() @ wv.abs()
        assert ((out[at:at + c].double() - rows @ wv).abs() <= size * (2.0 ** -16.9 + (blocks + 11) * 2.0 ** -24)).all(), e
        at += c
    return at


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("counts,tile", [
    ([140 + 7 * (i % 5) for i in range(300)], 0),        # more groups than CTA pairs take, a tile and more each
    ([129] * 257, 0), ([200] * 256, 0),                  # either side of that limit
    ([5000] + [1] * 511, 0), ([1] * 511 + [5000], 0),    # a mean share of 11 rows, and one group of 313 tiles of 16
    ([0] * 400 + [3000] + [0] * 624, 16), ([700, 0, 1] * 100, 32),
])
def test_many_and_skewed_groups(counts, tile, trans):
    N, K, G = 144, 272, len(counts)
    rows = sum(counts) + 13
    a, a_scale = ops.quant_fp8(randn(rows, N if trans else K, seed=G))
    w = ops.quant_fp8_weight(randn(G, N, K, seed=G + 1, scale=0.05))
    out = torch.full((rows, K if trans else N), 7.0, device=DEV)
    ops.gemm_fp8_grouped(a, a_scale, w, torch.tensor(counts, device=DEV), trans_w=trans, out=out, token_tile=tile)
    tb.check_status()
    at = check_grouped(out, a, a_scale, w, counts, trans)
    assert at == rows - 13 and (out[at:] == 7.0).all()


@pytest.mark.parametrize("G,each", [(256, 200), (257, 200), (300, 140)])
def test_gated_products_either_side_of_256_groups(G, each):
    """Fused up to 256 groups, a product in float32 and a quantiser above. The codes stand for the activation to half a
    step (2^-4, 2^-10 of the scale for the smallest) and what the product's bound, 2^-16.5 of the sum of magnitudes, moves
    it by (|silu'| <= 1.1)."""
    F, K = 128, 256
    a, a_scale = ops.quant_fp8(randn(G * each, K, seed=1))
    w = ops.quant_fp8_weight(randn(G, 2 * F, K, seed=2, scale=0.05))
    counts = torch.full((G,), each, device=DEV)
    codes, scales = ops.gemm_fp8_gated(a, a_scale, w, counts)
    tb.check_status()
    if G > 256:
        want = ops.silu_mul_quant_fp8(ops.gemm_fp8_grouped(a, a_scale, w, counts, out_dtype=torch.float32))
        assert torch.equal(codes.float(), want[0].float()) and torch.equal(scales, want[1])
    av = (a.double() * a_scale.double()[:, torch.arange(K, device=DEV) // 128]).view(G, each, K)
    wv = w.codes.double() * w.scales.double()[:, torch.arange(2 * F, device=DEV) // 128][:, :, torch.arange(K, device=DEV) // 128]
    ref, size = torch.bmm(av, wv.transpose(1, 2)).flatten(0, 1), torch.bmm(av.abs(), wv.abs().transpose(1, 2)).flatten(0, 1) * 2.0 ** -16.5
    (g, u), (dg, du) = ref.split(F, -1), size.split(F, -1)
    v = torch.sigmoid(g) * g * u
    slack = 1.1 * dg * u.abs() + g.abs() * du + 2.0 ** -20 * v.abs()
    s = scales.double()
    off = (codes.double() * s - v).abs()
    assert (off <= (v.abs() + slack) * 2.0 ** -4 + s * 2.0 ** -10 * 1.001 + slack).all()


@pytest.mark.parametrize("dtype,rows", [(torch.float8_e4m3fn, 2000), (torch.float8_e5m2, 2000), (torch.float8_e4m3fn, 40)])
def test_gated_codes_are_the_nearest_but_at_borders(dtype, rows):
    """Fused and not: a code other than that of the 64-bit quotient is its neighbour, and the border between the two is
    no further from the quotient than the product's bound (2^-16.5 of the sum of magnitudes) and 2^-20 of the value allow."""
    F, K = 256, 512
    a, a_scale = ops.quant_fp8(randn(rows, K, seed=1))
    w = ops.quant_fp8_weight(randn(2 * F, K, seed=2, scale=0.05))
    codes, scales = ops.gemm_fp8_gated(a, a_scale, w, dtype=dtype)
    av = a.double() * a_scale.double()[:, torch.arange(K, device=DEV) // 128]
    wv = w.codes.double() * w.scales.double()[torch.arange(2 * F, device=DEV) // 128][:, torch.arange(K, device=DEV) // 128]
    (g, u), (dg, du) = (av @ wv.t()).split(F, -1), ((av.abs() @ wv.abs().t()) * 2.0 ** -16.5).split(F, -1)
    s = scales.double()[:, torch.arange(F, device=DEV) // 128]
    v = torch.sigmoid(g) * g * u
    q, slack = v / s, (1.1 * dg * u.abs() + g.abs() * du + 2.0 ** -20 * v.abs()) / s
    nearest, got = q.to(dtype).double(), codes.double()
    other = got != nearest
    assert other.double().mean() <= 1e-3
    assert ((q - (got + nearest) / 2).abs() <= slack)[other].all()
    step = torch.maximum(nearest.abs(), got.abs()) * (2.0 ** -3 if dtype == torch.float8_e4m3fn else 2.0 ** -2) + 2.0 ** (-9 if dtype == torch.float8_e4m3fn else -16)
    assert ((got - nearest).abs() <= step).all()
    for _ in range(3):
        again = ops.gemm_fp8_gated(a, a_scale, w, dtype=dtype)
        assert torch.equal(again[0].float(), codes.float()) and torch.equal(again[1], scales)


@pytest.mark.parametrize("M,N,K", [(1, 72, 200), (5, 1, 100), (5, 72, 200), (200, 300, 1), (5, 72, 128)])
def test_factory_takes_rows_without_gaps(M, N, K):
    """As tensors come from elsewhere, the profiler's own among them."""
    a, a_scale = ops.quant_fp8(randn(M, K, seed=1))
    w = ops.quant_fp8_weight(randn(N, K, seed=2))
    kernel = tb.matmul_fp8_block(M, N, K, "float8_e4m3", "float32", "float32")
    want = ops.gemm_fp8(a, a_scale, w, out_dtype=torch.float32)
    packed = [t.clone(memory_format=torch.contiguous_format) for t in (a, a_scale, w.codes, w.scales)]
    assert all(t.is_contiguous() for t in packed)
    assert torch.equal(kernel(*packed), want) and torch.equal(kernel(a, a_scale, w.codes, w.scales), want)
    replay, out = kernel.capture(*packed)
    replay()
    assert torch.equal(out, want)
    profiler = kernel.get_profiler()
    profiler.assert_consistent(repeat=3)
    assert profiler.do_bench(n_warmup=1, n_repeat=2) > 0
    tb.check_status()
