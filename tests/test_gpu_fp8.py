"""GPU: products of 8-bit floats with a scale for each block of 128, and their quantisers, against the
definition in 64 bits.

Tolerances. Quantiser: a code is off by at most half a step, 2^-4 (e4m3) or 2^-3 (e5m2) of the value and half
the smallest subnormal (2^-10, 2^-17 of the scale) below the normal range, plus the float32 roundings in front of it
(at most 8 of 2^-24 for the silu forms; 2^-20 covers them). A scale carries the two roundings of the
product with 1/448 and those of the value it is the maximum of. Product: within a block of 128 the tensor core adds
four times 32 exact products to an accumulator, each term cut off at 2^-24 of the largest or better: at
most 4 * 33 * 2^-24 < 2^-16.9 of the sum of magnitudes S; the scales' product, the fma and the join of at
most 8 parts add a rounding of 2^-24 per block and part. The output's own rounding is half a step."""
import pytest
import torch

import tilelang_b200 as tb
from tilelang_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
LARGEST = {E4M3: 448.0, E5M2: 57344.0}
HALF_STEP = {E4M3: 2.0 ** -4, E5M2: 2.0 ** -3}
HALF_SUBNORMAL = {E4M3: 2.0 ** -10, E5M2: 2.0 ** -17}


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=gen(seed)) * scale).to(dtype)


def spread(codes, scales, rows=1):
    """Values in 64 bits, one scale per ``rows`` x 128."""
    n, k = codes.shape
    i, j = torch.arange(n, device=DEV) // rows, torch.arange(k, device=DEV) // 128
    return codes.double() * scales.double()[i][:, j]


def block_max(v):
    return torch.cat([b.abs().amax(-1, keepdim=True) for b in v.double().split(128, -1)], -1)


def check_quantised(codes, scales, v, dtype):
    """``codes`` and ``scales`` against the exact values ``v`` (64 bits)."""
    assert codes.shape == v.shape and codes.dtype == dtype and scales.dtype == torch.float32
    want = (block_max(v) / LARGEST[dtype]).clamp(min=2.0 ** -126)
    assert ((scales.double() - want).abs() <= want * 2.0 ** -20).all()
    s = scales.double()[:, torch.arange(v.shape[1], device=DEV) // 128]
    off = (codes.double() * s - v.double()).abs()
    assert (off <= v.double().abs() * (HALF_STEP[dtype] + 2.0 ** -20) + s * HALF_SUBNORMAL[dtype] * (1 + 2.0 ** -20)).all()


def check_product(c, a, a_scale, w, w_scale, trans=False):
    av, wv = spread(a, a_scale), spread(w, w_scale, 128)
    wv = wv if trans else wv.t()
    ref, size = av @ wv, av.abs() @ wv.abs()
    blocks = -(-av.shape[1] // 128)
    bound = size * (2.0 ** -16.9 + (blocks + 11) * 2.0 ** -24)
    if c.dtype != torch.float32:
        bound = bound + ref.abs() * torch.finfo(c.dtype).eps / 2 + 2.0 ** -25 * (c.dtype == torch.float16)
    assert c.shape == ref.shape
    worst = ((c.double() - ref).abs() - bound).max().item()
    assert worst <= 0, f"off by {worst:.3g} more than the bound"


# ---- quantisers ----------------------------------------------------------------------------------

@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (5, 129), (7, 16), (2, 144), (33, 1408), (64, 1000), (129, 2048)])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
def test_quantised_rows(M, K, dtype, kind):
    x = randn(M, K, seed=M + K, dtype=kind) * torch.logspace(-3, 2, M, device=DEV).unsqueeze(1).to(kind)
    x[-1, : min(K, 130)] = 0                                       # a block of zeros, or part of one
    codes, scales = ops.quant_fp8(x, dtype)
    check_quantised(codes, scales, x, dtype)
    # the same steps in torch float32 give the same bits
    pad = torch.nn.functional.pad(x.float(), (0, -K % 128)).view(M, -1, 128)
    s = (pad.abs().amax(-1) * (1.0 / LARGEST[dtype])).clamp(min=2.0 ** -126)
    q = (pad * s.reciprocal().unsqueeze(-1)).clamp(-LARGEST[dtype], LARGEST[dtype]).to(dtype).float().flatten(1)[:, :K]
    assert torch.equal(scales, s) and torch.equal(codes.float(), q)


def test_quantised_rows_that_are_views():
    big = randn(40, 700, seed=1, dtype=torch.bfloat16)
    for x in (big[:, 5:261], big[::3, :256], big[3:4, 1:], big[:, 16:272]):
        codes, scales = ops.quant_fp8(x)
        want, s = ops.quant_fp8(x.contiguous())
        assert torch.equal(codes.float(), want.float()) and torch.equal(scales, s)


def test_quantised_rows_with_infinities_and_nan():
    x = randn(4, 256, seed=2)
    x[1, 3], x[2, 200] = float("inf"), float("nan")
    codes, scales = ops.quant_fp8(x)
    assert torch.isinf(scales[1, 0]) and torch.isnan(scales[2, 1])
    fine = torch.isfinite(scales)
    assert fine.sum() == 6
    v = spread(codes, scales)
    assert not torch.isfinite(v[1, :128]).any() and torch.isnan(v[2, 128:]).all()
    assert torch.isfinite(v[[0, 3]]).all() and torch.isfinite(v[1, 128:]).all() and torch.isfinite(v[2, :128]).all()


def test_tiny_and_huge_rows():
    x = torch.tensor([[1e-38] * 128, [2.0 ** -140] * 128, [3e38] * 128, [0.0] * 128], device=DEV)
    codes, scales = ops.quant_fp8(x)
    check_quantised(codes, scales, x, E4M3)
    assert torch.equal(codes[3].float(), torch.zeros(128, device=DEV))


@pytest.mark.parametrize("M,F", [(1, 128), (3, 100), (5, 16), (9, 200), (17, 256), (40, 1408)])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_quantised_gate_and_its_gradient(M, F, kind, dtype):
    h = randn(M, 2 * F, seed=F, dtype=kind, scale=2.0)
    h[0, 0], h[0, F] = -60000.0 if kind == torch.float16 else -1e5, 3.0      # e^60000 is infinite: silu is -0
    d = randn(M, F, seed=F + 1, dtype=kind)
    g, u = h.double().split(F, -1)
    p = torch.sigmoid(g)
    check_quantised(*ops.silu_mul_quant_fp8(h, dtype), p * g * u, dtype)
    dd = d.double()
    check_quantised(*ops.silu_mul_backward_quant_fp8(h, d, dtype),
                    torch.cat((dd * u * p * (1 + g * (1 - p)), dd * g * p), -1), dtype)


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 200), (3, 257, 129)])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_quantised_weight(shape, dtype):
    x = randn(*shape, seed=5, dtype=torch.bfloat16)
    w = ops.quant_fp8_weight(x, dtype)
    assert w.codes.shape == x.shape and w.codes.stride(-2) % 16 == 0 and w.N == shape[-2] and w.K == shape[-1]
    for m, c, s in zip(x.reshape(-1, *shape[-2:]), w.codes.reshape(-1, *shape[-2:]), w.scales.reshape(-1, *w.scales.shape[-2:])):
        for i in range(0, shape[-2], 128):
            v = m[i:i + 128].double()
            want = block_max(v.amax(0, keepdim=True).maximum(-v.amin(0, keepdim=True)))[0] / LARGEST[dtype]
            assert ((s[i // 128].double() - want).abs() <= want * 2.0 ** -22).all()
            sv = s[i // 128].double()[torch.arange(shape[-1], device=DEV) // 128]
            off = (c[i:i + 128].double() * sv - v).abs()
            assert (off <= v.abs() * (HALF_STEP[dtype] + 2.0 ** -20) + sv * HALF_SUBNORMAL[dtype] * 1.001).all()


# ---- products ------------------------------------------------------------------------------------

def operands(M, N, K, seed, a_type=E4M3, w_type=E4M3, trans=False):
    a, a_scale = ops.quant_fp8(randn(M, N if trans else K, seed=seed), a_type)
    w = ops.quant_fp8_weight(randn(N, K, seed=seed + 1, scale=0.02), w_type)
    return a, a_scale, w


SIZES = [(1, 1, 1), (1, 128, 128), (3, 130, 64), (16, 256, 1000), (17, 300, 384), (33, 128, 2048), (64, 1000, 200),
         (65, 129, 512), (128, 256, 256), (200, 384, 1100), (300, 8640, 400)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_product(M, N, K, trans, out_dtype):
    a, a_scale, w = operands(M, N, K, seed=M + N + K, trans=trans)
    c = ops.gemm_fp8(a, a_scale, w, trans_w=trans, out_dtype=out_dtype)
    tb.check_status()
    check_product(c, a, a_scale, w.codes, w.scales, trans)
    assert torch.equal(c, ops.gemm_fp8(a, a_scale, w, trans_w=trans, out_dtype=out_dtype))


@pytest.mark.parametrize("a_type", [E4M3, E5M2])
@pytest.mark.parametrize("w_type", [E4M3, E5M2])
@pytest.mark.parametrize("M,trans", [(5, False), (5, True), (150, False), (150, True)])
def test_product_of_either_type(a_type, w_type, M, trans):
    a, a_scale, w = operands(M, 272, 400, 7, a_type, w_type, trans)
    c = ops.gemm_fp8(a, a_scale, w, trans_w=trans, out_dtype=torch.float32)
    check_product(c, a, a_scale, w.codes, w.scales, trans)


@pytest.mark.parametrize("token_tile", [16, 32, 128])
@pytest.mark.parametrize("split", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("trans", [False, True])
def test_every_tile_and_split(token_tile, split, trans):
    """150 tokens in every tile, contractions of 9 blocks (the last one ragged) cut into every number of parts."""
    M, N, K = (150, 1100, 272) if trans else (150, 272, 1100)
    a, a_scale, w = operands(M, N, K, 11, trans=trans)
    c = ops.gemm_fp8(a, a_scale, w, trans_w=trans, out_dtype=torch.float32, token_tile=token_tile, split=split)
    tb.check_status()
    check_product(c, a, a_scale, w.codes, w.scales, trans)


@pytest.mark.parametrize("M,N,K", [(1, 100, 64), (128, 256, 128), (129, 300, 400), (700, 656, 1100), (2500, 1600, 160)])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_tiles_of_cta_pairs(M, N, K, trans, out_dtype):
    """Pairs with one row, an empty half, several tiles to a pair, more blocks than stages."""
    M, N, K = (M, K, N) if trans and K % 16 == 0 else (M, N, K)
    a, a_scale, w = operands(M, N, K, 13, trans=trans)
    c = ops.gemm_fp8(a, a_scale, w, trans_w=trans, out_dtype=out_dtype, token_tile=256)
    tb.check_status()
    check_product(c, a, a_scale, w.codes, w.scales, trans)
    assert torch.equal(c, ops.gemm_fp8(a, a_scale, w, trans_w=trans, out_dtype=out_dtype, token_tile=256))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_leave_before_an_empty_slab_takes_their_place(out_dtype):
    """Contractions of one block: tiles follow so closely that a warp whose next 32 rows lie behind the last one comes
    to its staging while the rows before are still on their way out."""
    a, a_scale, w = operands(2476, 2936, 52, 3)
    first = ops.gemm_fp8(a, a_scale, w, out_dtype=out_dtype, token_tile=256)
    check_product(first, a, a_scale, w.codes, w.scales)
    for _ in range(30):
        assert torch.equal(first, ops.gemm_fp8(a, a_scale, w, out_dtype=out_dtype, token_tile=256))


@pytest.mark.parametrize("token_tile", [16, 32, 128, 256])
@pytest.mark.parametrize("trans", [False, True])
def test_one_hot_rows_read_the_weight_back(token_tile, trans):
    """A row of one 1 and scales that are powers of two give the weight's values, bit for bit."""
    N, K = 272, 400
    w = ops.quant_fp8_weight(randn(N, K, seed=3))
    w.scales.copy_(torch.exp2(torch.arange(w.scales.numel(), device=DEV).float().view_as(w.scales) - 5))
    inner = N if trans else K
    a = ops._fp8_rows(inner, inner, E4M3, torch.device(DEV, 0))
    a.copy_(torch.eye(inner, device=DEV).to(E4M3))
    scale = torch.exp2(torch.arange(inner, device=DEV).float() % 3).unsqueeze(1).expand(-1, -(-inner // 128)).contiguous()
    c = ops.gemm_fp8(a, scale, w, trans_w=trans, out_dtype=torch.float32, token_tile=token_tile)
    wv = spread(w.codes, w.scales, 128)
    assert torch.equal(c.double(), (wv if trans else wv.t()) * scale[:, :1].double())


def test_product_of_views():
    """Rows of A and of its scales any distance apart, a weight that is a slice of a larger one, an output given."""
    big, big_scale, w = operands(40, 256, 512, 5)
    a, a_scale = big[::2], big_scale[::2]
    want = ops.gemm_fp8(a.contiguous(), a_scale.contiguous(), w)
    assert torch.equal(ops.gemm_fp8(a, a_scale, w), want)
    part = ops.Fp8Weight(w.codes[128:], w.scales[1:])
    out = torch.empty(20, 128, dtype=torch.bfloat16, device=DEV)
    assert ops.gemm_fp8(a, a_scale, part, out=out) is out and torch.equal(out, want[:, 128:])
    column = ops.Fp8Weight(w.codes[:, 256:], w.scales[:, 2:].contiguous())
    c = ops.gemm_fp8(a[:, 256:], a_scale[:, 2:], column, out_dtype=torch.float32)
    check_product(c, a[:, 256:], a_scale[:, 2:], column.codes, column.scales)


def test_output_that_is_not_aligned_to_four_columns():
    a, a_scale, w = operands(20, 256, 256, 9)
    want = ops.gemm_fp8(a, a_scale, w)
    out = torch.empty(20 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(20, 256)
    assert torch.equal(ops.gemm_fp8(a, a_scale, w, out=out), want)


def test_infinities_stay_in_their_rows():
    x = randn(40, 512, seed=3)
    x[3, 5], x[7, 300] = float("inf"), float("nan")
    a, a_scale = ops.quant_fp8(x)
    w = ops.quant_fp8_weight(randn(256, 512, seed=4))
    for tile in (16, 32, 128, 256):
        c = ops.gemm_fp8(a, a_scale, w, token_tile=tile)
        bad = torch.zeros(40, dtype=torch.bool, device=DEV)
        bad[[3, 7]] = True
        assert not torch.isfinite(c[bad]).any() and torch.isfinite(c[~bad]).all()


def test_no_rows():
    w = ops.quant_fp8_weight(randn(256, 128, seed=1))
    a, s = ops.quant_fp8(torch.empty(0, 128, device=DEV))
    assert ops.gemm_fp8(a, s, w).shape == (0, 256)


# ---- grouped -------------------------------------------------------------------------------------

def grouped_operands(counts, N, K, seed, trans=False, extra=0):
    rows = sum(counts) + extra
    a, a_scale = ops.quant_fp8(randn(rows, N if trans else K, seed=seed))
    return a, a_scale, ops.quant_fp8_weight(randn(len(counts), N, K, seed=seed + 1, scale=0.05))


COUNTS = [[1], [0, 3, 0], [300, 0, 17, 256, 1], [40, 90, 33], [1] * 40, [0] * 35 + [70] + [0] * 40 + [5], [129, 127, 128]]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("token_tile", [0, 16, 32, 128, 256])
def test_grouped_product(counts, trans, token_tile):
    """Empty experts, single rows, exact tiles; rows behind the last expert stay as they were."""
    N, K = 144, 272
    a, a_scale, w = grouped_operands(counts, N, K, len(counts), trans, extra=9)
    for given in (counts, torch.tensor(counts, device=DEV), torch.tensor(counts, device=DEV, dtype=torch.int32)):
        out = torch.full((a.shape[0], K if trans else N), 7.0, device=DEV)
        ops.gemm_fp8_grouped(a, a_scale, w, given, trans_w=trans, out=out, token_tile=token_tile)
        tb.check_status()
        at = 0
        for e, c in enumerate(counts):
            if c:
                check_product(out[at:at + c], a[at:at + c], a_scale[at:at + c], w.codes[e], w.scales[e], trans)
            at += c
        assert (out[at:] == 7.0).all()


@pytest.mark.parametrize("token_tile", [0, 16, 128, 256])
def test_device_counts_that_ask_for_more_rows_than_there_are(token_tile):
    a, a_scale, w = grouped_operands([100, 60], 256, 256, 3)
    want = ops.gemm_fp8_grouped(a, a_scale, w, [100, 60], token_tile=token_tile)
    for counts in ([100, 1000], [100, 60]):
        got = ops.gemm_fp8_grouped(a, a_scale, w, torch.tensor(counts, device=DEV), token_tile=token_tile)
        assert torch.equal(got, want)
    got = ops.gemm_fp8_grouped(a, a_scale, w, torch.tensor([2 ** 40, -5], device=DEV), token_tile=token_tile)
    first = ops.gemm_fp8(a, a_scale, ops.Fp8Weight(w.codes[0], w.scales[0]), out_dtype=torch.float32)
    assert ((got.float() - first).abs() <= first.abs() * 2.0 ** -7 + 1e-3 * first.abs().max()).all()
    tb.check_status()


@pytest.mark.parametrize("F", [128, 200, 384])
@pytest.mark.parametrize("counts", [None, [30, 0, 45, 1], [300, 140, 0, 77], [4000, 0, 1, 3900], 7000])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_gated_product(F, counts, dtype):
    """The codes stand for the exact activation to half a step and what the product's own bound moves it by."""
    K = 400
    counts, rows = (None, counts) if isinstance(counts, int) else (counts, 70 if counts is None else sum(counts))
    a, a_scale = ops.quant_fp8(randn(rows, K, seed=F))
    x = randn(*(() if counts is None else (len(counts),)), 2 * F, K, seed=F + 1, scale=0.05)
    w = ops.quant_fp8_weight(x)
    codes, scales, h = ops.gemm_fp8_gated(a, a_scale, w, counts, dtype, keep_h=True)
    tb.check_status()
    again = ops.gemm_fp8_gated(a, a_scale, w, counts, dtype)
    assert torch.equal(codes.float(), again[0].float()) and torch.equal(scales, again[1])
    at = 0
    for e, c in enumerate([rows] if counts is None else counts):
        if c == 0:
            continue
        wc, ws = (w.codes, w.scales) if counts is None else (w.codes[e], w.scales[e])
        av, wv = spread(a[at:at + c], a_scale[at:at + c]), spread(wc, ws, 128).t()
        ref, size = av @ wv, (av.abs() @ wv.abs()) * 2.0 ** -16.5
        assert ((h[at:at + c].double() - ref).abs() <= size + ref.abs() * 2.0 ** -8).all()
        g, u = ref.split(F, -1)
        dg, du = size.split(F, -1)
        v = torch.sigmoid(g) * g * u
        slack = 1.1 * dg * u.abs() + g.abs() * du + 2.0 ** -20 * v.abs()            # |silu'| <= 1.1
        s = scales[at:at + c].double()[:, torch.arange(F, device=DEV) // 128]
        off = (codes[at:at + c].double() * s - v).abs()
        assert (off <= (v.abs() + slack) * HALF_STEP[dtype] + s * HALF_SUBNORMAL[dtype] * 1.001 + slack).all()
        at += c


# ---- streams, graphs -----------------------------------------------------------------------------

def test_two_streams_and_a_captured_graph():
    a, a_scale, w = operands(24, 512, 1024, 1)
    b, b_scale, v = operands(90, 640, 512, 2)
    want = ops.gemm_fp8(a, a_scale, w), ops.gemm_fp8(b, b_scale, v)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            got[0] = ops.gemm_fp8(a, a_scale, w)
        with torch.cuda.stream(streams[1]):
            got[1] = ops.gemm_fp8(b, b_scale, v)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = randn(24, 1024, seed=8, dtype=torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, scales = ops.quant_fp8(x)
        out = ops.gemm_fp8(codes, scales, w)
    for seed in (9, 10):
        x.copy_(randn(24, 1024, seed=seed, dtype=torch.bfloat16))
        graph.replay()
        assert torch.equal(out, ops.gemm_fp8(*ops.quant_fp8(x), w))
