"""GPU: the token exchange of a mixture-of-experts layer and its gradients against plain loops in 64 bits.

Sorting and copying are exact. A sum of k terms in float32 is off by at most k 2^-24 of the sum of magnitudes and
half a step of its type; a dot product of H terms, added in threads, shuffles and warps, by at most (H / 256 + 16)
2^-24 of its sum of magnitudes (H 2^-24 is asserted)."""
import pytest
import torch

import tilelang_b200 as tb
from tilelang_b200 import moe, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=gen(seed)).to(dtype)


def plain_sort(experts, E):
    """row_of and counts by Python loops over the pairs."""
    T, k = experts.shape
    ids = [i if 0 <= i < E else E for i in experts.flatten().tolist()]
    order = sorted(range(len(ids)), key=lambda p: (ids[p], p))
    row_of = [0] * len(ids)
    for row, pair in enumerate(order):
        row_of[pair] = row if ids[pair] < E else -1 - row
    return torch.tensor(row_of, device=DEV).view(T, k), torch.tensor([ids.count(e) for e in range(E)], device=DEV)


def pick(T, k, E, seed, dropped=0.0):
    experts = torch.randint(0, E, (T, k), device=DEV, generator=gen(seed))
    if dropped:
        lost = torch.rand(T, k, device=DEV, generator=gen(seed + 1)) < dropped
        experts = torch.where(lost, torch.where(experts % 2 == 0, -1, E + experts), experts)
    return experts


SIZES = [(1, 1, 1, 8), (1, 8, 8, 64), (5, 2, 4, 100), (33, 6, 64, 256), (300, 3, 7, 33), (512, 8, 256, 128),
         (700, 6, 64, 64), (1500, 8, 1024, 16), (4097, 1, 3, 8), (9000, 2, 33, 8)]


@pytest.mark.parametrize("T,k,E,H", SIZES)
@pytest.mark.parametrize("dropped", [0.0, 0.3])
@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
def test_rows_sorted_by_expert(T, k, E, H, dropped, ids):
    experts = pick(T, k, E, T + k, dropped).to(ids)
    x = randn(T, H, seed=T, dtype=torch.bfloat16)
    rows, plan = moe.dispatch(x, experts, E)
    row_of, counts = plain_sort(experts, E)
    assert torch.equal(plan.row_of, row_of) and torch.equal(plan.counts, counts)
    want = torch.zeros(T * k, H, dtype=x.dtype, device=DEV)
    kept = row_of >= 0
    want[row_of[kept]] = x.unsqueeze(1).expand(T, k, H)[kept]
    assert torch.equal(rows, want)
    codes, scales, plan8 = moe.dispatch_fp8(x, experts, E)
    assert torch.equal(plan8.row_of, row_of) and torch.equal(plan8.counts, counts)
    q, s = ops.quant_fp8(want)
    assert torch.equal(codes.float(), q.float()) and torch.equal(scales, s)


@pytest.mark.parametrize("kind", [torch.float16, torch.float32])
@pytest.mark.parametrize("H", [1, 7, 16, 200, 2048])
@pytest.mark.parametrize("T", [3, 1000])
def test_row_types_widths_and_views(kind, H, T):
    experts = pick(T, 5, 9, H)
    big = randn(T, 2 * H + 3, seed=H, dtype=kind)
    for x in (big[:, 1:H + 1], big[:, :H].contiguous()):
        rows, plan = moe.dispatch(x, experts, 9)
        assert torch.equal(rows[plan.row_of], x.unsqueeze(1).expand(T, 5, H))
        for dtype in (torch.float8_e4m3fn, torch.float8_e5m2):
            codes, scales, plan8 = moe.dispatch_fp8(x, experts, 9, dtype)
            q, s = ops.quant_fp8(rows, dtype)
            assert torch.equal(codes.float(), q.float()) and torch.equal(scales, s)


def test_one_expert_takes_everything_and_all_are_dropped():
    x = randn(600, 64, seed=1, dtype=torch.bfloat16)
    rows, plan = moe.dispatch(x, torch.full((600, 8), 3, device=DEV), 5)
    assert plan.counts.tolist() == [0, 0, 0, 4800, 0]
    assert torch.equal(plan.row_of, torch.arange(4800, device=DEV).view(600, 8))
    rows, plan = moe.dispatch(x, torch.full((600, 8), -1, device=DEV), 5)
    assert plan.counts.sum() == 0 and (plan.row_of < 0).all() and (rows == 0).all()
    assert (moe.combine(rows, plan, torch.ones(600, 8, device=DEV)) == 0).all()


def test_no_tokens():
    rows, plan = moe.dispatch(torch.empty(0, 16, device=DEV), torch.empty(0, 2, dtype=torch.int64, device=DEV), 4)
    assert rows.shape == (0, 16) and plan.counts.tolist() == [0, 0, 0, 0]
    assert moe.combine(rows, plan, torch.empty(0, 2, device=DEV)).shape == (0, 16)


@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 8), (7, 2, 4, 100), (40, 6, 64, 256), (64, 9, 16, 33), (900, 5, 8, 512), (3, 2, 4, 4104)])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dropped", [0.0, 0.3])
def test_exchange_and_its_gradients(T, k, E, H, kind, dropped):
    experts = pick(T, k, E, T + H, dropped)
    x = randn(T, H, seed=1, dtype=kind).requires_grad_()
    y = randn(T * k, H, seed=2, dtype=kind).requires_grad_()
    w = torch.rand(T, k, device=DEV, generator=gen(3)).requires_grad_()
    d_rows, d_out = randn(T * k, H, seed=4, dtype=kind), randn(T, H, seed=5, dtype=kind)
    with torch.no_grad():
        y[-1] = float("nan") if dropped and bool((experts[0] < 0).any()) else y[-1]
    rows, plan = moe.dispatch(x, experts, E)
    out = moe.combine(y, plan, w)
    d_x, d_y, d_w = torch.autograd.grad((rows, out), (x, y, w), (d_rows, d_out))
    kept = plan.row_of >= 0
    at = plan.row_of.clamp(min=0)
    half = torch.finfo(kind).eps / 2

    def near(got, terms, dim):
        """A float32 sum of the 64-bit ``terms`` along ``dim``, rounded to the type."""
        ref, size = terms.sum(dim), terms.abs().sum(dim)
        bound = size * terms.shape[dim] * 2.0 ** -24 + ref.abs() * (half if got.dtype == kind else 2.0 ** -24) + 2.0 ** -25 * (kind == torch.float16)
        assert ((got.double() - ref).abs() <= bound).all()

    yk = torch.where(kept.unsqueeze(-1), y.detach().double()[at], 0.0)
    near(out.detach(), yk * w.detach().double().unsqueeze(-1), 1)
    near(d_x, torch.where(kept.unsqueeze(-1), d_rows.double()[at], 0.0), 1)
    near(d_w, yk * d_out.double().unsqueeze(1), 2)
    assert (d_w[~kept] == 0).all()
    want = torch.zeros(T * k, H, dtype=torch.float64, device=DEV)
    want[plan.row_of[kept]] = (w.detach().double().unsqueeze(-1) * d_out.double().unsqueeze(1))[kept]
    assert ((d_y.double() - want).abs() <= want.abs() * (half + 2.0 ** -24) + 2.0 ** -25 * (kind == torch.float16)).all()


def test_gradients_against_differences():
    """The layer's exchange is linear in x and y, and in the weights: a central difference is exact but for
    rounding, so float32 with a step of 1 is held to 1e-4 of the largest."""
    T, k, E, H = 20, 3, 5, 48
    experts = pick(T, k, E, 7, 0.2)
    x, w = randn(T, H, seed=1).requires_grad_(), torch.rand(T, k, device=DEV, generator=gen(2)).requires_grad_()
    v = randn(T, H, seed=3)

    def f(x, w):
        rows, plan = moe.dispatch(x, experts, E)
        return (moe.combine(rows, plan, w) * v).sum()

    d_x, d_w = torch.autograd.grad(f(x, w), (x, w))
    with torch.no_grad():
        for d, at, i in ((d_x, x, (3, 5)), (d_x, x, (19, 47)), (d_w, w, (0, 0)), (d_w, w, (19, 2))):
            step = torch.zeros_like(at)
            step[i] = 1.0
            diff = ((f(x + step, w) - f(x - step, w)) if at is x else (f(x, w + step) - f(x, w - step))) / 2
            assert (diff - d[i]).abs() <= 1e-4 * d.abs().max()


def test_only_the_gradients_that_are_asked_for():
    experts = pick(30, 2, 4, 1)
    y, w = randn(60, 32, seed=1), torch.rand(30, 2, device=DEV)
    _, plan = moe.dispatch(randn(30, 32, seed=2), experts, 4)
    d = randn(30, 32, seed=3)
    full = torch.autograd.grad(moe.combine(y.requires_grad_(), plan, w.requires_grad_()), (y, w), d)
    assert torch.equal(torch.autograd.grad(moe.combine(y, plan, w.detach()), y, d)[0], full[0])
    assert torch.equal(torch.autograd.grad(moe.combine(y.detach(), plan, w), w, d)[0], full[1])
    # a gradient that arrives with stride zero, weights of another type
    moe.combine(y, plan, w.detach().half()).sum().backward()
    assert torch.equal(y.grad, torch.autograd.grad(moe.combine(y, plan, w.detach().half().float()), y, torch.ones_like(d))[0])


def test_rows_outside_the_tensor_are_not_followed():
    """Indices that no dispatch gives add nothing; in the backward pass they are neither read nor written."""
    y = randn(12, 40, seed=1).requires_grad_()
    row_of = torch.tensor([[0, 5], [12, 3], [2 ** 40, -1], [7, -2 ** 50], [1, 2], [-13, 4]], device=DEV)
    w = torch.ones(6, 2, device=DEV).requires_grad_()
    plan = moe.ExchangePlan(row_of, torch.zeros(1, dtype=torch.int64, device=DEV))
    out = moe.combine(y, plan, w)
    kept = (row_of >= 0) & (row_of < 12)
    want = torch.where(kept.unsqueeze(-1), y.detach()[row_of.clamp(0, 11)], 0.0).sum(1)
    assert torch.equal(out.detach(), want)
    d_w, = torch.autograd.grad(out, w, torch.ones_like(out))
    assert (d_w[~kept] == 0).all() and (d_w[kept] != 0).all()


def test_rows_that_no_index_names_have_no_gradient():
    y, d = randn(12, 40, seed=1).requires_grad_(), randn(6, 40, seed=2)
    row_of = torch.tensor([[0, 5], [12, 3], [2 ** 40, -1], [7, -2 ** 50], [1, 2], [-13, 4]], device=DEV)
    w = torch.rand(6, 2, device=DEV, generator=gen(3))
    want = torch.zeros_like(y.detach())
    for t in range(6):
        for s in range(2):
            if 0 <= int(row_of[t, s]) < 12:
                want[int(row_of[t, s])] = w[t, s] * d[t]
    for _ in range(3):
        torch.full((4096,), float("nan"), device=DEV)                # what an allocation may find
        d_y, = torch.autograd.grad(moe.combine_rows(y, row_of, w), y, d)
        assert torch.equal(d_y, want)


def test_two_captured_graphs_share_nothing():
    experts = [pick(2000, 4, 16, 1), pick(2000, 4, 16, 2)]
    x = randn(2000, 64, seed=3, dtype=torch.bfloat16)
    w = torch.rand(2000, 4, device=DEV, generator=gen(4))
    moe.dispatch(x, experts[0], 16)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for e in experts:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            rows, plan = moe.dispatch(x, e, 16)
            outs.append((rows, plan.row_of, plan.counts, moe.combine(rows, plan, w)))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for e, out in zip(experts, outs):
        rows, plan = moe.dispatch(x, e, 16)
        for a, b in zip(out, (rows, plan.row_of, plan.counts, moe.combine(rows, plan, w))):
            assert torch.equal(a, b)


def test_backward_in_a_graph():
    x = randn(700, 64, seed=1, dtype=torch.bfloat16)
    w = torch.rand(700, 8, device=DEV, generator=gen(2))
    experts = pick(700, 8, 16, 3)

    def step():
        leaves = x.detach().requires_grad_(), w.detach().requires_grad_()
        rows, plan = moe.dispatch(leaves[0], experts, 16)
        out = moe.combine(rows, plan, leaves[1])
        return (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    x.copy_(randn(700, 64, seed=9, dtype=torch.bfloat16))
    g.replay()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)
    tb.check_status()
