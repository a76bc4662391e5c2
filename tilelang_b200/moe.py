"""Mixture-of-experts MLP on grouped W4A16 dequantize-GEMMs, single GPU and expert-parallel.

The reference has no W4A16 MoE kernel; its semantics come from
examples/fusedmoe/example_fusedmoe_torch.py (routing :26-40: softmax then
``topk(sorted=False)``; expert MLP :8-23: ``down(silu(gate(x)) * up(x))``; dispatch by
argsort/bincount and score-weighted combine :65-91) and from its grouped GEMM
(examples/grouped_gemm/example_grouped_gemm_fwd.py:8-36: rows sorted by expert, one
weight per expert). Here the two grouped GEMMs and the activation between them are this
library's kernels, and on a GPU so is what sorts, moves and adds up the rows (:func:`dispatch`,
:func:`combine`, both differentiable in reverse mode); routing is torch's. Torch's sort and gather take
over where more than the values is asked of a layer over torch functions (gradients of the tokens,
forward mode, vmap, traces) and across ranks. :class:`Fp8ExpertMLP` runs the experts in 8-bit floating point.

Expert parallelism: experts are split contiguously over the ranks, tokens start out
partitioned by rank; one all-to-all sends every (token, expert) row to the rank that
owns the expert, the local grouped GEMMs run, a second all-to-all returns the rows, and
the token's home rank does the weighted sum. ``torch.distributed`` (NCCL over NVLink on
GPUs, gloo in CPU tests) carries both exchanges.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, List, Optional, Sequence, Tuple

import torch
import torch.distributed as dist
from torch.autograd.function import once_differentiable

from . import _lib, ops


def route(logits: torch.Tensor, top_k: int):
    scores = torch.softmax(logits.float(), dim=-1)
    weights, experts = torch.topk(scores, top_k, dim=-1, sorted=False)
    return weights, experts


def sort_by_expert(experts: torch.Tensor, num_experts: int):
    """Flatten (token, slot) pairs and order them by expert (stable). Returns the
    permutation, the token of every sorted row and the per-expert counts."""
    flat = experts.reshape(-1)
    sorted_ids, order = torch.sort(flat, stable=True)
    token_of_row = order // experts.shape[1]
    # counts from the sorted ids (bincount would make the host wait for the largest id)
    edges = torch.searchsorted(sorted_ids, torch.arange(num_experts + 1, device=flat.device, dtype=flat.dtype))
    counts = edges[1:] - edges[:-1]
    return order, token_of_row, counts


class ExpertMLP:
    """``y = W2( silu(g) * u )`` with ``[g, u] = W1(x)`` for rows sorted by expert.

    ``gemm1`` / ``gemm2`` map (rows sorted by expert, per-expert counts) to outputs and
    ``act`` maps the (rows, 2H) intermediate to (rows, H); on a GPU they are
    ``ops.gemm_grouped`` and ``ops.silu_mul``, CPU tests inject stand-ins. ``combine``
    maps (rows, (T, k) row indices, (T, k) weights) to the (T, H) weighted sums
    (``ops.moe_combine`` on a GPU, a torch gather-and-sum otherwise)."""

    def __init__(self, gemm1: Callable, gemm2: Callable, act: Callable, combine: Optional[Callable] = None):
        self.gemm1, self.gemm2, self.act = gemm1, gemm2, act
        self.combine = combine or torch_combine

    def __call__(self, x_sorted: torch.Tensor, counts: Sequence[int]) -> torch.Tensor:
        h = self.gemm1(x_sorted, counts)
        return self.gemm2(self.act(h), counts)


def torch_combine(y: torch.Tensor, row_of: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
    return (y[row_of].float() * weights.unsqueeze(-1)).sum(1).to(y.dtype)


def rows_of_tokens(order: torch.Tensor, top_k: int) -> torch.Tensor:
    """(T, k) index of every (token, slot) pair's row in the expert-sorted order."""
    inv = torch.empty_like(order)
    inv[order] = torch.arange(order.numel(), device=order.device)
    return inv.view(-1, top_k)


def expert_token_tile(rows: int, num_groups: int, N: int, device=None, sms: Optional[int] = None) -> int:
    """Token tile of a grouped GEMM over ``rows`` rows: 128 when the problem has so many tiles that
    the schedule hands out whole tiles in short spans (at least 16 tiles per SM: no partial tiles,
    no fix-up pass, and an expert's ragged row count wastes half as much padding), else 256.
    ``sms``: the SM count, read from ``device`` when not given."""
    if sms is None:
        sms = torch.cuda.get_device_properties(device if device is not None else torch.cuda.current_device()).multi_processor_count
    tiles = (rows // 128 + num_groups) * ((N + 127) // 128)
    return 128 if tiles >= 16 * sms else 256


def make_gpu_expert_mlp(w1_packed, w2_packed, token_tile: Optional[int] = None) -> ExpertMLP:
    """The expert MLP on this library's kernels. ``token_tile=None`` picks the tile per call
    (:func:`expert_token_tile`): on the 64-expert, top-6 layer with 16384 tokens the 128-token tile
    measured 2.49 ms against 3.19 ms for the 256-token tile."""

    def gemm(w):
        def run(x, counts):
            tt = token_tile or expert_token_tile(x.shape[0], w.num_groups, w.N, x.device)
            return ops.gemm_grouped(x, w, counts, token_tile=tt)
        return run

    return ExpertMLP(gemm(w1_packed), gemm(w2_packed), ops.silu_mul, ops.moe_combine)


# ---------------------------------------------------------------------------
# token exchange: rows sorted by expert and back, with gradients
# ---------------------------------------------------------------------------

@dataclass
class ExchangePlan:
    """Where every (token, slot) pair went: ``row_of`` (T, k) int64, the pair's row in expert order, or -1 - row
    for a pair whose expert id was outside [0, E) (its row lies behind the last expert's); ``counts`` (E,)
    int64, the rows of each expert. Both stay on the device. ``whole``: every row is some pair's, as it is in
    the plans that :func:`dispatch` makes."""

    row_of: torch.Tensor
    counts: torch.Tensor
    whole: bool = False

    @property
    def tokens(self) -> int:
        return self.row_of.shape[0]

    @property
    def top_k(self) -> int:
        return self.row_of.shape[1]

    @property
    def num_experts(self) -> int:
        return self.counts.numel()


def _check_experts(x: torch.Tensor, experts: torch.Tensor, num_experts: int) -> torch.Tensor:
    ops._check_rows("x", x)
    if x.dtype not in ops._FLOAT_OF:
        raise TypeError(f"x must be float16, bfloat16 or float32, got {x.dtype}")
    if x.shape[1] == 0:
        raise ValueError("x must have at least one column")
    if not isinstance(experts, torch.Tensor) or experts.dtype not in (torch.int32, torch.int64):
        raise TypeError("experts must be an int32 or int64 tensor")
    if experts.device != x.device:
        raise ValueError(f"experts is on {experts.device}, x on {x.device}")
    if experts.dim() != 2 or experts.shape[0] != x.shape[0] or experts.shape[1] == 0:
        raise ValueError(f"experts must have shape ({x.shape[0]}, top_k) with top_k at least 1, got {tuple(experts.shape)}")
    if experts.numel() >= 1 << 31:
        raise ValueError(f"experts must have fewer than 2^31 entries, got {tuple(experts.shape)}")
    if not 1 <= num_experts <= 1024:
        raise ValueError(f"num_experts must lie in 1 .. 1024, got {num_experts}")
    return experts.contiguous()


def _exchange_out(x: torch.Tensor, experts: torch.Tensor, num_experts: int, out: torch.Tensor,
                  scales: Optional[torch.Tensor], dtype: Optional[torch.dtype]) -> ExchangePlan:
    """Sorts the pairs and moves the rows of ``x`` into ``out``, on the current stream."""
    lib = _lib.load()
    T, k = experts.shape
    plan = ExchangePlan(ops._new(T, k, torch.int64, x.device),
                        torch.empty_strided((num_experts,), (1,), dtype=torch.int64, device=x.device), True)
    if T == 0:
        plan.counts.zero_()
        return plan
    need = lib.b200dq_exchange_scratch_bytes(T, k, num_experts)
    # scratch of this call alone: calls on two streams, or in two graphs, share nothing
    scratch = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    width = x.shape[1]
    ops._call(lib.b200dq_exchange_dispatch, "b200dq_exchange_dispatch", x.device,
              experts.data_ptr(), 1 if experts.dtype == torch.int64 else 0, T, k, num_experts,
              x.data_ptr(), x.stride(0) if T > 1 else width, width, ops._FLOAT_OF[x.dtype], out.data_ptr(),
              out.stride(0), scales.data_ptr() if scales is not None else None, ops._FP8_OF[dtype] if dtype is not None else 0,
              plan.row_of.data_ptr(), plan.counts.data_ptr(), scratch.data_ptr() if need else None, need)
    return plan


def _wants_gradient(*tensors: torch.Tensor) -> bool:
    """Whether a call has to go through its autograd function: for a gradient, or because that refuses what it has no
    rule for (a forward-mode tangent, a functorch transform), where the kernels would drop it."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                return True
    return ops._transformed(*tensors)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, experts, num_experts):
        out = torch.empty((experts.numel(), x.shape[1]), dtype=x.dtype, device=x.device)
        plan = _exchange_out(x, experts, num_experts, out, None, None)
        ctx.save_for_backward(plan.row_of)
        ctx.mark_non_differentiable(plan.row_of, plan.counts)
        ctx.set_materialize_grads(False)
        return out, plan.row_of, plan.counts

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, _row_of, _counts):
        if d_out is None:
            return None, None, None
        return _exchange_sum(d_out.contiguous(), ctx.saved_tensors[0], None), None, None


def _exchange_sum(y: torch.Tensor, row_of: torch.Tensor, weights: Optional[torch.Tensor]) -> torch.Tensor:
    T, k = row_of.shape
    out = ops._new(T, y.shape[1], y.dtype, y.device)
    if T:
        ops._call(_lib.load().b200dq_exchange_sum, "b200dq_exchange_sum", y.device, y.data_ptr(), row_of.data_ptr(),
                  weights.data_ptr() if weights is not None else None, out.data_ptr(), T, k, y.shape[1],
                  ops._FLOAT_OF[y.dtype])
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, row_of, weights, whole):
        ctx.save_for_backward(y, row_of, weights)
        ctx.whole = whole
        return _exchange_sum(y, row_of, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        y, row_of, weights = ctx.saved_tensors
        T, k = row_of.shape
        d_out = d_out.contiguous()
        # The kernel writes the rows that the indices name, zeros where -1 - row names one: in a dispatch's plan
        # that is all of them. Elsewhere a negative index names none (-1 may stand for "no row").
        if not ctx.whole:
            row_of = row_of.masked_fill(row_of < 0, row_of.numel())
        d_y = (torch.empty_like if ctx.whole else torch.zeros_like)(y) if ctx.needs_input_grad[0] else None
        d_w = torch.empty_like(weights) if ctx.needs_input_grad[2] else None
        if T:
            ops._call(_lib.load().b200dq_exchange_sum_grad, "b200dq_exchange_sum_grad", y.device, d_out.data_ptr(),
                      y.data_ptr(), row_of.data_ptr(), weights.data_ptr(), d_y.data_ptr() if d_y is not None else None,
                      d_w.data_ptr() if d_w is not None else None, T, k, y.shape[1], ops._FLOAT_OF[y.dtype])
        return d_y, None, d_w, None


def dispatch(x: torch.Tensor, experts: torch.Tensor, num_experts: int) -> Tuple[torch.Tensor, ExchangePlan]:
    """Every token's row once for each of its experts, sorted by expert: returns ``(rows, plan)`` with rows
    (T * k, H) in x's dtype. ``x`` (T, H) float16, bfloat16 or float32, its rows any distance apart;
    ``experts`` (T, k) int32 or int64. Rows of one expert keep the order of their (token, slot) pairs. A pair
    whose id lies outside [0, num_experts) -- a padded token's, say -- takes part in nothing: it gets a row of
    zeros behind the last expert's. Differentiable in x (reverse mode; float32 sums over the slots, in their order)."""
    experts = _check_experts(x, experts, num_experts)
    if _wants_gradient(x):
        rows, row_of, counts = _Dispatch.apply(x, experts, num_experts)
        return rows, ExchangePlan(row_of, counts, True)
    rows = ops._new(experts.numel(), x.shape[1], x.dtype, x.device)
    return rows, _exchange_out(x, experts, num_experts, rows, None, None)


def dispatch_fp8(x: torch.Tensor, experts: torch.Tensor, num_experts: int,
                 dtype: torch.dtype = torch.float8_e4m3fn) -> Tuple[torch.Tensor, torch.Tensor, ExchangePlan]:
    """:func:`dispatch` with every token quantised once on its way, as :func:`ops.quant_fp8` does it: returns
    ``(codes (T * k, H), scales (T * k, ceil(H / 128)), plan)``. Not differentiable. A dropped pair's row has
    zero codes."""
    ops._check_fp8_target(dtype)
    experts = _check_experts(x, experts, num_experts)
    rows = experts.numel()
    codes = ops._fp8_rows(rows, x.shape[1], dtype, x.device)
    scales = ops._new(rows, ops._blocks128(x.shape[1]), torch.float32, x.device)
    return codes, scales, _exchange_out(x.detach(), experts, num_experts, codes, scales, dtype)


def combine_rows(y: torch.Tensor, row_of: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
    """:func:`combine` from the (T, k) row indices alone. For a gradient of ``y`` no row may be named twice; rows
    that no index names have the gradient zero."""
    return combine(y, ExchangePlan(row_of, row_of.new_empty(0)), weights)


def combine(y: torch.Tensor, plan: ExchangePlan, weights: torch.Tensor) -> torch.Tensor:
    """Back from expert order: ``out[t] = sum_s weights[t, s] * y[plan.row_of[t, s]]``, float32 sums in slot order
    rounded once to y's dtype; dropped pairs add nothing. ``y`` (T * k, H) contiguous float16, bfloat16 or float32,
    ``weights`` (T, k) of any floating type. Differentiable in y and weights (reverse mode)."""
    ops._check_cuda_contig("y", y)
    if y.dim() != 2 or y.dtype not in ops._FLOAT_OF:
        raise ValueError("y must be a 2-D float16, bfloat16 or float32 tensor")
    row_of = plan.row_of
    if row_of.device != y.device or weights.device != y.device:
        raise ValueError("y, the plan and the weights must be on one device")
    if row_of.dtype != torch.int64 or row_of.dim() != 2 or not row_of.is_contiguous():
        raise ValueError("row indices must be a contiguous int64 tensor of shape (tokens, top_k)")
    if not weights.dtype.is_floating_point or weights.shape != row_of.shape:
        raise ValueError(f"weights must be floating point of shape {tuple(row_of.shape)}, got {weights.dtype} {tuple(weights.shape)}")
    if y.shape[0] != row_of.numel() or y.shape[1] == 0:
        raise ValueError(f"y must have {row_of.numel()} rows of at least one column, got {tuple(y.shape)}")
    if y.shape[1] > 1 << 28 or row_of.shape[1] >= 1 << 31:           # the C call counts both in 32 bits
        raise ValueError(f"rows have at most 2^28 columns and tokens fewer than 2^31 slots, got y {tuple(y.shape)} and row indices {tuple(row_of.shape)}")
    weights = weights.float().contiguous()
    if not _wants_gradient(y, weights):
        return _exchange_sum(y, row_of, weights)
    return _Combine.apply(y, row_of, weights, plan.whole)


class _Fp8Mlp(torch.autograd.Function):
    """The expert MLP on rows sorted by expert; gradient of the rows (the quantised weights are constants)."""

    @staticmethod
    def forward(ctx, x_sorted, counts, mlp, rows_behind):
        codes, scales = ops.quant_fp8(x_sorted)
        act, act_scales, h = ops.gemm_fp8_gated(codes, scales, mlp.w1, counts, keep_h=True)
        y = ops.gemm_fp8_grouped(act, act_scales, mlp.w2, counts, out_dtype=x_sorted.dtype)
        ctx.save_for_backward(h, counts, mlp.w1.codes, mlp.w1.scales, mlp.w2.codes, mlp.w2.scales)
        ctx.grad_dtype, ctx.rows_behind = mlp.grad_dtype, rows_behind
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        h, counts, *w = ctx.saved_tensors
        w1, w2 = ops.Fp8Weight(*w[:2]), ops.Fp8Weight(*w[2:])
        d_codes, d_scales = ops.quant_fp8(d_y.contiguous(), ctx.grad_dtype)
        d_act = ops.gemm_fp8_grouped(d_codes, d_scales, w2, counts, trans_w=True, out_dtype=h.dtype)
        d_codes, d_scales = ops.silu_mul_backward_quant_fp8(h, d_act, ctx.grad_dtype)
        # the products do not write rows behind the last expert's
        d_x = (torch.zeros if ctx.rows_behind else torch.empty)((h.shape[0], w1.K), dtype=d_y.dtype, device=h.device)
        ops.gemm_fp8_grouped(d_codes, d_scales, w1, counts, trans_w=True, out=d_x)
        return d_x, None, None, None


class Fp8ExpertMLP(ExpertMLP):
    """``y = W2( silu(g) * u )`` with ``[g, u] = W1(x)``, experts' weights in 8-bit floating point
    (:class:`ops.Fp8Weight`: ``w1`` (E, 2F, H) with the gate's rows first, ``w2`` (E, H, F)), activations
    quantised per row and 128 columns on their way: tokens by the dispatch, the gated intermediate by the
    first product. Goes where :func:`make_gpu_expert_mlp`'s result goes (:func:`moe_forward`,
    :func:`moe_forward_ep`).

    Tokens are float16 or bfloat16: the backward pass keeps h, and the gradient that meets it, in bfloat16. Differentiable
    in the tokens (on one GPU) and the routing weights, in reverse mode; the experts' weights are constants. The gradient is
    quantised like the activations, to ``grad_dtype``, and multiplied with the same weight bytes; the
    quantiser itself counts as the identity."""

    def __init__(self, w1: "ops.Fp8Weight", w2: "ops.Fp8Weight", grad_dtype: torch.dtype = torch.float8_e4m3fn):
        ops._check_fp8_target(grad_dtype)
        if w1.codes.dim() != 3 or w2.codes.dim() != 3:
            raise ValueError("w1 and w2 hold one matrix per expert: codes of shape (E, 2F, H) and (E, H, F)")
        if w1.num_groups != w2.num_groups or w1.N != 2 * w2.K or w1.K != w2.N:
            raise ValueError(f"w1 {tuple(w1.codes.shape)} and w2 {tuple(w2.codes.shape)} are not (E, 2F, H) and (E, H, F)")
        self.w1, self.w2, self.grad_dtype = w1, w2, grad_dtype
        self.combine = combine_rows

    def _check(self, x: torch.Tensor) -> None:
        if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2 or x.shape[1] != self.w1.K:
            raise ValueError(f"rows must be float16 or bfloat16 of width {self.w1.K}, got {x.dtype} {tuple(x.shape)}")

    def __call__(self, x_sorted: torch.Tensor, counts) -> torch.Tensor:
        """Rows sorted by expert -> rows. Rows behind the last expert's are undefined, their gradient is zero."""
        self._check(x_sorted)
        counts = ops._device_counts(counts, self.w1.num_groups, x_sorted.shape[0], x_sorted.device)
        if _wants_gradient(x_sorted):
            return _Fp8Mlp.apply(x_sorted, counts, self, True)
        return self._run(*ops.quant_fp8(x_sorted), counts, x_sorted.dtype)

    def _run(self, codes, scales, counts, dtype):
        act, act_scales = ops.gemm_fp8_gated(codes, scales, self.w1, counts)
        return ops.gemm_fp8_grouped(act, act_scales, self.w2, counts, out_dtype=dtype)

    def layer(self, x: torch.Tensor, experts: torch.Tensor, weights: torch.Tensor, num_experts: int) -> torch.Tensor:
        """The layer behind the router: tokens (T, H), their experts and weights (T, k) -> (T, H)."""
        if num_experts != self.w1.num_groups:
            raise ValueError(f"the router has {num_experts} experts, the weights {self.w1.num_groups}")
        self._check(x)
        if _wants_gradient(x):
            rows, plan = dispatch(x, experts, num_experts)
            # the dispatch's gradient reads no row behind the last expert's
            return combine(_Fp8Mlp.apply(rows, plan.counts, self, False), plan, weights)
        codes, scales, plan = dispatch_fp8(x, experts, num_experts)
        return combine(self._run(codes, scales, plan.counts, x.dtype), plan, weights)


def _fits_exchange(x: torch.Tensor, logits: torch.Tensor, top_k: int, num_experts: int) -> bool:
    """Whether :func:`dispatch` takes these tokens and routes. A router wider than the experts drops pairs, whose negative
    row indices an ``ExpertMLP.combine`` need not know; one of fewer rows than ``x`` leaves the other tokens out."""
    return (x.dtype in ops._FLOAT_OF and x.dim() == 2 and 0 < x.shape[1] <= 1 << 28 and num_experts <= 1024
            and x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1])
            and logits.dim() == 2 and logits.shape[0] == x.shape[0] and logits.shape[1] <= num_experts
            and logits.shape[0] * top_k < 1 << 31)


def moe_forward(x: torch.Tensor, logits: torch.Tensor, top_k: int, num_experts: int, mlp: ExpertMLP) -> torch.Tensor:
    """Single-device MoE layer: route, gather rows by expert, expert MLP, weighted combine."""
    if logits.shape[0] > x.shape[0]:
        raise ValueError(f"{logits.shape[0]} rows of logits for {x.shape[0]} tokens")
    weights, experts = route(logits, top_k)
    if isinstance(mlp, Fp8ExpertMLP):
        return mlp.layer(x, experts, weights, num_experts)
    if (ops._ordinary(x, logits) and x.is_cuda and _fits_exchange(x, logits, top_k, num_experts) and ops._may_launch(x.device)
            and not (torch.is_grad_enabled() and x.requires_grad)):
        # the same order of rows as below, in one to three launches instead of some ten (torch's gather can be
        # differentiated more than once, forwards, batched and recorded: all of these go on below)
        x_sorted, plan = dispatch(x, experts, num_experts)
        return mlp.combine(mlp(x_sorted, plan.counts), plan.row_of, weights.contiguous())
    order, token_of_row, counts = sort_by_expert(experts, num_experts)
    x_sorted = x.index_select(0, token_of_row)
    # on a GPU the counts stay on the device: the grouped GEMMs plan their work there
    y = mlp(x_sorted, counts if counts.is_cuda else counts.tolist())
    return mlp.combine(y, rows_of_tokens(order, top_k), weights.contiguous())


def expert_ranges(num_experts: int, world_size: int) -> List[range]:
    per = (num_experts + world_size - 1) // world_size
    return [range(min(r * per, num_experts), min((r + 1) * per, num_experts)) for r in range(world_size)]


def moe_forward_ep(x_local: torch.Tensor, logits_local: torch.Tensor, top_k: int, num_experts: int,
                   local_mlp: ExpertMLP, group: Optional[dist.ProcessGroup] = None) -> torch.Tensor:
    """Expert-parallel MoE layer. ``x_local`` are this rank's tokens; ``local_mlp`` runs this
    rank's experts (counts are given for the local experts only, in order). The exchange between the
    ranks carries no gradient of the tokens."""
    if isinstance(local_mlp, Fp8ExpertMLP) and _wants_gradient(x_local):
        raise ValueError("moe_forward_ep gives no gradient of the tokens (moe_forward does): call it under torch.no_grad(), or detach them")
    world = dist.get_world_size(group)
    rank = dist.get_rank(group)
    ranges = expert_ranges(num_experts, world)
    weights, experts = route(logits_local, top_k)
    order, token_of_row, counts = sort_by_expert(experts, num_experts)     # rows sorted by global expert id
    x_sorted = x_local.index_select(0, token_of_row)

    # the full count matrix (every rank learns what it will receive): one collective, one sync
    flat_counts = counts.new_empty(world * num_experts)
    dist.all_gather_into_tensor(flat_counts, counts.contiguous(), group=group)
    all_counts_dev = flat_counts.view(world, num_experts)
    # The one host wait of the layer: the split sizes of the two all-to-alls are host
    # arguments. Only the per-rank totals come to the host (2 * world numbers); the per-expert
    # counts stay on the device and the grouped GEMMs plan their work there.
    my = ranges[rank]
    bounds = torch.tensor([r.start for r in ranges] + [ranges[-1].stop], device=counts.device)
    csum = torch.cat((all_counts_dev.new_zeros(world, 1), all_counts_dev.cumsum(1)), dim=1)    # (world, E + 1)
    per_rank = csum[:, bounds[1:]] - csum[:, bounds[:-1]]                  # [source rank, owner rank] rows
    totals = torch.stack((per_rank[rank], per_rank[:, rank])).cpu()        # what I send to / receive from each rank
    send_rows, recv_rows = totals[0].tolist(), totals[1].tolist()
    mine_dev = all_counts_dev[:, my.start:my.stop]                         # (world, local experts)

    recv = x_sorted.new_empty((sum(recv_rows), x_sorted.shape[1]))
    dist.all_to_all_single(recv, x_sorted.contiguous(), recv_rows, send_rows, group=group)

    # received rows are ordered (source rank, expert); regroup them by expert for the grouped GEMM
    local_ids = torch.arange(len(my), device=recv.device).repeat(world)
    src_expert = torch.repeat_interleave(local_ids, mine_dev.reshape(-1), output_size=sum(recv_rows))
    regroup = torch.argsort(src_expert, stable=True)
    local_counts = mine_dev.sum(0)
    y_grouped = local_mlp(recv.index_select(0, regroup), local_counts if local_counts.is_cuda else local_counts.tolist())
    ungroup = torch.empty_like(regroup)
    ungroup[regroup] = torch.arange(regroup.numel(), device=regroup.device)
    y = y_grouped.index_select(0, ungroup)                                 # back to (source rank, expert) order

    back = y.new_empty((x_sorted.shape[0], y.shape[1]))
    dist.all_to_all_single(back, y.contiguous(), send_rows, recv_rows, group=group)

    return local_mlp.combine(back, rows_of_tokens(order, top_k), weights.contiguous())
