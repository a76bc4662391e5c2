"""The measured cases of the 8-bit floating point expert layer: block-scaled products (dense, grouped by expert, with
the gate fused, and the gradient of their input), the quantisers around them, and the exchange that sorts tokens by
expert and brings them back with their weights, forward and backward.

``run`` computes each operator in plain torch operations in 32 bits, or with ``own`` through ``tilelang_b200``.
"""
import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 128
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
OUT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one new token through a 14336 x 4096 projection: the latency of a decode step
        {"name": "product_one_token", "op": "product", "m": 1, "n": 14336, "k": 4096, "a": "e4m3", "out": "bf16"},
        # a batch of 16 decoding sequences through the 28672 x 8192 projection of the benchmark
        {"name": "product_batch_16", "op": "product", "m": 16, "n": 28672, "k": 8192, "a": "e4m3", "out": "bf16"},
        # a chunk of a prompt, no size a multiple of the tile: half a scale block of rows, sums kept in 32 bits
        {"name": "product_ragged", "op": "product", "m": 333, "n": 8640, "k": 3200, "a": "e4m3", "out": "f32"},
        # a long prompt through the benchmark's projection
        {"name": "product_prompt", "op": "product", "m": 4096, "n": 28672, "k": 8192, "a": "e4m3", "out": "bf16"},
        # the gradient of a projection's input: dY in the wide-range type, the weight read along its rows
        {"name": "product_gradient", "op": "gradient", "m": 2048, "n": 14336, "k": 4096, "a": "e5m2", "out": "bf16"},
        # 16 decoding sequences, six of 64 experts each: almost every expert's weight for a row or two
        {"name": "grouped_decode", "op": "grouped", "t": 16, "e": 64, "top": 6, "n": 2816, "k": 2048, "out": "bf16"},
        # the experts' second product over a prompt batch of 16384 tokens
        {"name": "grouped_prompt", "op": "grouped", "t": 16384, "e": 64, "top": 6, "n": 2048, "k": 1408, "out": "bf16"},
        # the experts' first product over that batch, gated and quantised for the second one
        {"name": "gated_prompt", "op": "gated", "t": 16384, "e": 64, "top": 6, "n": 1408, "k": 2048},
        # hidden states of a prompt batch quantised in front of a projection
        {"name": "quantise_rows", "op": "quantise", "m": 16384, "k": 2048, "x": "bf16", "to": "e4m3"},
        # the gradient of the gate, quantised in front of the product that follows it in the backward pass
        {"name": "quantise_gate_gradient", "op": "gate_gradient", "m": 24576, "k": 1408, "x": "bf16", "to": "e5m2"},
        # a decode step's exchange: 32 tokens to six experts each, quantised on the way, and back
        {"name": "exchange_decode", "op": "exchange", "t": 32, "e": 64, "top": 6, "h": 2048, "x": "bf16"},
        # a training step's exchange, out and back with both gradients
        {"name": "exchange_train", "op": "exchange_train", "t": 16384, "e": 64, "top": 6, "h": 2048, "x": "bf16"},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["product", "product", "gradient", "grouped", "grouped", "gated", "quantise", "gate_gradient",
                     "exchange", "exchange_train"])
    a = rng.choice(["e4m3", "e4m3", "e5m2"])
    if op in ("product", "gradient"):
        m = _spread(rng, 1, 8192)
        n, k = _spread(rng, 256, 28672), 16 * _spread(rng, 16, 512)
        if op == "gradient":
            n, k = 16 * max(16, n // 16), k + 16 * rng.randrange(2)
        m = min(m, max(1, int(0.9e12 / (n * k))))
        return {"op": op, "m": m, "n": n, "k": k, "a": a, "out": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "grouped" or op == "gated":
        e = rng.choice([4, 8, 16, 32, 64, 128])
        top = rng.randint(1, min(8, e))
        t = _spread(rng, 1, 16384)
        n = 128 * _spread(rng, 2, 16) if op == "gated" else _spread(rng, 256, 4096)
        k = 16 * _spread(rng, 16, 160)
        t = min(t, max(1, int(2.5e11 / (top * n * k * (2 if op == "gated" else 1)))))
        case = {"op": op, "t": t, "e": e, "top": top, "n": n, "k": k}
        return case if op == "gated" else dict(case, out=rng.choice(["bf16", "f16", "f32"]))
    x = rng.choice(["bf16", "bf16", "f16"])
    if op in ("quantise", "gate_gradient"):
        return {"op": op, "m": _spread(rng, 1, 16384), "k": _spread(rng, 128, 2048), "x": x, "to": a}
    e = rng.choice([4, 8, 16, 32, 64, 128, 256])
    case = {"op": op, "e": e, "top": rng.randint(1, min(8, e)), "h": 8 * _spread(rng, 32, 512), "x": x}
    return dict(case, t=_spread(rng, 1, 512) if op == "exchange" else min(_spread(rng, 1, 16384), int(2e8 / (case["top"] * case["h"]))))


# ---- what a program has in hand ------------------------------------------------------------------

def _blocks(n):
    return -(-n // BLOCK)


def _amounts(x, kind, rows):
    """``x`` (..., R, C) in blocks of ``rows`` x 128: its codes and the (..., R blocks, C blocks) scales."""
    r, c = x.shape[-2:]
    pad = torch.nn.functional.pad(x, (0, _blocks(c) * BLOCK - c, 0, -r % rows))
    split = pad.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, rows))
    scale = (split.abs().amax((-3, -1)) / LARGEST[kind]).clamp(min=2.0 ** -126)
    codes = (split / scale[..., :, None, :, None]).to(FP8[kind])
    return codes.view(torch.uint8).flatten(-4, -3).flatten(-2, -1)[..., :r, :c].contiguous().view(FP8[kind]), scale


def _rows(m, k, kind, gen):
    return _amounts(torch.randn(m, k, device=DEVICE, generator=gen), kind, 1)


def _weight(e, n, k, gen):
    if e is None:
        return _amounts(torch.randn(n, k, device=DEVICE, generator=gen) * 0.02, "e4m3", BLOCK)
    codes = torch.empty(e, n, k, dtype=FP8["e4m3"], device=DEVICE)
    scales = torch.empty(e, _blocks(n), _blocks(k), device=DEVICE)
    for i in range(e):
        codes[i], scales[i] = _amounts(torch.randn(n, k, device=DEVICE, generator=gen) * 0.02, "e4m3", BLOCK)
    return codes, scales


def _experts(t, e, top, gen):
    """Each token's experts, some more in demand than others, and their weights."""
    logits = torch.randn(t, e, device=DEVICE, generator=gen) + 0.5 * torch.randn(e, device=DEVICE, generator=gen)
    weights, experts = torch.topk(torch.softmax(logits, -1), top, -1)
    return experts, weights


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    s = dict(case)
    op = case["op"]
    if op in ("product", "gradient"):
        s["codes"], s["scale"] = _rows(case["m"], case["k"] if op == "product" else case["n"], case["a"], gen)
        s["w"], s["w_scale"] = _weight(None, case["n"], case["k"], gen)
    elif op in ("grouped", "gated"):
        s["codes"], s["scale"] = _rows(case["t"] * case["top"], case["k"], "e4m3", gen)
        s["w"], s["w_scale"] = _weight(case["e"], case["n"] * (2 if op == "gated" else 1), case["k"], gen)
        s["counts"] = torch.bincount(_experts(case["t"], case["e"], case["top"], gen)[0].flatten(), minlength=case["e"])
        s["most"] = int(s["counts"].max())
    elif op in ("quantise", "gate_gradient"):
        kind = OUT[case["x"]]
        width = case["k"] * (1 if op == "quantise" else 2)
        s["x"] = (torch.randn(case["m"], width, device=DEVICE, generator=gen) *
                  torch.exp2(torch.randint(-3, 4, (case["m"], 1), device=DEVICE, generator=gen).float())).to(kind)
        if op == "gate_gradient":
            s["d"] = (torch.randn(case["m"], case["k"], device=DEVICE, generator=gen) * 1e-3).to(kind)
    else:
        kind = OUT[case["x"]]
        t, h, rows = case["t"], case["h"], case["t"] * case["top"]
        s["x"] = torch.randn(t, h, device=DEVICE, generator=gen).to(kind)
        s["y"] = torch.randn(rows, h, device=DEVICE, generator=gen).to(kind)
        s["experts"], s["weights"] = _experts(t, case["e"], case["top"], gen)
        if op == "exchange_train":
            s["d_sorted"] = torch.randn(rows, h, device=DEVICE, generator=gen).to(kind)
            s["d_out"] = torch.randn(t, h, device=DEVICE, generator=gen).to(kind)
    return s


# ---- the operators in plain form -----------------------------------------------------------------

def _spread_rows(codes, scale):
    """The values that codes with a scale per row and 128 columns stand for."""
    return codes.float() * scale.repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]


def _spread_blocks(codes, scale):
    n, k = codes.shape[-2:]
    return codes.float() * scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _quantised(x, kind):
    """Codes and scales of the rows of ``x``."""
    c = x.shape[-1]
    split = torch.nn.functional.pad(x, (0, _blocks(c) * BLOCK - c)).unflatten(-1, (-1, BLOCK))
    scale = (split.abs().amax(-1) * (1.0 / LARGEST[kind])).clamp(min=2.0 ** -126)
    codes = (split * torch.reciprocal(scale).unsqueeze(-1)).clamp(-LARGEST[kind], LARGEST[kind]).to(FP8[kind])
    return codes.flatten(-2)[..., :c], scale


def _grouped(a, w, counts, most):
    """Rows sorted by expert times their expert's weight: the experts' rows side by side, padded to the most."""
    rows, e = a.shape[0], w.shape[0]
    group = torch.repeat_interleave(torch.arange(e, device=a.device), counts, output_size=rows)
    place = torch.arange(rows, device=a.device) - (counts.cumsum(0) - counts)[group]
    padded = torch.zeros(e, most, a.shape[1], device=a.device)
    padded[group, place] = a
    return torch.bmm(padded, w.transpose(1, 2))[group, place]


def _sorted_by_expert(experts, e):
    """Rows in expert order (equal ones in token order): the place of every (token, slot) pair, the token of every
    row, and the rows of each expert."""
    flat = experts.flatten()
    order = torch.sort(flat, stable=True).indices
    row_of = torch.empty_like(order)
    row_of[order] = torch.arange(order.numel(), device=order.device)
    counts = (flat.unsqueeze(1) == torch.arange(e, device=flat.device)).sum(0)
    return row_of.view(experts.shape), order // experts.shape[1], counts


def _plain(s):
    op = s["op"]
    if op == "product":
        return (_spread_rows(s["codes"], s["scale"]) @ _spread_blocks(s["w"], s["w_scale"]).t()).to(OUT[s["out"]])
    if op == "gradient":
        return (_spread_rows(s["codes"], s["scale"]) @ _spread_blocks(s["w"], s["w_scale"])).to(OUT[s["out"]])
    if op == "grouped":
        y = _grouped(_spread_rows(s["codes"], s["scale"]), _spread_blocks(s["w"], s["w_scale"]), s["counts"], s["most"])
        return y.to(OUT[s["out"]])
    if op == "gated":
        h = _grouped(_spread_rows(s["codes"], s["scale"]), _spread_blocks(s["w"], s["w_scale"]), s["counts"], s["most"])
        g, u = h.chunk(2, -1)
        return _quantised(g / (1 + torch.exp(-g)) * u, "e4m3")
    if op == "quantise":
        return _quantised(s["x"].float(), s["to"])
    if op == "gate_gradient":
        g, u = s["x"].float().chunk(2, -1)
        d, p = s["d"].float(), 1 / (1 + torch.exp(-g))
        return _quantised(torch.cat((d * u * (p * (1 + g * (1 - p))), d * (g * p)), -1), s["to"])
    row_of, token, counts = _sorted_by_expert(s["experts"], s["e"])
    y = s["y"].float()
    back = (y[row_of] * s["weights"].unsqueeze(-1)).sum(1).to(s["y"].dtype)
    if op == "exchange":
        codes, scale = _quantised(s["x"].float(), "e4m3")
        return codes[token], scale[token], row_of, counts, back
    d_out = s["d_out"].float()
    d_x = s["d_sorted"].float()[row_of].sum(1).to(s["x"].dtype)
    d_y = torch.empty_like(y)
    d_y[row_of] = d_out.unsqueeze(1) * s["weights"].unsqueeze(-1)
    d_w = (d_out.unsqueeze(1) * y[row_of]).sum(-1)
    return s["x"][token], counts, back, d_x, d_y.to(s["y"].dtype), d_w


# ---- the same through the framework --------------------------------------------------------------

def _framework(s):
    from tilelang_b200 import moe, ops
    op = s["op"]
    if op == "product":
        return ops.gemm_fp8(s["codes"], s["scale"], ops.Fp8Weight(s["w"], s["w_scale"]), out_dtype=OUT[s["out"]])
    if op == "gradient":
        return ops.gemm_fp8(s["codes"], s["scale"], ops.Fp8Weight(s["w"], s["w_scale"]), trans_w=True,
                            out_dtype=OUT[s["out"]])
    if op == "grouped":
        return ops.gemm_fp8_grouped(s["codes"], s["scale"], ops.Fp8Weight(s["w"], s["w_scale"]), s["counts"],
                                    out_dtype=OUT[s["out"]])
    if op == "gated":
        return ops.gemm_fp8_gated(s["codes"], s["scale"], ops.Fp8Weight(s["w"], s["w_scale"]), s["counts"])
    if op == "quantise":
        return ops.quant_fp8(s["x"], dtype=FP8[s["to"]])
    if op == "gate_gradient":
        return ops.silu_mul_backward_quant_fp8(s["x"], s["d"], dtype=FP8[s["to"]])
    if op == "exchange":
        codes, scale, plan = moe.dispatch_fp8(s["x"], s["experts"], s["e"])
        return codes, scale, plan.row_of, plan.counts, moe.combine(s["y"], plan, s["weights"])
    x, y, weights = (s[n].detach().requires_grad_() for n in ("x", "y", "weights"))
    x_sorted, plan = moe.dispatch(x, s["experts"], s["e"])
    back = moe.combine(y, plan, weights)
    d_x, d_y, d_w = torch.autograd.grad((x_sorted, back), (x, y, weights), (s["d_sorted"], s["d_out"]))
    return x_sorted.detach(), plan.counts, back.detach(), d_x, d_y, d_w


def run(state):
    if own:
        return _framework(state)
    return _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("product", "gradient"):
        m, n, k = case["m"], case["n"], case["k"]
        inner, outer = (k, n) if op == "product" else (n, k)
        scales = 4 * (m * _blocks(inner) + _blocks(n) * _blocks(k))
        return {"bytes": m * inner + n * k + scales + m * outer * OUT[case["out"]].itemsize, "flops": 2.0 * m * n * k}
    if op in ("grouped", "gated"):
        rows, k, e = case["t"] * case["top"], case["k"], case["e"]
        n = case["n"] * (2 if op == "gated" else 1)
        used = e * (1 - (1 - case["top"] / e) ** case["t"])          # experts that some token chose
        written = rows * n * OUT[case["out"]].itemsize if op == "grouped" else rows * (case["n"] + 4 * _blocks(case["n"]))
        return {"bytes": rows * (k + 4 * _blocks(k)) + used * (n * k + 4 * _blocks(n) * _blocks(k)) + written,
                "flops": 2.0 * rows * n * k}
    if op == "quantise":
        return {"bytes": case["m"] * (3 * case["k"] + 4 * _blocks(case["k"])), "flops": 3.0 * case["m"] * case["k"]}
    if op == "gate_gradient":
        return {"bytes": case["m"] * (8 * case["k"] + 4 * _blocks(2 * case["k"])), "flops": 20.0 * case["m"] * case["k"]}
    t, h, rows = case["t"], case["h"], case["t"] * case["top"]
    ids = 8 * rows * 2 + 4 * rows
    if op == "exchange":
        return {"bytes": 2 * t * h + rows * (h + 4 * _blocks(h)) + 2 * rows * h + 2 * t * h + ids, "flops": 2.0 * rows * h}
    # x, y and the two gradients that come in are read, and as much is written
    return {"bytes": 2 * h * 4 * (t + rows) + 2 * ids, "flops": 7.0 * rows * h}


# ---- the definition in 64 bits -------------------------------------------------------------------

def _full(codes, scale, rows):
    """Values in 64 bits of codes with one scale per ``rows`` x 128."""
    n, k = codes.shape
    i = torch.arange(n, device=codes.device) // rows
    j = torch.arange(k, device=codes.device) // BLOCK
    return codes.double() * scale.double()[i[:, None], j[None, :]]


def _largest(x, kind):
    """A row's scale of each 128 columns, in 64 bits."""
    parts = [p.abs().amax(-1, keepdim=True) for p in x.double().split(BLOCK, -1)]
    return torch.cat(parts, -1) / LARGEST[kind]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "product":
        return _full(s["codes"], s["scale"], 1) @ _full(s["w"], s["w_scale"], BLOCK).T
    if op == "gradient":
        return _full(s["codes"], s["scale"], 1) @ _full(s["w"], s["w_scale"], BLOCK)
    if op in ("grouped", "gated"):
        parts, start = [], 0
        for e, c in enumerate(s["counts"].tolist()):
            rows = _full(s["codes"][start:start + c], s["scale"][start:start + c], 1)
            parts.append(rows @ _full(s["w"][e], s["w_scale"][e], BLOCK).T)
            start += c
        y = torch.cat(parts)
        if op == "grouped":
            return y
        g, u = y[:, :case["n"]], y[:, case["n"]:]
        return None, _largest(torch.sigmoid(g) * g * u, "e4m3")      # codes are rounded: a border decides otherwise
    if op == "quantise":
        return None, _largest(s["x"], case["to"])
    if op == "gate_gradient":
        g, u = s["x"].double().chunk(2, -1)
        p, d = torch.sigmoid(g), s["d"].double()
        return None, _largest(torch.cat((d * u * p * (1 + g * (1 - p)), d * g * p), -1), case["to"])
    ids = s["experts"].flatten().tolist()
    order = sorted(range(len(ids)), key=ids.__getitem__)
    row = [0] * len(ids)
    for place, pair in enumerate(order):
        row[pair] = place
    row_of = torch.tensor(row, device=DEVICE).view(s["experts"].shape)
    token = torch.tensor([pair // case["top"] for pair in order], device=DEVICE)
    counts = torch.tensor([ids.count(e) for e in range(case["e"])], device=DEVICE)
    weights, back, d_x, d_w = s["weights"].double(), 0, 0, []
    for k in range(case["top"]):
        back = back + weights[:, k:k + 1] * s["y"][row_of[:, k]].double()
    if op == "exchange":
        return None, _largest(s["x"], "e4m3")[token], row_of, counts, back
    d_y = torch.zeros(len(ids), case["h"], dtype=torch.float64, device=DEVICE)
    for k in range(case["top"]):
        d_x = d_x + s["d_sorted"][row_of[:, k]].double()
        d_y[row_of[:, k]] = weights[:, k:k + 1] * s["d_out"].double()
        d_w.append((s["d_out"].double() * s["y"][row_of[:, k]].double()).sum(-1))
    return s["x"][token], counts, back, d_x, d_y, torch.stack(d_w, 1)
