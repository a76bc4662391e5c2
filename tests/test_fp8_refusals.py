"""CPU: the 8-bit floating point entry points refuse wrong arguments before anything is launched, through the C ABI
and through Python; the argument struct follows the header."""
import ctypes
import os
import re

import pytest
import torch

import tilelang_b200 as tb
from tilelang_b200 import _lib, moe, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20                                  # an address that is never read: every call here is refused first


def test_struct_matches_header_field_order():
    text = open(os.path.join(ROOT, "include", "b200dq.h")).read()
    body = text[text.index("typedef struct b200dq_fp8_gemm_args {"):text.index("} b200dq_fp8_gemm_args;")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    names = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        parts = [p.strip().lstrip("*") for p in decl.split(",")]
        names += [parts[0].split()[-1].lstrip("*"), *parts[1:]]
    assert names == [f[0] for f in _lib.Fp8GemmArgs._fields_]


def good():
    return dict(a=FAKE, a_scale=FAKE, w=FAKE, w_scale=FAKE, c=FAKE, lda=256, ld_a_scale=2, ldw=256, w_group_stride=0,
                M=8, N=256, K=256, out_type=_lib.OUT_BF16)


BAD_GEMM = [
    dict(a=0), dict(a_scale=0), dict(w=0), dict(w_scale=0), dict(c=0), dict(M=0), dict(N=-1), dict(K=0), dict(lda=248),
    dict(lda=240), dict(ldw=264), dict(ldw=128), dict(ld_a_scale=1), dict(a=FAKE + 8), dict(w=FAKE + 1),
    dict(a_scale=FAKE + 2), dict(c=FAKE + 1), dict(a_type=2), dict(w_type=-1), dict(out_type=_lib.OUT_I32),
    dict(token_tile=64), dict(token_tile=256, split=2), dict(split=9), dict(split=-1), dict(num_groups=-1),
    dict(num_groups=2), dict(num_groups=70000, counts=FAKE), dict(num_groups=2, counts=FAKE, w_group_stride=1024),
    dict(num_groups=300, counts=FAKE, w_group_stride=65536, token_tile=256), dict(trans_w=1, lda=128),
    dict(gate_codes=FAKE), dict(gate_codes=FAKE, gate_scales=FAKE, ld_gate=64), dict(gate_codes=FAKE + 4, gate_scales=FAKE, ld_gate=128),
    dict(gate_codes=FAKE, gate_scales=FAKE, ld_gate=128, N=128), dict(gate_codes=FAKE, gate_scales=FAKE, ld_gate=128, trans_w=1),
    dict(gate_codes=FAKE, gate_scales=FAKE, ld_gate=128, gate_type=5), dict(gate_codes=FAKE, gate_scales=FAKE, ld_gate=128, token_tile=16),
    dict(gate_codes=FAKE, gate_scales=FAKE, ld_gate=128, out_type=_lib.OUT_F32),
]


@pytest.mark.parametrize("change", BAD_GEMM)
def test_products_refuse(change):
    lib = _lib.load()
    args = _lib.Fp8GemmArgs(**{**good(), **change})
    assert lib.b200dq_gemm_fp8(ctypes.byref(args), None) == -1
    assert _lib.last_error().startswith("gemm_fp8")


def test_null_struct():
    assert _lib.load().b200dq_gemm_fp8(None, None) == -1 and "null" in _lib.last_error()


def test_quantisers_refuse():
    f = _lib.load().b200dq_quant_fp8
    ok = [0, FAKE, 64, None, 0, FAKE, 64, FAKE, 8, 64, _lib.BF16, _lib.FP8_E4M3, None]
    for at, value in ((0, 3), (0, -1), (1, None), (5, None), (7, None), (8, -1), (9, 0), (2, 63), (6, 63), (10, 3), (11, 2),
                      (1, FAKE + 1), (7, FAKE + 2), (0, 1), (0, 2)):
        args = list(ok)
        args[at] = value
        assert f(*args) == -1 and _lib.last_error().startswith("quant_fp8"), (at, value)
    args = list(ok)
    args[8] = 0
    assert f(*args) == 0                                             # no rows, nothing to do
    g = _lib.load().b200dq_quant_fp8_blocks
    ok = [FAKE, FAKE, 64, FAKE, 1, 64, 64, _lib.F32, _lib.FP8_E5M2, None]
    for at, value in ((0, None), (1, None), (3, None), (2, 63), (4, 0), (4, 65536), (5, 0), (6, -4), (7, 9), (8, 9), (0, FAKE + 2)):
        args = list(ok)
        args[at] = value
        assert g(*args) == -1 and _lib.last_error().startswith("quant_fp8_blocks"), (at, value)


def test_exchange_refuses():
    lib = _lib.load()
    ok = [FAKE, 1, 8, 2, 4, FAKE, 64, 64, _lib.BF16, FAKE, 64, None, 0, FAKE, FAKE, None, 0, None]
    for at, value in ((0, None), (5, None), (9, None), (13, None), (14, None), (2, 0), (3, 0), (4, 0), (4, 1025), (6, 63), (7, 0),
                      (8, 7), (10, 63), (10, 65), (5, FAKE + 1), (2, 1 << 31), (2, 4096)):      # 4096 x 2 pairs need scratch
        args = list(ok)
        args[at] = value
        assert lib.b200dq_exchange_dispatch(*args) == -1 and _lib.last_error().startswith("exchange_dispatch"), (at, value)
    assert lib.b200dq_exchange_scratch_bytes(8, 2, 4) == 0
    assert lib.b200dq_exchange_scratch_bytes(4096, 2, 4) > 0
    ok = [FAKE, FAKE, None, FAKE, 8, 2, 64, _lib.F16, None]
    for at, value in ((0, None), (1, None), (3, None), (4, -1), (5, 0), (6, 0), (7, 3), (0, FAKE + 1)):
        args = list(ok)
        args[at] = value
        assert lib.b200dq_exchange_sum(*args) == -1 and _lib.last_error().startswith("exchange_sum"), (at, value)
    ok = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 8, 2, 64, _lib.F16, None]
    for at, value in ((0, None), (1, None), (2, None), (3, None), (6, -1), (7, 0), (8, 0), (9, 5), (4, FAKE + 1)):
        args = list(ok)
        args[at] = value
        assert lib.b200dq_exchange_sum_grad(*args) == -1 and _lib.last_error().startswith("exchange_sum_grad"), (at, value)


def test_gated_products_are_fused_where_the_pairs_take_them():
    lib = _lib.load()
    assert lib.b200dq_fp8_gated_fuses(98304, 2816, 2048, 64) == 1
    assert lib.b200dq_fp8_gated_fuses(96, 2816, 2048, 64) == 0       # one or two rows an expert
    assert lib.b200dq_fp8_gated_fuses(98304, 2800, 2048, 64) == 0    # halves that are no whole blocks
    assert lib.b200dq_fp8_gated_fuses(0, 2816, 2048, 64) == 0


def test_there_is_no_cpu_path():
    x = torch.zeros(4, 128)
    codes = x.to(torch.float8_e4m3fn)
    w = ops.Fp8Weight(codes, torch.ones(1, 1))
    for f in (lambda: ops.quant_fp8(x), lambda: ops.silu_mul_quant_fp8(x), lambda: ops.quant_fp8_weight(x),
              lambda: ops.gemm_fp8(codes, torch.ones(4, 1), w), lambda: moe.dispatch(x, torch.zeros(4, 1, dtype=torch.int64), 2),
              lambda: moe.combine(x, moe.ExchangePlan(torch.zeros(4, 1, dtype=torch.int64), torch.zeros(2)), torch.ones(4, 1))):
        with pytest.raises(ValueError):
            f()


def test_factory_checks():
    k = tb.matmul_fp8_block(4, 300, 200, "float8_e4m3", "bfloat16", "float32")
    assert [p.name for p in k.params] == ["A", "A_scale", "B", "B_scale", "C"] and k.out_idx == [-1]
    assert k.params[1].shape == (4, 2) and k.params[3].shape == (3, 2)
    with pytest.raises(ValueError):
        k(torch.zeros(4, 200))                                       # wrong input count
    for bad in (dict(in_dtype="int8"), dict(out_dtype="int32"), dict(accum_dtype="float16"), dict(block_size=64),
                dict(weight_dtype="bfloat16")):
        with pytest.raises(ValueError):
            tb.matmul_fp8_block(**{**dict(M=4, N=8, K=16), **bad})


def test_sizes_whose_last_tile_would_pass_32_bits():
    lib = _lib.load()
    for change in (dict(M=2 ** 31 - 1), dict(N=2 ** 31 - 100, trans_w=1, lda=2 ** 31, ld_a_scale=2 ** 24), dict(M=2 ** 31 - 511),
                   dict(K=2 ** 31 - 1, lda=2 ** 31, ldw=2 ** 31, ld_a_scale=2 ** 24)):
        args = _lib.Fp8GemmArgs(**{**good(), **change})
        assert lib.b200dq_gemm_fp8(ctypes.byref(args), None) == -1 and "2^31 - 512" in _lib.last_error(), change
    wide = 2 ** 28 + 16                                              # rows of more than 2^30 bytes
    for f, args in ((lib.b200dq_exchange_dispatch, [FAKE, 1, 1, 1, 4, FAKE, wide, wide, _lib.F32, FAKE, wide, None, 0, FAKE, FAKE, None, 0, None]),
                    (lib.b200dq_exchange_sum, [FAKE, FAKE, None, FAKE, 1, 1, wide, _lib.F32, None]),
                    (lib.b200dq_exchange_sum_grad, [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1, 1, wide, _lib.F32, None])):
        assert f(*args) == -1 and "2^28" in _lib.last_error()


def test_no_gradient_of_tokens_across_ranks():
    w1 = ops.Fp8Weight(torch.zeros(2, 256, 128).to(torch.float8_e4m3fn), torch.ones(2, 2, 1))
    w2 = ops.Fp8Weight(torch.zeros(2, 128, 128).to(torch.float8_e4m3fn), torch.ones(2, 1, 1))
    x = torch.zeros(4, 128, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient of the tokens"):
        moe.moe_forward_ep(x, torch.zeros(4, 2), 1, 2, moe.Fp8ExpertMLP(w1, w2))
