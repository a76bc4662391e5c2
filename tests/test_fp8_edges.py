"""CPU: calls of the 8-bit floating point C entries that have to be refused on the host, since no kernel takes them."""
import ctypes

import pytest
import torch
from torch._subclasses import FakeTensorMode

from tilelang_b200 import _lib, moe, ops

FAKE = 1 << 20                                  # an address that is never read: every call here is refused first


def product(**change):
    args = dict(a=FAKE, a_scale=FAKE, w=FAKE, w_scale=FAKE, c=FAKE, lda=256, ld_a_scale=2, ldw=256, w_group_stride=256 * 256,
                M=4096, N=256, K=256, out_type=_lib.OUT_BF16)
    args.update(change)
    return _lib.Fp8GemmArgs(**args)


GATED = dict(gate_codes=FAKE, gate_scales=FAKE, ld_gate=128, counts=FAKE)


@pytest.mark.parametrize("groups", [257, 300, 65535])
@pytest.mark.parametrize("more", [dict(token_tile=0), dict(token_tile=256), dict(token_tile=0, c=None)])
def test_gated_products_of_more_groups_than_the_tile_table_holds(groups, more):
    lib = _lib.load()
    args = product(num_groups=groups, **GATED, **more)
    assert lib.b200dq_gemm_fp8(ctypes.byref(args), None) == -1 and "at most 256 groups" in _lib.last_error()
    assert lib.b200dq_fp8_gated_fuses(1 << 20, 256, 256, groups) == 0
    assert lib.b200dq_fp8_gated_fuses(1 << 20, 256, 256, 256) == 1


@pytest.mark.parametrize("change", [dict(a_scale=FAKE + 2), dict(w_scale=FAKE + 1), dict(c=FAKE + 1), dict(**{**GATED, "gate_scales": FAKE + 2}),
                                    dict(num_groups=2, counts=FAKE + 2), dict(num_groups=2, counts=FAKE + 4, counts_int64=1),
                                    dict(out_type=_lib.OUT_F32, c=FAKE + 2)])
def test_products_refuse_pointers_between_elements(change):
    args = product(**change)
    assert _lib.load().b200dq_gemm_fp8(ctypes.byref(args), None) == -1 and "aligned" in _lib.last_error()


def test_the_exchange_refuses_pointers_between_elements():
    """Every array of a call: an address inside an element would be a misaligned access."""
    lib = _lib.load()
    # experts 0, int64 1, x 5, out 9, scales 11, row_of 13, counts 14, scratch 15
    dispatch = [FAKE, 1, 8, 2, 4, FAKE, 64, 64, _lib.BF16, FAKE, 64, FAKE, 0, FAKE, FAKE, FAKE, 0, None]
    total = [FAKE, FAKE, FAKE, FAKE, 8, 2, 64, _lib.F32, None]
    grad = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 8, 2, 64, _lib.F32, None]
    for f, args, wrong in ((lib.b200dq_exchange_dispatch, dispatch, [(0, 4), (5, 1), (11, 2), (13, 4), (14, 4), (15, 2)]),
                           (lib.b200dq_exchange_sum, total, [(0, 2), (1, 4), (2, 2), (3, 2)]),
                           (lib.b200dq_exchange_sum_grad, grad, [(0, 2), (1, 2), (2, 4), (3, 2), (4, 2), (5, 1)])):
        for at, by in wrong:
            bad = list(args)
            bad[at] += by
            assert f(*bad) == -1 and "aligned" in _lib.last_error(), (f.__name__, at)
    ids32 = list(dispatch)
    ids32[0], ids32[1] = FAKE + 2, 0
    assert lib.b200dq_exchange_dispatch(*ids32) == -1 and "aligned" in _lib.last_error()


def test_sizes_that_the_c_calls_would_cut_to_32_bits():
    """2^32 + 8 columns would arrive as 8 of them."""
    with FakeTensorMode():                                           # sizes alone: nothing is allocated
        def new(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        one = new(1, 1, dtype=torch.int64)
        for width in (2 ** 28 + 8, 2 ** 32 + 8):
            with pytest.raises(ValueError, match="2\\^28"):
                moe.combine_rows(new(1, width), one, new(1, 1))
        many = 2 ** 32 + 2
        with pytest.raises(ValueError, match="2\\^31"):
            moe.combine_rows(new(many, 8), new(1, many, dtype=torch.int64), new(1, many))
        for dispatch in (moe.dispatch, moe.dispatch_fp8):
            with pytest.raises(ValueError, match="2\\^31"):
                dispatch(new(1, 8), new(1, many, dtype=torch.int64), 4)
            with pytest.raises(ValueError, match="2\\^31"):
                dispatch(new(2 ** 28, 8), new(2 ** 28, 8, dtype=torch.int64), 4)
        for shape in ((1, 2 ** 32 + 8), (2 ** 32 + 8, 1), (1, 2 ** 31, 1)):
            with pytest.raises(ValueError, match="2\\^31"):
                ops.quant_fp8_weight(new(*shape))
        for f in (ops.quant_fp8, ops.silu_mul_quant_fp8):
            with pytest.raises(ValueError, match="2\\^31"):
                f(new(1, 2 ** 32 + 256))
