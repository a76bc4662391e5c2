"""CPU: calls of the 8-bit floating point C entries that have to be refused on the host, since no kernel takes them."""
import ctypes

import pytest

from tilelang_b200 import _lib

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
