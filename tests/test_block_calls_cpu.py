"""Refusals of the calls on 8-bit floating-point blocks that need no device, beside those in test_blocks_cpu.py."""
import pytest

from test_blocks_cpu import AT, BF16, matrix, refused
from vpux_plugin_b200 import abi


@pytest.mark.parametrize("offsets", [8 * AT, 8 * AT + 8, 8 * AT - 24, 8 * AT + 64 - 8])
def test_a_result_over_its_offsets(offsets):
    x, w = matrix(4, 256, 1), matrix(8, 256, 128, codes=4 * AT, scales=5 * AT, count=3)
    name = "vf_matmul_blocks_grouped"
    refused(abi.VF_ERR_INVALID_ARG, "the result and the offsets overlap", name, x, w, offsets, 8 * AT, BF16, 0, 4 * 8 * 2)
    for apart in (8 * AT - 32, 8 * AT + 64):  # four offsets in front of the result, or behind it
        refused(abi.VF_ERR_INVALID_ARG, "ctx is NULL", name, x, w, apart, 8 * AT, BF16, 0, 4 * 8 * 2)


def test_more_tiles_than_can_be_counted():
    """Refused before anything is enqueued, whichever kernel would run; the count is of tiles of 16 rows by 64 columns."""
    wide = dict(out=1 << 60, dt=BF16, ld=0, nbytes=1 << 62)

    def call(status, words, rows, outputs, experts=0, ld=0):
        x = matrix(rows, 16, 1, codes=1 << 40, scales=2 << 40)
        w = matrix(outputs, 16, 128, codes=3 << 40, scales=7 << 40, count=experts or 1, ld=ld)
        args = tuple(wide.values())
        if experts:
            refused(status, words, "vf_matmul_blocks_grouped", x, w, 15 << 50, *args)
        else:
            refused(status, words, "vf_matmul_blocks", x, w, *args)

    too_many, fine = (abi.VF_ERR_CAPACITY, "too many tiles"), (abi.VF_ERR_INVALID_ARG, "ctx is NULL")
    call(*too_many, 1 << 30, 1 << 21)
    call(*too_many, 1 << 30, 1 << 21, ld=17)
    call(*fine, 1 << 26, 32 * 511 * 2)          # 2^22 * 511
    call(*too_many, 1 << 26, 32 * 512 * 2)
    call(*too_many, 1 << 30, 128, 1 << 30)      # every expert may end inside a tile
    call(*fine, 1 << 30, 64, 1 << 29)
    call(*fine, 1 << 30, 0)
    call(*fine, 0, 1 << 30)
