"""Refusals of the calls on 8-bit floating-point blocks that need no device, beside those in test_blocks_cpu.py."""
import numpy as np
import pytest

from test_blocks_cpu import AT, BF16, DEV, E4M3, F32, HOST, matrix, refused
from vpux_plugin_b200 import abi
from vpux_plugin_b200.lib import Library


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


def test_arrays_are_host_memory():
    """A host address is never handed on as one of device memory."""
    q, s = np.zeros((4, 256), np.uint8), np.zeros((4, 2), np.float32)
    assert abi.block_matrix(q, s, E4M3, 1, 4, 256).mem_kind == HOST
    assert abi.block_matrix(AT, 2 * AT, E4M3, 1, 4, 256).mem_kind == DEV
    assert abi.block_matrix(None, None, E4M3, 1, 0, 256).mem_kind == DEV
    assert abi.block_matrix(q, 2 * AT, E4M3, 1, 4, 256, mem_kind=abi.VF_MEM_HOST_PINNED).mem_kind == abi.VF_MEM_HOST_PINNED
    for args, kw in (((q, s), {"mem_kind": DEV}), ((q, 2 * AT), {}), ((AT, s), {}), ((AT, s), {"mem_kind": DEV}),
                     ((q, s.astype(np.float64)), {}), ((q.astype(np.int32), s), {}), ((np.zeros((4, 512), np.uint8)[:, ::2], s), {})):
        with pytest.raises(ValueError):
            abi.block_matrix(*args, E4M3, 1, 4, 256, **kw)


def test_reading_back_into_an_array():
    """Checked before the library is called: the object below has no context."""
    lib = Library.__new__(Library)
    lib.ctx = None
    m = matrix(4, 256, 1)
    y = np.zeros((4, 256), np.float32)
    for dst, nbytes, kw in ((y, y.nbytes, {"dst_mem_kind": DEV}), (y, y.nbytes + 1, {}), (y[:, ::2], 2048, {})):
        with pytest.raises(ValueError):
            lib.dequantize_blocks(m, dst, F32, nbytes, **kw)
