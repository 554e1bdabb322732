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
