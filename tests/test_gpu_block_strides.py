"""Layouts that the strides of vf_block_matrix allow beside the dense ones: matrices of a stack whose rows lie in turn, strides of
matrices, scales that share a row with others."""
import numpy as np
import pytest

import block_reference as br
from test_gpu_blocks import E4M3, F32, check_product, device_content, operands, torch, weight_values  # noqa: F401 - torch is a fixture
from vpux_plugin_b200 import abi

pytestmark = pytest.mark.gpu


class Strided:
    """codes[i][r][c] and scales[i][rb][cb] on the device at the strides given (in elements), 0xA5 and -7 elsewhere"""

    def __init__(self, torch, count, rows, cols, block_rows, ld, matrix_stride, scale_strides, codes=None, scales=None):  # noqa: F811
        self.rb, self.cb = -(-rows // block_rows), -(-cols // 128)
        sms, srs, scs = scale_strides
        n = (count - 1) * matrix_stride + (rows - 1) * ld + cols
        ns = (count - 1) * sms + (self.rb - 1) * srs + (self.cb - 1) * scs + 1
        self.buf = torch.full((n + 32,), 0xA5, dtype=torch.uint8, device="cuda")
        self.sbuf = torch.full((ns + 32,), -7.0, device="cuda")
        self.codes = self.buf.as_strided((count, rows, cols), (matrix_stride, ld, 1))
        self.scales = self.sbuf.as_strided((count, self.rb, self.cb), (sms, srs, scs))
        if codes is not None:
            self.codes.copy_(torch.from_numpy(codes).view(count, rows, cols))
            self.scales.copy_(torch.from_numpy(scales).view(count, self.rb, self.cb))
        torch.cuda.synchronize()
        self.pod = abi.block_matrix(self.buf.data_ptr(), self.sbuf.data_ptr(), E4M3, block_rows, rows, cols, count=count, ld=ld, matrix_stride=matrix_stride,
                                    scale_matrix_stride=sms, scale_row_stride=srs, scale_col_stride=scs)

    def untouched_elsewhere(self):
        b, s = self.buf.clone(), self.sbuf.clone()
        b.as_strided(self.codes.shape, self.codes.stride()).fill_(0xA5)
        s.as_strided(self.scales.shape, self.scales.stride()).fill_(-7.0)
        return bool((b == 0xA5).all()) and bool((s == -7.0).all())


def layouts(count, rows, cols, block_rows):
    """ld, matrix stride, scale strides (matrix, row block, column block)"""
    rb, cb, p = -(-rows // block_rows), -(-cols // 128), -(-cols // 16) * 16
    return [(count * p, p, (cb, count * cb, 1)),                      # rows of all matrices in turn, scales as well
            (p + 32, (p + 32) * rows + 64, (rb * cb + 3, 1, rb)),     # gaps everywhere, scales column block by column block
            (count * p + 16, p, (1, count * cb, count)),              # in turn with a gap, the matrices' scales innermost
            (cols + 1, (cols + 1) * rows, (rb * (cb + 2), cb + 2, 1))]


@pytest.mark.parametrize("layout", range(4))
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantise_and_read_back(gpu, torch, layout, block_rows):  # noqa: F811
    rng = np.random.default_rng(500 + layout)
    count, rows, cols = 3, 140, 300
    x = weight_values(rng, (count, rows, cols))
    src = torch.from_numpy(x).cuda()
    m = Strided(torch, count, rows, cols, block_rows, *layouts(count, rows, cols, block_rows)[layout])
    c, keep = device_content(torch, src, F32, (count, rows, cols))
    gpu.quantize_blocks(c, m.pod)
    codes, scales = br.quantize(x, block_rows, E4M3)
    assert np.array_equal(m.codes.cpu().numpy(), codes) and np.array_equal(m.scales.cpu().numpy(), scales)
    assert m.untouched_elsewhere()
    back = torch.zeros(count, rows, cols, device="cuda")
    torch.cuda.synchronize()
    gpu.dequantize_blocks(m.pod, back.data_ptr(), F32, back.nbytes)
    assert np.array_equal(back.cpu().numpy(), br.values(codes, scales, block_rows, E4M3).astype(np.float32))


@pytest.mark.parametrize("layout", range(4))
@pytest.mark.parametrize("rows,k", [(5, 300), (40, 2100), (333, 300), (1200, 1100)])
def test_grouped_product(gpu, torch, layout, rows, k):  # noqa: F811
    rng = np.random.default_rng(600 + layout)
    count, n = 3, 270
    xc, xs, wc, ws = operands(rng, rows, n, k, E4M3, E4M3, count)
    w = Strided(torch, count, n, k, 128, *layouts(count, n, k, 128)[layout], codes=wc, scales=ws)
    ld, _, (_, srs, scs) = layouts(1, rows, k, 1)[layout]
    x = Strided(torch, 1, rows, k, 1, ld, rows * ld, (1 << 20, srs, scs), codes=xc, scales=xs)
    offsets = [0, rows // 3, rows // 3, rows]
    offs = torch.tensor(offsets, device="cuda")
    out = torch.zeros(rows, n, device="cuda")
    torch.cuda.synchronize()
    gpu.matmul_blocks_grouped(x.pod, w.pod, offs.data_ptr(), out.data_ptr(), F32, out.nbytes)
    for e in range(count):
        check_product(out.double().cpu().numpy(), xc, xs, wc, ws, E4M3, E4M3, F32, offsets[e], offsets[e + 1], e)
