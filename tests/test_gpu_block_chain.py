"""Calls that wait for nothing in between, each reading what the one before wrote and rewriting what the one before that read, give
the same bits as the same calls one by one."""
import numpy as np
import pytest

import block_reference as br
from test_gpu_blocks import E4M3, F32, Matrix, device_content, torch  # noqa: F401 - torch is a fixture
from vpux_plugin_b200 import abi
from vpux_plugin_b200.lib import Library

pytestmark = pytest.mark.gpu

N = 256
STEPS = 150


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("m", [1, 7, 40, 300])
def test_a_chain(torch, m, offset, grouped):  # noqa: F811
    rng = np.random.default_rng(700 + m)
    turn = np.linalg.qr(rng.standard_normal((N, N)))[0].astype(np.float32)  # keeps a row's length, so 150 steps neither grow nor fade
    wc, ws = br.quantize(np.stack([turn, turn.T]), 128, E4M3)
    w = Matrix(torch, N, N, 128, count=2, codes=wc, scales=ws)
    one = abi.block_matrix(w.buf.data_ptr(), w.sbuf.data_ptr(), E4M3, 128, N, N)
    x = Matrix(torch, m, N, 1, col_major=True)
    start = torch.from_numpy(rng.standard_normal((m, N)).astype(np.float32))
    buf = torch.zeros(m * N + 8, device="cuda")
    y = buf[offset:offset + m * N].view(m, N)  # at offset 1 the quantiser takes single elements
    c, keep = device_content(torch, y, F32, (m, N))
    offs = torch.tensor([0, m // 2, m], device="cuda")

    def run(lib):
        y.copy_(start)
        torch.cuda.synchronize()
        for _ in range(STEPS):
            lib.quantize_blocks(c, x.pod)
            if grouped:
                lib.matmul_blocks_grouped(x.pod, w.pod, offs.data_ptr(), y.data_ptr(), F32, y.nbytes)
            else:
                lib.matmul_blocks(x.pod, one, y.data_ptr(), F32, y.nbytes)
            lib.quantize_blocks(c, x.pod)
            lib.dequantize_blocks(x.pod, y.data_ptr(), F32, y.nbytes)
        lib.synchronize()
        return y.clone()

    waiting, pipelined = Library(device=0), Library(device=0, pipelined=True)
    want = run(waiting)
    assert 0.1 < float(want.norm() / start.norm()) < 10
    for _ in range(3):
        assert torch.equal(run(pipelined), want)
    waiting.close()
    pipelined.close()
