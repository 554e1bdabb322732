"""What kernels find is reported once, by the right call: around recorded and replayed graphs, and behind calls that failed."""
import ctypes as C

import numpy as np
import pytest

import block_reference as br
from test_gpu_blocks import E4M3, F32, Matrix, device_content, torch, weight_values  # noqa: F401 - torch is a fixture
from vpux_plugin_b200 import abi
from vpux_plugin_b200.lib import Library, VfoldError

pytestmark = pytest.mark.gpu


class Tokens:
    """A pipelined context on a stream of its own, whose quantising call is recorded into a graph."""

    def __init__(self, torch, seed):  # noqa: F811
        rng = np.random.default_rng(seed)
        self.torch, self.stream = torch, torch.cuda.Stream()
        self.lib = Library(device=0, stream=self.stream.cuda_stream, pipelined=True)
        self.good = torch.from_numpy(weight_values(rng, (5, 300)))
        self.bad = self.good.clone()
        self.bad[3, 200] = float("nan")
        self.src = self.good.cuda()
        self.m = Matrix(torch, 5, 300, 1)
        self.content, self.keep = device_content(torch, self.src, F32, (5, 300))
        torch.cuda.synchronize()

    def quantize(self):
        self.lib.quantize_blocks(self.content, self.m.pod)

    def put(self, x):
        self.src.copy_(x)
        self.torch.cuda.synchronize()

    def record(self):
        self.graph = self.torch.cuda.CUDAGraph()
        with self.torch.cuda.graph(self.graph, stream=self.stream):
            self.quantize()

    def replay(self, x):
        self.put(x)
        self.graph.replay()
        self.torch.cuda.synchronize()

    def waits_for(self, status):
        if status is None:
            return self.lib.synchronize()
        with pytest.raises(VfoldError) as e:
            self.lib.synchronize()
        assert e.value.status == status

    def close(self):
        self.graph = None
        self.lib.close()


def refused(lib):
    """A call that fails when it is under way, before it has enqueued anything."""
    with pytest.raises(VfoldError) as e:
        lib.weights_table_batch((abi.WeightsTableJob * 1)(), out_mem_kind=abi.VF_MEM_DEVICE)
    assert e.value.status == abi.VF_ERR_INVALID_ARG and "table is NULL" in str(e.value)


def test_a_graph_recorded_behind_an_error_keeps_what_its_replays_find(torch):  # noqa: F811
    t = Tokens(torch, 1)
    t.put(t.bad)
    t.quantize()
    t.waits_for(abi.VF_ERR_NAN)
    t.record()  # nothing in it may clear the flags
    t.replay(t.bad)
    t.replay(t.good)
    t.quantize()
    t.waits_for(abi.VF_ERR_NAN)
    t.quantize()
    t.waits_for(None)
    t.close()


def test_a_call_behind_an_error_keeps_what_a_replay_found(torch):  # noqa: F811
    t = Tokens(torch, 2)
    t.record()
    t.waits_for(None)
    t.put(t.bad)
    t.quantize()
    t.waits_for(abi.VF_ERR_NAN)
    t.replay(t.bad)
    t.put(t.good)
    t.quantize()
    t.waits_for(abi.VF_ERR_NAN)
    t.replay(t.good)
    t.quantize()
    t.waits_for(None)
    t.close()


def test_a_refused_call_keeps_what_a_replay_found(torch):  # noqa: F811
    t = Tokens(torch, 3)
    t.record()
    t.waits_for(None)
    t.replay(t.bad)
    refused(t.lib)
    t.put(t.good)
    t.quantize()
    t.waits_for(abi.VF_ERR_NAN)
    t.close()


def test_a_refused_call_does_not_end_a_recording(torch):  # noqa: F811
    t = Tokens(torch, 5)
    t.graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(t.graph, stream=t.stream):
        refused(t.lib)
        t.quantize()
        refused(t.lib)
    t.replay(t.good)
    codes, scales = br.quantize(t.good.numpy(), 1, E4M3)
    assert np.array_equal(t.m.codes()[0], codes) and np.array_equal(t.m.scales()[0], scales)
    t.waits_for(None)
    t.close()


def test_an_error_is_reported_once(gpu, torch):  # noqa: F811
    """Errors of synchronous calls, of every kind of call in turn, are not seen by the calls behind them."""
    rng = np.random.default_rng(4)
    x = weight_values(rng, (6, 256))
    good = torch.from_numpy(x).cuda()
    bad = good.clone()
    bad[2, 2] = float("inf")
    m = Matrix(torch, 6, 256, 1)
    cg, k1 = device_content(torch, good, F32, (6, 256))
    cb, k2 = device_content(torch, bad, F32, (6, 256))
    torch.cuda.synchronize()
    data, counts = torch.zeros(8, dtype=torch.uint8, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    weights = torch.ones(6, 64, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        with pytest.raises(VfoldError) as e:
            gpu.quantize_blocks(cb, m.pod)
        assert e.value.status == abi.VF_ERR_QUANT_RANGE
        gpu.quantize_blocks(cg, m.pod)
        written, err = C.c_uint64(0), C.create_string_buffer(512)  # too small a buffer: the kernel notices as well
        st = gpu.lib.vf_sparsify_noalloc(gpu.ctx, C.c_void_p(weights.data_ptr()), C.c_int32(abi.VF_DT_U8), C.c_int64(6), C.c_int64(64), C.c_int64(0),
                                         C.c_void_p(data.data_ptr()), C.c_uint64(8), C.byref(written), None, C.c_uint64(0),
                                         C.c_void_p(counts.data_ptr()), err, C.c_size_t(512))
        assert st == abi.VF_ERR_BUFFER_TOO_SMALL and written.value >= 6 * 64
        gpu.quantize_blocks(cg, m.pod)
