"""8-bit floating-point blocks on the GPU against their restatement in 64 bits (block_reference.py): quantising and
reading back bit for bit, products within the error their arithmetic can make, each at the sizes, strides, types and
group borders where a kernel can go wrong, and a run of them together."""
import os
import threading

import numpy as np
import pytest

import block_reference as br
from vpux_plugin_b200 import abi
from vpux_plugin_b200.lib import Library, VfoldError

pytestmark = pytest.mark.gpu

E4M3, E5M2 = abi.VF_DT_F8E4M3FN, abi.VF_DT_F8E5M2
F32, F16, BF16 = abi.VF_DT_F32, abi.VF_DT_F16, abi.VF_DT_BF16
DEV, HOST = abi.VF_MEM_DEVICE, abi.VF_MEM_HOST
GUARD = 0xA5
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def wide_type(torch, dt):
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[dt]


def to_device(torch, x, dt=None, offset=0):
    """A device buffer that holds x (numpy) as `dt`, `offset` elements from an aligned start; returns (view, keepalive)."""
    t = torch.from_numpy(np.ascontiguousarray(x))
    if dt is not None:
        t = t.to(wide_type(torch, dt))
    buf = torch.empty(t.numel() + offset + 64, dtype=t.dtype, device="cuda")
    v = buf[offset:offset + t.numel()].view(t.shape)
    v.copy_(t)
    return v, buf


def host_f32(torch, x, dt):
    """What the device sees after x (float32) was stored as dt."""
    return torch.from_numpy(x).to(wide_type(torch, dt)).float().numpy()


class Matrix:
    """A vf_block_matrix on the device with guard bytes around and between its elements."""

    def __init__(self, torch, rows, cols, block_rows, dtype=E4M3, count=1, ld=0, col_major=False, offset=0, codes=None, scales=None):
        self.torch, self.dtype, self.block_rows, self.count, self.rows, self.cols = torch, dtype, block_rows, count, rows, cols
        self.ld = ld or cols
        self.offset, self.col_major = offset, col_major
        self.rb, self.cb = -(-rows // block_rows), -(-cols // 128)
        self.buf = torch.full((offset + count * rows * self.ld + 64,), GUARD, dtype=torch.uint8, device="cuda")
        self.sbuf = torch.full((count * self.rb * self.cb + 16,), -7.0, device="cuda")
        if codes is not None:
            self.code_view().copy_(torch.from_numpy(codes).view(count, rows, cols))
            self.scale_view().copy_(torch.from_numpy(scales.astype(np.float32)).view(count, self.rb, self.cb))
        torch.cuda.synchronize()
        strides = {"scale_row_stride": 1, "scale_col_stride": self.rb} if col_major else {}
        self.pod = abi.block_matrix(self.buf.data_ptr() + offset, self.sbuf.data_ptr(), dtype, block_rows, rows, cols, count=count, ld=ld, **strides)

    def code_view(self):
        n = self.count * self.rows * self.ld
        return self.buf[self.offset:self.offset + n].view(self.count, self.rows, self.ld)[:, :, :self.cols]

    def scale_view(self):
        n = self.count * self.rb * self.cb
        if self.col_major:
            return self.sbuf[:n].view(self.count, self.cb, self.rb).transpose(1, 2)
        return self.sbuf[:n].view(self.count, self.rb, self.cb)

    def codes(self):
        return self.code_view().cpu().numpy().copy()

    def scales(self):
        return self.scale_view().cpu().numpy().copy()

    def guards_intact(self):
        b = self.buf.clone()
        n = self.count * self.rows * self.ld
        b[self.offset:self.offset + n].view(self.count, self.rows, self.ld)[:, :, :self.cols] = GUARD
        return bool((b == GUARD).all()) and bool((self.sbuf[self.count * self.rb * self.cb:] == -7.0).all())


def weight_values(rng, shape, sigma=0.02):
    x = rng.standard_normal(shape) * sigma
    return np.where(rng.random(shape) < 0.01, x * 20, x).astype(np.float32)


def device_content(torch, x, dt, shape, base_ld=0):
    es = abi.DTYPE_BITS[dt] // 8
    n = int(np.prod(shape[:-1])) * (base_ld or shape[-1]) * es
    return abi.make_content(abi.TType(list(shape), dt), None, ptr=x.data_ptr(), nbytes=n, mem_kind=DEV)


# ---- quantising ----------------------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (1, 128), (1, 4096), (3, 127), (5, 129), (33, 256), (130, 257), (128, 128), (129, 384), (300, 1000)]


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_is_the_definition(gpu, torch, block_rows, dt, dtype):
    rng = np.random.default_rng(7)
    for rows, cols in SHAPES:
        x = host_f32(torch, weight_values(rng, (rows, cols)), dt)
        src, keep = to_device(torch, x, dt)
        m = Matrix(torch, rows, cols, block_rows, dtype, ld=-(-cols // 16) * 16, col_major=block_rows == 1)
        c, k = device_content(torch, src, dt, (rows, cols))
        gpu.quantize_blocks(c, m.pod)
        codes, scales = br.quantize(x, block_rows, dtype)
        assert np.array_equal(m.scales()[0], scales), (rows, cols)
        assert np.array_equal(m.codes()[0], codes), (rows, cols)
        assert m.guards_intact()
        assert gpu.last_stats.kernels_launched == 1


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dt,src_offset,src_ld,ld,offset", [(BF16, 0, 300, 300, 0), (BF16, 1, 257, 272, 0), (F16, 0, 264, 257, 3), (F32, 3, 261, 263, 1), (F32, 0, 260, 264, 8)])
def test_quantize_strides_and_alignments(gpu, torch, block_rows, dt, src_offset, src_ld, ld, offset):
    rng = np.random.default_rng(8)
    rows, cols = 131, 257
    full = host_f32(torch, weight_values(rng, (rows, src_ld)), dt)
    src, keep = to_device(torch, full, dt, offset=src_offset)
    for col_major in (False, True):
        m = Matrix(torch, rows, cols, block_rows, ld=ld, offset=offset, col_major=col_major)
        c, k = device_content(torch, src, dt, (rows, cols), src_ld)
        gpu.quantize_blocks(c, m.pod, base_ld=src_ld)
        codes, scales = br.quantize(full[:, :cols], block_rows, E4M3)
        assert np.array_equal(m.scales()[0], scales) and np.array_equal(m.codes()[0], codes) and m.guards_intact()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_a_stack_of_matrices(gpu, torch, block_rows):
    rng = np.random.default_rng(9)
    x = weight_values(rng, (3, 150, 200))
    src, keep = to_device(torch, x, F32)
    m = Matrix(torch, 150, 200, block_rows, count=3, ld=208)
    c, k = device_content(torch, src, F32, (3, 150, 200))
    gpu.quantize_blocks(c, m.pod)
    codes, scales = br.quantize(x, block_rows, E4M3)
    assert np.array_equal(m.scales(), scales) and np.array_equal(m.codes(), codes) and m.guards_intact()


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extreme_magnitudes(gpu, torch, block_rows, dtype):
    """Zeros of both signs, subnormal numbers, the largest number, ties between two codes."""
    x = np.zeros((260, 384), np.float32)
    x[0, :128] = -0.0
    x[130, 3] = 1e-45
    x[131, 130:140] = np.float32(2.0 ** -140) * np.arange(10)
    x[132, 256:] = np.finfo(np.float32).max * np.linspace(-1, 1, 128).astype(np.float32)
    top = br.code_values(dtype)
    mid = np.sort(top[np.isfinite(top)])
    ties = ((mid[1:] + mid[:-1]) / 2).astype(np.float32)
    x[3, 256:256 + 127] = ties[:127]
    x[3, 383] = br.LARGEST[dtype]
    src, keep = to_device(torch, x, F32)
    m = Matrix(torch, 260, 384, block_rows, dtype)
    c, k = device_content(torch, src, F32, (260, 384))
    gpu.quantize_blocks(c, m.pod)
    codes, scales = br.quantize(x, block_rows, dtype)
    assert np.array_equal(m.scales()[0], scales) and np.array_equal(m.codes()[0], codes)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("bad,status", [(np.nan, abi.VF_ERR_NAN), (np.inf, abi.VF_ERR_QUANT_RANGE), (-np.inf, abi.VF_ERR_QUANT_RANGE)])
def test_quantize_reports_what_is_not_finite(gpu, torch, block_rows, dt, bad, status):
    rng = np.random.default_rng(10)
    x = host_f32(torch, weight_values(rng, (140, 300)), dt)
    codes, scales = br.quantize(x, block_rows, E4M3)
    x[135, 140] = bad
    src, keep = to_device(torch, x, dt)
    m = Matrix(torch, 140, 300, block_rows)
    c, k = device_content(torch, src, dt, (140, 300))
    with pytest.raises(VfoldError) as e:
        gpu.quantize_blocks(c, m.pod)
    assert e.value.status == status
    other = np.ones((140, 300), bool)  # the other blocks are complete
    other[135 if block_rows == 1 else slice(128, 140), 128:256] = False
    assert np.array_equal(m.codes()[0][other], codes[other])
    x[135, 140] = 0  # and the context goes on
    src.copy_(torch.from_numpy(x).to(src.dtype))
    torch.cuda.synchronize()
    gpu.quantize_blocks(c, m.pod)
    assert np.array_equal(m.codes()[0], br.quantize(x, block_rows, E4M3)[0])


@pytest.mark.parametrize("block_rows", [1, 128])
def test_host_memory_both_ways(gpu, block_rows):
    rng = np.random.default_rng(11)
    x = weight_values(rng, (2, 140, 300))
    c, keep = abi.make_content(abi.TType([2, 140, 300], F32), x)
    codes, scales = br.quantize(x, block_rows, E4M3)
    q, s = np.zeros((2, 140, 300), np.uint8), np.zeros_like(scales)
    m = abi.block_matrix(q, s, E4M3, block_rows, 140, 300, count=2, mem_kind=HOST)
    gpu.quantize_blocks(c, m)
    assert np.array_equal(q, codes) and np.array_equal(s, scales)
    assert gpu.last_stats.h2d_bytes == x.nbytes and gpu.last_stats.d2h_bytes == q.nbytes + s.nbytes
    back = np.zeros_like(x)
    gpu.dequantize_blocks(m, back, F32, back.nbytes, dst_mem_kind=HOST)
    assert np.array_equal(back, br.values(codes, scales, block_rows, E4M3).astype(np.float32))


def test_nothing_to_quantize(gpu, torch):
    src, keep = to_device(torch, np.zeros(8, np.float32), F32)
    c, k = device_content(torch, src, F32, (0, 256))
    gpu.quantize_blocks(c, abi.block_matrix(None, None, E4M3, 1, 0, 256))
    gpu.dequantize_blocks(abi.block_matrix(None, None, E4M3, 1, 0, 256), None, F32, 0)
    assert gpu.last_stats.kernels_launched == 0


# ---- reading back ----------------------------------------------------------------------------------------------------------

def rounded(torch, v, dt):
    """float64 values -> fp32 (the product of code and scale) -> dt, both to nearest even; as float32."""
    with np.errstate(over="ignore", invalid="ignore"):
        f = v.astype(np.float32)
    return torch.from_numpy(f).to(wide_type(torch, dt)).float().numpy()


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,block_rows,ld,offset,dst_ld,dst_offset", [
    (1, 1, 1, 0, 0, 0, 0), (3, 256, 1, 0, 0, 0, 0), (130, 300, 128, 304, 0, 320, 0), (130, 300, 1, 301, 5, 303, 1), (257, 1111, 128, 1120, 0, 1112, 0)])
def test_dequantize_every_code(gpu, torch, rows, cols, block_rows, ld, offset, dst_ld, dst_offset, dt, dtype):
    rng = np.random.default_rng(12)
    codes = rng.integers(0, 256, (rows, cols)).astype(np.uint8)  # NaN and infinity among them
    scales = np.exp2(rng.uniform(-12, 6, (-(-rows // block_rows), -(-cols // 128)))).astype(np.float32)
    scales.flat[0] = 2.0 ** -126
    m = Matrix(torch, rows, cols, block_rows, dtype, ld=ld, offset=offset, col_major=block_rows == 1, codes=codes, scales=scales)
    step = dst_ld or cols
    dst = torch.full((dst_offset + rows * step + 8,), 3.0, dtype=wide_type(torch, dt), device="cuda")
    torch.cuda.synchronize()
    view = dst[dst_offset:dst_offset + rows * step].view(rows, step)
    gpu.dequantize_blocks(m.pod, view.data_ptr(), dt, view.nbytes, dst_ld=dst_ld)
    want = rounded(torch, br.values(codes, scales, block_rows, dtype), dt)
    assert np.array_equal(view[:, :cols].float().cpu().numpy(), want, equal_nan=True)
    view[:, :cols] = 3.0
    assert bool((dst == 3.0).all())


# ---- products ------------------------------------------------------------------------------------------------------------

def operands(rng, m, n, k, xt, wt, count=1):
    xc, xs = br.quantize(rng.standard_normal((m, k)).astype(np.float32), 1, xt)
    wc, ws = br.quantize(weight_values(rng, (count, n, k)), 128, wt)
    return xc, xs, wc, ws


def up16(k):
    return -(-k // 16) * 16


def run_product(gpu, torch, xc, xs, wc, ws, xt, wt, out_dt, offsets=None, x_kw=None, w_kw=None, out_ld=0, out_offset=0):
    """out (float64) of the product, checked for writes outside of it; rows that no group owns keep the value 3."""
    m, k = xc.shape
    count, n = wc.shape[:2]
    x = Matrix(torch, m, k, 1, xt, codes=xc, scales=xs, **({"ld": up16(k), "col_major": True} if x_kw is None else x_kw))
    w = Matrix(torch, n, k, 128, wt, count=count, codes=wc, scales=ws, **({"ld": up16(k)} if w_kw is None else w_kw))
    step = out_ld or n
    out = torch.full((out_offset + m * step + 8,), 3.0, dtype=wide_type(torch, out_dt), device="cuda")
    view = out[out_offset:out_offset + m * step].view(m, step)
    offs = None if offsets is None else torch.tensor(offsets, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    try:
        if offs is None:
            gpu.matmul_blocks(x.pod, w.pod, view.data_ptr(), out_dt, view.nbytes, out_ld)
        else:
            gpu.matmul_blocks_grouped(x.pod, w.pod, offs.data_ptr(), view.data_ptr(), out_dt, view.nbytes, out_ld)
    finally:
        gpu.synchronize()
        got = view[:, :n].double().cpu().numpy()
        view[:, :n] = 3.0
        assert bool((out == 3.0).all())
        assert x.guards_intact() and w.guards_intact()
    return got


def check_product(got, xc, xs, wc, ws, xt, wt, out_dt, lo=0, hi=None, e=0):
    xv, wv = br.values(xc[lo:hi], xs[lo:hi], 1, xt), br.values(wc[e], ws[e], 128, wt)
    y = xv @ wv.T
    off = np.abs(got[lo:hi] - y) - br.product_tolerance(xv, wv, y, out_dt)
    assert off.size == 0 or off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 4096, 512), (1, 300, 2048), (2, 17, 16), (7, 129, 130), (16, 256, 384), (17, 128, 1000), (31, 1000, 128), (33, 200, 257),
            (64, 384, 640), (65, 130, 128), (100, 512, 1024), (128, 128, 128), (129, 257, 300), (200, 640, 400), (255, 256, 256),
            (256, 300, 1024), (257, 128, 144), (400, 1000, 512), (520, 2100, 272), (1000, 1111, 640)]


@pytest.mark.parametrize("xt,wt,out_dt", [(E4M3, E4M3, BF16), (E5M2, E4M3, F16), (E4M3, E5M2, F32), (E5M2, E5M2, BF16)])
def test_product(gpu, torch, xt, wt, out_dt):
    rng = np.random.default_rng(13)
    for m, n, k in PRODUCTS:
        ops = operands(rng, m, n, k, xt, wt)
        got = run_product(gpu, torch, *ops, xt, wt, out_dt)
        check_product(got, *ops, xt, wt, out_dt)


@pytest.mark.parametrize("m,n,k,out_ld", [(2300, 2500, 400, 0), (1100, 4099, 272, 0), (4097, 1300, 128, 1301), (1024, 5000, 1600, 5008)])
def test_product_with_many_tiles(gpu, torch, m, n, k, out_ld):
    """Enough tiles for every multiprocessor, several each: 256 rows by 256 columns on pairs of them."""
    rng = np.random.default_rng(24)
    for xt, wt, out_dt in ((E4M3, E4M3, BF16), (E5M2, E4M3, F32)):
        ops = operands(rng, m, n, k, xt, wt)
        got = run_product(gpu, torch, *ops, xt, wt, out_dt, out_ld=out_ld)
        check_product(got, *ops, xt, wt, out_dt)


@pytest.mark.parametrize("offsets,n", [([0, 700, 700, 701, 2000, 2256], 1500), ([7] + [7 + 60 * i for i in range(40)], 1100)])
def test_grouped_product_with_many_tiles(gpu, torch, offsets, n):
    rng = np.random.default_rng(25)
    m, experts = offsets[-1] + 11, len(offsets) - 1
    ops = operands(rng, m, n, 300, E4M3, E4M3, experts)
    got = run_product(gpu, torch, *ops, E4M3, E4M3, BF16, offsets=offsets)
    for e in range(experts):
        check_product(got, *ops, E4M3, E4M3, BF16, offsets[e], offsets[e + 1], e)
    assert (got[:offsets[0]] == 3).all() and (got[offsets[-1]:] == 3).all()


@pytest.mark.parametrize("k", [257, 640, 1153, 2100, 4480])
@pytest.mark.parametrize("m", [1, 5, 16, 17, 30, 33, 50, 64, 66, 100, 128, 140, 250])
def test_product_of_few_rows_and_long_sums(gpu, torch, m, k):
    """Column blocks that two to eight CTAs share, in numbers that do not divide evenly."""
    rng = np.random.default_rng(26)
    for n in (120, 300):
        ops = operands(rng, m, n, k, E4M3, E4M3)
        got = run_product(gpu, torch, *ops, E4M3, E4M3, F32)
        check_product(got, *ops, E4M3, E4M3, F32)


def test_elements_beyond_32_bits(gpu, torch):
    """Matrices of more than 2^31 elements: the last rows of quantising, reading back and both products."""
    rng = np.random.default_rng(27)
    rows, cols = 70000, 32000
    src = torch.zeros(rows * cols, dtype=torch.bfloat16, device="cuda").view(rows, cols)
    x = host_f32(torch, weight_values(rng, (130, cols)), BF16)
    src[-130:] = torch.from_numpy(x).to(torch.bfloat16)
    codes = torch.full((rows, cols), GUARD, dtype=torch.uint8, device="cuda")
    for block_rows in (1, 128):
        scales = torch.zeros(-(-rows // block_rows), 250, device="cuda")
        m = abi.block_matrix(codes.data_ptr(), scales.data_ptr(), E4M3, block_rows, rows, cols)
        c, keep = device_content(torch, src, BF16, (rows, cols))
        torch.cuda.synchronize()
        gpu.quantize_blocks(c, m)
        first = rows - 130 if block_rows == 1 else rows // 128 * 128  # the first row of a whole block of known values
        want_c, want_s = br.quantize(x[first - (rows - 130):], block_rows, E4M3)
        assert np.array_equal(codes[first:].cpu().numpy(), want_c)
        assert np.array_equal(scales[first // block_rows:].cpu().numpy(), want_s)
        codes[:1000] = 7
        src[:1000] = 0
        torch.cuda.synchronize()
        gpu.dequantize_blocks(m, src.data_ptr(), BF16, src.nbytes)
        want = rounded(torch, br.values(want_c, want_s, block_rows, E4M3), BF16)
        assert np.array_equal(src[first:].float().cpu().numpy(), want)
        src[-130:] = torch.from_numpy(x).to(torch.bfloat16)
    # results beyond 2^31 elements, and weights of as many codes (the last of nine experts)
    xc, xs = br.quantize(rng.standard_normal((rows, 16)).astype(np.float32), 1, E4M3)
    wc, ws = br.quantize(weight_values(rng, (cols, 16)), 128, E4M3)
    xm, wm = Matrix(torch, rows, 16, 1, codes=xc, scales=xs), Matrix(torch, cols, 16, 128, codes=wc, scales=ws)
    gpu.matmul_blocks(xm.pod, wm.pod, src.data_ptr(), BF16, src.nbytes)
    part = (xc[-40:], xs[-40:], wc[None], ws[None])
    check_product(src[-40:].double().cpu().numpy(), *part, E4M3, E4M3, BF16)
    del src
    experts, n, k = 9, 16384, 16384
    big = codes.view(-1)[:0].new_empty(experts * n * k)
    big.fill_(0)
    wc, ws = br.quantize(weight_values(rng, (1, 256, k)), 128, E4M3)
    big.view(experts, n, k)[-1, -256:] = torch.from_numpy(wc[0])
    all_s = torch.ones(experts, n // 128, k // 128, device="cuda")
    all_s[-1, -2:] = torch.from_numpy(ws[0])
    wm = abi.block_matrix(big.data_ptr(), all_s.data_ptr(), E4M3, 128, n, k, count=experts)
    xc, xs = br.quantize(rng.standard_normal((12, k)).astype(np.float32), 1, E4M3)
    xm = Matrix(torch, 12, k, 1, codes=xc, scales=xs)
    offs = torch.tensor([0] * 4 + [5] * 5 + [12], device="cuda")
    out = torch.zeros(12, n, device="cuda")
    torch.cuda.synchronize()
    gpu.matmul_blocks_grouped(xm.pod, wm, offs.data_ptr(), out.data_ptr(), F32, out.nbytes)
    check_product(out[:, -256:].double().cpu().numpy(), xc, xs, wc, ws, E4M3, E4M3, F32, 5, 12)
    assert (out[:5] == 0).all() and (out[5:, :-256] == 0).all()


@pytest.mark.parametrize("n", [1, 200])
def test_one_row_has_no_pitch(gpu, torch, n):
    """One token of odd width, dense: its row pitch is not a multiple of 16 and does not have to be."""
    rng = np.random.default_rng(30)
    for k in (1, 15, 1001, 4099):
        ops = operands(rng, 1, n, k, E4M3, E4M3)
        for w_kw in ({"ld": up16(k)}, {"ld": k}):
            got = run_product(gpu, torch, *ops, E4M3, E4M3, F32, x_kw={"ld": k}, w_kw=w_kw)
            check_product(got, *ops, E4M3, E4M3, F32)


def test_captured_without_a_call_before(torch, tmp_path):
    """The first calls of a process, recorded into a graph: nothing about them waits or allocates."""
    import subprocess
    import sys
    script = tmp_path / "first.py"
    script.write_text(FIRST_CALLS_CAPTURED)
    r = subprocess.run([sys.executable, str(script)], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("equal"), r.stdout + r.stderr


FIRST_CALLS_CAPTURED = """
import sys
sys.path.insert(0, ".")
import torch
from vpux_plugin_b200 import abi
from vpux_plugin_b200.lib import Library
stream = torch.cuda.Stream()
lib = Library(device=0, stream=stream.cuda_stream, pipelined=True)
outs = {}
keep = []
for m in (1, 20, 40, 100, 3000):
    x = torch.randn(m, 512, device="cuda")
    w = torch.randn(2, 3000, 512, device="cuda")
    xc, xs = torch.zeros(m, 512, dtype=torch.uint8, device="cuda"), torch.zeros(4, m, device="cuda")
    wc, ws = torch.zeros(2, 3000, 512, dtype=torch.uint8, device="cuda"), torch.zeros(2, 24, 4, device="cuda")
    y, yg = torch.zeros(m, 3000, device="cuda"), torch.zeros(m, 3000, device="cuda")
    off = torch.tensor([0, m // 2, m], device="cuda")
    xm = abi.block_matrix(xc.data_ptr(), xs.data_ptr(), abi.VF_DT_F8E4M3FN, 1, m, 512, scale_row_stride=1, scale_col_stride=m)
    wm = abi.block_matrix(wc.data_ptr(), ws.data_ptr(), abi.VF_DT_F8E4M3FN, 128, 3000, 512, count=2)
    w0 = abi.block_matrix(wc.data_ptr(), ws.data_ptr(), abi.VF_DT_F8E4M3FN, 128, 3000, 512)
    cx, k1 = abi.make_content(abi.TType([m, 512], abi.VF_DT_F32), None, ptr=x.data_ptr(), nbytes=x.nbytes, mem_kind=abi.VF_MEM_DEVICE)
    cw, k2 = abi.make_content(abi.TType([2, 3000, 512], abi.VF_DT_F32), None, ptr=w.data_ptr(), nbytes=w.nbytes, mem_kind=abi.VF_MEM_DEVICE)

    def calls():
        lib.quantize_blocks(cx, xm)
        lib.quantize_blocks(cw, wm)
        lib.matmul_blocks(xm, w0, y.data_ptr(), abi.VF_DT_F32, y.nbytes)
        lib.matmul_blocks_grouped(xm, wm, off.data_ptr(), yg.data_ptr(), abi.VF_DT_F32, yg.nbytes)
        lib.dequantize_blocks(wm, w.data_ptr(), abi.VF_DT_F32, w.nbytes)

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        calls()
    g.replay()
    torch.cuda.synchronize()
    first = (y.clone(), yg.clone(), w.clone())
    y.zero_(), yg.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        calls()
    lib.synchronize()
    for a, b in zip(first, (y, yg, w)):
        assert float(a.abs().max()) > 1 and torch.equal(a, b), m
    del g
print("equal")
"""


def test_a_claim_of_more_tiles_than_fit_is_refused(gpu):
    at = 1 << 40  # addresses that nothing looks at
    x = abi.block_matrix(at, 2 * at, E4M3, 1, 1 << 30, 16)
    w = abi.block_matrix(3 * at, 4 * at, E4M3, 128, 1 << 21, 16)
    with pytest.raises(VfoldError) as e:
        gpu.matmul_blocks(x, w, 1 << 60, BF16, 1 << 59)
    assert e.value.status == abi.VF_ERR_CAPACITY


def test_memory_kinds_mixed(gpu, torch):
    rng = np.random.default_rng(28)
    x = weight_values(rng, (40, 300))
    codes, scales = br.quantize(x, 1, E4M3)
    m = Matrix(torch, 40, 300, 1)
    c, keep = abi.make_content(abi.TType([40, 300], F32), x)  # from host memory to the device
    gpu.quantize_blocks(c, m.pod)
    assert np.array_equal(m.codes()[0], codes) and np.array_equal(m.scales()[0], scales)
    src, k1 = to_device(torch, x, F32)
    torch.cuda.synchronize()
    c, k2 = device_content(torch, src, F32, (40, 300))  # and back
    q, s = np.zeros((40, 300), np.uint8), np.zeros((3, 40), np.float32)
    gpu.quantize_blocks(c, abi.block_matrix(q, s, E4M3, 1, 40, 300, scale_row_stride=1, scale_col_stride=40, mem_kind=HOST))
    assert np.array_equal(q, codes) and np.array_equal(s.T, scales)
    back = np.zeros_like(x)
    gpu.dequantize_blocks(m.pod, back, F32, back.nbytes, dst_mem_kind=HOST)
    assert np.array_equal(back, br.values(codes, scales, 1, E4M3).astype(np.float32))


def test_on_the_legacy_default_stream(torch):
    """The handle 1 stands for the default stream, so calls line up with what torch enqueues there."""
    lib = Library(device=0, stream=1, pipelined=True)
    rng = np.random.default_rng(29)
    ops = operands(rng, 20, 300, 512, E4M3, E4M3)
    x, w = Matrix(torch, 20, 512, 1, codes=ops[0], scales=ops[1]), Matrix(torch, 300, 512, 128, codes=ops[2], scales=ops[3])
    y = torch.empty(20, 300, device="cuda")
    y.fill_(3)
    lib.matmul_blocks(x.pod, w.pod, y.data_ptr(), F32, y.nbytes)
    doubled = y * 2  # behind the product, without a wait
    check_product(doubled.double().cpu().numpy() / 2, *ops, E4M3, E4M3, F32)
    lib.close()


@pytest.mark.parametrize("m", [3, 70, 300])
@pytest.mark.parametrize("x_kw,w_kw,out_ld,out_offset", [
    ({"ld": 320, "col_major": False}, {"ld": 336, "col_major": True}, 0, 0),      # scales in the other orders, rows further apart
    ({"ld": 304, "offset": 16}, {"ld": 304, "offset": 32}, 203, 1),               # an odd result pitch, an odd start
    ({"ld": 304}, {"ld": 304}, 208, 0), ({"ld": 304}, {"ld": 304}, 216, 4),
    ({"ld": 300}, {"ld": 304}, 0, 0), ({"ld": 304}, {"ld": 303}, 0, 0),           # not for the tensor cores: pitch, start
    ({"ld": 304, "offset": 8}, {"ld": 304}, 0, 0), ({"ld": 304}, {"ld": 304, "offset": 1}, 0, 0)])
def test_product_strides_and_alignments(gpu, torch, m, x_kw, w_kw, out_ld, out_offset):
    rng = np.random.default_rng(14)
    ops = operands(rng, m, 201, 300, E4M3, E4M3)
    for out_dt in (BF16, F32):
        got = run_product(gpu, torch, *ops, E4M3, E4M3, out_dt, x_kw=x_kw, w_kw=w_kw, out_ld=out_ld, out_offset=out_offset)
        check_product(got, *ops, E4M3, E4M3, out_dt)


@pytest.mark.parametrize("m,n", [(0, 5), (5, 0), (0, 0)])
def test_product_of_nothing(gpu, torch, m, n):
    x = abi.block_matrix(None if m == 0 else torch.zeros(m * 16, dtype=torch.uint8, device="cuda").data_ptr(),
                         None if m == 0 else torch.zeros(m, device="cuda").data_ptr(), E4M3, 1, m, 16)
    w = abi.block_matrix(None if n == 0 else torch.zeros(n * 16, dtype=torch.uint8, device="cuda").data_ptr(),
                         None if n == 0 else torch.zeros(1, device="cuda").data_ptr(), E4M3, 128, n, 16)
    gpu.matmul_blocks(x, w, None, BF16, 0)
    assert gpu.last_stats.kernels_launched == 0


@pytest.mark.parametrize("m", [4, 300])
def test_codes_that_are_not_finite_stay_in_their_row_and_column(gpu, torch, m):
    rng = np.random.default_rng(15)
    xc, xs, wc, ws = operands(rng, m, 200, 512, E5M2, E4M3)
    xc[2, 200] = 0x7C  # infinity
    wc[0, 150, 3] = 0x7F  # NaN
    got = run_product(gpu, torch, xc, xs, wc, ws, E5M2, E4M3, F32)
    assert not np.isfinite(got[2]).any() and np.isnan(got[:, 150]).all()
    rest = np.ones(got.shape, bool)
    rest[2], rest[:, 150] = False, False
    assert np.isfinite(got[rest]).all()


@pytest.mark.parametrize("m", [2, 130])
def test_results_beyond_the_output_type(gpu, torch, m):
    """Sums past the largest fp16 number become infinite; scales of the smallest blocks leave zeros."""
    k = 256
    xc = np.full((m, k), 0x7E, np.uint8)  # 448
    xs = np.full((m, 2), 1.0, np.float32)
    wc = np.full((1, 128, k), 0x7E, np.uint8)
    ws = np.full((1, 1, 2), 1.0, np.float32)
    assert np.isinf(run_product(gpu, torch, xc, xs, wc, ws, E4M3, E4M3, F16)).all()
    assert (run_product(gpu, torch, xc, xs, wc, ws, E4M3, E4M3, F32) == 448.0 * 448.0 * k).all()
    ws[:] = br.SMALLEST_SCALE
    xs[:] = 2.0 ** -60
    assert (run_product(gpu, torch, xc, xs, wc, ws, E4M3, E4M3, F16) == 0).all()


GROUPS = [[0, 5], [0, 0, 0, 7, 7, 7], [3, 10, 10, 50, 51], [0, 128, 256, 257], [0, 1, 2, 3, 4, 5, 6, 7, 8], [10, 300, 300, 310],
          [0] * 33 + [1] * 33 + [40, 40, 90], list(range(0, 71)), [0] * 70, [5, 5, 6, 6, 500, 700]]


@pytest.mark.parametrize("xt,wt,out_dt", [(E4M3, E4M3, BF16), (E5M2, E4M3, F16), (E4M3, E4M3, F32)])
@pytest.mark.parametrize("offsets", GROUPS)
def test_grouped_product(gpu, torch, offsets, xt, wt, out_dt):
    rng = np.random.default_rng(16)
    for n, k, behind in ((130, 200, 0), (257, 384, 37)):
        m, experts = offsets[-1] + behind, len(offsets) - 1
        m = max(m, 1)
        ops = operands(rng, m, n, k, xt, wt, experts)
        got = run_product(gpu, torch, *ops, xt, wt, out_dt, offsets=offsets)
        for e in range(experts):
            check_product(got, *ops, xt, wt, out_dt, offsets[e], offsets[e + 1], e)
        assert (got[:offsets[0]] == 3).all() and (got[offsets[-1]:] == 3).all()


@pytest.mark.parametrize("x_kw,w_kw", [({"ld": 200}, {"ld": 201}), ({"ld": 208, "offset": 2}, {"ld": 208})])
def test_grouped_product_of_unaligned_operands(gpu, torch, x_kw, w_kw):
    rng = np.random.default_rng(17)
    offsets = [2, 2, 75, 76, 140]
    ops = operands(rng, 150, 90, 200, E4M3, E5M2, 4)
    got = run_product(gpu, torch, *ops, E4M3, E5M2, BF16, offsets=offsets, x_kw=x_kw, w_kw=w_kw)
    for e in range(4):
        check_product(got, *ops, E4M3, E5M2, BF16, offsets[e], offsets[e + 1], e)
    assert (got[:2] == 3).all() and (got[140:] == 3).all()


@pytest.mark.parametrize("offsets", [[0, 30, 20, 40], [-5, 10, 20, 30], [0, 10, 20, 41], [0, 10, 1 << 40, 1 << 41], [-(1 << 62), -3, -2, -1], [50, 60, 70, 80]])
def test_offsets_that_leave_the_operand_are_reported(gpu, torch, offsets):
    rng = np.random.default_rng(18)
    ops = operands(rng, 40, 64, 128, E4M3, E4M3, 3)
    for kw in (None, {"ld": 131}):
        with pytest.raises(VfoldError) as e:
            run_product(gpu, torch, *ops, E4M3, E4M3, BF16, offsets=offsets, w_kw=kw)
        assert e.value.status == abi.VF_ERR_RANGE
    good = [0, 10, 10, 40]
    got = run_product(gpu, torch, *ops, E4M3, E4M3, BF16, offsets=good)
    check_product(got, *ops, E4M3, E4M3, BF16, 10, 40, 2)


# ---- together, and as programs call them -----------------------------------------------------------------------------------

def test_a_layer_from_weights_to_answers(gpu, torch):
    """Weights folded to blocks, tokens quantised, both products, and the weights read back: as a program runs them,
    without waiting in between."""
    rng = np.random.default_rng(19)
    n, k, experts = 300, 640, 5
    w = host_f32(torch, weight_values(rng, (experts, n, k)), F16)
    x = host_f32(torch, rng.standard_normal((90, k)).astype(np.float32), BF16)
    wd, wk = to_device(torch, w, F16)
    xd, xk = to_device(torch, x, BF16)
    lib = Library(device=0, pipelined=True)
    wm = Matrix(torch, n, k, 128, count=experts)
    xm = Matrix(torch, 90, k, 1, col_major=True)
    offsets = [0, 20, 20, 61, 62, 90]
    offs = torch.tensor(offsets, device="cuda")
    y1, y2 = (torch.full((90, n), 3.0, device="cuda") for _ in range(2))
    back = torch.zeros((experts, n, k), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    wc, k1 = device_content(torch, wd, F16, (experts, n, k))
    xc, k2 = device_content(torch, xd, BF16, (90, k))
    first = abi.block_matrix(wm.buf.data_ptr(), wm.sbuf.data_ptr(), E4M3, 128, n, k)
    for _ in range(3):
        lib.quantize_blocks(wc, wm.pod)
        lib.quantize_blocks(xc, xm.pod)
        lib.matmul_blocks(xm.pod, first, y1.data_ptr(), F32, y1.nbytes)
        lib.matmul_blocks_grouped(xm.pod, wm.pod, offs.data_ptr(), y2.data_ptr(), F32, y2.nbytes)
        lib.dequantize_blocks(wm.pod, back.data_ptr(), F16, back.nbytes)
    lib.synchronize()
    qx, sx = br.quantize(x, 1, E4M3)
    qw, sw = br.quantize(w, 128, E4M3)
    check_product(y1.double().cpu().numpy(), qx, sx, qw, sw, E4M3, E4M3, F32)
    for e in range(experts):
        check_product(y2.double().cpu().numpy(), qx, sx, qw, sw, E4M3, E4M3, F32, offsets[e], offsets[e + 1], e)
    assert np.array_equal(back.float().cpu().numpy(), rounded(torch, br.values(qw, sw, 128, E4M3), F16))
    assert lib.launch_count == 15
    lib.close()


def test_pipelined_calls_report_at_the_next_wait(torch):
    lib = Library(device=0, pipelined=True)
    rng = np.random.default_rng(20)
    x = weight_values(rng, (4, 256))
    x[1, 1] = np.nan
    src, keep = to_device(torch, x, F32)
    m = Matrix(torch, 4, 256, 1)
    c, k = device_content(torch, src, F32, (4, 256))
    torch.cuda.synchronize()
    lib.quantize_blocks(c, m.pod)
    with pytest.raises(VfoldError) as e:
        lib.synchronize()
    assert e.value.status == abi.VF_ERR_NAN
    lib.synchronize()
    lib.close()


@pytest.mark.parametrize("m", [1, 40, 300])
def test_captured_on_the_callers_stream_and_replayed(torch, m):
    """Two captured graphs of one context, replayed in turn with new inputs in the same buffers."""
    rng = np.random.default_rng(21)
    n, k, experts = 200, 512, 3
    stream = torch.cuda.Stream()
    lib = Library(device=0, stream=stream.cuda_stream, pipelined=True)
    src = torch.zeros((m, k), device="cuda")
    xm = Matrix(torch, m, k, 1, col_major=True)
    ops = operands(rng, m, n, k, E4M3, E4M3, experts)
    wm = Matrix(torch, n, k, 128, count=experts, codes=ops[2], scales=ops[3])
    first = abi.block_matrix(wm.buf.data_ptr(), wm.sbuf.data_ptr(), E4M3, 128, n, k)
    offsets = [0, m // 2, m // 2, m]
    offs = torch.tensor(offsets, device="cuda")
    y1, y2 = (torch.zeros((m, n), device="cuda") for _ in range(2))
    c, keep = device_content(torch, src, F32, (m, k))
    calls = (lambda: lib.matmul_blocks(xm.pod, first, y1.data_ptr(), F32, y1.nbytes),
             lambda: lib.matmul_blocks_grouped(xm.pod, wm.pod, offs.data_ptr(), y2.data_ptr(), F32, y2.nbytes))
    torch.cuda.synchronize()
    graphs = []
    for f in calls:
        with torch.cuda.stream(stream):
            lib.quantize_blocks(c, xm.pod)
            f()
            lib.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                lib.quantize_blocks(c, xm.pod)
                f()
        graphs.append(g)
    for turn in range(3):
        x = rng.standard_normal((m, k)).astype(np.float32)
        src.copy_(torch.from_numpy(x))
        y1.fill_(3)
        y2.fill_(3)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        qx, sx = br.quantize(x, 1, E4M3)
        check_product(y1.double().cpu().numpy(), qx, sx, ops[2], ops[3], E4M3, E4M3, F32)
        for e in range(experts):
            check_product(y2.double().cpu().numpy(), qx, sx, ops[2], ops[3], E4M3, E4M3, F32, offsets[e], offsets[e + 1], e)
    del graphs
    lib.close()


def test_two_contexts_at_once(torch):
    """Two threads, each with a context (and stream) of its own, and a third that shares the first one's."""
    rng = np.random.default_rng(22)
    libs = [Library(device=0), Library(device=0)]
    work = []
    for lib, (m, n, k) in ((libs[0], (3, 500, 1024)), (libs[1], (300, 260, 512)), (libs[0], (50, 300, 768))):
        ops = operands(rng, m, n, k, E4M3, E4M3)
        x = Matrix(torch, m, k, 1, codes=ops[0], scales=ops[1])
        w = Matrix(torch, n, k, 128, codes=ops[2], scales=ops[3])
        work.append((lib, x, w, torch.zeros((m, n), device="cuda"), ops))
    torch.cuda.synchronize()
    failed = []

    def go(lib, x, w, y, ops):
        try:
            for _ in range(20):
                lib.matmul_blocks(x.pod, w.pod, y.data_ptr(), F32, y.nbytes)
        except Exception as e:  # noqa: BLE001 - handed to the test's thread
            failed.append(e)

    threads = [threading.Thread(target=go, args=a) for a in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for lib, x, w, y, ops in work:
        check_product(y.double().cpu().numpy(), *ops, E4M3, E4M3, F32)
    for lib in libs:
        lib.close()


def test_the_same_call_gives_the_same_bits(gpu, torch):
    rng = np.random.default_rng(23)
    for m, n, k in ((1, 4096, 2048), (40, 1000, 1111), (600, 600, 600)):
        ops = operands(rng, m, n, k, E4M3, E4M3)
        a = run_product(gpu, torch, *ops, E4M3, E4M3, F32)
        b = run_product(gpu, torch, *ops, E4M3, E4M3, F32)
        assert np.array_equal(a, b)
