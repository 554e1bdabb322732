"""8-bit floating-point blocks without a device: every refusal of the four entry points (arguments are checked before the
context is looked at, so a NULL context reaches them all), and the numpy restatement against torch's conversions."""
import numpy as np
import pytest

import block_reference as br
from vpux_plugin_b200 import abi, lib

E4M3, E5M2, I8 = abi.VF_DT_F8E4M3FN, abi.VF_DT_F8E5M2, abi.VF_DT_I8
BF16, F32, I32 = abi.VF_DT_BF16, abi.VF_DT_F32, abi.VF_DT_I32
AT = 1 << 20  # addresses that nothing looks at
DEV, HOST = abi.VF_MEM_DEVICE, abi.VF_MEM_HOST


def matrix(rows, cols, block_rows, codes=AT, scales=2 * AT, dtype=E4M3, **kw):
    return abi.block_matrix(codes, scales, dtype, block_rows, rows, cols, **kw)


def content(shape, dtype=BF16, ptr=16 * AT, nbytes=None, mem_kind=DEV, **kw):
    t = abi.TType(shape, dtype, kw.pop("order", 0))
    return abi.make_content(t, None, ptr=ptr, nbytes=t.nbytes() if nbytes is None else nbytes, mem_kind=mem_kind, **kw)


def call(name, *args):
    import ctypes as C
    err = C.create_string_buffer(512)
    args = [C.byref(a) if isinstance(a, C.Structure) else a for a in args]
    st = getattr(lib.raw(), name)(None, *args, None, err, 512)
    return st, err.value.decode()


def refused(status, words, name, *args):
    st, msg = call(name, *args)
    assert st == status and words in msg, (st, msg)


def test_good_arguments_reach_the_context():
    q, _ = content([4, 256])
    x, w = matrix(4, 256, 1), matrix(8, 256, 128)
    for name, args in (("vf_quantize_blocks", (q, 0, matrix(4, 256, 1))), ("vf_dequantize_blocks", (x, 8 * AT, BF16, 0, 4 * 256 * 2, DEV)),
                       ("vf_matmul_blocks", (x, w, 8 * AT, BF16, 0, 4 * 8 * 2)),
                       ("vf_matmul_blocks_grouped", (x, matrix(8, 256, 128, count=3), 9 * AT, 8 * AT, BF16, 0, 4 * 8 * 2))):
        refused(abi.VF_ERR_INVALID_ARG, "ctx is NULL", name, *args)


@pytest.mark.parametrize("change,status,words", [
    ({"dtype": I8}, abi.VF_ERR_UNSUPPORTED, "e4m3 or e5m2"),
    ({"block_rows": 64}, abi.VF_ERR_UNSUPPORTED, "blocks of 64 rows"),
    ({"mem_kind": 7}, abi.VF_ERR_INVALID_ARG, "memory kind"),
    ({"count": 0}, abi.VF_ERR_SHAPE, "shape"),
    ({"rows": -1}, abi.VF_ERR_SHAPE, "shape"),
    ({"cols": 0}, abi.VF_ERR_SHAPE, "shape"),
    ({"cols": 1 << 31}, abi.VF_ERR_SHAPE, "shape"),
    ({"rows": (1 << 31) - 1}, abi.VF_ERR_SHAPE, "shape"),
    ({"ld": 255}, abi.VF_ERR_SHAPE, "hold no 256 columns"),
    ({"ld": -256}, abi.VF_ERR_SHAPE, "hold no 256 columns"),
    ({"ld": 1 << 62}, abi.VF_ERR_SHAPE, "too large"),
    ({"count": 2, "matrix_stride": 1000}, abi.VF_ERR_SHAPE, "elements meet"),
    ({"count": 2, "matrix_stride": -1024}, abi.VF_ERR_INVALID_ARG, "negative stride"),
    ({"scale_row_stride": 1, "scale_col_stride": 3}, abi.VF_ERR_SHAPE, "elements meet"),
    ({"scale_row_stride": -2, "scale_col_stride": 1}, abi.VF_ERR_INVALID_ARG, "negative stride"),
    ({"codes": None}, abi.VF_ERR_BUFFER_TOO_SMALL, "codes need 1024 bytes"),
    ({"codes_bytes": 1023}, abi.VF_ERR_BUFFER_TOO_SMALL, "codes need 1024 bytes, buffer holds 1023"),
    ({"scales": None}, abi.VF_ERR_BUFFER_TOO_SMALL, "scales need 32 bytes"),
    ({"scales_bytes": 31}, abi.VF_ERR_BUFFER_TOO_SMALL, "scales need 32 bytes"),
    ({"scales": 2 * AT + 2}, abi.VF_ERR_ALIGNMENT, "4-byte aligned"),
    ({"mem_kind": HOST, "ld": 272}, abi.VF_ERR_UNSUPPORTED, "no gaps"),
    ({"mem_kind": HOST, "scale_row_stride": 4, "scale_col_stride": 1}, abi.VF_ERR_UNSUPPORTED, "no gaps"),
])
def test_matrices_that_are_refused(change, status, words):
    m = matrix(4, 256, 1)
    for k, v in change.items():
        setattr(m, k, v)
    refused(status, words, "vf_dequantize_blocks", m, 8 * AT, F32, 0, 1 << 30, DEV)


def test_null_pointers():
    m = matrix(4, 256, 1)
    refused(abi.VF_ERR_INVALID_ARG, "in is NULL", "vf_dequantize_blocks", None, 8 * AT, F32, 0, 1 << 30, DEV)
    refused(abi.VF_ERR_INVALID_ARG, "base is NULL", "vf_quantize_blocks", None, 0, m)
    refused(abi.VF_ERR_INVALID_ARG, "x is NULL", "vf_matmul_blocks", None, m, 8 * AT, F32, 0, 1 << 30)
    refused(abi.VF_ERR_INVALID_ARG, "w is NULL", "vf_matmul_blocks", m, None, 8 * AT, F32, 0, 1 << 30)
    w = matrix(8, 256, 128, count=2)
    refused(abi.VF_ERR_INVALID_ARG, "offsets is NULL", "vf_matmul_blocks_grouped", m, w, None, 8 * AT, F32, 0, 1 << 30)
    refused(abi.VF_ERR_ALIGNMENT, "offsets", "vf_matmul_blocks_grouped", m, w, 9 * AT + 4, 8 * AT, F32, 0, 1 << 30)


def test_quantize_refusals():
    m = matrix(4, 256, 1)
    q = "vf_quantize_blocks"
    for c, status, words in ((content([4, 256], I32), abi.VF_ERR_UNSUPPORTED, "f32, f16 or bf16"),
                             (content([4, 255]), abi.VF_ERR_SHAPE, "different shapes"),
                             (content([1024]), abi.VF_ERR_SHAPE, "different shapes"),
                             (content([2, 4, 256]), abi.VF_ERR_SHAPE, "different shapes"),
                             (content([4, 256], nbytes=2047), abi.VF_ERR_BUFFER_TOO_SMALL, "base needs 2048 bytes"),
                             (content([4, 256], ptr=16 * AT + 1), abi.VF_ERR_ALIGNMENT, "aligned to its elements"),
                             (content([4, 256], ptr=AT - 2000), abi.VF_ERR_INVALID_ARG, "base and codes overlap"),
                             (content([4, 256], ptr=2 * AT), abi.VF_ERR_INVALID_ARG, "base and scales overlap"),
                             (content([4, 256], order=0x21), abi.VF_ERR_UNSUPPORTED, "row-major"),
                             (content([4, 256], is_splat=True), abi.VF_ERR_SPLAT, "splat"),
                             (content([4, 256], storage_dtype=F32), abi.VF_ERR_UNSUPPORTED, "plain f32")):
        refused(status, words, q, c[0], 0, m)
    good = content([4, 256])[0]
    refused(abi.VF_ERR_SHAPE, "hold no 256 columns", q, good, 200, m)
    refused(abi.VF_ERR_INVALID_ARG, "negative stride", q, good, -256, m)
    refused(abi.VF_ERR_BUFFER_TOO_SMALL, "base needs", q, good, 257, m)
    refused(abi.VF_ERR_UNSUPPORTED, "no gaps", q, content([4, 256], mem_kind=HOST, nbytes=1 << 20)[0], 257, m)
    refused(abi.VF_ERR_INVALID_ARG, "codes and scales overlap", q, good, 0, matrix(4, 256, 1, scales=AT + 1020))
    elem = abi.Elem.uniform(abi.VF_DT_U8, F32, 0.1, 0, 0, 255)
    c, keep = abi.make_content(abi.TType([4, 256], elem), None, ptr=16 * AT, nbytes=1024, mem_kind=DEV)
    refused(abi.VF_ERR_UNSUPPORTED, "plain", q, c, 0, m)


def test_dequantize_refusals():
    m = matrix(4, 256, 1)
    d = "vf_dequantize_blocks"
    refused(abi.VF_ERR_UNSUPPORTED, "f32, f16 or bf16", d, m, 8 * AT, I8, 0, 1 << 20, DEV)
    refused(abi.VF_ERR_BUFFER_TOO_SMALL, "dst needs 2048 bytes", d, m, 8 * AT, BF16, 0, 2047, DEV)
    refused(abi.VF_ERR_BUFFER_TOO_SMALL, "dst needs 2048 bytes", d, m, None, BF16, 0, 2048, DEV)
    refused(abi.VF_ERR_SHAPE, "hold no 256 columns", d, m, 8 * AT, BF16, 128, 1 << 20, DEV)
    refused(abi.VF_ERR_ALIGNMENT, "aligned", d, m, 8 * AT + 2, F32, 0, 1 << 20, DEV)
    refused(abi.VF_ERR_INVALID_ARG, "memory kind", d, m, 8 * AT, F32, 0, 1 << 20, 5)
    refused(abi.VF_ERR_UNSUPPORTED, "no gaps", d, m, 8 * AT, F32, 300, 1 << 20, HOST)
    refused(abi.VF_ERR_INVALID_ARG, "dst and codes overlap", d, m, AT + 1000, F32, 0, 1 << 20, DEV)


def test_product_refusals():
    x, w = matrix(4, 256, 1), matrix(8, 256, 128, codes=4 * AT, scales=5 * AT)
    mm = "vf_matmul_blocks"

    def bad(status, words, x=x, w=w, out=8 * AT, dt=BF16, ld=0, nbytes=1 << 20):
        refused(status, words, mm, x, w, out, dt, ld, nbytes)

    bad(abi.VF_ERR_SHAPE, "x has 256 columns, w 300", w=matrix(8, 300, 128))
    bad(abi.VF_ERR_SHAPE, "x is one matrix", x=matrix(4, 256, 1, count=2))
    bad(abi.VF_ERR_SHAPE, "w is one matrix", w=matrix(8, 256, 128, codes=4 * AT, scales=5 * AT, count=2))
    bad(abi.VF_ERR_UNSUPPORTED, "block_rows 1", x=w, w=w)
    bad(abi.VF_ERR_UNSUPPORTED, "block_rows 128", x=x, w=x)
    bad(abi.VF_ERR_UNSUPPORTED, "device memory", x=matrix(4, 256, 1, mem_kind=HOST))
    bad(abi.VF_ERR_UNSUPPORTED, "f32, f16 or bf16", dt=E4M3)
    bad(abi.VF_ERR_UNSUPPORTED, "f32, f16 or bf16", dt=E4M3, w=matrix(0, 256, 128))
    bad(abi.VF_ERR_SHAPE, "hold no 8 columns", ld=7)
    bad(abi.VF_ERR_INVALID_ARG, "negative stride", ld=-8)
    bad(abi.VF_ERR_BUFFER_TOO_SMALL, "out needs 64 bytes", nbytes=63)
    bad(abi.VF_ERR_BUFFER_TOO_SMALL, "out needs 64 bytes", out=None)
    bad(abi.VF_ERR_ALIGNMENT, "aligned", out=8 * AT + 1)
    for at in (AT, 2 * AT, 4 * AT, 5 * AT):
        bad(abi.VF_ERR_INVALID_ARG, "overlap", out=at)


def test_numpy_handles_without_gaps_only():
    with pytest.raises(ValueError):
        abi.block_matrix(np.zeros((4, 512), np.uint8)[:, ::2], np.zeros((4, 2), np.float32), E4M3, 1, 4, 256, mem_kind=HOST)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_restated_codes_match_the_formats(dtype):
    import torch
    t = torch.float8_e4m3fn if dtype == E4M3 else torch.float8_e5m2
    v = torch.arange(256, dtype=torch.uint8).view(t).double().numpy()
    assert np.array_equal(v, br.code_values(dtype), equal_nan=True)
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.standard_normal(4000) * s for s in (1e-6, 1e-3, 1.0, 50.0)] + [v[np.isfinite(v)], -v[np.isfinite(v)], np.zeros(1)])
    mid = np.sort(v[np.isfinite(v)])
    x = np.concatenate([x, (mid[1:] + mid[:-1]) / 2]).astype(np.float32)  # ties among them
    x = np.clip(x, -br.LARGEST[dtype], br.LARGEST[dtype])
    want = torch.from_numpy(x).to(t).view(torch.uint8).numpy()
    assert np.array_equal(br.nearest_codes(x.astype(np.float64), dtype), want)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_restated_quantization_returns_what_it_was_given(block_rows):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((130, 300)).astype(np.float32)
    x[5, 128:256] = 0
    codes, scales = br.quantize(x, block_rows, E4M3)
    back = br.values(codes, scales, block_rows, E4M3)
    # half a step of the code, and half a step 2^-24 each of the scale, its reciprocal and their product
    step = np.maximum(np.abs(x), 2.0 ** -6 * br.expand(scales, 130, 300, block_rows))
    assert np.all(np.abs(back - x) <= step * (2.0 ** -4 + 4 * 2.0 ** -24))
