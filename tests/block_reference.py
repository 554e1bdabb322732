"""Matrices of 8-bit floats with a scale per block of 128 columns, restated with numpy in 64 bits: the values of the
codes from the format's definition, quantising, reading back, and the product. Used by the CPU and the GPU tests."""
import numpy as np

from vpux_plugin_b200 import abi

BLOCK = 128
E4M3, E5M2 = abi.VF_DT_F8E4M3FN, abi.VF_DT_F8E5M2
LARGEST = {E4M3: 448.0, E5M2: 57344.0}
SMALLEST_SCALE = np.float32(2.0 ** -126)
HALF_STEP = {abi.VF_DT_F32: 2.0 ** -24, abi.VF_DT_F16: 2.0 ** -11, abi.VF_DT_BF16: 2.0 ** -8}


def code_values(dtype):
    """float64 [256]: the value of every code."""
    exp_bits, man_bits = (4, 3) if dtype == E4M3 else (5, 2)
    bias = 2 ** (exp_bits - 1) - 1
    b = np.arange(256)
    e, m = (b >> man_bits) & (2 ** exp_bits - 1), b & (2 ** man_bits - 1)
    v = np.where(e == 0, np.ldexp(m.astype(np.float64), 1 - bias - man_bits),
                 np.ldexp((2 ** man_bits + m).astype(np.float64), e - bias - man_bits))
    if dtype == E5M2:
        v = np.where(e == 31, np.where(m == 0, np.inf, np.nan), v)
    else:
        v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


def nearest_codes(v, dtype):
    """uint8 codes of the 8-bit floats nearest to v (float64, finite), ties to the even code, saturating."""
    table = code_values(dtype)[:128]
    table = table[np.isfinite(table)]  # ascending: codes of non-negative numbers are ordered as the numbers
    a = np.abs(v)
    hi = np.minimum(np.searchsorted(table, a, side="left"), len(table) - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - table[lo], table[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(a >= table[-1], len(table) - 1, code)
    return (code | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def expand(scales, rows, cols, block_rows):
    """scales [..., row blocks, col blocks] -> [..., rows, cols]"""
    r, c = np.arange(rows) // block_rows, np.arange(cols) // BLOCK
    return scales[..., r, :][..., c]


def quantize(x, block_rows, dtype):
    """x [..., rows, cols] float32 -> (codes uint8, scales float32), by the definition in vfold.h: the scale is the
    correctly rounded quotient, the code is that of fl32(x * fl32(1 / scale))."""
    rows, cols = x.shape[-2:]
    pad = [(0, 0)] * (x.ndim - 2) + [(0, -rows % block_rows), (0, -cols % BLOCK)]
    p = np.pad(x, pad)
    b = p.reshape(*p.shape[:-2], p.shape[-2] // block_rows, block_rows, p.shape[-1] // BLOCK, BLOCK)
    top = np.abs(b).max((-3, -1)).astype(np.float32)
    scales = np.maximum((top / np.float32(LARGEST[dtype])).astype(np.float32), SMALLEST_SCALE)
    inverse = (np.float32(1) / scales).astype(np.float32)
    q = (x * expand(inverse, rows, cols, block_rows)).astype(np.float32)
    return nearest_codes(q.astype(np.float64), dtype), scales


def values(codes, scales, block_rows, dtype):
    """float64 values of a matrix (or a stack of them)."""
    return code_values(dtype)[codes] * expand(scales.astype(np.float64), *codes.shape[-2:], block_rows)


def product_tolerance(x, w, y, out_dtype):
    """Largest error of y = x @ w.T (float64 values of the operands) that the operator's arithmetic can make.
    Products of two codes are exact in fp32 (4 + 4 significant bits). A column block's sum has at most 128 of them: 127
    additions, each wrong by at most one step 2^-23 of the magnitudes added so far (hardware sums may truncate
    instead of rounding). The scales' product, its multiplication with the sum and the addition of the K / 128 blocks
    round by half a step 2^-24 each, the result once more by half a step of its type (or, below its normal range, by half
    its smallest step)."""
    mass = np.abs(x) @ np.abs(w).T
    blocks = -(-x.shape[-1] // BLOCK)
    least = {abi.VF_DT_F32: 2.0 ** -150, abi.VF_DT_F16: 2.0 ** -25, abi.VF_DT_BF16: 2.0 ** -134}[out_dtype]
    inner = mass * (127 * 2.0 ** -23 + (blocks + 2) * 2.0 ** -24)
    return inner + HALF_STEP[out_dtype] * (np.abs(y) + inner) + least
