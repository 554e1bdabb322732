// Kernels on matrices of 8-bit floats with a scale per block of 128 columns (vf_block_matrix): launch wrappers and
// the checked form of the descriptor that they take.
#pragma once

#include "common.h"

namespace vf {

constexpr int kBlock = 128;  // columns per scale, and rows per scale of a weight matrix

struct Blocks {  // a vf_block_matrix whose strides are resolved and whose extents are known to lie in its buffers
    int dtype = VF_DT_INVALID;
    int block_rows = 1;
    int64_t count = 0, rows = 0, cols = 0, ld = 0, matrix_stride = 0;
    int64_t row_blocks = 0, col_blocks = 0;
    int64_t srs = 0, scs = 0, sms = 0;  // scale strides: row block, column block, matrix
    uint8_t* codes = nullptr;
    float* scales = nullptr;
    uint64_t codes_span = 0, scales_span = 0;  // bytes from the first element to behind the last one
};

// `base` is on the device: [count * rows][base_ld] elements of f32 / f16 / bf16
void launch_quantize_blocks(vf_ctx* ctx, const void* base, int base_dt, int64_t base_ld, const Blocks& out);
// rows of `dst` (f32 / f16 / bf16) are dst_ld elements apart
void launch_dequantize_blocks(vf_ctx* ctx, const Blocks& in, void* dst, int dst_dt, int64_t dst_ld);

struct BlockProduct {  // out[m][n] = sum_k x[m][k] w[n][k]; with `offsets`, matrix e of w for rows offsets[e] .. offsets[e + 1]
    Blocks x, w;
    const int64_t* offsets = nullptr;
    void* out = nullptr;
    int out_dt = VF_DT_INVALID;
    int64_t out_ld = 0;
    uint64_t out_span = 0;  // bytes from the first result to behind the last one
};
void launch_matmul_blocks(vf_ctx* ctx, const BlockProduct& p);

}  // namespace vf
