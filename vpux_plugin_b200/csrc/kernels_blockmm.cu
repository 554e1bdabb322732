// Products of matrices of 8-bit floats with a scale per block of 128 columns, plain or grouped by expert.
//
//   y[m][n] = sum over column blocks b of  (sx[m][b] * sw[n / 128][b]) * sum over k in b of cx[m][k] * cw[n][k]
#include "block_device.cuh"

namespace vf {

namespace {

constexpr int kPlain = 64;   // rows and columns of a tile of the plain kernel
constexpr int kDepth = 32;   // k per step of it

// The plain kernel: 64 x 64 results per CTA, 4 x 4 per thread, codes decoded into shared memory, fp32 multiply-adds on
// the ordinary cores. It makes no demand on alignment.
template <class T>
__global__ void __launch_bounds__(256) k_matmul_blocks_plain(BlockProduct p, int n_tiles, int* flags) {
    __shared__ float xs[kDepth][kPlain + 1], ws[kDepth][kPlain + 1];
    TileWalk walk;
    walk.start(p.offsets, p.offsets ? int(p.w.count) : 1, p.x.rows, kPlain, n_tiles, flags);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const bool x5 = p.x.dtype == VF_DT_F8E5M2, w5 = p.w.dtype == VF_DT_F8E5M2;
    for (int64_t t = blockIdx.x; walk.find(t); t += gridDim.x) {
        const int m0 = walk.row0, m_end = walk.row_end, n0 = walk.n_tile * kPlain;
        const uint8_t* w = p.w.codes + walk.expert * p.w.matrix_stride;
        const float* wscale = p.w.scales + walk.expert * p.w.sms + (n0 / kBlock) * p.w.srs;
        float acc[4][4] = {};
        for (int64_t b = 0; b < p.x.col_blocks; ++b) {
            float part[4][4] = {};
            const int64_t k_end = min(p.x.cols, (b + 1) * kBlock);
            for (int64_t k0 = b * kBlock; k0 < k_end; k0 += kDepth) {
                __syncthreads();
                for (int i = threadIdx.x; i < kPlain * kDepth; i += 256) {
                    const int r = i / kDepth, k = i % kDepth;
                    const bool kin = k0 + k < k_end;
                    xs[k][r] = kin && m0 + r < m_end ? from_codes(p.x.codes[(m0 + r) * p.x.ld + k0 + k], x5).x : 0.f;
                    ws[k][r] = kin && n0 + r < p.w.rows ? from_codes(w[(n0 + r) * p.w.ld + k0 + k], w5).x : 0.f;
                }
                __syncthreads();
#pragma unroll 8
                for (int k = 0; k < kDepth; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) part[i][j] = __fmaf_rn(xs[k][ty + 16 * i], ws[k][tx + 16 * j], part[i][j]);
            }
            const float sw = wscale[b * p.w.scs];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = m0 + ty + 16 * i;
                const float s = m < m_end ? p.x.scales[m * p.x.srs + b * p.x.scs] * sw : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(part[i][j], s, acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
                if (m < m_end && n < p.w.rows) static_cast<T*>(p.out)[m * p.out_ld + n] = to_wide<T>(acc[i][j]);
            }
    }
}

// Row tiles of `bm` rows: exact without offsets; with them an upper bound (every expert may end inside a tile).
int64_t most_row_tiles(const BlockProduct& p, int bm) {
    const int64_t whole = (p.x.rows + bm - 1) / bm;
    return p.offsets ? std::min(p.x.rows, whole + p.w.count) : whole;
}

template <class T>
void launch_plain(vf_ctx* ctx, const BlockProduct& p) {
    const int64_t n_tiles = (p.w.rows + kPlain - 1) / kPlain;
    const int64_t tiles = most_row_tiles(p, kPlain) * n_tiles;
    k_matmul_blocks_plain<T><<<unsigned(std::min<int64_t>(tiles, 8 * ctx->sm_count)), 256, 0, ctx->stream>>>(p, int(n_tiles), ctx->d_flags);
}

}  // namespace

void launch_matmul_blocks(vf_ctx* ctx, const BlockProduct& p) {
    if (p.out_dt == VF_DT_F32) launch_plain<float>(ctx, p);
    else if (p.out_dt == VF_DT_F16) launch_plain<__half>(ctx, p);
    else launch_plain<__nv_bfloat16>(ctx, p);
    VF_CUDA(cudaGetLastError());
    ctx->launches += 1;
}

}  // namespace vf
