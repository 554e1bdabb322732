// Quantising to 8-bit floats with a scale per block of 128 columns, and reading such a matrix back.
//
// Both are one pass: quantising reads an element once (4 or 2 bytes), holds it in registers until its block's largest
// magnitude is known, and writes one byte. They are bound by memory. A block's largest magnitude is found on the bit
// patterns with the sign cleared: for floats their order as integers is the order of the magnitudes, 16-bit types are
// compared two at a time, and infinities and NaN sort above every number, so the maximum also tells whether there was one.
#include "block_device.cuh"
#include "tensor_core.cuh"

namespace vf {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// (The kernels' inputs are not declared __restrict__: the compiler would read them through the path for data that nobody writes while
// the kernel runs, but these kernels start while the one that writes their input still does.)
template <class T>
struct Eight {  // eight consecutive elements of a row, as 32-bit words
    static constexpr int kWords = sizeof(T) * 2;
    uint32_t w[kWords];
};

template <class T>
__device__ __forceinline__ float value_of(const Eight<T>& v, int i) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(v.w[i]);
    } else {
        const uint32_t h = (i & 1) ? v.w[i / 2] >> 16 : v.w[i / 2] & 0xFFFFu;
        if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(uint16_t(h)));
        else return __uint_as_float(h << 16);
    }
}

// `n` of the eight elements at p exist; the others read as zero
template <class T, bool Aligned>
__device__ __forceinline__ Eight<T> load_eight(const T* p, int n) {
    Eight<T> v;
    if (Aligned && n >= 8) {
        const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int i = 0; i < Eight<T>::kWords / 4; ++i) {
            const uint4 x = __ldcs(q + i);
            v.w[4 * i] = x.x;
            v.w[4 * i + 1] = x.y;
            v.w[4 * i + 2] = x.z;
            v.w[4 * i + 3] = x.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.w[i] = i < n ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
    } else {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v.w[i] = (2 * i < n ? uint32_t(q[2 * i]) : 0u) | (2 * i + 1 < n ? uint32_t(q[2 * i + 1]) << 16 : 0u);
    }
    return v;
}

// Largest bit pattern without its sign: one 32-bit pattern, or two 16-bit ones side by side
template <class T>
__device__ __forceinline__ uint32_t top_of(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) return max(a, b);
    else return __vmaxu2(a, b);
}
template <class T>
__device__ __forceinline__ uint32_t top_bits(const Eight<T>& v) {
    constexpr uint32_t kAbs = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
    uint32_t m = v.w[0] & kAbs;
#pragma unroll
    for (int i = 1; i < Eight<T>::kWords; ++i) m = top_of<T>(m, v.w[i] & kAbs);
    return m;
}
template <class T>
__device__ __forceinline__ float magnitude(uint32_t m) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(m);
    const uint32_t h = max(m >> 16, m & 0xFFFFu);
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(uint16_t(h)));
    else return __uint_as_float(h << 16);
}

// two products, each rounded as the single multiplication rounds
__device__ __forceinline__ float2 times(float2 a, float s) {
    const uint64_t r = mul2(pack2(__float_as_uint(a.x), __float_as_uint(a.y)), pack2(__float_as_uint(s), __float_as_uint(s)));
    return make_float2(__uint_as_float(uint32_t(r)), __uint_as_float(uint32_t(r >> 32)));
}

struct Scale {
    float scale, inverse;
};
// The division and the reciprocal are IEEE ones: the scale is the correctly rounded quotient.
template <bool E5M2>
__device__ __forceinline__ Scale scale_of(float top, int* flags) {
    if (__float_as_uint(top) >= 0x7F800000u) set_flag(flags, __float_as_uint(top) == 0x7F800000u ? VF_FLAG_INFINITE : VF_FLAG_NAN);
    Scale s;
    s.scale = fmaxf(__fdiv_rn(top, largest_code(E5M2)), kSmallestScale);
    s.inverse = __frcp_rn(s.scale);
    return s;
}

template <class T, bool E5M2>
__device__ __forceinline__ uint2 codes_of(const Eight<T>& v, float inverse) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 q = times(make_float2(value_of<T>(v, 2 * i), value_of<T>(v, 2 * i + 1)), inverse);
        c[i] = to_codes<E5M2>(q.x, q.y);
    }
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

template <bool Aligned>
__device__ __forceinline__ void store_codes(uint8_t* p, uint2 c, int n) {
    if (Aligned && n >= 8) {
        *reinterpret_cast<uint2*>(p) = c;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = uint8_t((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
}

// Token blocks: half a warp owns 128 columns of a row (8 elements per lane, one 16-byte load of a 16-bit type), a warp
// 256 columns of Rows rows, whose loads are in flight together. The rows' maxima are found by halves: lanes that differ in
// bit 3 of their position exchange what the other one keeps, then bit 2, bit 1, so that after Rows - 1 exchanges instead of
// 4 * Rows a lane is left with one row, for which it alone divides.
//   [8192, 11008] bf16: 43.9 us with eight rows (6.2 TB/s), 54.9 with four, 60.6 with two; 59 us with four when every lane divided
//   for every row. [1, 4096]: 2.5 us with eight, 1.6 with two. Bound by memory (issue slots 62 % busy).
template <class T, int Rows, bool E5M2, bool Aligned>
__global__ void __launch_bounds__(kThreads, 4) k_quantize_tokens(const T* base, int64_t base_ld, Blocks b, int64_t col_tiles, int64_t tiles,
                                                                 int* flags) {
    chain_enter();
    constexpr int kShare = 16 / Rows;  // lanes that end up with the same row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l16 = lane & 15;
    const int64_t all_rows = b.count * b.rows;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t kb = (t % col_tiles) * 2 + (lane >> 4);
        const int64_t c = kb * kBlock + l16 * 8;
        const int64_t r0 = ((t / col_tiles) * kWarps + warp) * Rows;
        const int n = int(min(int64_t(8), b.cols - c));  // elements of this lane, not positive beyond the row
        Eight<T> v[Rows];
        uint32_t m[Rows];
#pragma unroll
        for (int i = 0; i < Rows; ++i) {
            const bool in = r0 + i < all_rows;
            v[i] = load_eight<T, Aligned>(base + (in ? (r0 + i) * base_ld + c : 0), in ? n : 0);
        }
#pragma unroll
        for (int i = 0; i < Rows; ++i) m[i] = top_bits<T>(v[i]);
#pragma unroll
        for (int d = 8, left = Rows / 2; d; d >>= 1, left >>= 1) {
            if (left == 0) {
                m[0] = top_of<T>(m[0], __shfl_xor_sync(0xffffffffu, m[0], d));
            } else {
                const bool upper = l16 & d;
#pragma unroll
                for (int i = 0; i < left; ++i) {
                    const uint32_t keep = upper ? m[i + left] : m[i], give = upper ? m[i] : m[i + left];
                    m[i] = top_of<T>(keep, __shfl_xor_sync(0xffffffffu, give, d));
                }
            }
        }
        const Scale mine = scale_of<E5M2>(magnitude<T>(m[0]), flags);
#pragma unroll
        for (int i = 0; i < Rows; ++i) {
            const float inverse = __shfl_sync(0xffffffffu, mine.inverse, i * kShare, 16);
            if (r0 + i >= all_rows || n <= 0) continue;
            int64_t at = (r0 + i) * b.ld;
            if (b.count > 1) {
                const int64_t mat = (r0 + i) / b.rows;
                at = mat * b.matrix_stride + (r0 + i - mat * b.rows) * b.ld;
            }
            store_codes<Aligned>(b.codes + at + c, codes_of<T, E5M2>(v[i], inverse), n);
        }
        const int64_t r = r0 + l16 / kShare;
        if (l16 % kShare == 0 && r < all_rows && kb < b.col_blocks) {
            const int64_t mat = b.count > 1 ? r / b.rows : 0;
            b.scales[mat * b.sms + (r - mat * b.rows) * b.srs + kb * b.scs] = mine.scale;
        }
    }
}

// Weight blocks: a CTA owns 128 x 128 elements, eight loads of eight elements per thread, all in flight before the
// maximum is taken; the elements stay in registers until the codes are written. [11008, 4096] f16: 26.3 us (5.1 TB/s; [28672, 8192]
// 118 us, 6.0 TB/s: 2752 tiles make 4.6 rounds). Tried: 512 threads with four loads each 27.7, five CTAs per multiprocessor 28.7 (it
// spills), a persistent grid 26.9, rows of blocks before columns 28.0.
template <class T, bool E5M2, bool Aligned>
__global__ void __launch_bounds__(kThreads) k_quantize_weights(const T* base, int64_t base_ld, Blocks b, int64_t tiles, int* flags) {
    chain_enter();
    constexpr int kIter = kBlock / (kThreads / 16);
    __shared__ uint32_t tops[2][kThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int turn = 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, turn ^= 1) {
        const int64_t kb = t % b.col_blocks, u = t / b.col_blocks;
        const int64_t rb = u % b.row_blocks, mat = u / b.row_blocks;
        const int64_t c = kb * kBlock + (threadIdx.x & 15) * 8;
        const int64_t r0 = rb * kBlock + (threadIdx.x >> 4);
        const int n = int(min(int64_t(8), b.cols - c));
        Eight<T> v[kIter];
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const int64_t r = r0 + i * (kThreads / 16);
            const bool in = r < b.rows;
            v[i] = load_eight<T, Aligned>(base + (in ? (mat * b.rows + r) * base_ld + c : 0), in ? n : 0);
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kIter; ++i) m = top_of<T>(m, top_bits<T>(v[i]));
#pragma unroll
        for (int d = 16; d; d >>= 1) m = top_of<T>(m, __shfl_xor_sync(0xffffffffu, m, d));
        if (lane == 0) tops[turn][warp] = m;
        __syncthreads();  // (two sets of slots: a warp that is a tile ahead writes the other one)
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) m = top_of<T>(m, tops[turn][w]);
        const Scale s = scale_of<E5M2>(magnitude<T>(m), flags);
        if (threadIdx.x == 0) b.scales[mat * b.sms + rb * b.srs + kb * b.scs] = s.scale;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const int64_t r = r0 + i * (kThreads / 16);
            if (r < b.rows && n > 0) store_codes<Aligned>(b.codes + mat * b.matrix_stride + r * b.ld + c, codes_of<T, E5M2>(v[i], s.inverse), n);
        }
    }
}

// Reading back: a lane turns the codes behind one 16-byte store into it (8 codes for a 16-bit type, 4 for f32), so that
// every store instruction of a warp is one run of 512 bytes; Rows rows are in flight per warp.
// 11008 x 4096 to f16: 23.7 us with eight, 25.3 with four, 28.3 with two; [1003, 1111] to f32: 4.0 us with eight, 3.2 with two.
template <class T, int Rows, bool E5M2, bool Aligned>
__global__ void __launch_bounds__(kThreads, 4) k_dequantize_blocks(Blocks b, T* __restrict__ dst, int64_t dst_ld, int64_t col_tiles, int64_t tiles) {
    chain_enter();
    constexpr int kPer = 16 / sizeof(T);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t all_rows = b.count * b.rows;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t c = (t % col_tiles) * (32 * kPer) + lane * kPer;
        const int64_t r0 = ((t / col_tiles) * kWarps + warp) * Rows;
        const int n = int(min(int64_t(kPer), b.cols - c));
        if (n <= 0) continue;
        uint32_t w[Rows][kPer / 4];
        float s[Rows];
#pragma unroll
        for (int i = 0; i < Rows; ++i) {
            const int64_t rr = min(r0 + i, all_rows - 1);
            const int64_t mat = b.count > 1 ? rr / b.rows : 0, r = rr - mat * b.rows;
            const uint8_t* p = b.codes + mat * b.matrix_stride + r * b.ld + c;
            s[i] = b.scales[mat * b.sms + (b.block_rows == 1 ? r : r / kBlock) * b.srs + c / kBlock * b.scs];
            if (Aligned && n == kPer) {
                if constexpr (kPer == 8) {
                    const uint2 x = __ldcs(reinterpret_cast<const uint2*>(p));
                    w[i][0] = x.x;
                    w[i][1] = x.y;
                } else {
                    w[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
                }
            } else {
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    if ((k & 3) == 0) w[i][k / 4] = 0;
                    if (k < n) w[i][k / 4] |= uint32_t(p[k]) << (8 * (k & 3));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < Rows; ++i) {
            if (r0 + i >= all_rows) break;
            alignas(16) T out[kPer];
#pragma unroll
            for (int k = 0; k < kPer; k += 2) {
                const float2 f = times(from_codes((w[i][k / 4] >> (8 * (k & 3))) & 0xFFFFu, E5M2), s[i]);
                out[k] = to_wide<T>(f.x);
                out[k + 1] = to_wide<T>(f.y);
            }
            T* q = dst + (r0 + i) * dst_ld + c;
            if (Aligned && n == kPer) {
                *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(out);
            } else {
#pragma unroll
                for (int k = 0; k < kPer; ++k)
                    if (k < n) q[k] = out[k];
            }
        }
    }
}

bool aligned_to(const void* p, int64_t step_bytes, int64_t step2_bytes, int64_t a) {
    return reinterpret_cast<uintptr_t>(p) % uintptr_t(a) == 0 && step_bytes % a == 0 && step2_bytes % a == 0;
}

unsigned grid_for(int64_t tiles) {
    return unsigned(std::min<int64_t>(tiles, 1 << 30));
}

void launched(vf_ctx* ctx) {
    VF_CUDA(cudaGetLastError());
    ctx->launches += 1;
}

template <class F>
void with_flag(bool f, F&& body) {
    if (f) body(std::true_type{});
    else body(std::false_type{});
}

template <class F>
void with_wide(int dt, F&& body) {
    if (dt == VF_DT_F32) body(float{});
    else if (dt == VF_DT_F16) body(__half{});
    else body(__nv_bfloat16{});
}

// Rows per warp: many keep more loads in flight, few spread a small matrix over more multiprocessors
bool is_small(vf_ctx* ctx, int64_t elements) {
    return elements < int64_t(ctx->sm_count) * kThreads * 8 * 8;
}

}  // namespace

void launch_quantize_blocks(vf_ctx* ctx, const void* base, int base_dt, int64_t base_ld, const Blocks& b) {
    const int es = dtype_bits(base_dt) / 8;
    const bool al = aligned_to(base, base_ld * es, 0, 16) && aligned_to(b.codes, b.ld, b.count > 1 ? b.matrix_stride : 0, 8);
    const int64_t rows = b.count * b.rows;
    with_wide(base_dt, [&](auto t) {
        with_flag(b.dtype == VF_DT_F8E5M2, [&](auto e5) {
            with_flag(al, [&](auto vec) {
                using T = decltype(t);
                constexpr int kMany = sizeof(T) == 4 || !vec.value ? 4 : 8;  // (registers)
                const T* src = static_cast<const T*>(base);
                if (b.block_rows == 1) {
                    const bool small = is_small(ctx, rows * b.cols);
                    const int64_t per = kWarps * (small ? 2 : kMany), ct = (b.col_blocks + 1) / 2, tiles = ct * ((rows + per - 1) / per);
                    VF_CUDA(launch_chained(small ? k_quantize_tokens<T, 2, e5.value, vec.value> : k_quantize_tokens<T, kMany, e5.value, vec.value>,
                                           dim3(grid_for(tiles)), dim3(kThreads), 0, ctx->stream, src, base_ld, b, ct, tiles, ctx->d_flags));
                } else {
                    const int64_t tiles = b.count * b.row_blocks * b.col_blocks;
                    VF_CUDA(launch_chained(k_quantize_weights<T, e5.value, vec.value>, dim3(grid_for(tiles)), dim3(kThreads), 0, ctx->stream, src, base_ld, b,
                                           tiles, ctx->d_flags));
                }
            });
        });
    });
    launched(ctx);
}

void launch_dequantize_blocks(vf_ctx* ctx, const Blocks& b, void* dst, int dst_dt, int64_t dst_ld) {
    const int es = dtype_bits(dst_dt) / 8, per = 16 / es;
    const bool al = aligned_to(dst, dst_ld * es, 0, 16) && aligned_to(b.codes, b.ld, b.count > 1 ? b.matrix_stride : 0, per);
    const bool small = is_small(ctx, b.count * b.rows * b.cols);
    const int64_t rows = kWarps * (small ? 2 : 8), ct = (b.cols + 32 * per - 1) / (32 * per), tiles = ct * ((b.count * b.rows + rows - 1) / rows);
    with_wide(dst_dt, [&](auto t) {
        with_flag(b.dtype == VF_DT_F8E5M2, [&](auto e5) {
            with_flag(al, [&](auto vec) {
                using T = decltype(t);
                VF_CUDA(launch_chained(small ? k_dequantize_blocks<T, 2, e5.value, vec.value> : k_dequantize_blocks<T, 8, e5.value, vec.value>,
                                       dim3(grid_for(tiles)), dim3(kThreads), 0, ctx->stream, b, static_cast<T*>(dst), dst_ld, ct, tiles));
            });
        });
    });
    launched(ctx);
}

}  // namespace vf
