// Device code shared by the kernels on 8-bit floating-point blocks: conversions, and the walk over the tiles of a
// product whose rows are grouped by expert.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "block_plan.h"
#include "blocks.h"
#include "device_utils.cuh"

namespace vf {

constexpr float kSmallestScale = 1.1754943508222875e-38f;  // 2^-126

__host__ __device__ inline float largest_code(bool e5m2) {
    return e5m2 ? 57344.f : 448.f;
}

// Two values to two 8-bit codes (lo in the low byte): nearest, ties to even, magnitudes beyond the largest saturate.
template <bool E5M2>
__device__ __forceinline__ uint32_t to_codes(float lo, float hi) {
    uint16_t r;
    if constexpr (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two 8-bit codes to floats; exact (every value of either type is an fp16 number).
__device__ __forceinline__ float2 from_codes(uint32_t two, bool e5m2) {
    if (e5m2) {  // e5m2 is the upper half of an fp16
        const uint32_t h = __byte_perm(two, 0u, 0x1404);
        return __half22float2(*reinterpret_cast<const __half2*>(&h));
    }
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(two)));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// fp32 results to the output type: nearest, ties to even, overflow to infinity. (The fold's own bf16 conversion drops
// half of the ties downwards as the reference does; these operators have no such model and round as IEEE 754 says.)
template <class T>
__device__ __forceinline__ T to_wide(float v);
template <>
__device__ __forceinline__ float to_wide<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half to_wide<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 to_wide<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Walks the tiles of a product in ascending order. A tile is `bm` rows of one expert by one of `n_tiles` column tiles;
// the tiles of expert e come before those of e + 1, and within an expert the row tiles of a column tile follow one
// another, so that tiles which run at the same time share the weights. Without offsets all rows form one group. Every method is
// called by whole warps; the number of tiles fits 32 bits (too_many_tiles() sees to it). Offsets are read 32 at a time, one expert
// per lane. Offsets that break the rules are moved as rows_of() says and set a flag; those that keep them cost one vote.
struct TileWalk {
    const int64_t* offsets;
    int* flags;
    int experts, bm, n_tiles;
    int64_t rows;
    int e0;                // expert of lane 0
    int base;              // tiles before expert e0
    int through;           // tiles of experts e0 .. e0 + lane
    int lo, hi;            // this lane's rows
    int reach;             // where the ranges before expert e0 end
    // the tile found
    int expert, row0, row_end, n_tile;

    __device__ __forceinline__ void load() {
        const int lane = int(threadIdx.x & 31), e = e0 + lane;
        const bool in = e < experts;
        const int64_t a = in ? offsets[e] : 0, b = in ? offsets[e + 1] : 0;
        lo = int(a);
        hi = int(b);
        int before = __shfl_up_sync(0xffffffffu, hi, 1);
        if (lane == 0) before = reach;
        if (__all_sync(0xffffffffu, !in || (a >= 0 && a <= b && b <= rows && lo >= before))) {
            reach = __shfl_sync(0xffffffffu, hi, 31);  // (looked at only if there are experts behind these)
        } else {
            int to = max(reach, in ? row_reach(a, b, rows) : 0);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, to, d);
                if (lane >= d) to = max(to, o);
            }
            before = __shfl_up_sync(0xffffffffu, to, 1);
            if (lane == 0) before = reach;
            const RowRange r = rows_of(a, b, rows, before);
            if (in && r.moved) set_flag(flags, VF_FLAG_OFFSETS);
            lo = in ? r.lo : 0;
            hi = in ? r.hi : 0;
            reach = __shfl_sync(0xffffffffu, to, 31);
        }
        through = tiles_of_rows(lo, hi, bm) * n_tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, through, d);
            if (lane >= d) through += o;
        }
    }
    __device__ __forceinline__ void start(const int64_t* offs, int n_experts, int64_t n_rows, int tile_rows, int col_tiles, int* err_flags) {
        offsets = offs;
        experts = n_experts;
        rows = n_rows;
        bm = tile_rows;
        n_tiles = col_tiles;
        flags = err_flags;
        e0 = 0;
        base = 0;
        reach = 0;
        if (offsets) load();
    }
    // Finds tile `t` (not below the one found before); false behind the last tile.
    __device__ __forceinline__ bool find(int t) {
        if (!offsets) {  // one group: nothing to search
            const int m_tiles = (int(rows) + bm - 1) / bm;
            if (t >= m_tiles * n_tiles) return false;
            n_tile = int(uint32_t(t) / uint32_t(m_tiles));
            expert = 0;
            row0 = (t - n_tile * m_tiles) * bm;
            row_end = int(rows);
            return true;
        }
        for (;;) {
            const int here = __shfl_sync(0xffffffffu, through, 31);
            if (t - base < here) break;
            base += here;
            e0 += 32;
            if (e0 >= experts) {
                e0 -= 32;  // a later call ends here again
                base -= here;
                return false;
            }
            load();
        }
        const int rel = t - base;
        const int src = __ffs(__ballot_sync(0xffffffffu, through > rel)) - 1;
        const int l = __shfl_sync(0xffffffffu, lo, src), h = __shfl_sync(0xffffffffu, hi, src);
        const int before = __shfl_sync(0xffffffffu, through, src ? src - 1 : 0);
        const int m_tiles = tiles_of_rows(l, h, bm);
        const int in_expert = src ? rel - before : rel;
        n_tile = int(uint32_t(in_expert) / uint32_t(m_tiles));
        expert = e0 + src;
        row0 = l + (in_expert - n_tile * m_tiles) * bm;
        row_end = h;
        return true;
    }
};

}  // namespace vf
