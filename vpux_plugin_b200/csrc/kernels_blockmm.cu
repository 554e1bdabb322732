// Products of matrices of 8-bit floats with a scale per block of 128 columns, plain or grouped by expert.
//
//   y[m][n] = sum over column blocks b of  (sx[m][b] * sw[n / 128][b]) * sum over k in b of cx[m][k] * cw[n][k]
#include <atomic>

#include "block_device.cuh"
#include "tensor_core.cuh"

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
    for (int t = blockIdx.x; walk.find(t); t += gridDim.x) {
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

// Tiles of bm rows by bn columns, as an upper bound (below kTileLimit: the entry points have refused what is not)
int64_t most_tiles(const BlockProduct& p, int bm, int bn) {
    return most_row_tiles(p.x.rows, p.offsets ? p.w.count : 0, bm) * ((p.w.rows + bn - 1) / bn);
}

template <class T>
void launch_plain(vf_ctx* ctx, const BlockProduct& p) {
    const int64_t n_tiles = (p.w.rows + kPlain - 1) / kPlain;
    const int64_t tiles = most_tiles(p, kPlain, kPlain);
    k_matmul_blocks_plain<T><<<unsigned(std::min<int64_t>(tiles, 8 * ctx->sm_count)), 256, 0, ctx->stream>>>(p, int(n_tiles), ctx->d_flags);
}


// ---- tensor cores ------------------------------------------------------------------------------------------------------
// One column block is four matrix instructions of 32 k. It starts from zero in one of NBUF accumulators in tensor memory; while
// the tensor core fills the next one, the epilogue warps read it, multiply it by the column block's scales and add it to the
// running sums, which stay in registers:   sum += part * (sx * sw)
// Weights have one scale per 128 rows, activations one per row. That decides which operand is which:
//   many rows    the 128-row operand is 128 activations, one per thread of a group of four epilogue warps, and a thread multiplies
//                all of its columns (outputs) by the same number. (With the weights there, a 256-column tile reads 256 scales
//                per column block and thread from shared memory: [4096, 11008, 4096] 281 us against 228 at that stage.)
//   few rows     the 128-row operand is 128 outputs, the other one 16 to 128 activations, so that no matrix instruction works on
//                rows that are not there; the scales are one per column.
// Few rows make few tiles as well: the column blocks of a tile are then spread over the CTAs of a cluster, which push their sums
// to each other's shared memory, four columns to the CTA that owns them, where they are added in the order of the ranks.
//
// Warps: the first ones are the epilogue, in groups of four that read a quarter of tensor memory's lanes each; then one that finds
// tiles and copies them in (bulk tensor copies into a ring of STAGES), one that issues the matrix instructions, and one that
// brings the scales of eight column blocks at a time into a ring of their own.
//
// Measured ([rows, outputs, columns]): [4096, 11008, 4096] 192 us in calls that follow one another for seconds, 1.93 PFLOP/s, at the
// 1.43 GHz that the power limit then leaves; 166 us in bursts of 84 launches from idle. That is about 860 cycles per column block and
// tile, of which the tensor core needs 512 (tensor pipe active 64 % of the time). What bounds it: two accumulators of 256 columns fill the
// tensor memory, and from one use of an accumulator to the next pass the instructions (512), the epilogue's 480 cycles of reading it
// and three hand-overs through barriers; and the power limit.
// Tried before the issuing warp became uniform, when this size took 180 in bursts, and not since: pairs of CTAs (256 x 256 tiles) 177-184 us, 128 x 192 tiles
// 206, four epilogue groups 193-199, 32 columns per load 190, the column-block loop unrolled twice 221-290 (it spills).
// [1, 11008, 4096] 10.1 us and [48, 4096, 11008] 13.9 us at 4.5 and 3.3 TB/s of weights; [1, 32000, 8192] 43.4 us at 6.0 TB/s: a
// launch costs 3.5 us of its own, and joining the CTAs of a cluster 1 to 3.
constexpr int kGiven = 72, kTaken = 216;  // registers per thread after the trade: 128 * 72 + 256 * 216 = 384 * 168

template <bool SWAP_, int BN_, int STAGES_, int NBUF_, int GROUPS_, int PER_SM_, int LOAD_ = 32>
struct Shape {
    static constexpr bool SWAP = SWAP_;  // the weights are the 128-row operand; else the activations are
    static constexpr int BN = BN_, STAGES = STAGES_, NBUF = NBUF_, GROUPS = GROUPS_, PER_SM = PER_SM_, LOAD = LOAD_;
    static constexpr int kCols = BN / GROUPS;               // columns of the accumulator per epilogue warp
    static constexpr int kTokens = SWAP ? BN : 128, kOutputs = SWAP ? 128 : BN;  // a tile's results
    static constexpr int kEpilogue = 4 * GROUPS, kCopies = kEpilogue, kIssue = kEpilogue + 1, kScaling = kEpilogue + 2;  // warps
    static constexpr bool kTrades = kCols > 64;             // the warps behind the epilogue's give it registers, as a group of four
    static constexpr int kThreads = 32 * (kEpilogue + (kTrades ? 4 : 3));
    // scales of kAhead column blocks at a time: [kAhead][kTileRows] of the activations, then [kTileBlocks][kAhead] of the weights,
    // one row for each epilogue group's columns
    static constexpr int kAhead = 8, kSlots = 2, kTileRows = SWAP ? BN : 128, kTileBlocks = SWAP ? 1 : GROUPS;
    static constexpr int kSlotBytes = kAhead * (kTileRows + kTileBlocks) * 4;
    static constexpr int kStageBytes = (128 + BN) * kBlock;
    static constexpr int kTmem = NBUF * BN;  // a power of two
    // clusters share a tile's column blocks: four columns of a tile at a time, the CTAs of a cluster own them in turn
    static constexpr int kFours = BN / 4, kParts = BN == 16 ? 8 : (BN == 32 ? 10 : BN / 4);
    static constexpr int kRing = STAGES * kStageBytes;
    static constexpr int kScales = kSlots * kSlotBytes;
    static constexpr int kExtra = SWAP ? kParts * 128 * 16 : 4 * GROUPS * 4096;  // partial sums; results on their way out
    static constexpr int kBars = 2 * STAGES + 2 * NBUF + 2 + 2 * 2 + 2 * kSlots;
    static constexpr int kSmem = 1024 + kRing + kScales + kExtra + 2 * 16 + kBars * 8 + 16;
};

// A warp's 32 rows x N results (one row per lane) to memory, 128 bytes of every row at a time: through shared memory, so that
// eight lanes write one row's 128 bytes, in 16-byte units where every row allows them. `rows` and `cols` of them exist.
template <class T, int N>
__device__ __forceinline__ void store_rows(char* stage, T* out, int64_t ld, const uint64_t (&acc)[N / 2], int rows, int cols, int lane) {
    constexpr int kPer = 16 / sizeof(T), kChunk = 8 * kPer;  // elements per 16 bytes, per 128 bytes
    const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15u) == 0 && (ld * sizeof(T)) % 16 == 0;
#pragma unroll
    for (int c = 0; c < N; c += kChunk) {
        __syncwarp();  // the chunk before has been read
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            alignas(16) T v[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int k = c + u * kPer + i;
                v[i] = to_wide<T>(__uint_as_float(uint32_t(acc[k / 2] >> (32 * (k & 1)))));
            }
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ lane) & 7) * 16) = *reinterpret_cast<const uint4*>(v);
        }
        __syncwarp();
        if (aligned && c + kChunk <= cols) {
            const int u = lane & 7;
#pragma unroll
            for (int r = lane >> 3; r < 32; r += 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((u ^ r) & 7) * 16);
                if (r < rows) *reinterpret_cast<uint4*>(out + r * ld + c + u * kPer) = v;
            }
        } else {
#pragma unroll 8
            for (int r = 0; r < 32; ++r)
#pragma unroll
                for (int k = lane; k < kChunk; k += 32)
                    if (r < rows && c + k < cols) out[r * ld + c + k] = *reinterpret_cast<const T*>(stage + r * 128 + ((k / kPer ^ r) & 7) * 16 + k % kPer * sizeof(T));
        }
    }
}

// Position in a ring of N and the phase of its barriers; the producer of a ring waits for the other phase than its consumer.
template <int N>
struct RingAt {
    uint32_t i = 0, phase = 0;
    __device__ __forceinline__ void next() {
        if (++i == N) {
            i = 0;
            phase ^= 1;
        }
    }
};

template <class S, class T>
__global__ void __launch_bounds__(S::kThreads, S::PER_SM)
    k_matmul_blocks(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ BlockProduct p, int n_tiles,
                    uint32_t idesc, int* flags) {
    constexpr int BN = S::BN, STAGES = S::STAGES, NBUF = S::NBUF;
    extern __shared__ char raw[];
    char* const base = raw + (1024 - (smem_addr(raw) & 1023)) % 1024;  // the swizzle works on 1024-byte units
    char* const ring = base;
    float* const scales = reinterpret_cast<float*>(base + S::kRing);
    char* const extra = base + S::kRing + S::kScales;
    int4* const tiles = reinterpret_cast<int4*>(extra + S::kExtra);  // expert (-1: no more tiles), row0, row_end, n_tile
    uint64_t* const bars = reinterpret_cast<uint64_t*>(tiles + 2);
    uint32_t* const tmem_at = reinterpret_cast<uint32_t*>(bars + S::kBars);
    volatile int* const gave_up = reinterpret_cast<volatile int*>(tmem_at + 1);
    const uint32_t full = smem_addr(bars), empty = full + 8 * STAGES;                      // ring
    const uint32_t done = empty + 8 * STAGES, taken = done + 8 * NBUF;                     // accumulators
    const uint32_t parts_full = taken + 8 * NBUF, drained = parts_full + 8;
    const uint32_t tile_there = drained + 8, tile_read = tile_there + 16;
    const uint32_t slot_full = tile_read + 16, slot_read = slot_full + 8 * S::kSlots;

    // What is the same for a whole warp comes from one lane: the compiler then knows that it is, keeps the warps' branches and the
    // operands of the matrix and copy instructions uniform, and a column block's four instructions and two commits are issued in
    // half the time ([4096, 11008, 4096] 180 -> 165 us in bursts, [400, 4096, 11008] 37 -> 26 us).
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t ranks = S::SWAP ? __shfl_sync(0xffffffffu, cluster_size(), 0) : 1, rank = S::SWAP ? __shfl_sync(0xffffffffu, cluster_rank(), 0) : 0;  // CTAs that share a tile's column blocks
    const bool in_cluster = ranks > 1;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            bar_init(full + 8 * i, 1);
            bar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < NBUF; ++i) {
            bar_init(done + 8 * i, 1);
            bar_init(taken + 8 * i, 4 * S::GROUPS);
        }
        bar_init(parts_full, 1);
        bar_init(drained, 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(tile_there + 8 * i, 1);
            bar_init(tile_read + 8 * i, S::kEpilogue + 2);
        }
        for (int i = 0; i < S::kSlots; ++i) {
            bar_init(slot_full + 8 * i, 32);
            bar_init(slot_read + 8 * i, S::kEpilogue);
        }
        *gave_up = 0;
        bar_init_fence();
        tma_prefetch_map(&xmap);
        tma_prefetch_map(&wmap);
    }
    if (warp == S::kIssue) tmem_alloc(smem_addr(tmem_at), S::kTmem);
    tc_fence_before();
    __syncthreads();
    if (in_cluster) cluster_arrive();  // waited for before anything goes to another CTA
    bool joined = !in_cluster, left = !in_cluster;
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);
    const int kbs = int(p.x.col_blocks), kb0 = int(rank * uint32_t(kbs) / ranks), kb1 = int((rank + 1) * uint32_t(kbs) / ranks);
    // Set up while the kernel before this one was ending; from chain_enter() on its results are read. The weights of the first
    // tile are asked for before that: into the L2 cache, where it does not matter whether that kernel writes them.
    if (warp == S::kCopies && !p.offsets) {
        const int64_t t = blockIdx.x / ranks;
        const int n_tile = int(t / ((p.x.rows + S::kTokens - 1) / S::kTokens));
        if (lane < STAGES && kb0 + lane < kb1 && n_tile < n_tiles) tma_prefetch_3d(&wmap, (kb0 + lane) * kBlock, n_tile * S::kOutputs, 0);
        __syncwarp();
    }
    chain_enter();

    // The next tile, as the copying warp has found it; by whole warps
    int4 tile;
    uint32_t turn = 0;
    auto next_tile = [&]() {
        const uint32_t i = turn & 1;
        if (!__all_sync(0xffffffffu, bar_wait(tile_there + 8 * i, (turn >> 1) & 1, gave_up))) return false;
        tile = tiles[i];
        __syncwarp();
        if (lane == 0) bar_arrive(tile_read + 8 * i);
        ++turn;
        return tile.x >= 0;
    };

    if (warp >= S::kEpilogue) {
        if constexpr (S::kTrades) regs_give<kGiven>();
        if (warp == S::kCopies) {  // ---- finding tiles, copying them in
            TileWalk walk;
            walk.start(p.offsets, p.offsets ? int(p.w.count) : 1, p.x.rows, S::kTokens, n_tiles, flags);
            uint32_t it = 0;
            RingAt<STAGES> at_stage;
            bool ok = true;
            for (int t = blockIdx.x / ranks; ok; t += gridDim.x / ranks, ++turn) {
                bool more = walk.find(t);
                if (in_cluster && turn && more) {  // a cluster joins its sums once; the launch has one for every tile that there can be
                    set_flag(flags, VF_FLAG_OFFSETS);
                    more = false;
                }
                const uint32_t i = turn & 1;
                ok = __all_sync(0xffffffffu, bar_wait(tile_read + 8 * i, ((turn >> 1) & 1) ^ 1, gave_up));
                if (!ok) break;
                if (lane == 0) {
                    tiles[i] = more ? make_int4(walk.expert, walk.row0, walk.row_end, walk.n_tile) : make_int4(-1, 0, 0, 0);
                    bar_arrive(tile_there + 8 * i);
                }
                if (!more) break;
                for (int kb = kb0; kb < kb1; ++kb, ++it, at_stage.next()) {
                    const uint32_t s = at_stage.i, at = smem_addr(ring) + s * S::kStageBytes;
                    ok = __all_sync(0xffffffffu, bar_wait(empty + 8 * s, at_stage.phase ^ 1, gave_up));
                    if (!ok) break;
                    if (elect_one()) {
                        bar_expect(full + 8 * s, S::kStageBytes);
                        tma_load_3d(S::SWAP ? at : at + 128 * kBlock, &wmap, full + 8 * s, kb * kBlock, walk.n_tile * S::kOutputs, walk.expert);
                        tma_load_2d(S::SWAP ? at + 128 * kBlock : at, &xmap, full + 8 * s, kb * kBlock, walk.row0);
                    }
                }
            }
            if (ok && lane == 0)  // every arrival at the ring's barriers has happened before the CTA ends
                for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i) bar_wait(empty + 8 * (i % STAGES), (i / STAGES) & 1, gave_up);
            if (!ok && lane == 0)  // the copies in flight land before the CTA ends
                for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i) {
                    const uint64_t t0 = global_ns();
                    while (!bar_try(full + 8 * (i % STAGES), (i / STAGES) & 1) && global_ns() - t0 < kDrainLimitNs) {
                    }
                }
        } else if (warp == S::kIssue) {  // ---- matrix instructions
            RingAt<STAGES> at_stage;
            RingAt<NBUF> at_sum;
            bool ok = true;
            while (ok && next_tile()) {
                for (int kb = kb0; kb < kb1; ++kb, at_stage.next(), at_sum.next()) {
                    const uint32_t s = at_stage.i, b = at_sum.i;
                    const uint32_t at = smem_addr(ring) + s * S::kStageBytes;
                    const uint64_t ad = tc_operand(at), bd = tc_operand(at + 128 * kBlock);
                    // Both are asked at once, since an answer takes time even if it is yes; else the accumulator last: the tensor core waits for it.
                    const bool filled = bar_try(full + 8 * s, at_stage.phase), free = bar_try(taken + 8 * b, at_sum.phase ^ 1);
                    if (!__all_sync(0xffffffffu, filled && free))
                        ok = __all_sync(0xffffffffu, bar_wait(full + 8 * s, at_stage.phase, gave_up) && bar_wait(taken + 8 * b, at_sum.phase ^ 1, gave_up));
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < kBlock / 32; ++k) tc_mma_f8(tmem + b * BN, ad + 2 * k, bd + 2 * k, idesc, k > 0);
                        tc_commit(done + 8 * b);
                        tc_commit(empty + 8 * s);
                    }
                }
            }
            if (!ok && elect_one()) {  // the instructions in flight end before their memory is given back
                tc_commit(drained);
                const uint64_t t0 = global_ns();
                while (!bar_try(drained, 0) && global_ns() - t0 < kDrainLimitNs) {
                }
            }
        } else if (warp == S::kScaling) {  // ---- scales of kAhead column blocks into the next slot, by asynchronous copies
            RingAt<S::kSlots> at_slot;
            bool ok = true;
            while (ok && next_tile()) {
                const int row = tile.y + lane;
                const float* const sx = p.x.scales + row * p.x.srs;
                for (int kb = kb0; kb < kb1; kb += S::kAhead, at_slot.next()) {
                    const uint32_t slot = at_slot.i, at = smem_addr(scales) + slot * S::kSlotBytes;
                    ok = __all_sync(0xffffffffu, bar_wait(slot_read + 8 * slot, at_slot.phase ^ 1, gave_up));
                    if (!ok) break;
#pragma unroll
                    for (int a = 0; a < S::kAhead; ++a)
#pragma unroll
                        for (int i = 0; i < (S::kTileRows + 31) / 32; ++i) {
                            if (S::kTileRows < 32 && lane >= S::kTileRows) break;
                            const bool in = kb + a < kb1 && row + 32 * i < tile.z;
                            copy_word_async(at + (a * S::kTileRows + 32 * i + lane) * 4, in ? sx + 32 * i * p.x.srs + (kb + a) * p.x.scs : p.x.scales, in);
                        }
                    if (lane < S::kTileBlocks * S::kAhead) {
                        const int a = lane % S::kAhead;
                        const bool in = kb + a < kb1;
                        const int64_t wb = min((int64_t(tile.w) * S::kOutputs + (S::SWAP ? 0 : lane / S::kAhead * S::kCols)) / 128, p.w.row_blocks - 1);
                        copy_word_async(at + (S::kAhead * S::kTileRows + lane) * 4, in ? p.w.scales + tile.x * p.w.sms + wb * p.w.srs + (kb + a) * p.w.scs : p.w.scales, in);
                    }
                    bar_arrive_copies(slot_full + 8 * slot);
                }
            }
            copies_wait_all();
        }
    } else {  // ---- epilogue
        if constexpr (S::kTrades) regs_take<kTaken>();
        constexpr int kCols = S::kCols;
        const int quarter = warp & 3, col0 = warp / 4 * kCols;
        const uint32_t my_tmem = tmem + (uint32_t(quarter) << 21) + col0;
        RingAt<NBUF> at_sum;
        RingAt<S::kSlots> at_slot;
        bool ok = true;
        while (ok && next_tile()) {
            uint64_t acc[kCols / 2];
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) acc[i] = 0;
            const float* const my_scale = scales + (S::SWAP ? col0 : quarter * 32 + lane);
            const float* const my_weight = scales + S::kAhead * S::kTileRows + (S::SWAP ? 0 : warp / 4 * S::kAhead);
            // A wait that gave up is looked at once per tile (a vote after every wait cost 80 cycles per column block): what the warps
            // read until then is not meant, but lies where it should.
            for (int kb = kb0; kb < kb1; kb += S::kAhead, at_slot.next()) {
                bar_wait(slot_full + 8 * at_slot.i, at_slot.phase, gave_up);
                const float* sx = my_scale + at_slot.i * (S::kSlotBytes / 4);
                const float* sw = my_weight + at_slot.i * (S::kSlotBytes / 4);
                for (int todo = min(S::kAhead, kb1 - kb); todo > 0; --todo, sx += S::kTileRows, ++sw, at_sum.next()) {
                    const uint32_t b = at_sum.i;
                    float scale = *sw;
                    if (!S::SWAP) scale = __fmul_rn(*sx, scale);
                    const uint64_t s2 = pack2(__float_as_uint(scale), __float_as_uint(scale));
                    bar_wait(done + 8 * b, at_sum.phase, gave_up);
                    __syncwarp();
                    tc_fence_after();
                    uint32_t v[2][S::LOAD];  // one part being multiplied, the next one on its way
                    tmem_load(v[0], my_tmem + b * BN);
#pragma unroll
                    for (int c = 0; c < kCols; c += S::LOAD) {
                        uint32_t(&u)[S::LOAD] = v[c / S::LOAD & 1];
                        tmem_load_wait(u);
                        if (c + S::LOAD < kCols) tmem_load(v[(c / S::LOAD + 1) & 1], my_tmem + b * BN + c + S::LOAD);
                        if (c + S::LOAD == kCols) {  // all of it is in registers: the accumulator may be written again
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive(taken + 8 * b);
                        }
                        if constexpr (S::SWAP) {
#pragma unroll
                            for (int i = 0; i < S::LOAD; i += 4) {
                                const uint4 s4 = *reinterpret_cast<const uint4*>(sx + c + i);
                                fma2(acc[(c + i) / 2], pack2(u[i], u[i + 1]), mul2(pack2(s4.x, s4.y), s2));
                                fma2(acc[(c + i) / 2 + 1], pack2(u[i + 2], u[i + 3]), mul2(pack2(s4.z, s4.w), s2));
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < S::LOAD; i += 2) fma2(acc[(c + i) / 2], pack2(u[i], u[i + 1]), s2);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) bar_arrive(slot_read + 8 * at_slot.i);
            }
            ok = !__any_sync(0xffffffffu, *gave_up);
            if (!ok) break;
            const int here = tile.z - tile.y;
            if constexpr (!S::SWAP) {
                const int m = tile.y + quarter * 32, n = tile.w * S::kOutputs + col0;
                if (m < tile.z && n < p.w.rows)
                    store_rows<T, kCols>(extra + warp * 4096, static_cast<T*>(p.out) + m * p.out_ld + n, p.out_ld, acc, min(32, tile.z - m),
                                         int(min(int64_t(kCols), p.w.rows - n)), lane);
                continue;
            }
            const int n = tile.w * 128 + quarter * 32 + lane;
            T* const out = static_cast<T*>(p.out) + int64_t(tile.y) * p.out_ld + n;
            if (S::SWAP && ranks > 1) {
                // Four columns go to the CTA that owns them, which has a place for every rank's; the only tile of this
                // cluster (the copying warp sees to it), so nobody has to be asked whether a place is free.
                if constexpr (S::SWAP) {
                    const int fours = (min(here, BN) + 3) / 4, mine = fours > int(rank) ? (fours - int(rank) - 1) / int(ranks) + 1 : 0;
                    const int places = (S::kFours + int(ranks) - 1) / int(ranks);
                    if (threadIdx.x == 0 && mine) bar_expect(parts_full, mine * int(ranks) * 128 * 16);
                    __syncwarp();
                    cluster_wait();
                    joined = true;
                    const uint32_t my_place = smem_addr(extra) + (rank * places * 128 + quarter * 32 + lane) * 16;
                    uint32_t owner = uint32_t(col0 / 4) % ranks, place = my_place + uint32_t(col0 / 4) / ranks * 128 * 16;
#pragma unroll
                    for (int i = 0; i < kCols / 4; ++i) {
                        if (col0 / 4 + i < fours)
                            push_to_rank(place, parts_full, owner, uint32_t(acc[2 * i]), uint32_t(acc[2 * i] >> 32), uint32_t(acc[2 * i + 1]),
                                         uint32_t(acc[2 * i + 1] >> 32));
                        if (++owner == ranks) {
                            owner = 0;
                            place += 128 * 16;
                        }
                    }
                    __syncwarp();
                    cluster_arrive_relaxed();
                    left = true;
                    if (!mine) continue;
                    ok = __all_sync(0xffffffffu, bar_wait(parts_full, 0, gave_up));
                    if (!ok) break;
                    const float4* const parts = reinterpret_cast<const float4*>(extra) + quarter * 32 + lane;
                    for (int j = warp / 4; j < mine; j += S::GROUPS) {
                        float4 q[8];  // all of them on their way before the first is added
#pragma unroll
                        for (int r = 0; r < 8; ++r) q[r] = r < int(ranks) ? parts[(r * places + j) * 128] : make_float4(0.f, 0.f, 0.f, 0.f);
                        float4 v = q[0];
#pragma unroll
                        for (int r = 1; r < 8; ++r) {
                            v.x = __fadd_rn(v.x, q[r].x);
                            v.y = __fadd_rn(v.y, q[r].y);
                            v.z = __fadd_rn(v.z, q[r].z);
                            v.w = __fadd_rn(v.w, q[r].w);
                        }
                        const int i = 4 * (int(rank) + j * int(ranks));
                        if (n >= p.w.rows) continue;
                        out[int64_t(i) * p.out_ld] = to_wide<T>(v.x);
                        if (i + 1 < here) out[int64_t(i + 1) * p.out_ld] = to_wide<T>(v.y);
                        if (i + 2 < here) out[int64_t(i + 2) * p.out_ld] = to_wide<T>(v.z);
                        if (i + 3 < here) out[int64_t(i + 3) * p.out_ld] = to_wide<T>(v.w);
                    }
                }
            } else if (n < p.w.rows) {
#pragma unroll
                for (int i = 0; i < kCols; ++i)
                    if (col0 + i < here) out[int64_t(col0 + i) * p.out_ld] = to_wide<T>(__uint_as_float(uint32_t(acc[i / 2] >> (32 * (i & 1)))));
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == S::kIssue) tmem_free(tmem, S::kTmem);
    if (threadIdx.x == 0 && *gave_up) set_flag(flags, VF_FLAG_GAVE_UP);
    __syncwarp();
    // no CTA ends while another one may still write to it
    if (!joined) cluster_wait();
    if (!left) cluster_arrive_relaxed();
    if (in_cluster) cluster_wait();
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            raise(VF_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return f;
}

// A single row has no second one to be a pitch away from.
int64_t row_pitch(const Blocks& b) {
    return b.rows == 1 ? align_up(b.cols, 16) : b.ld;
}

// Boxes of `box_rows` rows by 128 columns of a matrix (rank 2) or a stack of them (rank 3); what lies outside reads as zero.
CUtensorMap map_codes(const Blocks& b, int rank, int box_rows) {
    CUtensorMap m;
    const cuuint64_t dim[3] = {cuuint64_t(b.cols), cuuint64_t(b.rows), cuuint64_t(b.count)};
    const int64_t ld = row_pitch(b);
    const cuuint64_t stride[2] = {cuuint64_t(ld), cuuint64_t(b.count > 1 ? b.matrix_stride : ld)};
    const cuuint32_t box[3] = {kBlock, cuuint32_t(box_rows), 1}, one[3] = {1, 1, 1};
    CUresult r = CUDA_SUCCESS;
    for (int attempt = 0; attempt < 2; ++attempt) {
        r = encode_tiled()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, cuuint32_t(rank), b.codes, dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_ERROR_INVALID_CONTEXT) break;
        int dev = 0;  // a thread's first call of the driver: let the runtime make its context current
        VF_CUDA(cudaGetDevice(&dev));
        VF_CUDA(cudaSetDevice(dev));
    }
    if (r != CUDA_SUCCESS) raise(VF_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
    return m;
}

bool fits_bulk_copies(const Blocks& b) {  // start and pitches of 16-byte units, pitches below 2^40 bytes
    return (reinterpret_cast<uintptr_t>(b.codes) & 15u) == 0 && row_pitch(b) % 16 == 0 && row_pitch(b) < (int64_t(1) << 40) &&
           (b.count == 1 || (b.matrix_stride % 16 == 0 && b.matrix_stride < (int64_t(1) << 40)));
}

template <class S, class T>
struct Kernel {
    static constexpr int kDevices = 64;
    static cudaLaunchConfig_t config(cudaLaunchAttribute (&attr)[2], int64_t ctas, int ranks, cudaStream_t st) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(unsigned(ctas));
        cfg.blockDim = dim3(S::kThreads);
        cfg.dynamicSmemBytes = S::kSmem;
        cfg.stream = st;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = unsigned(ranks);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // (see chain_enter)
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        return cfg;
    }
    static void prepare(vf_ctx* ctx) {  // what a device has to be told once
        static std::atomic<bool> ready[kDevices];
        if (ctx->device < kDevices && ready[ctx->device].load(std::memory_order_acquire)) return;
        auto kernel = k_matmul_blocks<S, T>;
        VF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        if (S::kTrades) {  // warps that take registers wait until they are there: what is taken has to have been given
            cudaFuncAttributes fa;
            VF_CUDA(cudaFuncGetAttributes(&fa, kernel));
            if (fa.numRegs * S::kThreads < 128 * kGiven + 128 * S::GROUPS * kTaken) raise(VF_ERR_CUDA, "the kernel was built with too few registers");
        }
        if (ctx->device < kDevices) ready[ctx->device].store(true, std::memory_order_release);
    }
};

template <class S, class T>
void launch_tensor(vf_ctx* ctx, const BlockProduct& p, int ranks = 1) {
    Kernel<S, T>::prepare(ctx);
    const int64_t n_tiles = (p.w.rows + S::kOutputs - 1) / S::kOutputs;
    const int64_t tiles = most_tiles(p, S::kTokens, S::kOutputs);
    const int64_t clusters = S::SWAP && ranks > 1 ? tiles : std::min<int64_t>(tiles, ctx->sm_count * S::PER_SM);
    cudaLaunchAttribute attr[2] = {};
    const cudaLaunchConfig_t cfg = Kernel<S, T>::config(attr, clusters * ranks, ranks, ctx->stream);
    const uint32_t idesc = tc_f8_shape((S::SWAP ? p.w : p.x).dtype == VF_DT_F8E5M2, (S::SWAP ? p.x : p.w).dtype == VF_DT_F8E5M2, S::BN);
    VF_CUDA(cudaLaunchKernelEx(&cfg, k_matmul_blocks<S, T>, map_codes(p.x, 2, S::kTokens), map_codes(p.w, 3, S::kOutputs), p, int(n_tiles), idesc, ctx->d_flags));
}

// Forms of block_plan.h: BN, stages, accumulators, epilogue groups of four warps, CTAs per SM, columns per load
using Swap16 = Shape<true, 16, 5, 4, 1, 2, 16>;
using Swap32 = Shape<true, 32, 4, 4, 1, 2, 16>;
using Swap128 = Shape<true, 128, 4, 2, 2, 1, 16>;
using Wide128 = Shape<false, 128, 5, 2, 2, 1, 32>;
using Wide256 = Shape<false, 256, 3, 2, 2, 1, 16>;

template <class S, class T>
void launch_swapped(vf_ctx* ctx, const BlockProduct& p) {
    launch_tensor<S, T>(ctx, p, ranks_of(most_tiles(p, S::BN, 128), p.x.col_blocks, S::PER_SM, ctx->sm_count, S::kFours, S::kParts));
}

template <class T>
void launch_for(vf_ctx* ctx, const BlockProduct& p) {
    if (!fits_bulk_copies(p.x) || !fits_bulk_copies(p.w)) return launch_plain<T>(ctx, p);
    switch (form_of(p.x.rows, p.offsets ? p.w.count : 0, p.w.rows, ctx->sm_count)) {
    case Form::Swap16: return launch_swapped<Swap16, T>(ctx, p);
    case Form::Swap32: return launch_swapped<Swap32, T>(ctx, p);
    case Form::Swap128: return launch_swapped<Swap128, T>(ctx, p);
    case Form::Wide128: return launch_tensor<Wide128, T>(ctx, p);
    case Form::Wide256: return launch_tensor<Wide256, T>(ctx, p);
    }
}

}  // namespace

void launch_matmul_blocks(vf_ctx* ctx, const BlockProduct& p) {
    if (p.out_dt == VF_DT_F32) launch_for<float>(ctx, p);
    else if (p.out_dt == VF_DT_F16) launch_for<__half>(ctx, p);
    else launch_for<__nv_bfloat16>(ctx, p);
    VF_CUDA(cudaGetLastError());
    ctx->launches += 1;
}

}  // namespace vf
