// Entry points on 8-bit floating-point blocks. All checks of arguments come before the context is looked at, so they
// hold (and are tested) without a device.
#include <algorithm>

#include "block_plan.h"
#include "blocks.h"
#include "call_scope.h"

namespace vf {

namespace {

// a + b * c without overflow; everything here is non-negative
int64_t mul_add(int64_t a, int64_t b, int64_t c, const char* what) {
    int64_t p, r;
    if (__builtin_mul_overflow(b, c, &p) || __builtin_add_overflow(a, p, &r)) raise(VF_ERR_SHAPE, "%s is too large", what);
    return r;
}

// Bytes that `extent[i]` steps of `stride[i]` elements span; refuses strides with which two elements meet.
uint64_t span_of(const int64_t* extent, const int64_t* stride, int n, int elem_bytes, const char* what) {
    int order[3], m = 0;
    for (int i = 0; i < n; ++i) {
        if (extent[i] == 0) return 0;
        if (stride[i] < 0) raise(VF_ERR_INVALID_ARG, "%s: negative stride", what);
        if (extent[i] > 1) order[m++] = i;
    }
    std::sort(order, order + m, [&](int a, int b) { return stride[a] < stride[b]; });
    int64_t reach = 1;  // elements from the first to behind the last one of the dims taken so far
    for (int i = 0; i < m; ++i) {
        if (stride[order[i]] < reach) raise(VF_ERR_SHAPE, "%s: a stride of %lld makes elements meet", what, (long long)stride[order[i]]);
        reach = mul_add(reach, extent[order[i]] - 1, stride[order[i]], what);
    }
    return uint64_t(mul_add(0, reach, elem_bytes, what));
}

void check_mem_kind(int k) {
    if (k != VF_MEM_HOST && k != VF_MEM_HOST_PINNED && k != VF_MEM_DEVICE) raise(VF_ERR_INVALID_ARG, "unknown memory kind %d", k);
}

Blocks checked(const vf_block_matrix* m, const char* name) {
    if (!m) raise(VF_ERR_INVALID_ARG, "%s is NULL", name);
    Blocks b;
    if (m->dtype != VF_DT_F8E4M3FN && m->dtype != VF_DT_F8E5M2) raise(VF_ERR_UNSUPPORTED, "%s: block codes are e4m3 or e5m2, not type %d", name, m->dtype);
    if (m->block_rows != 1 && m->block_rows != kBlock) raise(VF_ERR_UNSUPPORTED, "%s: blocks of %d rows (1 or %d are supported)", name, m->block_rows, kBlock);
    check_mem_kind(m->mem_kind);
    constexpr int64_t kMost = INT32_MAX - 2 * kBlock;  // coordinates of tiles stay 32-bit
    if (m->count < 1 || m->rows < 0 || m->cols < 1 || m->count > kMost || m->rows > kMost || m->cols > kMost)
        raise(VF_ERR_SHAPE, "%s: shape [%lld, %lld, %lld]", name, (long long)m->count, (long long)m->rows, (long long)m->cols);
    b.dtype = m->dtype;
    b.block_rows = m->block_rows;
    b.count = m->count;
    b.rows = m->rows;
    b.cols = m->cols;
    b.row_blocks = (m->rows + m->block_rows - 1) / m->block_rows;
    b.col_blocks = (m->cols + kBlock - 1) / kBlock;
    b.ld = m->ld ? m->ld : m->cols;
    if (b.ld < b.cols) raise(VF_ERR_SHAPE, "%s: rows %lld apart hold no %lld columns", name, (long long)b.ld, (long long)b.cols);
    b.matrix_stride = m->matrix_stride ? m->matrix_stride : mul_add(0, b.rows, b.ld, name);
    const int64_t ext[3] = {b.count, b.rows, b.cols}, st[3] = {b.matrix_stride, b.ld, 1};
    b.codes_span = span_of(ext, st, 3, 1, name);
    if (!m->scale_row_stride && !m->scale_col_stride && !m->scale_matrix_stride) {
        b.scs = 1;
        b.srs = b.col_blocks;
        b.sms = mul_add(0, b.row_blocks, b.col_blocks, name);
    } else {
        b.srs = m->scale_row_stride;
        b.scs = m->scale_col_stride;
        b.sms = m->scale_matrix_stride;
    }
    const int64_t sext[3] = {b.count, b.row_blocks, b.col_blocks}, sst[3] = {b.sms, b.srs, b.scs};
    b.scales_span = span_of(sext, sst, 3, 4, "scales");
    b.codes = static_cast<uint8_t*>(m->codes);
    b.scales = m->scales;
    if (m->mem_kind != VF_MEM_DEVICE && (b.codes_span != uint64_t(b.count * b.rows * b.cols) || b.scales_span != uint64_t(b.count * b.row_blocks * b.col_blocks) * 4))
        raise(VF_ERR_UNSUPPORTED, "%s: a matrix in host memory has no gaps between its elements", name);
    if (b.codes_span && (!m->codes || m->codes_bytes < b.codes_span))
        raise(VF_ERR_BUFFER_TOO_SMALL, "%s: codes need %llu bytes, buffer holds %llu", name, (unsigned long long)b.codes_span, (unsigned long long)(m->codes ? m->codes_bytes : 0));
    if (b.scales_span && (!m->scales || m->scales_bytes < b.scales_span))
        raise(VF_ERR_BUFFER_TOO_SMALL, "%s: scales need %llu bytes, buffer holds %llu", name, (unsigned long long)b.scales_span, (unsigned long long)(m->scales ? m->scales_bytes : 0));
    if (reinterpret_cast<uintptr_t>(m->scales) & 3u) raise(VF_ERR_ALIGNMENT, "%s: scales are not 4-byte aligned", name);
    return b;
}

bool is_wide(int dt) {
    return dt == VF_DT_F32 || dt == VF_DT_F16 || dt == VF_DT_BF16;
}

// [count * rows] rows of `cols` wide elements, `ld` apart: checked, and the bytes that they span
uint64_t wide_span(const void* p, int dt, int64_t n_rows, int64_t cols, int64_t& ld, uint64_t bytes, int mem_kind, const char* name) {
    if (!is_wide(dt)) raise(VF_ERR_UNSUPPORTED, "%s: f32, f16 or bf16 elements, not type %d", name, dt);
    check_mem_kind(mem_kind);
    if (ld < 0) raise(VF_ERR_INVALID_ARG, "%s: negative stride", name);
    if (!ld) ld = cols;
    if (ld < cols) raise(VF_ERR_SHAPE, "%s: rows %lld apart hold no %lld columns", name, (long long)ld, (long long)cols);
    const int es = dtype_bits(dt) / 8;
    const int64_t ext[2] = {n_rows, cols}, st[2] = {ld, 1};
    const uint64_t span = span_of(ext, st, 2, es, name);
    if (span && (!p || bytes < span)) raise(VF_ERR_BUFFER_TOO_SMALL, "%s needs %llu bytes, buffer holds %llu", name, (unsigned long long)span, (unsigned long long)(p ? bytes : 0));
    if (reinterpret_cast<uintptr_t>(p) & uintptr_t(es - 1)) raise(VF_ERR_ALIGNMENT, "%s is not aligned to its elements", name);
    if (mem_kind != VF_MEM_DEVICE && ld != cols) raise(VF_ERR_UNSUPPORTED, "%s: rows in host memory have no gaps between them", name);
    return span;
}

void check_apart(const void* a, uint64_t na, const void* b, uint64_t nb, const char* what) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (na && nb && x < y + nb && y < x + na) raise(VF_ERR_INVALID_ARG, "%s overlap", what);
}

// A matrix in host memory gets device buffers for the call.
struct Staged {
    DBuf codes, scales;
    Blocks on_device(vf_ctx* ctx, Blocks b, int mem_kind) {
        if (mem_kind == VF_MEM_DEVICE) return b;
        codes = DBuf(ctx, b.codes_span);
        scales = DBuf(ctx, b.scales_span);
        b.codes = codes.as<uint8_t>();
        b.scales = scales.as<float>();
        return b;
    }
};

BlockProduct checked_product(const vf_block_matrix* x, const vf_block_matrix* w, bool grouped, void* out, int32_t out_dtype, int64_t out_ld, uint64_t out_bytes) {
    BlockProduct p;
    p.x = checked(x, "x");
    p.w = checked(w, "w");
    if (x->mem_kind != VF_MEM_DEVICE || w->mem_kind != VF_MEM_DEVICE) raise(VF_ERR_UNSUPPORTED, "the operands of a product live in device memory");
    if (p.x.block_rows != 1 || p.w.block_rows != kBlock) raise(VF_ERR_UNSUPPORTED, "a product multiplies activations (block_rows 1) by weights (block_rows %d)", kBlock);
    if (p.x.count != 1) raise(VF_ERR_SHAPE, "x is one matrix, not %lld", (long long)p.x.count);
    if (p.x.cols != p.w.cols) raise(VF_ERR_SHAPE, "x has %lld columns, w %lld", (long long)p.x.cols, (long long)p.w.cols);
    const int64_t experts = grouped ? p.w.count : 0;
    if (too_many_tiles(p.x.rows, experts, p.w.rows))
        raise(VF_ERR_CAPACITY, "a product of %lld rows, %lld experts and %lld columns has too many tiles", (long long)p.x.rows, (long long)experts, (long long)p.w.rows);
    p.out = out;
    p.out_dt = out_dtype;
    p.out_ld = out_ld;
    p.out_span = p.w.rows ? wide_span(out, out_dtype, p.x.rows, p.w.rows, p.out_ld, out_bytes, VF_MEM_DEVICE, "out") : 0;
    if (!p.w.rows && !is_wide(out_dtype)) raise(VF_ERR_UNSUPPORTED, "out: f32, f16 or bf16 elements, not type %d", out_dtype);
    const char* what = "the result and an operand";
    check_apart(out, p.out_span, p.x.codes, p.x.codes_span, what);
    check_apart(out, p.out_span, p.x.scales, p.x.scales_span, what);
    check_apart(out, p.out_span, p.w.codes, p.w.codes_span, what);
    check_apart(out, p.out_span, p.w.scales, p.w.scales_span, what);
    return p;
}

void run_product(vf_ctx* ctx, const BlockProduct& p, vf_stats* stats) {
    CallScope scope(ctx, stats);
    if (p.x.rows && p.w.rows) launch_matmul_blocks(ctx, p);
    if (stats) {
        stats->bytes_in = p.x.codes_span + p.x.scales_span + p.w.codes_span + p.w.scales_span;
        stats->bytes_out = uint64_t(p.x.rows) * uint64_t(p.w.rows) * uint64_t(dtype_bits(p.out_dt) / 8);
    }
    scope.may_defer = true;
    scope.finish();
}

}  // namespace

}  // namespace vf

using namespace vf;

extern "C" {

int vf_quantize_blocks(vf_ctx* ctx, const vf_content* base, int64_t base_ld, const vf_block_matrix* out, vf_stats* stats,
                       char* err, size_t errlen) {
    return guard(err, errlen, [&] {
        if (!base) raise(VF_ERR_INVALID_ARG, "base is NULL");
        const Blocks b = checked(out, "out");
        const Type ty = Type::from(base->type);
        if (base->is_splat) raise(VF_ERR_SPLAT, "a splat has no blocks to quantise");
        if (ty.elem.quantized() || base->storage_dtype != ty.elem.dtype) raise(VF_ERR_UNSUPPORTED, "base: plain f32, f16 or bf16 elements");
        if (ty.order != identity_order(ty.rank)) raise(VF_ERR_UNSUPPORTED, "block quantization needs row-major input");
        const int64_t count = ty.rank == 3 ? ty.shape[0] : 1;
        if ((ty.rank != 2 && ty.rank != 3) || count != b.count || ty.shape[ty.rank - 2] != b.rows || ty.shape[ty.rank - 1] != b.cols)
            raise(VF_ERR_SHAPE, "base and out have different shapes");
        int64_t ld = base_ld;
        const uint64_t span = wide_span(base->data, ty.elem.dtype, mul_add(0, b.count, b.rows, "base"), b.cols, ld, base->nbytes, base->mem_kind, "base");
        if ((base->mem_kind == VF_MEM_DEVICE) == (out->mem_kind == VF_MEM_DEVICE)) {
            check_apart(base->data, span, b.codes, b.codes_span, "base and codes");
            check_apart(base->data, span, b.scales, b.scales_span, "base and scales");
        }
        check_apart(b.codes, b.codes_span, b.scales, b.scales_span, "codes and scales");

        CallScope scope(ctx, stats);
        if (b.rows) {
            DBuf up;
            const void* src = base->data;
            if (base->mem_kind != VF_MEM_DEVICE) {
                up = DBuf(ctx, span);
                copy_in(ctx, up.p, base->data, span, base->mem_kind);
                src = up.p;
            }
            Staged st;
            const Blocks d = st.on_device(ctx, b, out->mem_kind);
            launch_quantize_blocks(ctx, src, ty.elem.dtype, ld, d);
            if (out->mem_kind != VF_MEM_DEVICE) {
                copy_out(ctx, b.codes, out->mem_kind, d.codes, b.codes_span);
                copy_out(ctx, b.scales, out->mem_kind, d.scales, b.scales_span);
            }
        }
        if (stats) {
            stats->bytes_in = span;
            stats->bytes_out = uint64_t(b.count * b.rows * b.cols) + uint64_t(b.count * b.row_blocks * b.col_blocks) * 4;
            stats->h2d_bytes = base->mem_kind == VF_MEM_DEVICE ? 0 : span;
            stats->d2h_bytes = out->mem_kind == VF_MEM_DEVICE ? 0 : stats->bytes_out;
        }
        scope.may_defer = base->mem_kind == VF_MEM_DEVICE && out->mem_kind == VF_MEM_DEVICE;
        scope.finish();
    });
}

int vf_dequantize_blocks(vf_ctx* ctx, const vf_block_matrix* in, void* dst, int32_t dst_dtype, int64_t dst_ld,
                         uint64_t dst_bytes, int dst_mem_kind, vf_stats* stats, char* err, size_t errlen) {
    return guard(err, errlen, [&] {
        const Blocks b = checked(in, "in");
        int64_t ld = dst_ld;
        const uint64_t span = wide_span(dst, dst_dtype, mul_add(0, b.count, b.rows, "dst"), b.cols, ld, dst_bytes, dst_mem_kind, "dst");
        if ((in->mem_kind == VF_MEM_DEVICE) == (dst_mem_kind == VF_MEM_DEVICE)) {
            check_apart(dst, span, b.codes, b.codes_span, "dst and codes");
            check_apart(dst, span, b.scales, b.scales_span, "dst and scales");
        }

        CallScope scope(ctx, stats);
        if (b.rows) {
            Staged st;
            const Blocks d = st.on_device(ctx, b, in->mem_kind);
            if (in->mem_kind != VF_MEM_DEVICE) {
                copy_in(ctx, d.codes, b.codes, b.codes_span, in->mem_kind);
                copy_in(ctx, d.scales, b.scales, b.scales_span, in->mem_kind);
            }
            DBuf down;
            void* to = dst;
            if (dst_mem_kind != VF_MEM_DEVICE) {
                down = DBuf(ctx, span);
                to = down.p;
            }
            launch_dequantize_blocks(ctx, d, to, dst_dtype, ld);
            if (dst_mem_kind != VF_MEM_DEVICE) copy_out(ctx, dst, dst_mem_kind, to, span);
        }
        if (stats) {
            stats->bytes_in = uint64_t(b.count * b.rows * b.cols) + uint64_t(b.count * b.row_blocks * b.col_blocks) * 4;
            stats->bytes_out = uint64_t(b.count * b.rows * b.cols) * uint64_t(dtype_bits(dst_dtype) / 8);
            stats->h2d_bytes = in->mem_kind == VF_MEM_DEVICE ? 0 : stats->bytes_in;
            stats->d2h_bytes = dst_mem_kind == VF_MEM_DEVICE ? 0 : stats->bytes_out;
        }
        scope.may_defer = in->mem_kind == VF_MEM_DEVICE && dst_mem_kind == VF_MEM_DEVICE;
        scope.finish();
    });
}

int vf_matmul_blocks(vf_ctx* ctx, const vf_block_matrix* x, const vf_block_matrix* w, void* out, int32_t out_dtype,
                     int64_t out_ld, uint64_t out_bytes, vf_stats* stats, char* err, size_t errlen) {
    return guard(err, errlen, [&] {
        const BlockProduct p = checked_product(x, w, false, out, out_dtype, out_ld, out_bytes);
        if (p.w.count != 1) raise(VF_ERR_SHAPE, "w is one matrix, not %lld (vf_matmul_blocks_grouped takes a stack)", (long long)p.w.count);
        run_product(ctx, p, stats);
    });
}

int vf_matmul_blocks_grouped(vf_ctx* ctx, const vf_block_matrix* x, const vf_block_matrix* w, const int64_t* offsets, void* out,
                             int32_t out_dtype, int64_t out_ld, uint64_t out_bytes, vf_stats* stats, char* err,
                             size_t errlen) {
    return guard(err, errlen, [&] {
        BlockProduct p = checked_product(x, w, true, out, out_dtype, out_ld, out_bytes);
        if (!offsets) raise(VF_ERR_INVALID_ARG, "offsets is NULL");
        if (reinterpret_cast<uintptr_t>(offsets) & 7u) raise(VF_ERR_ALIGNMENT, "offsets are not 8-byte aligned");
        check_apart(out, p.out_span, offsets, uint64_t(p.w.count + 1) * 8, "the result and the offsets");
        p.offsets = offsets;
        run_product(ctx, p, stats);
    });
}

}  // extern "C"
