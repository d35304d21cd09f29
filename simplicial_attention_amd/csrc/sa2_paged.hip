// C entry points of the attention over paged caches (kernels: sa2_paged.hpp).
#include "sa2_paged.hpp"

#include <cmath>
#include <cstdlib>

#include "sa2.h"
#include "sa2_status.hpp"

namespace {

using namespace sa2;

#define SA2_TRY(expr)                  \
    do {                               \
        int rc_ = (expr);              \
        if (rc_ != SA2_OK) return rc_; \
    } while (0)

int kernel_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }

Divisor divisor(int by) {
    // floor(x / by) = (x * mul) >> (31 + s) with mul = floor(2^(31 + s) / by) + 1, s = ceil(log2 by): exact for x < 2^31
    uint32_t s = 0;
    while ((1ll << s) < by) ++s;
    return {(uint32_t)by, (uint32_t)((1ull << (31 + s)) / by + 1), 31 + s};
}

int check_problem(const sa2_paged_problem *p, bool simplicial) {
    if (!p) return fail_with(SA2_ERR_NULL_POINTER, "problem is NULL");
    if (p->batch < 1 || p->rows < 1 || p->heads < 1 || p->kv_heads < 1 || p->page_size < 1 || p->pages < 1 || p->table_width < 1)
        return fail_with(SA2_ERR_BAD_SHAPE, "batch=%d rows=%d heads=%d kv_heads=%d page_size=%d pages=%d table_width=%d must all be >= 1", p->batch, p->rows,
                         p->heads, p->kv_heads, p->page_size, p->pages, p->table_width);
    if (p->heads % p->kv_heads != 0) return fail_with(SA2_ERR_BAD_SHAPE, "heads=%d is not a multiple of kv_heads=%d", p->heads, p->kv_heads);
    if (p->dim_head < 8 || p->dim_head % 8 != 0 || p->pool_dim < p->dim_head || p->pool_dim > 256 || p->pool_dim % 8 != 0)
        return fail_with(SA2_ERR_UNSUPPORTED, "dim_head=%d in pools of %d channels: multiples of 8 up to 256, pools at least as wide as the head, are supported",
                         p->dim_head, p->pool_dim);
    if (p->dtype != SA2_ELEMENT_BF16 && p->dtype != SA2_ELEMENT_F16) return fail_with(SA2_ERR_UNSUPPORTED, "dtype %d is not supported (bf16 or fp16)", p->dtype);
    if (simplicial && (p->w1 < 1 || p->w2 < 1)) return fail_with(SA2_ERR_BAD_SHAPE, "windows w1=%d w2=%d must be >= 1", p->w1, p->w2);
    if (!(p->scale > 0.f) || !std::isfinite(p->scale)) return fail_with(SA2_ERR_BAD_SHAPE, "scale must be positive and finite");
    if (p->max_length < 0) return fail_with(SA2_ERR_BAD_SHAPE, "max_length=%d must be >= 0 (0: what the tables can name)", p->max_length);
    if (!product_within(p->batch, p->rows, p->heads, 0x3ffffff)) return fail_with(SA2_ERR_BAD_SHAPE, "problem too large for a 1-D grid");
    return SA2_OK;
}

// How the work is laid out: a function of the problem alone.
struct Plan {
    bool many, packed, even;
    int64_t batch;
    int unit_columns;
    int dim, row_tiles, splits, dblocks;
    int64_t grid, rows;      // workgroups (of the launch's first dimension); output rows
    int64_t bytes() const { return splits * dblocks > 1 ? splits * dblocks * rows * (dim * 4 + 8) + (even ? 0 : 8 * batch) : 0; }
};

Plan plan_of(const sa2_paged_problem *p, bool simplicial) {
    Plan x{};
    x.dim = kernel_dim(p->pool_dim);
    x.rows = (int64_t)p->batch * p->rows * p->heads;
    const int G = p->heads / p->kv_heads;
    const int64_t per = (int64_t)p->rows * G, seqs = (int64_t)p->batch * p->kv_heads;
    const int64_t reach = (int64_t)p->table_width * p->page_size;
    const int64_t most = p->max_length > 0 && p->max_length < reach ? p->max_length : reach;
    const int64_t keys = simplicial && p->w1 < most ? p->w1 : most;
    const int64_t tiles = (keys + 31) / 32;
    x.dblocks = simplicial ? (int)(((p->w2 < reach ? p->w2 : reach) + 31) / 32) : 1;
    const int waves = x.dim == 256 || simplicial ? 4 : 8;
    // 2-simplicial: a workgroup per (token, head) while all of them run at once, else units that share their keys (one sequence, 8 heads of 64 channels, w1 512,
    // w2 32: 64 tokens 14.5 and 16.6 us, 128 tokens 26.3 and 16.7; four sequences of 128 channels: 16 tokens 20.3 and 22.7, 64 tokens 75 and 30).  One token of many sequences follows the
    // same rule, though its workgroups have waves without a unit where a group has fewer heads than they have waves (64 sequences, w1 512, w2 32: 16 heads on 8, 64 channels 35.3
    // and 18.4, 128 channels 51.4 and 31.4; 16 heads on 16, 64 channels 38.7 and 35.1, 128 channels 59.9 and 61.6; 16 on 4, 128 channels 43.3 and 27.7)
    // Second windows up to 16 leave columns of a wave to other units: taken where there are more units than 256 workgroups of a unit per wave hold (8 heads, w1 512,
    // unit per wave and packed: four sequences of 1024 tokens, 128 channels, w2 16, 8 and 4: 433, 393, 387 and 244, 130, 72 us; one of 128 tokens, 64 channels,
    // w2 8: 15.7 and 16.5)
    x.many = simplicial ? seqs * per * x.dblocks > 512 : per > 32;
    x.packed = simplicial && seqs * per > 1024 && p->w2 <= 16;
    x.unit_columns = 32;
    while (x.packed && x.unit_columns > 1 && x.unit_columns / 2 >= p->w2) x.unit_columns /= 2;
    const int64_t per_wg = x.many ? (simplicial ? waves * (32 / x.unit_columns) : waves * 32) : (simplicial ? 1 : 32);
    x.row_tiles = (int)((per + per_wg - 1) / per_wg);
    const int64_t items = seqs * x.row_tiles * x.dblocks;
    int64_t splits = 1;
    if (x.many) {
        // The shares k of an item run on 256 CUs, one workgroup each (the 2-simplicial form two), in whole rounds; starting and ending a workgroup costs
        // about six tiles (sixteen), the merge six.  Measured and estimated agree in order: 128 items of 1008 tiles in 1, 2, 3, 4, 8 shares 797, 503, 600, 519, 573 us;
        // 2-simplicial, 256 items of 16 tiles in 1, 2, 4 shares 16.7, 18.4, 25.4
        const int64_t slots = simplicial && x.dim < 256 ? 512 : 256, around = simplicial ? 16 : 6;
        int64_t least = 0;
        for (int64_t k = 1; k <= 64 && (k == 1 || k * 8 <= tiles); ++k) {
            const int64_t cost = (items * k + slots - 1) / slots * (tiles / k + around) + (k > 1 ? 6 : 0);
            if (k == 1 || cost < least) {
                least = cost;
                splits = k;
            }
        }
    } else {
        // 2048 waves fill the chip, and twice as many balance sequences of different lengths where a wave keeps eight tiles (one token of 16
        // sequences of up to 32768 in 8, 16, 32 shares: 139, 131, 137 us; of 8 up to 8192: 17.6, 18.5, 23.3).  A wave has a tile at least, and short walks are not worth a
        // merge (one sequence of 1024 in 1, 4 shares: 11.0, 10.6; of 2048 in 1, 8: 17.1, 11.2)
        const int64_t waves = x.dim == 256 ? 2 : x.dim == 128 ? 4 : 8;
        if (tiles >= 4 * waves) {
            splits = (2048 + items * waves - 1) / (items * waves);
            if (2 * splits * waves * 8 <= tiles) splits *= 2;
            if (splits > tiles / waves) splits = tiles / waves;
            // ... and beyond 128 parts a wave's walk has to outweigh the longer merge (one token of 8 heads on one, 128 channels: 32768 rows in 128, 256 parts 15.0
            // and 16.7 us, 131072 rows 28.3 and 24.6; 256 channels, 32768 rows 26.9 and 22.2)
            const int64_t pays = tiles * x.dim / (512 * waves);
            if (splits > 128) splits = pays > 128 ? (splits < pays ? splits : pays) : 128;
        }
    }
    // (a dimension of the grid)
    const int64_t most_splits = x.dblocks < 255 ? 256 : x.dblocks < 65536 ? 65535 / x.dblocks : 1;
    x.splits = (int)(splits > most_splits ? most_splits : splits);
    // (a lane for each sequence, and lengths whose quotients are exact)
    x.even = simplicial || !x.many || x.splits == 1 || p->batch == 1 || p->batch > 64 || reach >= 1ll << 25;
    x.batch = p->batch;
    x.grid = x.many ? seqs * x.row_tiles : simplicial ? seqs : seqs * x.splits;
    return x;
}

int check_rows(const sa2_tensor *t, const char *name) {
    if (!t || !t->ptr) return fail_with(SA2_ERR_NULL_POINTER, "tensor %s is NULL", name);
    if ((reinterpret_cast<uintptr_t>(t->ptr) & 15) != 0 || (t->stride_b & 7) != 0 || (t->stride_n & 7) != 0 || (t->stride_h & 7) != 0)
        return fail_with(SA2_ERR_ALIGNMENT, "tensor %s: base pointer must be 16-byte aligned and strides multiples of 8 elements", name);
    return SA2_OK;
}

int check_pool(const sa2_pool *t, const char *name) {
    if (!t || !t->ptr) return fail_with(SA2_ERR_NULL_POINTER, "pool %s is NULL", name);
    if ((reinterpret_cast<uintptr_t>(t->ptr) & 15) != 0 || (t->stride_page & 7) != 0 || (t->stride_row & 7) != 0 || (t->stride_head & 7) != 0)
        return fail_with(SA2_ERR_ALIGNMENT, "pool %s: base pointer must be 16-byte aligned and strides multiples of 8 elements", name);
    return SA2_OK;
}

PagedPool pool_of(const sa2_pool *t) {
    PagedPool x{};
    if (t) x = {static_cast<const char *>(t->ptr), t->stride_page * 2, t->stride_row * 2, t->stride_head * 2};
    return x;
}

template <class E, int D, bool SIMP>
void launch(const Plan &x, const PagedParams &k, hipStream_t stream) {
    if (x.many) {
        const dim3 grid((unsigned)((int64_t)k.B * k.HK * x.row_tiles), (unsigned)(x.splits * x.dblocks)), block(ManyCfg<D, SIMP>::NW * 64);
        if (SIMP && x.packed) hipLaunchKernelGGL((paged_many_kernel<E, D, SIMP, SIMP>), grid, block, 0, stream, k);
        else hipLaunchKernelGGL((paged_many_kernel<E, D, SIMP, false>), grid, block, 0, stream, k);
    } else {
        const unsigned seqs = k.B * k.HK, parts = x.splits * x.dblocks;
        const dim3 grid(SIMP ? seqs : seqs * parts, (unsigned)x.row_tiles, SIMP ? parts : 1);
        if (!SIMP && k.n > 1) hipLaunchKernelGGL((paged_few_kernel<E, D, SIMP, !SIMP>), grid, dim3(FewCfg<D>::NW * 64), 0, stream, k);
        else hipLaunchKernelGGL((paged_few_kernel<E, D, SIMP, false>), grid, dim3(FewCfg<D>::NW * 64), 0, stream, k);
    }
    if (x.splits * x.dblocks > 1) {
        const int pg = x.splits * x.dblocks >= 8 && x.rows <= 1 << 20 ? 8 : 1, per = 256 / (D / 8) / pg;
        const dim3 grid((unsigned)((x.rows + per - 1) / per));
        if (pg > 1) hipLaunchKernelGGL((paged_merge_kernel<E, D, 8>), grid, dim3(256), 0, stream, k);
        else hipLaunchKernelGGL((paged_merge_kernel<E, D, 1>), grid, dim3(256), 0, stream, k);
    }
}

template <class E, bool SIMP>
void launch_dim(const Plan &x, const PagedParams &k, hipStream_t stream) {
    switch (x.dim) {
        case 32: launch<E, 32, SIMP>(x, k, stream); break;
        case 64: launch<E, 64, SIMP>(x, k, stream); break;
        case 128: launch<E, 128, SIMP>(x, k, stream); break;
        default: launch<E, 256, SIMP>(x, k, stream); break;
    }
}

int attend(bool simplicial, const sa2_paged_problem *p, const sa2_tensor *q, const sa2_pool *k1, const sa2_pool *k2, const sa2_pool *v1, const sa2_pool *v2,
           const sa2_paged_index *at, const sa2_tensor *out, void *workspace, int64_t workspace_bytes, void *stream) {
    SA2_TRY(check_problem(p, simplicial));
    SA2_TRY(check_pool(k1, simplicial ? "k1" : "k"));
    SA2_TRY(check_pool(v1, simplicial ? "v1" : "v"));
    if (simplicial) {
        SA2_TRY(check_pool(k2, "k2"));
        SA2_TRY(check_pool(v2, "v2"));
    }
    SA2_TRY(check_rows(q, "q"));
    SA2_TRY(check_rows(out, "out"));
    if (!at || !at->tables || !at->lengths) return fail_with(SA2_ERR_NULL_POINTER, "tables and lengths are required");
    const Plan x = plan_of(p, simplicial);
    if (x.dblocks > 65535) return fail_with(SA2_ERR_BAD_SHAPE, "w2=%d: at most %d offsets are supported", p->w2, 65535 * 32);
    // (a launch has fewer than 2^32 threads, 512 in a workgroup)
    if (x.grid > 0x7fffffll) return fail_with(SA2_ERR_BAD_SHAPE, "problem too large for a 1-D grid");
    if (x.bytes() > 0 && (!workspace || workspace_bytes < x.bytes()))
        return fail_with(SA2_ERR_BAD_SHAPE, "workspace of %lld bytes, %lld are needed", (long long)(workspace ? workspace_bytes : 0), (long long)x.bytes());
    if (x.bytes() > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return fail_with(SA2_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    PagedParams k{};
    k.q = static_cast<const char *>(q->ptr);
    k.q_sb = q->stride_b * 2;
    k.q_sn = q->stride_n * 2;
    k.q_sh = q->stride_h * 2;
    k.o = static_cast<char *>(out->ptr);
    k.o_sb = out->stride_b * 2;
    k.o_sn = out->stride_n * 2;
    k.o_sh = out->stride_h * 2;
    k.k1 = pool_of(k1);
    k.v1 = pool_of(v1);
    k.k2 = pool_of(k2);
    k.v2 = pool_of(v2);
    k.tables = at->tables;
    k.lengths = at->lengths;
    k.counts = at->counts;
    k.t_sb = at->table_stride;
    k.div = divisor(p->page_size);
    k.group = divisor(p->heads / p->kv_heads);
    k.heads = divisor(p->kv_heads);
    k.seqs = divisor(p->batch * p->kv_heads);
    k.parts = divisor(x.splits * x.dblocks);
    k.pages = p->pages;
    k.width = p->table_width;
    k.B = p->batch;
    k.n = p->rows;
    k.H = p->heads;
    k.HK = p->kv_heads;
    k.G = p->heads / p->kv_heads;
    k.dq = p->dim_head;
    k.dp = p->pool_dim;
    k.w1 = p->w1;
    k.w2 = p->w2;
    k.scale_log2e = p->scale * kLog2e;
    k.unit_columns = x.unit_columns;
    k.row_tiles = x.row_tiles;
    k.splits = x.splits;
    k.dblocks = x.dblocks;
    k.even = x.even;
    if (x.bytes() > 0) {
        k.part_o = static_cast<float *>(workspace);
        k.part_ml = reinterpret_cast<float2 *>(k.part_o + (int64_t)x.splits * x.dblocks * x.rows * x.dim);
        k.shares = reinterpret_cast<int2 *>(k.part_ml + (int64_t)x.splits * x.dblocks * x.rows);
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->dtype == SA2_ELEMENT_F16) {
        if (simplicial) launch_dim<ElemF16, true>(x, k, s);
        else launch_dim<ElemF16, false>(x, k, s);
    } else {
        if (simplicial) launch_dim<ElemBf16, true>(x, k, s);
        else launch_dim<ElemBf16, false>(x, k, s);
    }
    return launched(simplicial ? "paged 2-simplicial attention" : "paged attention");
}

}  // namespace

extern "C" {

int64_t sa2_paged_attn_workspace_bytes(const sa2_paged_problem *prob) { return check_problem(prob, false) == SA2_OK ? plan_of(prob, false).bytes() : -1; }

int sa2_paged_attn(const sa2_paged_problem *prob, const sa2_tensor *q, const sa2_pool *k, const sa2_pool *v, const sa2_paged_index *at, const sa2_tensor *out,
                   void *workspace, int64_t workspace_bytes, void *hip_stream) {
    return attend(false, prob, q, k, nullptr, v, nullptr, at, out, workspace, workspace_bytes, hip_stream);
}

int64_t sa2_paged_simplicial_attn_workspace_bytes(const sa2_paged_problem *prob) {
    return check_problem(prob, true) == SA2_OK ? plan_of(prob, true).bytes() : -1;
}

int sa2_paged_simplicial_attn(const sa2_paged_problem *prob, const sa2_tensor *q, const sa2_pool *k1, const sa2_pool *k2, const sa2_pool *v1, const sa2_pool *v2,
                              const sa2_paged_index *at, const sa2_tensor *out, void *workspace, int64_t workspace_bytes, void *hip_stream) {
    return attend(true, prob, q, k1, k2, v1, v2, at, out, workspace, workspace_bytes, hip_stream);
}

}  // extern "C"
