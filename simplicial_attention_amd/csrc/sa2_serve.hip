// C entry points of the page moves and of sampling (kernels: sa2_pages.hpp, sa2_sample.hpp).
#include <algorithm>
#include <new>
#include <vector>

#include "sa2.h"
#include "sa2_pages.hpp"
#include "sa2_sample.hpp"
#include "sa2_status.hpp"

namespace {

using namespace sa2;

bool pieces16(const void *ptr, int64_t a, int64_t b, int64_t c) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && a % 16 == 0 && b % 16 == 0 && c % 16 == 0; }

template <int TYPE>
void launch_sample(int64_t rows, const SampleParams &k, hipStream_t s) {
    const dim3 grid((unsigned)(rows * k.chunks));
    constexpr int N = kSampleThreads, E = kSampleEach;
    // one wave up to 1024 tokens (no barriers), a piece per thread where that is enough
    if (k.vocab <= 64 * Logits<TYPE>::PIECE) hipLaunchKernelGGL((sample_chunk_kernel<TYPE, 64, Logits<TYPE>::PIECE, true>), grid, dim3(64), 0, s, k);
    else if (k.vocab <= 64 * E) hipLaunchKernelGGL((sample_chunk_kernel<TYPE, 64, E, true>), grid, dim3(64), 0, s, k);
    else if (k.chunks == 1) hipLaunchKernelGGL((sample_chunk_kernel<TYPE, N, E, true>), grid, dim3(N), 0, s, k);
    else {
        hipLaunchKernelGGL((sample_chunk_kernel<TYPE, N, E, false>), grid, dim3(N), 0, s, k);
        hipLaunchKernelGGL(sample_row_kernel<TYPE>, dim3((unsigned)rows), dim3(kRowThreads), 0, s, k);
    }
}

// workgroups of a launch: fewer than 2^32 threads of 256 a group
constexpr int64_t kMostGroups = 0xffffff;

}  // namespace

extern "C" {

int sa2_paged_append(const sa2_paged_problem *p, const sa2_append_item *items, int32_t count, int32_t src_type, const sa2_paged_index *at, void *hip_stream) {
    if (!p || !items || !at || !at->tables || !at->lengths) return fail_with(SA2_ERR_NULL_POINTER, "problem, items, tables and lengths are required");
    if (count < 1 || count > SA2_APPEND_MOST) return fail_with(SA2_ERR_BAD_SHAPE, "%d pools, 1 to %d are supported", count, SA2_APPEND_MOST);
    if (p->batch < 1 || p->rows < 1 || p->kv_heads < 1 || p->page_size < 1 || p->pages < 1 || p->table_width < 1 || p->dim_head < 1 || p->pool_dim < p->dim_head ||
        p->pool_dim > 256 || p->pool_dim % 8 != 0)
        return fail_with(SA2_ERR_BAD_SHAPE, "batch=%d rows=%d kv_heads=%d page_size=%d pages=%d table_width=%d dim_head=%d pool_dim=%d", p->batch, p->rows,
                         p->kv_heads, p->page_size, p->pages, p->table_width, p->dim_head, p->pool_dim);
    if (src_type < 0 || src_type > 2 || (p->dtype != SA2_ELEMENT_BF16 && p->dtype != SA2_ELEMENT_F16))
        return fail_with(SA2_ERR_UNSUPPORTED, "rows of type %d into pools of type %d", src_type, p->dtype);
    AppendParams k{};
    const int size = src_type == SA2_ELEMENT_F32 ? 4 : 2;
    bool plain = src_type == p->dtype && p->dim_head == p->pool_dim;
    for (int i = 0; i < count; ++i) {
        const sa2_append_item &it = items[i];
        if (!it.pool.ptr || !it.rows.ptr) return fail_with(SA2_ERR_NULL_POINTER, "pool or rows %d is NULL", i);
        if (!pieces16(it.pool.ptr, it.pool.stride_page * 2, it.pool.stride_row * 2, it.pool.stride_head * 2))
            return fail_with(SA2_ERR_ALIGNMENT, "pool %d: base pointer must be 16-byte aligned and strides multiples of 8 elements", i);
        k.item[i] = {static_cast<char *>(it.pool.ptr), it.pool.stride_page * 2, it.pool.stride_row * 2, it.pool.stride_head * 2,
                     static_cast<const char *>(it.rows.ptr), it.rows.stride_b * size, it.rows.stride_n * size, it.rows.stride_h * size};
        plain = plain && pieces16(it.rows.ptr, it.rows.stride_b * size, it.rows.stride_n * size, it.rows.stride_h * size);
    }
    k.tables = at->tables;
    k.lengths = at->lengths;
    k.counts = at->counts;
    k.t_sb = at->table_stride;
    k.ps = p->page_size;
    k.pages = p->pages;
    k.width = p->table_width;
    k.B = p->batch;
    k.n = p->rows;
    k.HK = p->kv_heads;
    k.dim = p->dim_head;
    k.pieces = p->pool_dim / 8;
    k.count = count;
    if (p->kv_heads > (1 << 24) || !product_within(p->batch, p->rows, (int64_t)p->kv_heads * k.pieces, kMostGroups * 256))
        return fail_with(SA2_ERR_BAD_SHAPE, "problem too large for a 1-D grid");
    const int64_t threads = (int64_t)p->batch * p->rows * p->kv_heads * k.pieces;
    const dim3 grid((unsigned)((threads + 255) / 256));
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    if (plain) hipLaunchKernelGGL(paged_append_kernel<true>, grid, dim3(256), 0, s, k, src_type, p->dtype);
    else hipLaunchKernelGGL(paged_append_kernel<false>, grid, dim3(256), 0, s, k, src_type, p->dtype);
    return launched("paged append");
}

int sa2_copy_pages(const sa2_page_pool *pools, int32_t count, const int32_t *pairs, int64_t n_pairs, void *hip_stream) {
    if (!pools || (n_pairs > 0 && !pairs)) return fail_with(SA2_ERR_NULL_POINTER, "pools and pairs are required");
    if (count < 1 || n_pairs < 0) return fail_with(SA2_ERR_BAD_SHAPE, "%d pools, %lld pairs", count, (long long)n_pairs);
    int64_t least = 0x7fffffff, most_bytes = 0;
    bool wide = true;
    for (int i = 0; i < count; ++i) {
        const sa2_page_pool &t = pools[i];
        if (!t.ptr) return fail_with(SA2_ERR_NULL_POINTER, "pool %d is NULL", i);
        if (t.bytes < 2 || t.bytes % 2 != 0 || t.bytes > (1 << 30) || t.stride < t.bytes || t.stride % 2 != 0 || (reinterpret_cast<uintptr_t>(t.ptr) & 1) != 0 || t.pages < 1)
            return fail_with(SA2_ERR_BAD_SHAPE, "pool %d: %lld pages of %lld bytes, %lld apart", i, (long long)t.pages, (long long)t.bytes, (long long)t.stride);
        least = std::min(least, t.pages);
        most_bytes = std::max(most_bytes, t.bytes);
        wide = wide && t.bytes % 16 == 0 && pieces16(t.ptr, t.stride, 0, 0);
    }
    if (n_pairs > least) return fail_with(SA2_ERR_BAD_SHAPE, "%lld pairs of %lld pages: a page is written twice", (long long)n_pairs, (long long)least);
    // what is written may be neither read nor written again: the pairs run in no order
    try {
        std::vector<std::pair<int32_t, bool>> seen;      // (page, written)
        seen.reserve(2 * n_pairs);
        for (int64_t i = 0; i < n_pairs; ++i)
            for (int e = 0; e < 2; ++e) {
                if (pairs[2 * i + e] < 0 || pairs[2 * i + e] >= least)
                    return fail_with(SA2_ERR_BAD_SHAPE, "pair %lld names page %d of %lld", (long long)i, pairs[2 * i + e], (long long)least);
                seen.emplace_back(pairs[2 * i + e], e == 1);
            }
        std::sort(seen.begin(), seen.end());
        for (size_t i = 1; i < seen.size(); ++i)
            if (seen[i].first == seen[i - 1].first && seen[i].second)
                return fail_with(SA2_ERR_BAD_SHAPE, "page %d is written and read, or written twice", seen[i].first);
    } catch (const std::bad_alloc &) {
        return fail_with(SA2_ERR_BAD_SHAPE, "no memory for %lld pairs", (long long)n_pairs);
    }
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    CopyParams k{};
    k.chunks = (int)((most_bytes + kCopyChunk - 1) / kCopyChunk);
    for (int p0 = 0; p0 < count; p0 += kCopyPools) {
        k.pools = std::min(kCopyPools, count - p0);
        for (int i = 0; i < k.pools; ++i) {
            k.pool[i] = static_cast<char *>(pools[p0 + i].ptr);
            k.stride[i] = pools[p0 + i].stride;
            k.bytes[i] = (int32_t)pools[p0 + i].bytes;
        }
        const int64_t per_pair = (int64_t)k.pools * k.chunks;
        const int most = (int)std::max<int64_t>(1, std::min<int64_t>(kCopyPairs, kMostGroups / per_pair));
        for (int64_t i0 = 0; i0 < n_pairs; i0 += most) {
            k.pairs = (int)std::min<int64_t>(most, n_pairs - i0);
            for (int i = 0; i < k.pairs; ++i) {
                k.src[i] = pairs[2 * (i0 + i)];
                k.dst[i] = pairs[2 * (i0 + i) + 1];
            }
            const dim3 grid((unsigned)(k.pairs * per_pair));
            if (wide) hipLaunchKernelGGL(copy_pages_kernel<u32x4>, grid, dim3(256), 0, s, k);
            else hipLaunchKernelGGL(copy_pages_kernel<uint16_t>, grid, dim3(256), 0, s, k);
            const int rc = launched("page copy");
            if (rc != SA2_OK) return rc;
        }
    }
    return SA2_OK;
}

int64_t sa2_sample_workspace_bytes(int64_t rows, int64_t vocab) {
    if (rows < 1 || rows > 0x7fffffff || vocab < 1 || vocab > (1 << 24)) return -1;
    const int64_t chunks = (vocab + kSampleChunk - 1) / kSampleChunk;
    return chunks == 1 ? 0 : rows * chunks * (int64_t)(sizeof(SampleRecord) + 4 * kSampleThreads);
}

int sa2_sample(const void *logits, int32_t type, int64_t rows, int64_t vocab, int64_t stride, const float *noise, int64_t noise_stride,
               const sa2_sample_params *params, int64_t *tokens, float *logprobs, void *workspace, int64_t workspace_bytes, void *hip_stream) {
    if (!logits || !noise || !params || !tokens || !logprobs) return fail_with(SA2_ERR_NULL_POINTER, "logits, noise, params, tokens and logprobs are required");
    if (rows < 1 || rows > 0x7fffffff || vocab < 1 || vocab > (1 << 24)) return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld vocab=%lld (up to 2^24)", (long long)rows, (long long)vocab);
    if (type < 0 || type > 2) return fail_with(SA2_ERR_UNSUPPORTED, "logits of type %d", type);
    if ((reinterpret_cast<uintptr_t>(logits) & (type == SA2_ELEMENT_F32 ? 3 : 1)) != 0 || (reinterpret_cast<uintptr_t>(noise) & 3) != 0)
        return fail_with(SA2_ERR_ALIGNMENT, "logits and noise must be aligned to their elements");
    const int64_t bytes = sa2_sample_workspace_bytes(rows, vocab), chunks = (vocab + kSampleChunk - 1) / kSampleChunk;
    if (rows * chunks > kMostGroups || (chunks > 1 && rows > kMostGroups * 256 / kRowThreads)) return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld vocab=%lld: too large for a 1-D grid", (long long)rows, (long long)vocab);
    if (bytes > 0 && (!workspace || workspace_bytes < bytes))
        return fail_with(SA2_ERR_BAD_SHAPE, "workspace of %lld bytes, %lld are needed", (long long)(workspace ? workspace_bytes : 0), (long long)bytes);
    if (bytes > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return fail_with(SA2_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    SampleParams k{};
    k.logits = static_cast<const char *>(logits);
    k.stride = stride;
    k.noise = noise;
    k.noise_stride = noise_stride;
    k.temperature = params->temperature;
    k.top_p = params->top_p;
    k.min_p = params->min_p;
    k.top_k = params->top_k;
    k.temperature_all = params->temperature_all;
    k.top_p_all = params->top_p_all;
    k.min_p_all = params->min_p_all;
    k.top_k_all = params->top_k_all;
    k.vocab = (int)vocab;
    k.chunks = (int)chunks;
    if (bytes > 0) {
        k.records = static_cast<SampleRecord *>(workspace);
        k.tops = reinterpret_cast<float *>(k.records + rows * chunks);
    }
    k.tokens = tokens;
    k.logprobs = logprobs;
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    if (type == SA2_ELEMENT_BF16) launch_sample<0>(rows, k, s);
    else if (type == SA2_ELEMENT_F16) launch_sample<1>(rows, k, s);
    else launch_sample<2>(rows, k, s);
    return launched("sampling");
}

}  // extern "C"
