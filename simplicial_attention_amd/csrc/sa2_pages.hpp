// Rows into the pages of a cache, and pages to other pages.
//
// Both are bound by the bytes they read and write, and where these are few by the launch: 64 tokens into four pools 4.7 us (an empty launch 3.6), 8 x 2048 tokens
// into two pools of 8 x 64 channels (67 MB) 12 us; 512 pages of every pool (1.2 GB) 253 us, 4.8 TB/s where a copy of 2 GiB reaches 4.9; eight pages of
// 36 pools 7.5 us.
#pragma once

#include "sa2_common.hpp"

namespace sa2 {

struct AppendItem {
    char *pool;
    int64_t p_sp, p_sr, p_sh;      // bytes
    const char *rows;
    int64_t r_sb, r_sn, r_sh;      // bytes
};
constexpr int kAppendMost = 4;
struct AppendParams {
    AppendItem item[kAppendMost];
    const int32_t *tables, *lengths, *counts;
    int64_t t_sb;
    int ps, pages, width, B, n, HK, dim, pieces;      // dim: channels of a row; pieces: 16-byte pieces of a pool's row
    int count;
};

__device__ __forceinline__ float element(const char *at, int type) {
    if (type == 2) return *reinterpret_cast<const float *>(at);
    const uint16_t x = *reinterpret_cast<const uint16_t *>(at);
    return type == 1 ? (float)__builtin_bit_cast(_Float16, x) : as_f32((uint32_t)x << 16);
}
__device__ __forceinline__ uint32_t element_bits(float x, int type) {
    return type == 1 ? (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x) : (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x);
}

// One thread moves a 16-byte piece of a row of every pool: one look at the table for all of them.  PLAIN: rows of the pools' type in whole
// aligned pieces; else elements are converted (types: 0 bf16, 1 fp16, 2 fp32) and channels beyond `dim` are zero.  Converted, a thread loads its elements one by one: fp32 rows
// into bf16 pools 7.9 us for 64 tokens into four pools and 36 for 8 x 2048 into two (floor 20).
template <bool PLAIN>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p, int src_type, int dst_type) {
    const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int per_row = p.HK * p.pieces;
    const int64_t bt = x / per_row;
    if (bt >= (int64_t)p.B * p.n) return;
    const int rest = (int)(x - bt * per_row), h = rest / p.pieces, piece = rest - h * p.pieces;
    const int b = (int)(bt / p.n), t = (int)(bt - (int64_t)b * p.n);
    const int length = max(p.lengths[b], 0), count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    const int pos = length - count + t;
    if (t >= count || pos < 0) return;
    const int entry = pos / p.ps, row = pos - entry * p.ps;
    if (entry >= p.width) return;
    const int page = p.tables[b * p.t_sb + entry];
    if ((unsigned)page >= (unsigned)p.pages) return;
#pragma unroll
    for (int i = 0; i < kAppendMost; ++i) {
        if (i >= p.count) break;
        const AppendItem &it = p.item[i];
        const char *src = it.rows + b * it.r_sb + t * it.r_sn + h * it.r_sh;
        char *dst = it.pool + (int64_t)page * it.p_sp + (int64_t)row * it.p_sr + (int64_t)h * it.p_sh + piece * 16;
        if constexpr (PLAIN) {
            st_global16(dst, ld_global16(src + piece * 16));
        } else {
            const int size = src_type == 2 ? 4 : 2;
            u32x4 v;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int d = piece * 8 + 2 * w;
                const uint32_t a = d < p.dim ? element_bits(element(src + d * size, src_type), dst_type) : 0u;
                const uint32_t z = d + 1 < p.dim ? element_bits(element(src + (d + 1) * size, src_type), dst_type) : 0u;
                v[w] = a | (z << 16);
            }
            st_global16(dst, v);
        }
    }
}

// ---- pages to other pages: the list travels in the kernel's arguments, so a call is one launch and no transfer
constexpr int kCopyPools = 64, kCopyPairs = 240;
struct CopyParams {
    char *pool[kCopyPools];
    int64_t stride[kCopyPools];    // bytes between pages
    int32_t bytes[kCopyPools];     // of a page
    int32_t src[kCopyPairs], dst[kCopyPairs];
    int pools, pairs, chunks;      // chunks of kCopyChunk bytes of the largest page
};
static_assert(sizeof(CopyParams) <= 4096, "kernel arguments");
constexpr int kCopyChunk = 256 * 16 * 4;

template <typename T>
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyParams p) {
    const int chunk = blockIdx.x % p.chunks, rest = blockIdx.x / p.chunks;
    const int pool = rest % p.pools, pair = rest / p.pools;
    const int bytes = p.bytes[pool];
    const char *src = p.pool[pool] + p.src[pair] * p.stride[pool];
    char *dst = p.pool[pool] + p.dst[pair] * p.stride[pool];
    const int end = min(bytes, (chunk + 1) * kCopyChunk);
    constexpr int S = sizeof(T);
    for (int at = chunk * kCopyChunk + threadIdx.x * S; at < end; at += 256 * S * 4) {
        T v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i * 256 * S < end) v[i] = *reinterpret_cast<const T *>(src + at + i * 256 * S);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i * 256 * S < end) *reinterpret_cast<T *>(dst + at + i * 256 * S) = v[i];
    }
}

}  // namespace sa2
