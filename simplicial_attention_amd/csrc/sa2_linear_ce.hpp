// Softmax cross entropy of a read-out layer, and its gradients, without keeping the logits.
//
//   z = H W^T     lse_i = log sum_v exp z_iv     l_i = lse_i - z_{i, t_i}
//   dz_iv = g_i (exp(z_iv - lse_i) - [v = t_i])     dH = dz W     dW = dz^T H
//
// The forward keeps, of every tile of logits, a maximum and a sum per row; they are merged to lse.  The backward goes over the vocabulary in pieces: logits of a piece
// are formed again, become dz in the operands' type, and are multiplied both ways.  Four products of 2 N V D operations for the three that a
// gradient needs, and N x (a piece) of memory.  Bound by the matrix unit; with few channels by the exponentials of the two epilogues.
// 8192 rows of 2048 channels over 131072 tokens: 14.8 to 15.1 ms by card (logits 3.8, dz 4.1, dH 3.6, dW 3.3), 1.19 PFLOP/s; over 32000 of 512 channels 1.24 to 1.3 ms.  The smallest (60 rows, 256 tokens): 22 us in four
// launches.
//
// dz is rounded to the operands' type for its products.  To use that type's range well it is divided by the largest weight G of a row's loss
// (mean and sum: the one weight of all) and in fp16 multiplied by 1024, which the products' results are multiplied by again in 32 bits.  Where every row has a weight
// of its own (reduction none), that would leave rows of small weights the least steps of fp16 (over 32000 tokens dH of a row at a millionth of G was off by 9 %): there dH is made from a second
// dz without weights (1237 rows of 328 channels over 10007 tokens: ce_dz_kernel 26.4 -> 30.6 us), and the rows of the result are multiplied by theirs.  dW adds rows up, and what it loses of one (2^-35 G of each dz) is small beside G.
#pragma once

#include "sa2_product.hpp"

namespace sa2 {

constexpr int kCeNone = 0, kCeMean = 1, kCeSum = 2;

struct CeParams {
    ProductShape shape;
    ProductOperand w, h;                     // vocabulary x dim, rows x dim
    int rows, vocab, dim, first, reduction;  // first: token at which the piece begins
    int channels;                            // of the gradients' rows, at most dim
    const int64_t *targets;
    int64_t ignore;
    // forward
    float2 *parts;                           // [half tiles of the vocabulary][rows]: maximum, sum of exp(z - maximum)
    float *at_target;                        // [rows] logit of the target
    uint32_t *ticket;
    int n_parts;
    float *sums;                             // [blocks of 32 rows]: loss and number of rows that count
    float *loss, *lse, *count;               // count: mean and sum only
    uint32_t *mask;                          // [blocks of 32 rows]: rows that count
    // backward
    const float *up;                         // gradient of the loss: one number, or one per row
    const float *most;                       // largest finite |up| of a row that counts (reduction none)
    char *dz;                                // [rows][piece], or NULL
    char *dz_rows;                           // the same without the rows' weights, for dH (reduction none in fp16), or NULL
    int64_t dz_row;                          // bytes
};

// exp(z - ref) in one multiply-add and an exponential: the rounding of ref log2(e) enters the exponent, up to 2e-4 of the result where ref is 4096.  Beyond that
// (some row of the wave) the difference is formed first, exact for what is near ref.
constexpr float kCeFar = 4096.f;

template <int T>
constexpr float ce_scale = T == kF16 ? 1024.f : 1.f;
template <int T>
constexpr float ce_log2_scale = T == kF16 ? 10.f : 0.f;

// ---- forward: a tile of logits

template <int T, int NL, int NR>
__global__ __launch_bounds__(256, NL == 4 ? 1 : 2) void ce_logits_kernel(CeParams p) {
    using P = Product<T, NL, NR, true, true, false>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape, blockIdx.x, gridDim.x);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
    f32x16 acc[NL][NR];
    P::run(p.shape, p.w, p.h, at, nullptr, lds, acc);
    const int lane = threadIdx.x & 63, wave = wave_index(), hf = lane >> 5;
    const int v0 = at.tile_r * P::TILE_R + 32 * NR * (wave & 1);
    const bool ragged = v0 + 32 * NR > p.vocab;
#pragma unroll
    for (int a = 0; a < NL; ++a) {
        const int row = at.tile_l * P::TILE_L + 32 * (NL * (wave >> 1) + a) + dmap_row(lane & 31);
        take(acc[a]);
        if (ragged) {
#pragma unroll
            for (int b = 0; b < NR; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (v0 + 32 * b + 16 * hf + r >= p.vocab) acc[a][b][r] = -INFINITY;
        }
        const int64_t target = row < p.rows ? p.targets[row] : -1;
        const int mine = target >= v0 && target < v0 + 32 * NR && target < p.vocab ? (int)(target - v0) : -1;
        if (wave_any(mine >= 0)) {
            const int here = mine - 16 * hf;
            float x = 0.f;
#pragma unroll
            for (int b = 0; b < NR; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) x = here == 32 * b + r ? acc[a][b][r] : x;
            if (mine >= 0 && (mine >> 4 & 1) == hf) p.at_target[row] = x;
        }
        float m = -INFINITY;
#pragma unroll
        for (int b = 0; b < NR; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[a][b][r]);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float ref = m == -INFINITY ? 0.f : m, ref2 = ref * kLog2e;
        float s = 0.f;
        const bool far = fabsf(ref) > kCeFar;            // (a row's own matter: its neighbours' results do not depend on it)
        if (wave_any(far)) {
#pragma unroll
            for (int b = 0; b < NR; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s += fast_exp2(far ? (acc[a][b][r] - ref) * kLog2e : acc[a][b][r] * kLog2e - ref2);
        } else {
#pragma unroll
            for (int b = 0; b < NR; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s += fast_exp2(acc[a][b][r] * kLog2e - ref2);
        }
        s += __shfl_xor(s, 32, 64);
        if (hf == 0 && row < p.rows) p.parts[(int64_t)(2 * at.tile_r + (wave & 1)) * p.rows + row] = make_float2(m, s);
    }
}

// ROWS rows a workgroup, the parts of each merged by G threads; the last workgroup adds up the losses in order
template <int ROWS, int G>
__global__ __launch_bounds__(ROWS *G) void ce_merge_kernel(CeParams p) {
    constexpr int WAVES = ROWS * G / 64;
    __shared__ float2 parts[G > 1 ? G : 1][G > 1 ? ROWS + 1 : 1];
    __shared__ float2 totals[WAVES];
    __shared__ uint32_t two[WAVES];
    __shared__ uint32_t last;
    const int c = threadIdx.x % ROWS, g = threadIdx.x / ROWS;
    // the row that this thread says something about in the end (with G > 1: the first lane of each 32)
    const int row = blockIdx.x * ROWS + (G > 1 ? threadIdx.x / 32 : c);
    const bool says = row < p.rows && (G == 1 || (threadIdx.x & 31) == 0);
    int64_t target = -1;
    float at_target = 0.f;
    if (says) target = p.targets[row], at_target = p.at_target[row];
    float m = -INFINITY, s = 0.f;
    auto add = [&](float2 x) {
        const float top = fmaxf(m, x.x), ref = top == -INFINITY ? 0.f : top;
        s = s * fast_exp2((m - ref) * kLog2e) + x.y * fast_exp2((x.x - ref) * kLog2e);
        m = top;
    };
    if (blockIdx.x * ROWS + c < p.rows)
#pragma unroll 4
        for (int i = g; i < p.n_parts; i += G) add(p.parts[(int64_t)i * p.rows + blockIdx.x * ROWS + c]);
    if constexpr (G > 1) {
        static_assert(ROWS == 32 && G == 32, "a row's parts are the 32 lanes of half a wave then");
        parts[g][c] = make_float2(m, s);
        __syncthreads();
        const float2 x = parts[threadIdx.x & 31][threadIdx.x / 32];
        m = x.x, s = x.y;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) add(make_float2(__shfl_xor(m, off, 64), __shfl_xor(s, off, 64)));
    }
    float loss = 0.f;
    bool counts = false;
    if (says) {
        const float lse = m + logf(s);
        counts = target != p.ignore;
        // (a target that is no token: no number comes of it)
        if (counts) loss = target >= 0 && target < p.vocab ? lse - at_target : NAN;
        p.lse[row] = lse;
        if (p.reduction == kCeNone) p.loss[row] = loss;
    }
    const uint64_t bits = __ballot(counts);
    if constexpr (G == 1) {
        if ((threadIdx.x & 31) == 0 && row < p.rows) p.mask[row >> 5] = (uint32_t)(bits >> (threadIdx.x & 32));
    }
    loss = lanes_sum<64>(loss);
    if ((threadIdx.x & 63) == 0) totals[threadIdx.x >> 6] = make_float2(loss, (float)__popcll(bits)), two[threadIdx.x >> 6] = (uint32_t)(bits & 1) | (uint32_t)(bits >> 32 & 1) << 1;
    __syncthreads();
    if (threadIdx.x == 0) {
        float2 sum = totals[0];
        for (int i = 1; i < WAVES; ++i) sum.x += totals[i].x, sum.y += totals[i].y;
        if constexpr (G > 1) {
            uint32_t word = 0;
            for (int i = 0; i < WAVES; ++i) word |= two[i] << (2 * i);
            p.mask[blockIdx.x] = word;
        }
        if (p.reduction == kCeNone) {
            last = 0;                            // (nobody asks for the sums)
        } else {
            p.sums[2 * blockIdx.x] = sum.x;
            p.sums[2 * blockIdx.x + 1] = sum.y;
            __threadfence();
            last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    // (atomic loads at the device's scope: what the other XCDs have written, past this one's cache)
    loss = 0.f;
    float count = 0.f;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += ROWS * G) {
        loss += __hip_atomic_load(&p.sums[2 * i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        count += __hip_atomic_load(&p.sums[2 * i + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    loss = lanes_sum<64>(loss);
    count = lanes_sum<64>(count);
    if ((threadIdx.x & 63) == 0) totals[threadIdx.x >> 6] = make_float2(loss, count);
    __syncthreads();
    if (threadIdx.x == 0) {
        loss = count = 0.f;
        for (int i = 0; i < WAVES; ++i) loss += totals[i].x, count += totals[i].y;
        *p.count = count;
        if (p.reduction == kCeMean) *p.loss = loss / count;
        else if (p.reduction == kCeSum) *p.loss = loss;
    }
}

// ---- backward

// the largest finite |up| of a row that counts
static __global__ __launch_bounds__(1024) void ce_most_kernel(const float *up, const uint32_t *mask, int rows, float *most) {
    __shared__ uint32_t tops[16];
    uint32_t m = 0;
    for (int i = threadIdx.x; i < rows; i += 1024)
        if (const uint32_t x = magnitude(up[i]); x < 0x7f800000u && (mask[i >> 5] >> (i & 31) & 1)) m = max(m, x);
    m = lanes_max<64>(m);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 0; i < 16; ++i) m = max(m, tops[i]);
        *most = as_f32(m);
    }
}

// what results of the products with dz are multiplied by
template <int T>
__device__ __forceinline__ float ce_factor(const CeParams &p) {
    if (p.reduction == kCeNone) return *p.most * (1.f / ce_scale<T>);
    if (p.reduction == kCeMean) return *p.count > 0.f ? *p.up / *p.count * (1.f / ce_scale<T>) : 0.f;      // (no row counts: no gradient)
    return *p.up * (1.f / ce_scale<T>);
}

template <int T>
__device__ __forceinline__ float ce_row_factor(const CeParams &p, int row) {
    return p.up[row] * (1.f / ce_scale<T>);
}

// TWO: dz_rows too
template <int T, int NL, int NR, bool TWO>
__global__ __launch_bounds__(256, NL == 4 ? 1 : 2) void ce_dz_kernel(CeParams p) {
    using P = Product<T, NL, NR, true, true, false>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape, blockIdx.x, gridDim.x);
    f32x16 acc[NL][NR];
    P::run(p.shape, p.w, p.h, at, nullptr, lds, acc);
    const int lane = threadIdx.x & 63, wave = wave_index(), hf = lane >> 5;
    const int c0 = at.tile_r * P::TILE_R + 32 * NR * (wave & 1);           // column of the piece
    __syncthreads();                                                     // (the tiles have been read)
    const ProductRows<T, NR> rows(lds);
#pragma unroll
    for (int a = 0; a < NL; ++a) {
        const int row0 = at.tile_l * P::TILE_L + 32 * (NL * (wave >> 1) + a), row = min(row0 + rows.row, p.rows - 1);
        const int64_t target = p.targets[row];
        const bool counts = target != p.ignore;
        const float ref = p.lse[row], ref2 = ref * kLog2e - ce_log2_scale<T>;
        const bool far = fabsf(ref) > kCeFar;
        take(acc[a]);
        // (what only some rows or tiles need is asked of the wave: a tile in the middle takes a multiply-add, an exponential and half a packing per element)
        if (wave_any(far)) {
#pragma unroll
            for (int b = 0; b < NR; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[a][b][r] = fast_exp2(far ? (acc[a][b][r] - ref) * kLog2e + ce_log2_scale<T> : acc[a][b][r] * kLog2e - ref2);
        } else {
#pragma unroll
            for (int b = 0; b < NR; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[a][b][r] = fast_exp2(acc[a][b][r] * kLog2e - ref2);
        }
        const int64_t from = p.first + c0;
        const int mine = counts && target >= from && target < from + 32 * NR ? (int)(target - from) - 16 * hf : -100;
        if (wave_any(mine > -100)) {
#pragma unroll
            for (int b = 0; b < NR; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (mine == 32 * b + r) acc[a][b][r] -= ce_scale<T>;
        }
        const float valid = counts && !(target >= 0 && target < p.vocab) ? NAN : 1.f;
        const auto store = [&](char *dz, float by) {
            if (wave_any(by != 1.f)) {
#pragma unroll
                for (int b = 0; b < NR; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[a][b][r] *= by;
            }
            int end = p.vocab - p.first - c0 - 16 * hf, first_row = row0;   // columns of this half that are tokens
            asm("" : "+v"(end), "+s"(first_row));                           // (else the compiler keeps masks of all columns, and addresses for the next store, and spills them)
            if (wave_any(!counts || end < 32 * NR)) {
#pragma unroll
                for (int b = 0; b < NR; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (!counts || 32 * b + r >= end) acc[a][b][r] = 0.f;
            }
#pragma unroll
            for (int b = 0; b < NR; ++b) rows.put(b, acc[a][b]);
            rows.each([&](int r, int col, u32x4 v) {
                if (first_row + r < p.rows) st_global16(dz + (int64_t)(first_row + r) * p.dz_row + 2 * (c0 + col), v);
            });
        };
        if constexpr (TWO) store(p.dz_rows, valid);
        if (!TWO || p.dz) {
            float weight = TWO ? 1.f : valid;
            if (p.reduction == kCeNone) {
                const float most = *p.most;
                weight *= most > 0.f ? p.up[row] / most : p.up[row];          // (an infinite weight, or one that is no number, is its own row's matter)
            }
            store(p.dz, weight);
        }
    }
}

// N results of two bytes of a row of `channels`, from d on; the others are padding
template <int N, typename V>
__device__ __forceinline__ void put_channels(char *out, int row, int d, int channels, const V &v) {
    char *to = out + ((int64_t)row * channels + d) * 2;
    typedef V any __attribute__((aligned(2)));
    if (channels % N == 0) {
        if (d < channels) *reinterpret_cast<V *>(to) = v;
    } else if (d + N <= channels) {
        *reinterpret_cast<any *>(to) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (d + i < channels) *reinterpret_cast<uint16_t *>(to + 2 * i) = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
    }
}

// Where the results of a product with dz go.  DIRECT: rounded, times what they were divided by; else fp32, for ce_combine_kernel.
struct CeOutput {
    char *out;                     // DIRECT: [rows][dim] in the operands' type
    float *parts;                  // else: [share][rows][dim]
    int rows, add;                 // add: to what is in the parts
    int masked;                    // rows that do not count become zero
    int by_row;                    // rows of a dz without weights: each is multiplied by its own
};

template <int T, int NL, int NR, bool DIRECT>
__device__ __forceinline__ void ce_store(const CeParams &p, const CeOutput &o, const ProductPlace &at, char *lds, f32x16 (&acc)[NL][NR]) {
    const int wave = wave_index();
    const int c0 = 64 * NR * at.tile_r + 32 * NR * (wave & 1);
    char *const out = DIRECT ? o.out : reinterpret_cast<char *>(o.parts + (int64_t)at.share * o.rows * p.dim);
    const float factor = DIRECT ? ce_factor<T>(p) : 1.f;
    __syncthreads();                              // (the tiles have been read)
    const ProductRows<DIRECT ? T : kF32, NR> rows(lds);
#pragma unroll
    for (int a = 0; a < NL; ++a) {
        const int row0 = 64 * NL * at.tile_l + 32 * (NL * (wave >> 1) + a);
        take(acc[a]);
        float by = factor;
        if constexpr (DIRECT && T == kF16) {
            if (o.by_row) by = ce_row_factor<T>(p, min(row0 + rows.row, o.rows - 1));
        }
#pragma unroll
        for (int b = 0; b < NR; ++b) rows.put(b, acc[a][b], by);
        rows.each([&](int r, int col, u32x4 v) {
            const int row = row0 + r, d = c0 + col;
            if (row >= o.rows || d >= p.dim) return;
            [[maybe_unused]] char *to = out + ((int64_t)row * p.dim + d) * 4;
            if constexpr (DIRECT) {
                if (o.masked && !(p.mask[row >> 5] >> (row & 31) & 1)) v = (u32x4){0, 0, 0, 0};
                put_channels<8>(out, row, d, p.channels, v);
                return;
            } else if (o.add) {
                const float4 x = __builtin_bit_cast(float4, v), y = *reinterpret_cast<const float4 *>(to);
                v = __builtin_bit_cast(u32x4, make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w));
            }
            st_global16(to, v);
        });
    }
}

// Logits of few tiles over many channels (172 rows of 3816 over 745 tokens: 9.0 us and 4.6 for their sums instead of 33 to 38, of which twelve CUs wait for their rows): shares of the contraction, fp32 [share][rows][columns] (p.dim: columns, a multiple of 8; those behind the vocabulary may hold anything)
template <int T, int NL, int NR>
__global__ __launch_bounds__(256, NL == 4 ? 1 : 2) void ce_shares_kernel(CeParams p, CeOutput o) {
    using P = Product<T, NL, NR, true, true, false>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape, blockIdx.x, gridDim.x);
    f32x16 acc[NL][NR];
    P::run(p.shape, p.w, p.h, at, nullptr, lds, acc);
    ce_store<T, NL, NR, false>(p, o, at, lds, acc);
}

// What the epilogues of ce_logits_kernel (DZ: ce_dz_kernel) do, from the shares added in order: a wave takes 256 columns of a row, a lane four.
constexpr int kCeColumns = 256;
template <int T, bool DZ>
__global__ __launch_bounds__(256) void ce_shared_logits_kernel(CeParams p, CeOutput o, int chunks) {
    if (!DZ && blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave_index();
    const int row = (int)(unit / chunks), chunk = (int)(unit - (int64_t)row * chunks), lane = threadIdx.x & 63;
    if (row >= p.rows) return;
    const int c = chunk * kCeColumns + 4 * lane, end = p.vocab - p.first - c;              // (columns of the lane that are tokens)
    float z[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < p.dim) {
        const float *src = o.parts + (int64_t)row * p.dim + c;
        const int64_t all = (int64_t)p.rows * p.dim;
#pragma unroll 8
        for (int x = 0; x < p.shape.shares; ++x, src += all) {
            const float4 v = *reinterpret_cast<const float4 *>(src);
            z[0] += v.x, z[1] += v.y, z[2] += v.z, z[3] += v.w;
        }
    }
    const int64_t target = p.targets[row];
    const int mine = target >= p.first + c && target < p.first + (int64_t)c + 4 && target < p.vocab ? (int)(target - p.first - c) : -1;
    if constexpr (!DZ) {
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i == mine) p.at_target[row] = z[i];
            if (i >= end) z[i] = -INFINITY;
            m = fmaxf(m, z[i]);
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < 4; ++i) s += fast_exp2((z[i] - ref) * kLog2e);
        s = lanes_sum<64>(s);
        if (lane == 0) p.parts[(int64_t)chunk * p.rows + row] = make_float2(m, s);
    } else {
        if (c >= p.dim) return;
        const bool counts = target != p.ignore;
        const float lse = p.lse[row];
        const float valid = counts && !(target >= 0 && target < p.vocab) ? NAN : 1.f;
        float weight = valid;
        if (p.reduction == kCeNone) {
            const float most = *p.most;
            weight *= most > 0.f ? p.up[row] / most : p.up[row];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = fast_exp2((z[i] - lse) * kLog2e + ce_log2_scale<T>) - (i == mine ? ce_scale<T> : 0.f);
        const auto store = [&](char *dz, float by) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = !counts || i >= end ? 0.f : z[i] * by;
            *reinterpret_cast<u32x2 *>(dz + (int64_t)row * p.dz_row + 2 * c) = pack4<T>(v);
        };
        if (T == kF16 && p.dz_rows) store(p.dz_rows, valid);
        if (p.dz) store(p.dz, weight);
    }
}

// dH of a piece: rows x dim, contracted over the piece's tokens (r side: W read along dim)
template <int T, int NL, int NR, bool DIRECT>
__global__ __launch_bounds__(256, NL == 4 ? 1 : 2) void ce_dh_kernel(CeParams p, CeOutput o) {
    using P = Product<T, NL, NR, false, true, false>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape, blockIdx.x, gridDim.x);
    f32x16 acc[NL][NR];
    P::run(p.shape, p.w, p.h, at, nullptr, lds, acc);
    ce_store<T, NL, NR, DIRECT>(p, o, at, lds, acc);
}

// dW of a piece: tokens x dim, contracted over the rows that count
template <int T, int NL, int NR, bool DIRECT>
__global__ __launch_bounds__(256, NL == 4 ? 1 : 2) void ce_dw_kernel(CeParams p, CeOutput o) {
    using P = Product<T, NL, NR, false, false, true>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape, blockIdx.x, gridDim.x);
    f32x16 acc[NL][NR];
    P::run(p.shape, p.w, p.h, at, p.mask, lds, acc);
    ce_store<T, NL, NR, DIRECT>(p, o, at, lds, acc);
}

// Both of a piece in one launch, in tiles of 128 x 128: the first workgroups are dH's, from a multiple of eight on (so that each XCD still walks tiles next to each other) dW's.
// One launch fills the chip where two would each leave part of it idle at their ends: 1024 rows of 1024 channels over 1024 tokens 25.9 -> 14.4 us, 1237 of 328 over 10007 34.8 -> 27.7.
template <int T, bool H_DIRECT, bool W_DIRECT>
__global__ __launch_bounds__(256, 2) void ce_gradients_kernel(CeParams h, CeOutput ho, CeParams w, CeOutput wo, int h_groups) {
    using H = Product<T, 2, 2, false, true, false>;
    using W = Product<T, 2, 2, false, false, true>;
    __shared__ __attribute__((aligned(16))) char lds[W::LDS];
    static_assert(W::LDS >= H::LDS, "");
    const int w_first = (h_groups + 7) / 8 * 8, wg = blockIdx.x;
    f32x16 acc[2][2];
    if (wg < w_first) {
        if (wg >= h_groups) return;
        const ProductPlace at = product_place(h.shape, wg, h_groups);
        H::run(h.shape, h.w, h.h, at, nullptr, lds, acc);
        ce_store<T, 2, 2, H_DIRECT>(h, ho, at, lds, acc);
    } else {
        const ProductPlace at = product_place(w.shape, wg - w_first, gridDim.x - w_first);
        W::run(w.shape, w.w, w.h, at, w.mask, lds, acc);
        ce_store<T, 2, 2, W_DIRECT>(w, wo, at, lds, acc);
    }
}

// the shares added in order, four elements a thread (blockIdx.y: of dH or dW; z: beyond 2^32 threads)
struct CeSum {
    CeOutput o;
    char *out;
    int shares, dim;
};
template <int T>
__global__ __launch_bounds__(256) void ce_combine_kernel(CeParams p, CeSum a, CeSum b) {
    // (by value: pointers out of a chosen struct would be accessed as if they could be LDS)
    const bool second = blockIdx.y != 0;
    const float *const parts = second ? b.o.parts : a.o.parts;
    char *const out = second ? b.out : a.out;
    const int rows = second ? b.o.rows : a.o.rows, masked = second ? b.o.masked : a.o.masked, by_row = second ? b.o.by_row : a.o.by_row, shares = second ? b.shares : a.shares, dim = a.dim;
    const int64_t at = (((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * 256 + threadIdx.x) * 4, all = (int64_t)rows * dim;
    if (at >= all) return;
    const int row = (int)(at / dim), d = (int)(at - (int64_t)row * dim);
    const float factor = by_row ? ce_row_factor<T>(p, row) : ce_factor<T>(p);
    const bool counts = !masked || (p.mask[row >> 5] >> (row & 31) & 1);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    const float *src = parts + at;
#pragma unroll 8
    for (int x = 0; x < shares; ++x, src += all) {
        const float4 v = *reinterpret_cast<const float4 *>(src);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const float v[4] = {s.x * factor, s.y * factor, s.z * factor, s.w * factor};
    u32x2 w = pack4<T>(v);
    if (!counts) w = (u32x2){0, 0};
    put_channels<4>(out, row, d, p.channels, w);
}

}  // namespace sa2
