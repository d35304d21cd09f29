// Softmax cross entropy of a read-out layer, and its gradients, without keeping the logits.
//
//   z = H W^T     lse_i = log sum_v exp z_iv     l_i = lse_i - z_{i, t_i}
//   dz_iv = g_i (exp(z_iv - lse_i) - [v = t_i])     dH = dz W     dW = dz^T H
//
// The forward keeps, of every tile of logits, a maximum and a sum per row; they are merged to lse.  The backward goes over the vocabulary in pieces: logits of a piece
// are formed again, become dz in the operands' type, and are multiplied both ways.  Four products of 2 N V D operations for the three that a
// gradient needs, and N x (a piece) of memory.  Bound by the matrix unit; with few channels by the exponentials of the two epilogues.
//
// dz is rounded to the operands' type for its products.  To use that type's range well it is divided by the largest weight G of a row's loss
// (mean and sum: the one weight of all) and in fp16 multiplied by 1024, which the products' results are multiplied by again in 32 bits.
#pragma once

#include "sa2_product.hpp"

namespace sa2 {

constexpr int kCeNone = 0, kCeMean = 1, kCeSum = 2;

struct CeParams {
    ProductShape shape;
    ProductOperand w, h;                     // vocabulary x dim, rows x dim
    int rows, vocab, dim, first, reduction;  // first: token at which the piece begins
    const int64_t *targets;
    int64_t ignore;
    // forward
    float2 *parts;                           // [half tiles of the vocabulary][rows]: maximum, sum of exp(z - maximum)
    float *at_target;                        // [rows] logit of the target
    uint32_t *ticket;
    int n_parts;
    float *sums;                             // [blocks of 32 rows]: loss and number of rows that count
    float *loss, *lse, *count;
    uint32_t *mask;                          // [blocks of 32 rows]: rows that count
    // backward
    const float *up;                         // gradient of the loss: one number, or one per row
    const float *most;                       // largest |up| of a row that counts (reduction none)
    char *dz;                                // [rows][piece]
    int64_t dz_row;                          // bytes
};

// exp(z - ref) in one multiply-add and an exponential: the rounding of ref log2(e) enters the exponent, up to 2e-4 of the result where ref is 4096.  Beyond that
// (some row of the wave) the difference is formed first, exact for what is near ref.
constexpr float kCeFar = 4096.f;

template <int T>
constexpr float ce_scale = T == kF16 ? 1024.f : 1.f;

// ---- forward: a tile of logits

template <int T, int NB>
__global__ __launch_bounds__(256) void ce_logits_kernel(CeParams p) {
    using P = Product<T, NB, true, true, false>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
    f32x16 acc[NB][NB];
    P::run(p.shape, p.w, p.h, at, nullptr, lds, acc);
    const int lane = threadIdx.x & 63, wave = wave_index(), hf = lane >> 5;
    const int v0 = at.tile_r * P::TILE + 32 * NB * (wave & 1);
    const bool ragged = v0 + 32 * NB > p.vocab;
#pragma unroll
    for (int a = 0; a < NB; ++a) {
        const int row = at.tile_l * P::TILE + 32 * (NB * (wave >> 1) + a) + dmap_row(lane & 31);
        if (ragged) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (v0 + 32 * b + 16 * hf + r >= p.vocab) acc[a][b][r] = -INFINITY;
        }
        const int64_t target = row < p.rows ? p.targets[row] : -1;
        const int mine = target >= v0 && target < v0 + 32 * NB && target < p.vocab ? (int)(target - v0) : -1;
        if (wave_any(mine >= 0)) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (mine == 32 * b + 16 * hf + r) p.at_target[row] = acc[a][b][r];
        }
        float m = -INFINITY;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[a][b][r]);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float ref = m == -INFINITY ? 0.f : m, ref2 = ref * kLog2e;
        float s = 0.f;
        const bool far = fabsf(ref) > kCeFar;            // (a row's own matter: its neighbours' results do not depend on it)
        if (wave_any(far)) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s += fast_exp2(far ? (acc[a][b][r] - ref) * kLog2e : acc[a][b][r] * kLog2e - ref2);
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s += fast_exp2(acc[a][b][r] * kLog2e - ref2);
        }
        s += __shfl_xor(s, 32, 64);
        if (hf == 0 && row < p.rows) p.parts[(int64_t)(2 * at.tile_r + (wave & 1)) * p.rows + row] = make_float2(m, s);
    }
}

// 32 rows a workgroup: the parts of each merged by 32 threads; the last workgroup adds up the losses in order
static __global__ __launch_bounds__(1024) void ce_merge_kernel(CeParams p) {
    __shared__ float2 parts[32][33];
    __shared__ float2 totals[16];
    __shared__ uint32_t last;
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, row = blockIdx.x * 32 + c;
    float m = -INFINITY, s = 0.f;
    auto add = [&](float2 x) {
        const float top = fmaxf(m, x.x), ref = top == -INFINITY ? 0.f : top;
        s = s * fast_exp2((m - ref) * kLog2e) + x.y * fast_exp2((x.x - ref) * kLog2e);
        m = top;
    };
    if (row < p.rows)
#pragma unroll 4
        for (int i = g; i < p.n_parts; i += 32) add(p.parts[(int64_t)i * p.rows + row]);
    parts[g][c] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x < 64) {
        float loss = 0.f;
        bool counts = false;
        if (threadIdx.x < 32) {
            m = -INFINITY, s = 0.f;
#pragma unroll 4
            for (int i = 0; i < 32; ++i) add(parts[i][c]);
            if (row < p.rows) {
                const float lse = m + logf(s);
                const int64_t target = p.targets[row];
                counts = target != p.ignore;
                // (a target that is no token: no number comes of it)
                if (counts) loss = target >= 0 && target < p.vocab ? lse - p.at_target[row] : NAN;
                p.lse[row] = lse;
                if (p.reduction == kCeNone) p.loss[row] = loss;
            }
        }
        const uint32_t bits = (uint32_t)__ballot(counts);
        loss = lanes_sum<32>(loss);
        if (threadIdx.x == 0) {
            p.mask[blockIdx.x] = bits;
            p.sums[2 * blockIdx.x] = loss;
            p.sums[2 * blockIdx.x + 1] = (float)__popc(bits);
            __threadfence();
            last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    float loss = 0.f, count = 0.f;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 1024) {
        loss += __hip_atomic_load(&p.sums[2 * i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        count += __hip_atomic_load(&p.sums[2 * i + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    loss = lanes_sum<64>(loss);
    count = lanes_sum<64>(count);
    if ((threadIdx.x & 63) == 0) totals[threadIdx.x >> 6] = make_float2(loss, count);
    __syncthreads();
    if (threadIdx.x == 0) {
        loss = count = 0.f;
        for (int i = 0; i < 16; ++i) loss += totals[i].x, count += totals[i].y;
        *p.count = count;
        if (p.reduction == kCeMean) *p.loss = loss / count;
        else if (p.reduction == kCeSum) *p.loss = loss;
    }
}

// ---- backward

// the largest |up| of a row that counts
static __global__ __launch_bounds__(1024) void ce_most_kernel(const float *up, const uint32_t *mask, int rows, float *most) {
    __shared__ uint32_t tops[16];
    uint32_t m = 0;
    for (int i = threadIdx.x; i < rows; i += 1024)
        if (mask[i >> 5] >> (i & 31) & 1) m = max(m, magnitude(up[i]));
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

template <int T, int NB>
__global__ __launch_bounds__(256) void ce_dz_kernel(CeParams p) {
    using P = Product<T, NB, true, true, false>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape);
    f32x16 acc[NB][NB];
    P::run(p.shape, p.w, p.h, at, nullptr, lds, acc);
    const int lane = threadIdx.x & 63, wave = wave_index(), hf = lane >> 5;
    const int c0 = at.tile_r * P::TILE + 32 * NB * (wave & 1);           // column of the piece
#pragma unroll
    for (int a = 0; a < NB; ++a) {
        const int row = at.tile_l * P::TILE + 32 * (NB * (wave >> 1) + a) + dmap_row(lane & 31);
        if (row >= p.rows) continue;
        const int64_t target = p.targets[row];
        const bool counts = target != p.ignore;
        float weight = ce_scale<T>;
        if (p.reduction == kCeNone) {
            const float most = *p.most;
            weight *= most > 0.f ? p.up[row] / most : most;              // (all weights zero, or one that is no number)
        }
        if (counts && !(target >= 0 && target < p.vocab)) weight = NAN;
        const float ref = p.lse[row], ref2 = ref * kLog2e;
        const bool far = fabsf(ref) > kCeFar;
        const bool any_far = wave_any(far);
        const int64_t mine = target - p.first - c0;
        char *out = p.dz + row * p.dz_row + 2 * (c0 + 16 * hf);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float x[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int col = 32 * b + 16 * hf + r;
                float e = acc[a][b][r] * kLog2e - ref2;
                if (any_far) e = far ? (acc[a][b][r] - ref) * kLog2e : e;
                e = fast_exp2(e);
                if (mine == col) e -= 1.f;
                x[r] = counts && p.first + c0 + col < p.vocab ? e * weight : 0.f;
            }
            float lo[8], hi[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) lo[r] = x[r], hi[r] = x[8 + r];
            st_some8<T>(out + 64 * b, 8, lo);
            st_some8<T>(out + 64 * b + 16, 8, hi);
        }
    }
}

// where the results of a product with dz go
struct CeOutput {
    char *out;                     // [rows][dim] in the operands' type (the sum is complete), or NULL
    float *parts;                  // [share][rows][dim]
    int rows, add;                 // add: to what is in the parts
    int masked;                    // rows that do not count become zero
};

template <int T, int NB, typename P>
__device__ __forceinline__ void ce_store(const CeParams &p, const CeOutput &o, const ProductPlace &at, const f32x16 (&acc)[NB][NB]) {
    const float factor = o.out ? ce_factor<T>(p) : 1.f;
    P::each_run(at, acc, [&](int row, int col, const f32x16 &x) {
        if (row >= o.rows) return;
        const bool counts = !o.masked || (p.mask[row >> 5] >> (row & 31) & 1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int d = col + 8 * half;
            if (d >= p.dim) continue;
            float *part = o.parts + ((int64_t)at.share * o.rows + row) * p.dim + d;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = x[8 * half + i];
            if (o.add) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += part[i];
            }
            if (o.out) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = counts ? v[i] * factor : 0.f;
                st_some8<T>(o.out + ((int64_t)row * p.dim + d) * 2, 8, v);
            } else {
                st_some8<kF32>(reinterpret_cast<char *>(part), 8, v);
            }
        }
    });
}

// dH of a piece: rows x dim, contracted over the piece's tokens (r side: W read along dim)
template <int T, int NB>
__global__ __launch_bounds__(256) void ce_dh_kernel(CeParams p, CeOutput o) {
    using P = Product<T, NB, false, true, false>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape);
    f32x16 acc[NB][NB];
    P::run(p.shape, p.w, p.h, at, nullptr, lds, acc);
    ce_store<T, NB, P>(p, o, at, acc);
}

// dW of a piece: tokens x dim, contracted over the rows that count
template <int T, int NB>
__global__ __launch_bounds__(256) void ce_dw_kernel(CeParams p, CeOutput o) {
    using P = Product<T, NB, false, false, true>;
    __shared__ __attribute__((aligned(16))) char lds[P::LDS];
    const ProductPlace at = product_place(p.shape);
    f32x16 acc[NB][NB];
    P::run(p.shape, p.w, p.h, at, p.mask, lds, acc);
    ce_store<T, NB, P>(p, o, at, acc);
}

// the shares added in order, eight elements a thread
template <int T>
__global__ __launch_bounds__(256) void ce_combine_kernel(CeParams p, CeOutput o, char *out) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8, all = (int64_t)o.rows * p.dim;
    if (at >= all) return;
    const int row = (int)(at / p.dim);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const float *src = o.parts + at;
#pragma unroll 4
    for (int x = 0; x < p.shape.shares; ++x, src += all) {
        float v[8];
        ld_some8<kF32>(reinterpret_cast<const char *>(src), 8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] += v[i];
    }
    const float factor = ce_factor<T>(p);
    const bool counts = !o.masked || (p.mask[row >> 5] >> (row & 31) & 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = counts ? s[i] * factor : 0.f;
    st_some8<T>(out + at * 2, 8, s);
}

}  // namespace sa2
