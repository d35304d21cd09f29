// The residual's addition and the root-mean-square norm behind it, forward, backward, and with an output in e4m3.
//
//   t = round(x + r)      y = round(t rstd w)      rstd = (mean(t^2) + eps)^-1/2
//   dt = rstd (dy w - t^ mean(dy w t^)) + dt_up     dw = sum over rows of dy t^         t^ = t rstd
//
// What is normalised is the rounded sum, the one that the next layer adds to.  A row is held by L lanes (part of a wave, a wave, or a
// workgroup) in registers between its two uses, so every tensor crosses the memory bus once; bound by bytes.  A lane's pieces of eight channels are next to its
// neighbours', so that a load or store of a wave is 1 KiB in a run; the last piece of a row that ends inside one overlaps the piece in front instead of
// going element by element (65752 x 255 in bf16, forward and backward: 151 -> 66 us).  The weight's gradient is summed in registers over the rows that a lane
// takes, over the lanes of a wave, its workgroup's waves and then the workgroups, in a fixed order (rows one after another through LDS: 65536 x 32 38 us, now 16).
//
// Measured (bf16, a copy runs at 4.9 TB/s): 16384 x 512 forward 13.3 us (5.0 TB/s), backward 15.8 and 3.4 for the weight's; 8192 x 4096 in e4m3 by groups of 128 42 us; a token of 512
// channels 2.2 us.  What is left: the backward's second launch (3 to 5 us).
#pragma once

#include "sa2_elements.hpp"

namespace sa2 {

struct NormParams {
    const char *x, *r, *w;           // r: NULL without a residual; w: NULL for ones
    char *y, *t;                     // contiguous; t: NULL without a residual
    float *rstd;                     // [rows] or NULL
    int64_t rows, x_row, r_row;      // bytes between rows
    int dim, w_type;
    float eps;
    // 8-bit output: y in e4m3, `groups` scales per row
    float *scales;
    int group_lanes, groups;         // lanes that hold a group of channels (0: the row is one)
    // backward
    const char *dy, *dt;             // dt: gradient of t from behind, or NULL
    char *dx, *dr;                   // dr: NULL where dx is the residual's gradient too
    int64_t dy_row, dt_row;
    float *dw_parts;                 // [workgroups][dim], or NULL
};

// L lanes a row, E pieces of eight channels a lane: lane l holds the pieces l, l + L, ...
template <int L, int E>
struct NormShape {
    static constexpr int THREADS = L > 256 ? L : 256;
    static constexpr int ROWS = THREADS / L;         // rows of a workgroup
    static constexpr int MOST = L * E * 8;           // channels
};

// a value reduced over the lanes of a row; `scratch`: one word per wave, used where the row is a workgroup's
template <int L>
__device__ __forceinline__ float row_sum(float x, float *scratch) {
    if constexpr (L <= 64) return lanes_sum<L>(x);
    x = lanes_sum<64>(x);
    __syncthreads();                                 // (the last sum has been read)
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) s += scratch[i];
    return s;
}
template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t x, float *scratch) {
    if constexpr (L <= 64) return lanes_max<L>(x);
    x = lanes_max<64>(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = as_f32(x);
    __syncthreads();
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) s = max(s, as_u32(scratch[i]));
    return s;
}

// Eight channels of a row from `at` on, of which the first `skip` are the piece's before (the last piece of a row whose channels are no multiple of eight ends with
// the row: whole accesses, and what is stored twice is the same); `count` (1 to 8; 0: none) are there from `at` on if the row has fewer than eight.
struct NormPiece {
    int at, skip, count;
    __device__ NormPiece(int index, int dim, bool here) {
        const int d = index * 8;
        at = dim >= 8 ? min(d, dim - 8) : d;
        skip = d - at;
        count = here && d < dim ? (dim >= 8 ? 8 : dim) : 0;
    }
};

// e4m3 of eight values for a store of `count` from the `skip`-th on
__device__ __forceinline__ void store_e4m3(char *y, const NormPiece &piece, const float (&t)[8], float inv) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = t[i] * inv;
    const uint32_t a = pack_e4m3(q[0], q[1], q[2], q[3]), b = pack_e4m3(q[4], q[5], q[6], q[7]);
    // (those of the piece before may have another scale)
    if (piece.skip == 0 && piece.count == 8) *reinterpret_cast<u32x2_any *>(y) = (u32x2){a, b};
    else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i >= piece.skip && i < piece.count) y[i] = (char)((i < 4 ? a : b) >> (8 * (i & 3)));
}
__device__ __forceinline__ float e4m3_scale(uint32_t most) { return most > 0x7f800000u ? as_f32(most) : fmaxf(as_f32(most) * (float)(1 / 448.), 0x1p-126f); }

template <int TX, int TR, int L, int E, bool EIGHT>
__global__ __launch_bounds__((NormShape<L, E>::THREADS)) void norm_kernel(NormParams p) {
    using S = NormShape<L, E>;
    __shared__ float scratch[S::THREADS / 64];
    const int64_t row = (int64_t)blockIdx.x * S::ROWS + threadIdx.x / L;
    const int l = threadIdx.x % L;
    const bool here = row < p.rows;                  // (the others go along: the reductions are the whole wave's)
    const char *x = p.x + row * p.x_row, *r = p.r + row * p.r_row;
    float t[E][8];
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const NormPiece piece(e * L + l, p.dim, here);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[e][i] = 0.f;
        if (piece.count > 0) {
            ld_some8<TX>(x + (int64_t)piece.at * element_size<TX>, piece.count, t[e]);
            if (p.r) {
                float add[8];
                ld_some8<TR>(r + (int64_t)piece.at * element_size<TR>, piece.count, add);
#pragma unroll
                for (int i = 0; i < 8; ++i) t[e][i] = rounded<TR>(t[e][i] + add[i]);
                st_some8<TR>(p.t + (row * p.dim + piece.at) * element_size<TR>, piece.count, t[e]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += i >= piece.skip ? t[e][i] * t[e][i] : 0.f;
    }
    const float rstd = rsqrtf(row_sum<L>(sum, scratch) / (float)p.dim + p.eps);
    if (p.rstd && here && l == 0) p.rstd[row] = rstd;
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const NormPiece piece(e * L + l, p.dim, here);
        float w[8];
        if (piece.count > 0 && p.w) ld_some8(p.w_type, p.w + (int64_t)piece.at * (p.w_type == kF32 ? 4 : 2), piece.count, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[e][i] = piece.count > 0 ? (p.w ? t[e][i] * rstd * w[i] : t[e][i] * rstd) : 0.f;
        if constexpr (EIGHT) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i >= piece.skip && i < piece.count) m = max(m, magnitude(t[e][i]));
            if (p.group_lanes) {
                // (groups are aligned lanes of one piece index)
                for (int off = p.group_lanes / 2; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
                const float scale = e4m3_scale(m);
                if (piece.count > 0) {
                    if (l % p.group_lanes == 0) p.scales[row * p.groups + (e * L + l) / p.group_lanes] = scale;
                    store_e4m3(p.y + row * p.dim + piece.at, piece, t[e], 1.f / scale);
                }
            }
            most = max(most, m);
        } else {
            if (piece.count > 0) st_some8<TX>(p.y + (row * p.dim + piece.at) * element_size<TX>, piece.count, t[e]);
        }
    }
    if constexpr (EIGHT) {
        if (p.group_lanes) return;
        const float scale = e4m3_scale(row_max<L>(most, scratch)), inv = 1.f / scale;
        if (here && l == 0) p.scales[row] = scale;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const NormPiece piece(e * L + l, p.dim, here);
            if (piece.count > 0) store_e4m3(p.y + row * p.dim + piece.at, piece, t[e], inv);
        }
    }
}

// Rows strided over the workgroups, which add up their share of dw in registers and leave it in dw_parts.
template <int TX, int TR, int L, int E>
__global__ __launch_bounds__((NormShape<L, E>::THREADS)) void norm_bwd_kernel(NormParams p) {
    using S = NormShape<L, E>;
    constexpr int WAVES = S::THREADS / 64;
    __shared__ float scratch[WAVES];
    __shared__ __attribute__((aligned(16))) float sums[S::ROWS > 1 ? WAVES : 1][S::ROWS > 1 ? S::MOST : 4];
    const int l = threadIdx.x % L;
    float dw[E][8];
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[e][i] = 0.f;
    for (int64_t row0 = (int64_t)blockIdx.x * S::ROWS; row0 < p.rows; row0 += (int64_t)gridDim.x * S::ROWS) {
        const int64_t row = row0 + threadIdx.x / L;
        const bool here = row < p.rows;
        const float rstd = here ? p.rstd[row] : 0.f;
        float t[E][8], g[E][8], inner = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const NormPiece piece(e * L + l, p.dim, here);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[e][i] = g[e][i] = 0.f;
            if (piece.count <= 0) continue;
            float w[8];
            ld_some8<TR>(p.x + row * p.x_row + (int64_t)piece.at * element_size<TR>, piece.count, t[e]);
            ld_some8<TX>(p.dy + row * p.dy_row + (int64_t)piece.at * element_size<TX>, piece.count, g[e]);
            if (p.w) ld_some8(p.w_type, p.w + (int64_t)piece.at * (p.w_type == kF32 ? 4 : 2), piece.count, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t[e][i] *= rstd;
                dw[e][i] += g[e][i] * t[e][i];
                if (p.w) g[e][i] *= w[i];
                inner += i >= piece.skip ? g[e][i] * t[e][i] : 0.f;
            }
        }
        inner = row_sum<L>(inner, scratch) / (float)p.dim;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const NormPiece piece(e * L + l, p.dim, here);
            if (piece.count <= 0) continue;
            float up[8];
            if (p.dt) ld_some8<TR>(p.dt + row * p.dt_row + (int64_t)piece.at * element_size<TR>, piece.count, up);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                g[e][i] = rstd * (g[e][i] - t[e][i] * inner);
                if (p.dt) g[e][i] += up[i];
            }
            if (p.dx) st_some8<TX>(p.dx + (row * p.dim + piece.at) * element_size<TX>, piece.count, g[e]);
            if (p.dr) st_some8<TR>(p.dr + (row * p.dim + piece.at) * element_size<TR>, piece.count, g[e]);
        }
    }
    if (!p.dw_parts) return;
    if constexpr (S::ROWS > 1) {
        // the rows of a wave in its lanes, then the waves
#pragma unroll
        for (int off = L; off < 64; off *= 2)
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < 8; ++i) dw[e][i] += __shfl_xor(dw[e][i], off, 64);
        float *const mine = sums[threadIdx.x / 64];
        if ((threadIdx.x & 63) < L)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const NormPiece piece(e * L + l, p.dim, true);
                if (piece.count == 8 && piece.skip == 0) {
                    *reinterpret_cast<float4 *>(mine + piece.at) = make_float4(dw[e][0], dw[e][1], dw[e][2], dw[e][3]);
                    *reinterpret_cast<float4 *>(mine + piece.at + 4) = make_float4(dw[e][4], dw[e][5], dw[e][6], dw[e][7]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i >= piece.skip && i < piece.count) mine[piece.at + i] = dw[e][i];
                }
            }
        __syncthreads();
        for (int d = threadIdx.x; d < p.dim; d += S::THREADS) {
            float s = sums[0][d];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) s += sums[w][d];
            p.dw_parts[(int64_t)blockIdx.x * p.dim + d] = s;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const NormPiece piece(e * L + l, p.dim, true);
            float *to = p.dw_parts + (int64_t)blockIdx.x * p.dim + piece.at;
            if (piece.count == 8 && piece.skip == 0) {
                st_some8<kF32>(reinterpret_cast<char *>(to), 8, dw[e]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i >= piece.skip && i < piece.count) to[i] = dw[e][i];
            }
        }
    }
}

// dw = sum of the parts in a fixed order: 32 columns a workgroup, every 32nd part a row of threads
static __global__ __launch_bounds__(1024) void norm_dw_kernel(const float *parts, int count, int dim, int type, char *dw) {
    __shared__ float sums[32][33];
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5, d = blockIdx.x * 32 + c;
    float s = 0.f;
    if (d < dim)
#pragma unroll 8
        for (int i = r; i < count; i += 32) s += parts[(int64_t)i * dim + d];
    sums[r][c] = s;
    __syncthreads();
    if (r == 0 && d < dim) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += sums[i][c];
        if (type == kF32) put_element<kF32>(dw + 4 * (int64_t)d, s);
        else if (type == kF16) put_element<kF16>(dw + 2 * (int64_t)d, s);
        else put_element<kBf16>(dw + 2 * (int64_t)d, s);
    }
}

}  // namespace sa2
