// Tiles of a matrix product for gfx950: out[l][r] = sum over k of L(l, k) R(r, k), bf16 or fp16 operands, fp32 sums, what becomes of them is the caller's.
//
// Each operand is in memory as rows of k (ROW: k is the fast index) or as rows along l or r (k is the slow index: read transposed out of
// LDS).  A workgroup of four waves owns TILE x TILE results, a wave a quarter of them as NB x NB blocks of 32 x 32; k goes by in
// steps of 32, of which a ring of four is under way (direct-to-LDS loads, three steps ahead), one barrier a step.  The fragments of the next half step
// are read while the products of the present one run.
//
// Registers: column c of an MFMA result is row dmap_row(c) of the l side, register r of half hf column 16 hf + r of the r side, so a
// lane holds runs of 16 consecutive results of one row.
#pragma once

#include "sa2_elements.hpp"
#include "sa2_lds.hpp"

namespace sa2 {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int T>
__device__ __forceinline__ f32x16 mfma_of(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (T == kF16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return mfma32(a, b, c);
}

// one direct-to-LDS load from addresses of the lanes' own
__device__ __forceinline__ void load_to_lds16_from(const char *p, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds_addr) : "memory");
}

static __device__ __attribute__((aligned(16))) const uint32_t kZeroPiece[4] = {0, 0, 0, 0};

struct ProductOperand {
    const char *ptr;
    int64_t row;                  // bytes between its rows
    int extent;                   // l or r indices that there are (a multiple of 8 where k is the slow index)
};

// A TILE x 32 tile of one operand in chunks of 1 KiB, chunk w, w + 4, ... moved by wave w.
//   ROW: a chunk is 16 rows of 64 bytes; the 16-byte pieces of a row lie XOR-swizzled, so that the rows of a fragment read (permuted by
//        dmap_row) hit all banks;
//   else: four k of 128 columns, [32 columns][k][64 bytes].
template <bool ROW, int TILE>
struct ProductSide {
    static constexpr int CHUNKS = TILE / 64;        // of a wave
    static constexpr int BYTES = TILE * 64;
    const char *base;
    int64_t advance;                                // bytes of a step
    uint32_t off[CHUNKS];
    int k_of;                                       // ROW: first k of the lane's piece; else the k of the lane's row in chunk 0 of the wave (chunk i: + 16 (i & 1))
    int frag;

    __device__ static int swizzle(int row) {
        const int u = (row >> 2) & 7;
        return (u >> 2) | ((u & 1) << 1);
    }

    __device__ ProductSide(const ProductOperand &o, int start, int lane, int wave) {
        if constexpr (ROW) {
            const int origin = min(start, o.extent - 1);           // (indices beyond the last one read that one)
            base = o.ptr + (int64_t)origin * o.row;
            advance = 64;
            const int row0 = 16 * wave + (lane >> 2), piece = (lane & 3) ^ swizzle(row0);      // (the swizzle repeats every 32 rows)
            k_of = 8 * piece;
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) off[i] = (uint32_t)(min(start + row0 + 64 * i, o.extent - 1) - origin) * (uint32_t)o.row + 16 * piece;
            const int row = dmap_row(lane & 31);
            frag = (row >> 4) * 1024 + (row & 15) * 64 + 16 * ((lane >> 5) ^ swizzle(row));
        } else {
            const int origin = min(start, o.extent - 8);
            base = o.ptr + 2 * (int64_t)origin;
            advance = 32 * o.row;
            k_of = 4 * wave + ((lane >> 2) & 3);
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                const int col = min(start + 128 * (i >> 1) + 32 * (lane >> 4) + 8 * (lane & 3), o.extent - 8) - origin;
                off[i] = (uint32_t)(k_of + 16 * (i & 1)) * (uint32_t)o.row + 2 * col;
            }
            frag = 2048 * (lane >> 5) + 64 * ((lane & 15) >> 2) + 2 * (16 * (lane & 1) + 8 * ((lane >> 4) & 1) + 4 * ((lane & 3) >> 1));
        }
    }

    // chunk i of the wave, of step t; `lds`: the tile's place
    __device__ __forceinline__ void issue(int i, int t, uint32_t lds, int wave) const {
        load_to_lds16(uniform(base + t * advance), off[i], uniform((int)(lds + 1024 * (wave + 4 * i))));
    }
    // the same with zeros for k from `count` on and (not ROW) for k whose bit is clear
    __device__ __forceinline__ void issue_some(int i, int t, uint32_t lds, int wave, int count, uint32_t bits) const {
        const int k = ROW ? k_of : k_of + 16 * (i & 1);
        const char *p = base + t * advance + off[i];
        const bool ok = k < count && (ROW || (bits >> k & 1));
        load_to_lds16_from(ok ? p : reinterpret_cast<const char *>(kZeroPiece), uniform((int)(lds + 1024 * (wave + 4 * i))));
    }
    // ... of the step that begins at p, with zeros for k whose bit is clear
    __device__ __forceinline__ void issue_masked(int i, const char *p, uint32_t lds, int wave, uint32_t bits) const {
        const bool ok = bits >> (k_of + 16 * (i & 1)) & 1;
        load_to_lds16_from(ok ? p + off[i] : reinterpret_cast<const char *>(kZeroPiece), uniform((int)(lds + 1024 * (wave + 4 * i))));
    }
    // 32 indices (block b) x 16 k (half s) of the tile
    __device__ __forceinline__ u32x4 fragment(const char *tile, int s, int b) const {
        if constexpr (ROW) {
            // (piece 2 s + hf: the swizzle is an XOR of the two low bits)
            return ld_lds16(tile + 2048 * b + (frag ^ (32 * s)));
        } else {
            const char *p = tile + 8192 * (b >> 2) + 256 * (b & 3) + 4096 * s + frag;
            const u32x2 lo = lds_read_tr<32, 0>(p, 0, 0), hi = lds_read_tr<32, 0>(p + 1024, 0, 0);
            return (u32x4){lo[0], lo[1], hi[0], hi[1]};
        }
    }
};

struct ProductShape {
    int k;                                   // contracted length (a multiple of 8 where both operands are rows of k)
    int tiles_r, tiles_l;
    int shares, share_steps;                 // workgroups that divide the steps of a tile, and the steps of each
};

// what a workgroup owns: its tile and share
struct ProductPlace {
    int tile_r, tile_l, share;
};
// Consecutive workgroups of an XCD take eight l tiles by as many r tiles as there are, l first: what they read at a time fits its L2.
__device__ __forceinline__ ProductPlace product_place(const ProductShape &s) {
    const int item = xcd_contiguous(blockIdx.x, gridDim.x);
    const int per_share = s.tiles_r * s.tiles_l, share = uniform(item / per_share), at = item - share * per_share;
    const int group = uniform(at / (8 * s.tiles_r)), rest = at - group * 8 * s.tiles_r;
    const int wide = min(8, s.tiles_l - 8 * group);
    const int r = uniform(rest / wide);
    return {r, 8 * group + rest - r * wide, share};
}

constexpr int kProductMostSteps = 2048;       // of a share, where k has a mask

template <int T, int NB, bool R_ROW, bool L_ROW, bool MASKED>
struct Product {
    static constexpr int TILE = 64 * NB;
    static constexpr int RING = 4;
    static constexpr int STAGE = 2 * TILE * 64;
    static constexpr int LDS = RING * STAGE + (MASKED ? kProductMostSteps * 4 : 0);
    using R = ProductSide<R_ROW, TILE>;
    using L = ProductSide<L_ROW, TILE>;
    static constexpr int LOADS = R::CHUNKS + L::CHUNKS;      // of a wave and step

    // acc[l block][r block] of this wave, whose blocks begin at NB (wave & 1) on the r side and NB (wave >> 1) on the l side
    static __device__ __forceinline__ void run(const ProductShape &shape, const ProductOperand &ro, const ProductOperand &lo, const ProductPlace &at, const uint32_t *mask, char *lds,
                                               f32x16 (&acc)[NB][NB]) {
        const int lane = threadIdx.x & 63, wave = wave_index();
        const R r(ro, at.tile_r * TILE, lane, wave);
        const L l(lo, at.tile_l * TILE, lane, wave);
        const int t0 = at.share * shape.share_steps, all = (shape.k + 31) / 32;
        const int nt = min(shape.share_steps, all - t0);
        const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
        uint32_t *bits = reinterpret_cast<uint32_t *>(lds + RING * STAGE);
        if constexpr (MASKED) {
            for (int i = threadIdx.x; i < nt; i += 256) bits[i] = mask[t0 + i];
            __syncthreads();
        }
        const int rest = shape.k - 32 * (all - 1);          // k of the last step
        auto issue = [&](int t) {
            const uint32_t to = lds0 + (t % RING) * STAGE;
            if (MASKED || (t0 + t == all - 1 && rest != 32)) {
                const int count = t0 + t == all - 1 ? rest : 32;
                uint32_t b = 0xffffffffu;
                if constexpr (MASKED) b = bits[t];
#pragma unroll
                for (int i = 0; i < R::CHUNKS; ++i) r.issue_some(i, t0 + t, to, wave, count, b);
#pragma unroll
                for (int i = 0; i < L::CHUNKS; ++i) l.issue_some(i, t0 + t, to + R::BYTES, wave, count, b);
            } else {
#pragma unroll
                for (int i = 0; i < R::CHUNKS; ++i) r.issue(i, t0 + t, to, wave);
#pragma unroll
                for (int i = 0; i < L::CHUNKS; ++i) l.issue(i, t0 + t, to + R::BYTES, wave);
            }
        };
#pragma unroll
        for (int a = 0; a < NB; ++a)
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[a][b] = zero16();
        if (nt <= 0) return;
        issue(0);
        if (nt > 1) issue(1);
        if (nt > 2) issue(2);
        if (nt > 2) wait_loads<2 * LOADS>();
        else if (nt > 1) wait_loads<LOADS>();
        else wait_loads<0>();
        __syncthreads();
        u32x4 fr[2][NB], fl[2][NB];
        const int br = NB * (wave & 1), bl = NB * (wave >> 1);
        auto read = [&](int t, auto s) {
            const char *tile = lds + (t % RING) * STAGE;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                fr[s.value][b] = r.fragment(tile, s.value, br + b);
                fl[s.value][b] = l.fragment(tile + R::BYTES, s.value, bl + b);
            }
        };
        auto multiply = [&](auto s) {
#pragma unroll
            for (int a = 0; a < NB; ++a)
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[a][b] = mfma_of<T>(fr[s.value][b], fl[s.value][a], acc[a][b]);
        };
        using Zero = std::integral_constant<int, 0>;
        using One = std::integral_constant<int, 1>;
        read(0, Zero{});
        int t = 0;
        // The steps in the middle, in the order they are written: a product takes 32 clocks of the matrix unit, in whose shadow one read of the next
        // fragments or one direct load is issued; the barrier stands behind the first products of the second half.
        const int full = !MASKED && rest != 32 && t0 + nt == all ? nt - 1 : nt;      // (tiles that are filled up with zeros are the other loop's)
        const char *pr = r.base + (int64_t)(t0 + 3) * r.advance, *pl = l.base + (int64_t)(t0 + 3) * l.advance;
        uint32_t b3 = 0xffffffffu;
        if constexpr (MASKED) b3 = bits[min(3, nt - 1)];
        for (; t + 3 < full; ++t) {
            const char *now = lds + (t % RING) * STAGE, *next = lds + ((t + 1) % RING) * STAGE;
            const uint32_t to = lds0 + ((t + 3) % RING) * STAGE;
            constexpr int N = NB * NB, READS = 2 * NB, FIRST = NB == 4 ? 4 : 1;
            auto read_one = [&](const char *tile, auto half, auto i) {
                if constexpr (i.value % 2 == 0) fr[half.value][i.value / 2] = r.fragment(tile, half.value, br + i.value / 2);
                else fl[half.value][i.value / 2] = l.fragment(tile + R::BYTES, half.value, bl + i.value / 2);
            };
            auto multiply_one = [&](auto half, auto i) {
                constexpr int a = i.value / NB, b = i.value % NB;
                acc[a][b] = mfma_of<T>(fr[half.value][b], fl[half.value][a], acc[a][b]);
            };
            auto load_one = [&](auto i) {
                if constexpr (i.value < R::CHUNKS) {
                    if constexpr (MASKED) r.issue_masked(i.value, pr, to, wave, b3);
                    else load_to_lds16(pr, r.off[i.value], uniform((int)(to + 1024 * (wave + 4 * i.value))));
                } else {
                    constexpr int j = i.value - R::CHUNKS;
                    if constexpr (MASKED) l.issue_masked(j, pl, to + R::BYTES, wave, b3);
                    else load_to_lds16(pl, l.off[j], uniform((int)(to + R::BYTES + 1024 * (wave + 4 * j))));
                }
            };
            static_for<0, N>([&](auto i) {
                multiply_one(Zero{}, i);
                if constexpr (i.value < READS) read_one(now, One{}, i);
                if constexpr (i.value >= N - LOADS) load_one(std::integral_constant<int, i.value - (N - LOADS)>{});
                __builtin_amdgcn_sched_barrier(0);
            });
            pr += r.advance;
            pl += l.advance;
            static_for<0, FIRST>([&](auto i) { multiply_one(One{}, i); });
            __builtin_amdgcn_sched_barrier(0);
            // step t + 1 is in (two more are under way), and this wave has read all of step t
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
            if constexpr (MASKED) b3 = bits[min(t + 4, nt - 1)];
            static_for<FIRST, N>([&](auto i) {
                multiply_one(One{}, i);
                constexpr int per = NB == 4 ? 1 : 2, at = (i.value - FIRST) * per;
                static_for<0, per>([&](auto j) {
                    if constexpr (at + j.value < READS) read_one(next, Zero{}, std::integral_constant<int, at + j.value>{});
                });
                __builtin_amdgcn_sched_barrier(0);
            });
        }
        for (; t < nt; ++t) {
            read(t, One{});
            if (t + 3 < nt) issue(t + 3);
            multiply(Zero{});
            if (t + 1 < nt) {
                if (t + 3 < nt) wait_loads<2 * LOADS>();
                else if (t + 2 < nt) wait_loads<LOADS>();
                else wait_loads<0>();
                __syncthreads();                            // step t + 1 is in, and step t has been read by all
                read(t + 1, Zero{});
            }
            multiply(One{});
        }
    }

    // f(l index, first r index of a run of 16, the run) for every run of the lane
    template <typename F>
    static __device__ __forceinline__ void each_run(const ProductPlace &at, const f32x16 (&acc)[NB][NB], F &&f) {
        const int lane = threadIdx.x & 63, wave = wave_index();
#pragma unroll
        for (int a = 0; a < NB; ++a)
#pragma unroll
            for (int b = 0; b < NB; ++b)
                f(at.tile_l * TILE + 32 * (NB * (wave >> 1) + a) + dmap_row(lane & 31), at.tile_r * TILE + 32 * (NB * (wave & 1) + b) + 16 * (lane >> 5), acc[a][b]);
    }
};

}  // namespace sa2
