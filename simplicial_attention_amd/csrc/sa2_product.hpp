// Tiles of a matrix product for gfx950: out[l][r] = sum over k of L(l, k) R(r, k), bf16 or fp16 operands, fp32 sums, what becomes of them is the caller's.
//
// Each operand is in memory as rows of k (ROW: k is the fast index) or as rows along l or r (k is the slow index: read transposed out of
// LDS).  A workgroup of four waves owns 64 NL x 64 NR results, a wave a quarter of them as NL x NR blocks of 32 x 32; k goes by in
// steps of 32, of which a ring of three or four is in LDS (direct loads, two or three steps ahead), one barrier a step.  The fragments of the next half step
// are read while the products of the present one run.
//
// Bound by the matrix unit and the power that it draws: 8192 x 16384 results over 2048 (256 x 256 tiles) run at 1.1 to 1.27 PFLOP/s with the unit busy 60 to 68 % of the clocks at 1.7 GHz,
// and neither a ring of five, nor another place of the barrier, nor loads two workgroups deep changes the time by more than 2 %.  Launches of fewer
// workgroups than CUs take 0.24 to 0.31 us a step of 128 x 128, which is the rate at which one CU gets rows that are not in its L2 (40 to 67 bytes a ns, from memory 20 to 40, however far ahead
// the loads run: fragments read a whole step ahead and loads eight steps ahead leave it as it is).  Rows that
// are not 64 bytes apart have their lines fetched twice (256 x 256: 11595 x 7910 over 2032 478 us, over 2048 387).
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

    // chunk i of the wave, of the step that begins at p; `lds`: the tile's place
    __device__ __forceinline__ void issue(int i, const char *p, uint32_t lds, int wave) const { load_to_lds16(p, off[i], uniform((int)(lds + 1024 * (wave + 4 * i)))); }
    // the same with zeros for k whose bit is clear
    __device__ __forceinline__ void issue_some(int i, const char *p, uint32_t lds, int wave, uint32_t bits) const {
        const bool ok = bits >> (ROW ? k_of : k_of + 16 * (i & 1)) & 1;
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
// Grid index -> item such that every XCD (which gets each eighth workgroup) walks items next to each other, whatever their number.
__device__ __forceinline__ int xcd_run(int wg, int total) {
    const int x = wg % 8, each = total / 8;
    return x * each + min(x, total % 8) + wg / 8;
}
// Consecutive workgroups of an XCD take eight l tiles by as many r tiles as there are, l first: what they read at a time fits its L2.
__device__ __forceinline__ ProductPlace product_place(const ProductShape &s, int wg, int total) {
    const int item = xcd_run(wg, total);
    const int per_share = s.tiles_r * s.tiles_l, share = uniform(item / per_share), at = item - share * per_share;
    const int group = uniform(at / (8 * s.tiles_r)), rest = at - group * 8 * s.tiles_r;
    const int wide = min(8, s.tiles_l - 8 * group);
    const int r = uniform(rest / wide);
    return {r, 8 * group + rest - r * wide, share};
}

constexpr int kProductMostSteps = 2048;       // of a share, where k has a mask

template <int T, int NL, int NR, bool R_ROW, bool L_ROW, bool MASKED>
struct Product {
    static constexpr int TILE_L = 64 * NL, TILE_R = 64 * NR;
    static constexpr int RING = NL != NR ? 3 : 4;            // (two workgroups of 128 x 256 on a CU)
    static constexpr int AHEAD = RING - 1;                   // steps that the loads run ahead
    static constexpr int STAGE = (TILE_L + TILE_R) * 64;
    static constexpr int LDS = RING * STAGE + (MASKED ? kProductMostSteps * 4 : 0);
    using R = ProductSide<R_ROW, TILE_R>;
    using L = ProductSide<L_ROW, TILE_L>;
    static constexpr int LOADS = R::CHUNKS + L::CHUNKS;      // of a wave and step

    // acc[l block][r block] of this wave, whose blocks begin at NR (wave & 1) on the r side and NL (wave >> 1) on the l side
    static __device__ __forceinline__ void run(const ProductShape &shape, const ProductOperand &ro, const ProductOperand &lo, const ProductPlace &at, const uint32_t *mask, char *lds,
                                               f32x16 (&acc)[NL][NR]) {
        const int lane = threadIdx.x & 63, wave = wave_index();
        const R r(ro, at.tile_r * TILE_R, lane, wave);
        const L l(lo, at.tile_l * TILE_L, lane, wave);
        const int t0 = at.share * shape.share_steps, all = (shape.k + 31) / 32;
        const int nt = min(shape.share_steps, all - t0);
        if constexpr (MASKED) {
            uint32_t *bits = reinterpret_cast<uint32_t *>(lds + RING * STAGE);
            for (int i = threadIdx.x; i < nt; i += 256) bits[i] = mask[t0 + i];
            __syncthreads();
        }
        // Steps whose k do not all count: those with a mask, or the last one of k where it is not whole (pieces of eight k: what a piece holds beyond k is zero)
        const uint32_t last = 0xffffffffu >> (32 * all - shape.k);
        if (MASKED || (t0 + nt == all && last != 0xffffffffu)) steps<true>(r, l, t0, nt, t0 + nt == all ? last : 0xffffffffu, lds, acc);
        else steps<false>(r, l, t0, nt, 0xffffffffu, lds, acc);
    }

    // `last`: bits of the k of the last step that count
    template <bool SOME>
    static __device__ __forceinline__ void steps(const R &r, const L &l, int t0, int nt, uint32_t last, char *lds, f32x16 (&acc)[NL][NR]) {
        const int wave = wave_index();
        const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
        [[maybe_unused]] const uint32_t *bits = reinterpret_cast<const uint32_t *>(lds + RING * STAGE);
#pragma unroll
        for (int a = 0; a < NL; ++a)
#pragma unroll
            for (int b = 0; b < NR; ++b) acc[a][b] = zero16();
        if (nt <= 0) return;
        const char *pr = r.base + t0 * r.advance, *pl = l.base + t0 * l.advance;      // of the step that is loaded next
        uint32_t next_bits = MASKED ? bits[0] : nt == 1 ? last : 0xffffffffu;
        auto load_one = [&](uint32_t to, auto i) {
            if constexpr (i.value < R::CHUNKS) {
                if constexpr (SOME) r.issue_some(i.value, pr, to, wave, next_bits);
                else r.issue(i.value, pr, to, wave);
            } else {
                if constexpr (SOME) l.issue_some(i.value - R::CHUNKS, pl, to + R::BYTES, wave, next_bits);
                else l.issue(i.value - R::CHUNKS, pl, to + R::BYTES, wave);
            }
        };
        // after step t has been issued: the next one, or behind the last step that one again (into a place that nobody reads; so every step is alike)
        auto go_on = [&](int t) {
            const bool more = t + 1 < nt;
            pr += more ? r.advance : 0;
            pl += more ? l.advance : 0;
            if constexpr (MASKED) next_bits = bits[min(t + 1, nt - 1)];
            else if constexpr (SOME) next_bits = t + 1 >= nt - 1 ? last : 0xffffffffu;
        };
#pragma unroll
        for (int t = 0; t < AHEAD; ++t) {
            static_for<0, LOADS>([&](auto i) { load_one(lds0 + t * STAGE, i); });
            go_on(t);
        }
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((AHEAD - 1) * LOADS) : "memory");
        u32x4 fr[2][NR], fl[2][NL];
        const int br = NR * (wave & 1), bl = NL * (wave >> 1);
        using Zero = std::integral_constant<int, 0>;
        using One = std::integral_constant<int, 1>;
        constexpr int N = NL * NR, READS = NL + NR, FIRST = N / 4, PER = (READS + N - FIRST - 1) / (N - FIRST);
        static_assert(NR >= NL && READS <= N && LOADS <= N, "one of each in the shadow of a product");
        auto read_one = [&](const char *tile, auto half, auto i) {
            // (by turns, as the products take them)
            if constexpr (i.value >= 2 * NL) fr[half.value][i.value - NL] = r.fragment(tile, half.value, br + i.value - NL);
            else if constexpr (i.value % 2 == 0) fr[half.value][i.value / 2] = r.fragment(tile, half.value, br + i.value / 2);
            else fl[half.value][i.value / 2] = l.fragment(tile + R::BYTES, half.value, bl + i.value / 2);
        };
        auto multiply_one = [&](auto half, auto i) {
            constexpr int a = i.value / NR, b = i.value % NR;
            acc[a][b] = mfma_of<T>(fr[half.value][b], fl[half.value][a], acc[a][b]);
        };
        static_for<0, READS>([&](auto i) { read_one(lds, Zero{}, i); });
        // In the order in which it is written: a product takes 32 clocks of the matrix unit, in whose shadow one read of the next fragments or one direct load is
        // issued; the barrier stands behind the first products of the second half.
        for (int t = 0; t < nt; ++t) {
            const char *now = lds + (t % RING) * STAGE, *next = lds + ((t + 1) % RING) * STAGE;
            const uint32_t to = lds0 + ((t + AHEAD) % RING) * STAGE;
            static_for<0, N>([&](auto i) {
                multiply_one(Zero{}, i);
                if constexpr (i.value < READS) read_one(now, One{}, i);
                if constexpr (i.value >= N - LOADS) load_one(to, std::integral_constant<int, i.value - (N - LOADS)>{});
                __builtin_amdgcn_sched_barrier(0);
            });
            static_for<0, FIRST>([&](auto i) { multiply_one(One{}, i); });
            __builtin_amdgcn_sched_barrier(0);
            // step t + 1 is in (those behind it are under way), and this wave has read all of step t
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((AHEAD - 1) * LOADS) : "memory");
            go_on(t + AHEAD);
            static_for<FIRST, N>([&](auto i) {
                multiply_one(One{}, i);
                constexpr int at = (i.value - FIRST) * PER;
                static_for<0, PER>([&](auto j) {
                    if constexpr (at + j.value < READS) read_one(next, Zero{}, std::integral_constant<int, at + j.value>{});
                });
                __builtin_amdgcn_sched_barrier(0);
            });
        }
        wait_loads<0>();      // (the last loads may still be on their way into LDS)
    }

};

// the blocks of a row of tiles, from here on (the compiler would read those of all rows out of the accumulation registers at once, and spill)
template <int NB>
__device__ __forceinline__ void take(f32x16 (&acc)[NB]) {
#pragma unroll
    for (int b = 0; b < NB; ++b) pin_acc(acc[b]);
}

// Results of a wave on their way to memory: a block of 32 rows goes through LDS, its 16-byte pieces XORed with the row, so that a store writes whole rows of
// the wave's 32 NB columns.  (From the registers it would be 16 bytes of 64 rows: an epilogue of 8192 x 16384 results of two bytes took 190 us of 628.)
// TO: kF32, or the type that the results are rounded to.
template <int TO, int NB>
struct ProductRows {
    static constexpr int PIECES = 2 * NB * element_size<TO>;      // of a row
    static constexpr int BYTES = 4 * 32 * PIECES * 16;            // of the four waves
    static constexpr int EACH = 16 / element_size<TO>;            // results of a piece
    char *block, *mine;
    int row, lane;

    __device__ ProductRows(char *lds) {
        lane = threadIdx.x & 63;
        block = lds + wave_index() * 32 * PIECES * 16;
        row = dmap_row(lane & 31);
        mine = block + row * PIECES * 16;
    }
    static __device__ int place(int row, int piece) { return 16 * (piece ^ (row & (PIECES < 16 ? PIECES - 1 : 15))); }
    // the lane's run of block b, times `factor`
    __device__ __forceinline__ void put(int b, const f32x16 &x, float factor = 1.f) const {
        const int first = PIECES / NB * b + PIECES / NB / 2 * (lane >> 5);
        if constexpr (TO == kF32) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4 *>(mine + place(row, first + q)) = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = x[8 * q + i] * factor;
                *reinterpret_cast<u32x4 *>(mine + place(row, first + q)) = pack8<TO>(v);
            }
        }
    }
    // f(row of the block, first column of the wave's, the piece) for every piece that the lane stores
    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < PIECES / 2; ++i) {
            const int r = 64 / PIECES * i + lane / PIECES, piece = lane % PIECES;
            f(r, EACH * piece, ld_lds16(block + r * PIECES * 16 + place(r, piece)));
        }
        __builtin_amdgcn_wave_barrier();
    }
};

}  // namespace sa2
