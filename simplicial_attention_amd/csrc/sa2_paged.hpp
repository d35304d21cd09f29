// Attention of new tokens over a paged cache: dense causal attention and its sliding-window 2-simplicial form.
//
// A pool holds pages of `ps` rows; position x of a sequence is row x % ps of page table[x / ps].  Row t of a sequence's chunk sits at
// position p = length - count + t.  Both operators are one product pair over 32-row key tiles and 32 columns,
//     S^T = K A^T      P^T = exp2(c S^T - M)      O^T += V^T P^T        (c = scale log2(e), M the column's reference)
// and differ in what a column is:
//   dense        column = (token, query head of the group):  A = q, keys 0 .. p, the column's O is an output row
//   2-simplicial column = offset d = p - k of ONE (token, query head):  A = c q * k2[p - d] (the chain of products starts from -M), keys (p - w1, p] of the first set,
//                o = sum over columns of v2[p - d] * O, so the 32 offsets of a token share its window and one product does them all
// Softmax: the reference M of a column moves only when a tile's weights outgrow 2^60 (fp16: 2^14) on it, the first tile included
// (M starts at the lowest number), so the ordinary tile has no maximum and no rescale.  Sums and accumulators are fp32; the weights
// are rounded to the element type for the second product, as the training kernels round theirs (in two parts they would double its length; with it the error is 2.3e-3 of the
// result in bf16 and 2.9e-4 in fp16, where rounding nothing but the result gives 1.7e-3 and 2.1e-4); c q * k2 enters the first in two parts of that type (rounded to one, its error
// would be the largest of the output's; the logits' products double).  Where fp16 does not hold a product, both parts of its column are divided by powers of two and
// its wave walks by plain steps; what is infinite or no number stays so.
//
// Keys that are not there (beyond the walked range, missing pages) are fetched from a row of zeros and masked; a value row that a
// column does not attend never reaches it, whatever it holds (0 * NaN is not 0: see PagedWave::values).
#pragma once

#include "sa2_common.hpp"
#include "sa2_lds.hpp"

namespace sa2 {

struct ElemBf16 {
    static constexpr float kBig = 1.152921504606846976e18f;      // 2^60
    static constexpr uint32_t kExp = 0x7f80u;
    static constexpr bool kNarrow = false;                       // products of two numbers are in the type's range
    static constexpr float kMost = 3.3895313892515355e38f;       // the largest number
    static __device__ __forceinline__ float lo(uint32_t w) { return bf16_lo(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return bf16_hi(w); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) { return mfma32(a, b, c); }
    static __device__ __forceinline__ void mfma_in_place(f32x16 &acc, u32x4 a, u32x4 b) {
        asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(a), "v"(b));
    }
};

struct ElemF16 {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    static constexpr float kBig = 16384.f;                       // 2^14: weights stay below the largest fp16 number
    static constexpr uint32_t kExp = 0x7c00u;
    static constexpr bool kNarrow = true;
    static constexpr float kMost = 65504.f;
    static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
    static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        f16x2 v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void mfma_in_place(f32x16 &acc, u32x4 a, u32x4 b) {
        asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(acc) : "v"(a), "v"(b));
    }
};
// mfma_in_place: the accumulator's registers are the result's.  (Left to itself the compiler gives a product of the loop below other registers than its
// addend, and copies 16 of them per product and step.)  Written as assembly, so the wait states it needs are this code's business: two
// behind a VALU write of an operand are in it, and PagedWave::settle stands behind a run of them.  The compiler must not move an accumulator between two of them: kernels that use it are held to ordinary registers
// (-amdgpu-mfma-vgpr-form, two waves per SIMD or more; tests/test_in_place_products.py reads the assembly).

struct PagedPool {
    const char *ptr;
    int64_t sp, sr, sh;       // bytes between pages, rows of a page, heads
};

// division by a number that the host knows as a multiplication (dividends below 2^31)
struct Divisor {
    uint32_t by, mul, shift;
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (uint32_t)(((uint64_t)x * mul) >> shift); }
};

struct PagedParams {
    const char *q;
    int64_t q_sb, q_sn, q_sh;
    char *o;
    int64_t o_sb, o_sn, o_sh;
    PagedPool k1, v1, k2, v2;                 // (k2, v2: 2-simplicial form only)
    const int32_t *tables, *lengths, *counts; // (counts nullptr: n for every sequence)
    int64_t t_sb;
    Divisor div, group, heads, seqs, parts;   // by the page size, G, HK, B HK, splits * dblocks
    int pages, width;                         // pages of a pool, entries of a table
    int B, n, H, HK, G;
    int dq, dp;                               // channels of q and the output, and of a pool's row (multiples of 8)
    int w1, w2;
    float scale_log2e;
    int unit_columns;                         // 2-simplicial, packed: columns of a (token, head)
    int row_tiles;                            // workgroups (per sequence and key/value head) that the rows take
    int splits, dblocks;                      // shares of the keys; blocks of 32 offsets
    int even;                                 // every sequence has `splits` shares; else see PagedShares
    // partial results where splits * dblocks > 1: fp32 [place][n H][D] and [place][n H] (reference, sum), B places per share and block of offsets
    float *part_o;
    float2 *part_ml;
    int2 *shares;                             // (not even) of a sequence: its first place, their number
};

constexpr float kNoRef = -3.402823466e38f;    // reference of a column that has met no key yet
// Beyond it (log2 units) a reference is a logit rounded so far that what is formed relative to it, by a chain of products or a fused multiplication, shows it: logits are
// formed and rounded as the reference was, and it is subtracted then
constexpr float kFarRef = 1048576.f;
// c times a logit, rounded: not fused into what is subtracted from it
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}
__device__ __attribute__((aligned(16))) uint32_t g_paged_zero_row[128];

// One direct-to-LDS load of 16 bytes per lane from addresses of its own (load_to_lds16 with 64-bit lane addresses)
__device__ __forceinline__ void load_to_lds16_from(const char *addr, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(addr), "s"(lds_addr) : "memory");
}
// LDS reads issued before have left the memory (a direct load may overwrite what they read)
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// ---- what a workgroup knows about its sequence
struct PagedSeq {
    const int32_t *table;
    int first, count;        // position of row 0 of the chunk (negative: rows before the sequence attend to nothing), rows that are there
    int reach;               // positions that the table can name
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams &p, int b) {
    PagedSeq s;
    s.table = p.tables + b * p.t_sb;
    const int length = p.lengths[b];
    int count = p.counts ? p.counts[b] : p.n;
    count = count < 0 ? 0 : (count > p.n ? p.n : count);
    s.first = (length < 0 ? 0 : length) - count;
    s.count = count;
    const int64_t reach = (int64_t)p.width * p.div.by;
    s.reach = reach > 0x7fffffff ? 0x7fffffff : (int)reach;
    return s;
}
// page of a position, -1 where there is none
__device__ __forceinline__ int paged_page(const PagedParams &p, const PagedSeq &s, int x) {
    if (x < 0 || x >= s.reach) return -1;
    const int id = s.table[p.div((uint32_t)x)];
    return (unsigned)id < (unsigned)p.pages ? id : -1;
}
// 2-simplicial: first key of a position (of position 0, for one in front of the sequence: windows may be as large as an int)
__device__ __forceinline__ int first_key_of(const PagedParams &p, int pos) { return max(0, max(0, pos) - p.w1 + 1); }
__device__ __forceinline__ const char *paged_row(const PagedPool &pool, int page, int row) {
    return pool.ptr + (int64_t)page * pool.sp + (int64_t)row * pool.sr;
}

// Shares of the keys of sequences of different lengths (up to 64 of them): the B splits places that even shares would take go to the sequences as their lengths
// ask, so that the longest share is as short as it gets.  Every wave of the walk forms them from the lengths, a lane for each sequence.  Measured, even shares
// and these: 1131 tokens of four sequences, 4 heads on 2 of 128 channels, up to 17739 rows of different lengths 177 and 119 us, all of 17739 rows 181 and 184; 256 tokens of eight
// sequences, 8 heads on 2 of 128 channels, up to 8192 rows 71 and 55, all of 8192 rows 83 and 85.
struct PagedShares {
    PagedSeq s;
    int count, behind;       // (of the lane's sequence) shares; places up to its last
    template <typename OP>
    static __device__ __forceinline__ int scan(int x, OP op) {
        x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));          // the row's lanes 1, 2, 4 and 8 before this one
        x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
        x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
        x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
        x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));          // lane 15 of a row into the next row
        x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));          // lane 31 into the upper half
        return x;
    }
    static __device__ __forceinline__ int plus(int a, int b) { return a + b; }
    static __device__ __forceinline__ int of(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
    __device__ __forceinline__ PagedShares(const PagedParams &p, int lane) {
        s = paged_seq(p, lane < p.B ? lane : 0);
        const int end = min(s.first + s.count, s.reach), tiles = lane < p.B && s.count > 0 && end > 0 ? (end + 31) / 32 : 0;
        const int most = of(scan(tiles, [](int a, int b) { return max(a, b); }), 63), all = of(scan(tiles, plus), 63);
        // (fewer than 2^20 tiles: the quotient is exact)
        auto shares = [&](int size) { return tiles > 0 ? (int)(((float)tiles - .5f) * __builtin_amdgcn_rcpf((float)size)) + 1 : 0; };
        const int places = p.B * p.splits;
        int size = max(kLeast, (most + p.splits - 1) / p.splits);      // (even shares of the longest fit)
        int least = min(size, max(kLeast, (all + places - 1) / places));
        while (least < size) {
            const int middle = (least + size) >> 1;
            if (of(scan(shares(middle), plus), 63) <= places) size = middle;
            else least = middle + 1;
        }
        count = shares(size);
        behind = scan(count, plus);
    }
    static constexpr int kLeast = 8;             // tiles of a share that are worth a place
};

// channels d0 .. d0 + 7 of a row of `channels`; zeros beyond them, and of a row that is not there.  (An address is chosen, not a branch taken: the
// pieces of a row are then in flight together)
__device__ __forceinline__ u32x4 paged_piece(const char *row, int d0, int channels, bool there) {
    const char *zero = reinterpret_cast<const char *>(g_paged_zero_row), *at = row + d0 * 2;
    asm volatile("" : "+v"(at));
    return ld_global16(there && d0 < channels ? at : zero);
}
template <class E>
__device__ __forceinline__ void paged_store8(const PagedParams &p, char *row, int d0, const float (&x)[8]) {
    if (d0 < p.dq) st_global16(row + d0 * 2, (u32x4){E::pack(x[0], x[1]), E::pack(x[2], x[3]), E::pack(x[4], x[5]), E::pack(x[6], x[7])});
}

// Products q * k2 beyond a narrow type's range: some column of the wave has them, and its two parts hold them divided by ratio * up and by up (powers of two; 1 for
// the wave's other columns)
template <bool THERE>
struct WideProducts {
    static constexpr bool wide = false;
};
template <>
struct WideProducts<true> {
    bool wide = false;
    float ratio = 1.f, up = 1.f;
};

// ---- one wave's 32 columns
// TWO: the operand of the logits in two parts (q * k2 has twice the digits of an element: rounded to one part it would double the error of
// the output, in two its error is 2^-17 of it)   IN_PLACE: value products by mfma_in_place
template <class E, int D, bool TWO, bool IN_PLACE = false>
struct PagedWave : WideProducts<TWO && E::kNarrow> {
    using RT = DmaTile<D>;
    static constexpr int KS = D / 16, DT = D / 32;
    u32x4 A[KS], A2[TWO ? KS : 1];
    f32x16 O[DT];
    float M, l;              // reference (log2 units) and this half's sum of the column's weights
    int lo, hi;              // keys the column attends (empty: lo > hi)
    int most_lo, least_hi;   // over the columns that attend to anything: keys between them need no mask

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) O[dt] = zero16();
        M = kNoRef;
        l = 0.f;
    }
    // this column's keys, and the bounds over all columns (`any`: there is one that attends to something)
    __device__ __forceinline__ void limits(int lo_, int hi_, bool on, bool any, int most_lo_, int least_hi_) {
        on = on && lo_ <= hi_;
        lo = on ? lo_ : 1;
        hi = on ? hi_ : 0;
        if (!on) M = 0.f;        // (nothing of it is used: it must not look like a column whose weights outgrow its reference)
        most_lo = any ? most_lo_ : -0x7fffffff;
        least_hi = any ? least_hi_ : 0x7fffffff;
    }

    __device__ __forceinline__ static float both_halves_max(float x) {
        auto sw = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
        return fmaxf(as_f32(sw[0]), as_f32(sw[1]));
    }

    __device__ __forceinline__ void add_product(int dt, u32x4 v, u32x4 w) {
        if constexpr (IN_PLACE) E::mfma_in_place(O[dt], v, w);
        else O[dt] = E::mfma(v, w, O[dt]);
    }
    // behind in-place products, in front of whatever else reads or copies the accumulators: 18 wait states (a product of 32 x 32 x 16 takes 8 passes, behind which the
    // compiler leaves 12 of them; the others are a margin)
    __device__ __forceinline__ void settle() {
        if constexpr (IN_PLACE) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) asm volatile("s_nop 15\n\ts_nop 1" : "+v"(O[dt]));
        }
    }

    __device__ __forceinline__ f32x16 logit(u32x4 k, int kk, f32x16 S) const {
        S = E::mfma(k, A[kk], S);
        if constexpr (TWO) S = E::mfma(k, A2[kk], S);
        return S;
    }
    // TWO: relative to `from` (c is in the operand); else the plain products
    __device__ __forceinline__ f32x16 logits(const char *k_lane, float from) const {
        if constexpr (TWO && E::kNarrow) {
            if (__builtin_expect(this->wide, 0)) {
                f32x16 S = zero16();
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) S = E::mfma(RT::row_frag(k_lane, kk), A[kk], S);
#pragma unroll
                for (int r = 0; r < 16; ++r) S[r] *= this->ratio;
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) S = E::mfma(RT::row_frag(k_lane, kk), A2[kk], S);
#pragma unroll
                for (int r = 0; r < 16; ++r) S[r] = S[r] * this->up - from;
                return S;
            }
        }
        f32x16 S = TWO ? splat16(-from) : zero16();
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) S = logit(RT::row_frag(k_lane, kk), kk, S);
        return S;
    }
    // some column has no reference yet, or a far one
    __device__ __forceinline__ bool no_near_reference() const { return wave_any(fabsf(M) > kFarRef); }

    // keys a .. z of the tile at `tile`, bit j for key tile + j
    __device__ __forceinline__ static uint32_t keys_of(int tile, int a, int z) {
        a = a - tile < 0 ? 0 : a - tile;
        z = z - tile > 31 ? 31 : z - tile;
        return a > z ? 0u : (0xffffffffu >> (31 - z)) & (0xffffffffu << a);
    }
    // S of the keys that a column does not attend; `there`: bit j of the keys that are there.  ONE: all columns attend to the same keys, so the masks of
    // the registers are formed by the scalar unit (row 8 (r / 4) + 4 hf + r % 4 of register r: a bit for either half of the lanes)
    template <bool ONE>
    __device__ __forceinline__ void mask(f32x16 &S, int tile, uint32_t there, int hf) const {
        if constexpr (ONE) {
            const uint32_t keys = there & keys_of(tile, most_lo, least_hi);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int j = 8 * (r >> 2) + (r & 3);
                const uint32_t low = (uint32_t)((int)(keys << (31 - j)) >> 31), high = (uint32_t)((int)(keys << (27 - j)) >> 31);
                const uint64_t lanes = ((uint64_t)high << 32) | low;
                S[r] = __builtin_amdgcn_inverse_ballot_w64(lanes) ? S[r] : -INFINITY;
            }
        } else {
            const int a = lo - tile - 4 * hf, z = hi - tile - 4 * hf;
            const uint32_t bits = there >> (4 * hf);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int j = 8 * (r >> 2) + (r & 3);
                S[r] = j >= a && j <= z && ((bits >> j) & 1u) ? S[r] : -INFINITY;
            }
        }
    }

    // weights of a tile, packed, and their sum; false (in every lane) if some column's outgrow its reference.  (TWO: logits relative to the reference; else SCALED
    // ones in log2 units, or products where every reference is near)
    template <bool SCALED = false>
    __device__ __forceinline__ bool weights(const f32x16 &S, float c, u32x4 (&pb)[2], float &sum) const {
        sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float e0 = fast_exp2(TWO ? S[r] : SCALED ? S[r] - M : S[r] * c - M), e1 = fast_exp2(TWO ? S[r + 1] : SCALED ? S[r + 1] - M : S[r + 1] * c - M);
            sum += e0 + e1;
            pb[r >> 3][(r & 7) >> 1] = E::pack(e0, e1);
        }
        return !wave_any(!(sum < E::kBig));
    }
    // the column's largest logit of a tile (TWO: relative to what S is relative to)
    __device__ __forceinline__ float top_of(const f32x16 &S) const {
        float top = S[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, S[r]);
        return both_halves_max(top);
    }
    // Weights of a masked tile whatever the references are.  Columns without one take the tile's largest logit (they hold nothing yet; S of TWO is then
    // relative to 0, as it is beside a far reference); where weights outgrow a reference, all move up to the tile's largest logits.  (Dense logits are scaled before anything is taken from them: the largest
    // one's weight is 1 whatever its size)
    __device__ __forceinline__ void any_weights(f32x16 &S, float c, bool fresh, u32x4 (&pb)[2], float &sum) {
        if constexpr (!TWO) {
#pragma unroll
            for (int r = 0; r < 16; ++r) S[r] = rounded_product(S[r], c);
        }
        if (fresh) {
            const float top = fmaxf(kNoRef, top_of(S));
            M = M == kNoRef ? top : M;
            if constexpr (TWO) {
#pragma unroll
                for (int r = 0; r < 16; ++r) S[r] -= M;
            }
        }
        if (__builtin_expect(!weights<true>(S, c, pb, sum), 0)) {
            const float top = top_of(S), up = TWO ? fmaxf(top, 0.f) : fmaxf(top, M) - M, f = fast_exp2(-up);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) O[dt][r] *= f;
            l *= f;
            M += up;
            if constexpr (TWO) {
#pragma unroll
                for (int r = 0; r < 16; ++r) S[r] -= up;
            }
            weights<true>(S, c, pb, sum);
        }
    }
    // the plain form of a step
    template <bool ONE>
    __device__ __forceinline__ void step(const char *k_lane, const char *v_lane, float c, bool masked, bool guard, int tile, uint32_t there, int hf) {
        const bool fresh = no_near_reference();
        f32x16 S = logits(k_lane, fresh ? 0.f : M);
        if (masked) mask<ONE>(S, tile, there, hf);
        u32x4 pb[2];
        float sum;
        any_weights(S, c, fresh, pb, sum);
        l += sum;
        values<ONE>(v_lane, pb, guard, tile, there, hf);
    }

    // O^T += V^T P^T.  `guard`: some column does not attend some key of the tile, so a value that is not finite must be kept from it.
    // `ONE` (all columns attend to the same keys): those the columns do not attend are cleared in the operand.  Otherwise, where the tile
    // holds such a value, every group of columns with keys of its own gets a product of its own.
    template <bool ONE>
    __device__ __forceinline__ void values(const char *v_lane, const u32x4 (&pb)[2], bool guard, int tile, uint32_t there, int hf) {
        if (!guard) {
#pragma unroll
            for (int k2s = 0; k2s < 2; ++k2s)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) add_product(dt, RT::tr_frag(v_lane, k2s, dt), pb[k2s]);
            settle();
            return;
        }
        auto key_masks = [&](uint32_t keys, u32x4 (&m)[2]) {
            const uint32_t bits = keys >> (4 * hf);
#pragma unroll
            for (int k2s = 0; k2s < 2; ++k2s)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int j = 16 * k2s + 8 * (w >> 1) + 2 * (w & 1);
                    m[k2s][w] = ((bits >> j) & 1u ? 0xffffu : 0u) | ((bits >> (j + 1)) & 1u ? 0xffff0000u : 0u);
                }
        };
        if (ONE) {
            u32x4 m[2];
            key_masks(there & keys_of(tile, most_lo, least_hi), m);
#pragma unroll
            for (int k2s = 0; k2s < 2; ++k2s)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) add_product(dt, RT::tr_frag(v_lane, k2s, dt) & m[k2s], pb[k2s]);
            settle();
            return;
        }
        uint32_t odd = 0u;
#pragma unroll
        for (int k2s = 0; k2s < 2; ++k2s)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const u32x4 v = RT::tr_frag(v_lane, k2s, dt);
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= (uint32_t)((v[w] & E::kExp) == E::kExp) | (uint32_t)(((v[w] >> 16) & E::kExp) == E::kExp);
                __builtin_amdgcn_sched_barrier(0);
            }
        asm volatile("" ::: "memory");         // (the products read the tile again: held, it would take all registers)
        if (__builtin_expect(!wave_any(odd != 0u), 1)) {
#pragma unroll
            for (int k2s = 0; k2s < 2; ++k2s)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) add_product(dt, RT::tr_frag(v_lane, k2s, dt), pb[k2s]);
            settle();
            return;
        }
        const int first = max(0, lo - tile), end = min(31, hi - tile);
        for (uint64_t left = __builtin_amdgcn_ballot_w64(lo <= hi && first <= end); left != 0;) {
            const int one = (int)__builtin_ctzll(left), a = __builtin_amdgcn_readlane(first, one), z = __builtin_amdgcn_readlane(end, one);
            const bool mine = lo <= hi && first == a && end == z;
            left &= ~__builtin_amdgcn_ballot_w64(mine);
            u32x4 m[2];
            key_masks(there & keys_of(tile, tile + a, tile + z), m);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                f32x16 x = zero16();
#pragma unroll
                for (int k2s = 0; k2s < 2; ++k2s) x = E::mfma(RT::tr_frag(v_lane, k2s, dt) & m[k2s], pb[k2s], x);
#pragma unroll
                for (int r = 0; r < 16; ++r) O[dt][r] = mine ? O[dt][r] + x[r] : O[dt][r];
                asm volatile("" ::: "memory");
            }
        }
    }

    __device__ __forceinline__ bool needs_mask(int tile, uint32_t there) const { return tile < most_lo || tile + 31 > least_hi || there != 0xffffffffu; }

    // the sum of the column's weights, in both halves
    __device__ __forceinline__ float whole_sum() const {
        auto sw = __builtin_amdgcn_permlane32_swap(as_u32(l), as_u32(l), false, false);
        return as_f32(sw[0]) + as_f32(sw[1]);
    }
};

// ---- 2-simplicial form: from the columns (offsets) of one (token, head) to its output row
//
// y[v] of a lane: channel 32 (v / 16) + 16 hf + v % 16 of its column.  Adds the columns of a half and leaves NV / 32 (at least one) sums per
// lane: y[i] of lane c is the sum for v = base(c) + i.  Every step halves what a lane holds: it gives one half away and adds the other lane's
// share of the half it keeps.  Rows of 16 lanes trade by a swap, lanes of a row with their mirror image in 16, 8, 4 and 2.
template <int NV>
struct ColumnSum {
    static constexpr int LEFT = NV > 32 ? NV / 32 : 1;
    static __device__ __forceinline__ int base(int c) {
        int b = 0, n = NV;
#pragma unroll
        for (int bit = 16; bit >= 1; bit >>= 1)
            if (n > 1) {
                n /= 2;
                b += c & bit ? n : 0;
            }
        return b;
    }
    template <int CTRL>
    static __device__ __forceinline__ float other(float x) {
        return as_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)as_u32(x), CTRL, 0xf, 0xf, false));
    }
    template <int N, int BIT>
    static __device__ __forceinline__ void step(float (&y)[NV], int c) {
        if constexpr (BIT >= 1) {
            constexpr int CTRL = BIT == 8 ? 0x140 : BIT == 4 ? 0x141 : BIT == 2 ? 0x1b : 0xb1;      // row_mirror, row_half_mirror, quad_perm 3210, 1032
            if constexpr (N > 1) {
                const bool up = c & BIT;
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    if constexpr (BIT == 16) {
                        auto sw = __builtin_amdgcn_permlane16_swap(as_u32(y[i]), as_u32(y[i + N / 2]), false, false);
                        y[i] = as_f32(sw[0]) + as_f32(sw[1]);
                    } else {
                        const float keep = up ? y[i + N / 2] : y[i], send = up ? y[i] : y[i + N / 2];
                        y[i] = keep + other<CTRL>(send);
                    }
                }
                step<N / 2, BIT / 2>(y, c);
            } else {
                y[0] += other<CTRL>(y[0]);
                step<1, BIT / 2>(y, c);
            }
        }
    }
    static __device__ __forceinline__ void add(float (&y)[NV], int c) { step<NV, 16>(y, c); }
    // sum and maximum over the 32 lanes of a half, in all of them
    template <typename OP>
    static __device__ __forceinline__ float all(float x, OP op) {
        x = op(x, other<0xb1>(x));
        x = op(x, other<0x1b>(x));
        x = op(x, other<0x141>(x));
        x = op(x, other<0x140>(x));
        auto sw = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
        return op(as_f32(sw[0]), as_f32(sw[1]));
    }
};

template <class E, int D>
struct SimplicialColumns {
    static constexpr int KS = D / 16, DT = D / 32;
    int page2, row2;          // place of the column's second row (page2 < 0: there is none)

    // A = q * k2 of the column's offset
    template <class W>
    __device__ __forceinline__ void build(const PagedParams &p, const PagedSeq &s, W &w, const char *q_row, int pos, int d, int hk, int hf, bool on) {
        const int x = pos - d;
        page2 = on && d < p.w2 ? paged_page(p, s, x) : -1;
        row2 = page2 >= 0 ? x - (int)p.div((uint32_t)x) * (int)p.div.by : 0;
        const char *k2 = paged_row(p.k2, page2, row2) + hk * p.k2.sh;
        constexpr int AT_ONCE = KS < 8 ? KS : 8;
        const float c = p.scale_log2e;
        float most = 0.f;         // the column's largest product (NaN left out)
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += AT_ONCE) {
            u32x4 f[AT_ONCE], k[AT_ONCE];
#pragma unroll
            for (int x = 0; x < AT_ONCE; ++x) {
                f[x] = paged_piece(q_row, 16 * (k0 + x) + 8 * hf, p.dq, true);
                k[x] = paged_piece(k2, 16 * (k0 + x) + 8 * hf, p.dp, page2 >= 0);
            }
#pragma unroll
            for (int x = 0; x < AT_ONCE; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = E::lo(f[x][i]) * c * E::lo(k[x][i]), b = E::hi(f[x][i]) * c * E::hi(k[x][i]);
                    most = fmaxf(fmaxf(fabsf(a), fabsf(b)), most);
                    const uint32_t high = E::pack(a, b);
                    w.A[k0 + x][i] = high;
                    w.A2[k0 + x][i] = E::pack(a - E::lo(high), b - E::hi(high));
                }
        }
        most = W::both_halves_max(most);
        if (__builtin_expect(!wave_any(most > E::kMost), 1)) return;
        // Products that the type does not hold.  An infinite one has no second part (inf - inf is no number).  Finite ones (fp16) are kept divided by powers of two, the second
        // parts by one of their own, so that small products beside a large one lose no digits to its range
        float up1 = 1.f, down1 = 1.f, down2 = 1.f;
        if constexpr (E::kNarrow) {
            // (beside an infinite product, what two finite factors can reach)
            const int exponent = most < INFINITY ? exponent_of(most) : exponent_of(c) + 33, e = most > E::kMost ? max(-100, min(100, exponent - 14)) : 0, e2 = max(0, e - 13);
            w.wide = true;
            w.ratio = two_to(e - e2);
            w.up = two_to(e2);
            up1 = two_to(e);
            down1 = two_to(-e);
            down2 = two_to(-e2);
        }
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            const u32x4 f = paged_piece(q_row, 16 * kk + 8 * hf, p.dq, true), k = paged_piece(k2, 16 * kk + 8 * hf, p.dp, page2 >= 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = E::lo(f[i]) * c * E::lo(k[i]), b = E::hi(f[i]) * c * E::hi(k[i]);
                const uint32_t high = E::pack(a * down1, b * down1);
                const float ah = E::lo(high), bh = E::hi(high);
                w.A[kk][i] = high;
                w.A2[kk][i] = E::pack(fabsf(ah) < INFINITY ? (a - ah * up1) * down2 : 0.f, fabsf(bh) < INFINITY ? (b - bh * up1) * down2 : 0.f);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    static __device__ __forceinline__ int exponent_of(float x) { return (int)(as_u32(x) >> 23 & 255u) - 127; }
    static __device__ __forceinline__ float two_to(int e) { return as_f32((uint32_t)(127 + e) << 23); }

    // the sum or the maximum over the `width` neighbouring lanes of a unit, in all of them (a power of two up to 16)
    template <typename OP>
    static __device__ __forceinline__ float over(int width, float x, OP op) {
        using C = ColumnSum<16 * DT>;
        if (width > 1) x = op(x, C::template other<0xb1>(x));
        if (width > 2) x = op(x, C::template other<0x1b>(x));
        if (width > 4) x = op(x, C::template other<0x141>(x));
        if (width > 8) x = op(x, C::template other<0x140>(x));
        return x;
    }

    // The columns of a unit as one row relative to one reference: y, ref, sum.  PACKED: a unit has `width` columns, and each of them ends with the whole
    // row, y[v] of channel 32 (v / 16) + 16 hf + v % 16; else all 32, and the row is shared out as ColumnSum says
    template <bool PACKED, class W>
    __device__ __forceinline__ void finish(const PagedParams &p, const W &w, int hk, int c, int hf, int width, float (&y)[16 * DT], float &ref, float &sum) const {
        const auto most = [](float a, float b) { return fmaxf(a, b); };
        const auto plus = [](float a, float b) { return a + b; };
        const char *v2 = paged_row(p.v2, page2, row2) + hk * p.v2.sh;
        u32x4 v[2 * DT];
#pragma unroll
        for (int x = 0; x < 2 * DT; ++x) {
            const int d0 = 32 * (x >> 1) + 16 * hf + 8 * (x & 1);
            v[x] = paged_piece(v2, d0, p.dp, page2 >= 0);
        }
        // (columns without a second row, and those that met no key, hold nothing that counts)
        const float column = w.whole_sum();
        const bool live = page2 >= 0 && column != 0.f;
        const float own = live ? w.M : kNoRef;
        ref = PACKED ? over(width, own, most) : ColumnSum<16 * DT>::all(own, most);
        const float f = live ? fast_exp2(w.M - ref) : 0.f, part = live ? column * f : 0.f;
        sum = PACKED ? over(width, part, plus) : ColumnSum<16 * DT>::all(part, plus);
        // (a factor of zero does not set aside what a column holds that does not count: its values, its weights where a key is infinite, or its second
        // value may be no numbers)
        const bool aside = wave_any(!live);
#pragma unroll
        for (int x = 0; x < 2 * DT; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 8 * x + 2 * i;
                y[at] = w.O[x >> 1][at & 15] * (f * E::lo(v[x][i]));
                y[at + 1] = w.O[x >> 1][(at & 15) + 1] * (f * E::hi(v[x][i]));
            }
        if (aside) {
#pragma unroll
            for (int at = 0; at < 16 * DT; ++at) y[at] = live ? y[at] : 0.f;
        }
        if constexpr (PACKED) {
            using C = ColumnSum<16 * DT>;
            auto stage = [&](auto ctrl) {
#pragma unroll
                for (int at = 0; at < 16 * DT; ++at) y[at] += C::template other<decltype(ctrl)::value>(y[at]);
            };
            if (width > 1) stage(std::integral_constant<int, 0xb1>{});
            if (width > 2) stage(std::integral_constant<int, 0x1b>{});
            if (width > 4) stage(std::integral_constant<int, 0x141>{});
            if (width > 8) stage(std::integral_constant<int, 0x140>{});
        } else {
            ColumnSum<16 * DT>::add(y, c);
        }
    }
};

// ---- few rows: every wave walks key tiles of its own
//
// A workgroup has 32 columns (dense: up to 32 rows of one sequence and key/value head; 2-simplicial: one token and head) and a share
// of their keys; its waves take the tiles in turn, each with a K and a V tile of its own in LDS, and merge at the end.  No barrier in the walk: the
// next K tile is requested when the logits of a tile are formed, the next V tile behind its second product, so a wave always has
// a tile in flight and a CU sixteen waves of them.
//
// Bound by the cache's bytes: one token of 16 sequences of up to 32768, 16 heads on 4 of 128 channels (602 MB) 131 us with its merge, 4.6 TB/s where a copy of 2 GiB
// reaches 4.9.  The smallest calls are bound by a chain of dependent loads (length, table, rows): 5.8 us for one token over 300 rows, 10.3 for one 2-simplicial
// token, whose second rows come in front of its keys; an empty launch takes 3.6.  Several tokens (MIXED; their masks differ by column) spill registers outside the
// products, 42 at 64 channels and 3 at 128: 4 tokens of 16 sequences of 8192, 16 heads on 4 of 128 channels 63 us at a floor of 54; 8 heads on 4 of 64 channels 32 at 27.
template <int D>
struct FewCfg {
    using RT = DmaTile<D>;
    static constexpr int NW = D == 256 ? 2 : D == 128 ? 4 : 8;
    static constexpr int WPE = D == 256 ? 1 : D == 128 ? 2 : 4;     // two workgroups per CU
    static constexpr int SEG = 2048;                                // positions whose pages are kept in LDS at a time
    static constexpr int RING = NW * 2 * RT::BYTES;
    static_assert(RING - RT::CP < 65536, "the LDS address of a direct load travels in 16 bits of M0");
    static constexpr int OP = D + 4;                                // floats per row of the merge
    static constexpr int MERGE = NW * 32 * OP * 4;
    static constexpr int WALK = RING + SEG * 4;
    static constexpr int XCH = MERGE > WALK ? MERGE : WALK;         // references and sums of the waves
    static constexpr int LDS = XCH + 2 * NW * 32 * 4;
};

// MIXED: the columns are rows at different positions (dense, more than one token)
template <class E, int D, bool SIMP, bool MIXED>
__global__ __launch_bounds__(FewCfg<D>::NW * 64) __attribute__((amdgpu_waves_per_eu(FewCfg<D>::WPE, FewCfg<D>::WPE))) void paged_few_kernel(PagedParams p) {
    using C = FewCfg<D>;
    using RT = DmaTile<D>;
    constexpr int NW = C::NW, DT = D / 32;
    __shared__ __attribute__((aligned(16))) char lds[C::LDS];
    int *seg = reinterpret_cast<int *>(lds + C::RING);
    const int tid = threadIdx.x, wave = wave_index(), lane = tid & 63, c = lane & 31, hf = lane >> 5;

    // Grid.  Dense: the parts of a sequence and key/value head next to each other (their pages are, as a rule: one token of 16 sequences of up to 32768 131 us, heads
    // next to each other 143).  2-simplicial: (sequence and key/value head, row tile, part), so that the heads of a group are on one XCD
    const int parts = p.splits * p.dblocks, tile_r = blockIdx.y;
    const int seq = SIMP ? (int)blockIdx.x : uniform((int)p.parts(blockIdx.x)), part = SIMP ? (int)blockIdx.z : (int)blockIdx.x - seq * parts;
    const int b = uniform((int)p.heads(seq)), hk = seq - b * p.HK;
    const int db = p.dblocks == 1 ? 0 : uniform(part / p.splits), split = part - db * p.splits;
    const PagedSeq s = paged_seq(p, b);

    // the columns: token t, head of the group g
    const int R = SIMP ? tile_r : tile_r * 32 + c;
    const int t = (int)p.group((uint32_t)R), g = R - t * p.G, h = hk * p.G + g;
    const int pos = s.first + t;
    const bool row_there = R < p.n * p.G;
    const bool on = row_there && t < s.count && pos >= 0;
    // (first and last token of the columns)
    const int t_first = MIXED ? max((int)p.group((uint32_t)(tile_r * 32)), -s.first) : (SIMP ? t : 0);
    const int t_last = MIXED ? min((int)p.group((uint32_t)(tile_r * 32 + 31)), s.count - 1) : t_first;
    const int last = min(s.first + t_last, s.reach - 1);              // last key of any column
    const int first_key = SIMP ? first_key_of(p, s.first + t) : 0;
    const bool any = t_first < s.count && t_first <= t_last && last >= first_key;
    const int tiles = any ? (last - first_key) / 32 + 1 : 0;
    const int tile_a = p.splits == 1 ? 0 : (int)((int64_t)tiles * split / p.splits), tile_z = p.splits == 1 ? tiles : (int)((int64_t)tiles * (split + 1) / p.splits);

    const char *q_row = p.q + b * p.q_sb + (int64_t)(row_there ? t : 0) * p.q_sn + (int64_t)(row_there ? h : 0) * p.q_sh;
    PagedWave<E, D, SIMP> w;
    SimplicialColumns<E, D> cols;
    w.clear();
    cols.page2 = -1;
    cols.row2 = 0;
    char *const kt = lds + wave * 2 * RT::BYTES, *const vt = kt + RT::BYTES;
    const uint32_t kt_at = (uint32_t)(uintptr_t)kt;
    const char *const zero = reinterpret_cast<const char *>(g_paged_zero_row);
    const int st_col = RT::st_col(lane);
    const bool col_there = st_col < p.dp * 2;
    constexpr int SEG_TILES = C::SEG / 32;
    int seg_a = tile_a, seg_z = tile_a, u = tile_a;
    // requests a tile's rows of K or V (four transfers at a time: their pages are looked up together)
    auto request = [&](int is_v, int tile) {
        const char *const base = (is_v ? p.v1.ptr : p.k1.ptr) + hk * (is_v ? p.v1.sh : p.k1.sh) + st_col;
        const int64_t sp = is_v ? p.v1.sp : p.k1.sp, sr = is_v ? p.v1.sr : p.k1.sr;
        const uint32_t to = kt_at + is_v * RT::BYTES;
        int x = 32 * (tile - seg_a) + RT::st_row(0, lane);
        constexpr int AT_ONCE = RT::NCH < 4 ? RT::NCH : 4;
#pragma unroll 1
        for (int ch = 0; ch < RT::NCH; ch += AT_ONCE, x += AT_ONCE * RT::RPC) {
            int page[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) page[i] = seg[x + i * RT::RPC];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int at = first_key + 32 * seg_a + x + i * RT::RPC;
                const int row = at - (int)p.div((uint32_t)at) * (int)p.div.by;
                const char *from = base + (int64_t)page[i] * sp + (int64_t)row * sr;
                load_to_lds16_from(page[i] >= 0 && col_there ? from : zero, to + (ch + i) * RT::CP);
            }
        }
    };
    // pages of the next positions, and the wave's first tile of them
    auto open_segment = [&](int early) {
        seg_z = min(tile_z, seg_a + SEG_TILES);
        for (int x = tid; x < (seg_z - seg_a) * 32; x += NW * 64) {
            const int at = first_key + seg_a * 32 + x;
            seg[x] = at > last ? -1 : early >= -1 && x < NW * 64 ? early : paged_page(p, s, at);
        }
        __syncthreads();
        u = seg_a + wave;
        if (u < seg_z) {
#pragma unroll 1
            for (int is_v = 0; is_v < 2; ++is_v) request(is_v, u);
        }
    };
    // (an undivided walk starts at position 0: its first pages are looked up beside the length)
    const int early = !SIMP && p.splits == 1 ? paged_page(p, s, tid) : -2;
    if (tile_a < tile_z) {
        open_segment(early);
        // the columns, read behind the first transfers
        if constexpr (SIMP) {
            cols.build(p, s, w, q_row, pos, 32 * db + c, hk, hf, on);
            w.limits(first_key, last, on && cols.page2 >= 0, true, first_key, last);
        } else {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) w.A[kk] = paged_piece(q_row, 16 * kk + 8 * hf, p.dq, on);
            w.limits(0, min(pos, last), on, true, 0, min(s.first + t_first, last));
        }
        for (;;) {
            for (; u < seg_z; u += NW) {
                const int tile = first_key + 32 * u, next = u + NW;
                const uint32_t there = (uint32_t)__builtin_amdgcn_ballot_w64(seg[32 * (u - seg_a) + c] >= 0);
                wait_loads<RT::NCH>();
                const bool fresh = w.no_near_reference();
                f32x16 S = w.logits(kt + RT::row_lane(lane), fresh ? 0.f : w.M);
                wait_lds_reads();
                if (next < seg_z) request(0, next);
                const bool masked = w.needs_mask(tile, there);
                if (masked) w.template mask<!MIXED>(S, tile, there, hf);
                u32x4 pb[2];
                float sum;
                w.any_weights(S, p.scale_log2e, fresh, pb, sum);
                w.l += sum;
                if (next < seg_z) wait_loads<RT::NCH>();
                else wait_loads<0>();
                // (a workgroup with one token has no key that some of its columns attend and others do not)
                w.template values<!MIXED>(vt + RT::tr_lane(lane), pb, MIXED && masked, tile, there, hf);
                wait_lds_reads();
                if (next < seg_z) request(1, next);
            }
            seg_a += SEG_TILES;
            if (seg_a >= tile_z) break;
            __syncthreads();
            open_segment(-2);
        }
    }

    // ---- merge of the waves
    __syncthreads();
    float *xm = reinterpret_cast<float *>(lds + C::XCH), *xl = xm + NW * 32;
    float *mo = reinterpret_cast<float *>(lds);
    const int64_t rows = (int64_t)p.B * p.n * p.H;
    if constexpr (SIMP) {
        float y[16 * DT], ref, sum;
        cols.template finish<false>(p, w, hk, c, hf, 32, y, ref, sum);
        if (lane == 0) {
            xm[wave] = ref;
            xl[wave] = sum;
        }
        const int base = ColumnSum<16 * DT>::base(c);
#pragma unroll
        for (int i = 0; i < ColumnSum<16 * DT>::LEFT; ++i) {
            const int v = base + i;
            mo[wave * D + 32 * (v >> 4) + 16 * hf + (v & 15)] = y[i];
        }
        __syncthreads();
        float top = xm[0], total = 0.f;
#pragma unroll
        for (int x = 1; x < NW; ++x) top = fmaxf(top, xm[x]);
#pragma unroll
        for (int x = 0; x < NW; ++x) total += xl[x] * fast_exp2(xm[x] - top);
        const int64_t row = ((int64_t)b * p.n + t) * p.H + h;
        for (int d0 = tid * 8; d0 < D; d0 += NW * 64 * 8) {
            float z[8] = {};
#pragma unroll
            for (int x = 0; x < NW; ++x) {
                const float f = fast_exp2(xm[x] - top);
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] += f * mo[x * D + d0 + e];
            }
            if (parts == 1) {
                const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] *= inv;
                paged_store8<E>(p, p.o + b * p.o_sb + t * p.o_sn + h * p.o_sh, d0, z);
            } else {
                float *dst = p.part_o + ((int64_t)part * rows + row) * D + d0;
                *reinterpret_cast<float4 *>(dst) = make_float4(z[0], z[1], z[2], z[3]);
                *reinterpret_cast<float4 *>(dst + 4) = make_float4(z[4], z[5], z[6], z[7]);
            }
        }
        if (parts > 1 && tid == 0) p.part_ml[part * rows + row] = make_float2(top, total);
    } else {
        if (!on) w.clear();
        const float sum = w.whole_sum();
        if (hf == 0) {
            xm[wave * 32 + c] = w.M;
            xl[wave * 32 + c] = sum;
        }
        if (row_there) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<float4 *>(mo + (wave * 32 + c) * C::OP + 32 * dt + 16 * hf + r) =
                        make_float4(w.O[dt][r], w.O[dt][r + 1], w.O[dt][r + 2], w.O[dt][r + 3]);
        }
        __syncthreads();
        const int rows_here = min(32, p.n * p.G - tile_r * 32);
        for (int x = tid; x < rows_here * (D / 8); x += NW * 64) {
            const int rr = x / (D / 8), d0 = 8 * (x % (D / 8));
            float top = xm[rr], total = 0.f, z[8] = {};
#pragma unroll
            for (int y = 1; y < NW; ++y) top = fmaxf(top, xm[y * 32 + rr]);
#pragma unroll
            for (int y = 0; y < NW; ++y) {
                const float f = fast_exp2(xm[y * 32 + rr] - top);
                total += f * xl[y * 32 + rr];
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] += f * mo[(y * 32 + rr) * C::OP + d0 + e];
            }
            const int R2 = tile_r * 32 + rr, t2 = (int)p.group((uint32_t)R2), h2 = hk * p.G + R2 - t2 * p.G;
            if (parts == 1) {
                const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] *= inv;
                paged_store8<E>(p, p.o + b * p.o_sb + t2 * p.o_sn + h2 * p.o_sh, d0, z);
            } else {
                const int64_t row = ((int64_t)b * p.n + t2) * p.H + h2;
                float *dst = p.part_o + ((int64_t)part * rows + row) * D + d0;
                *reinterpret_cast<float4 *>(dst) = make_float4(z[0], z[1], z[2], z[3]);
                *reinterpret_cast<float4 *>(dst + 4) = make_float4(z[4], z[5], z[6], z[7]);
                if (d0 == 0) p.part_ml[part * rows + row] = make_float2(top, total);
            }
        }
    }
}

// ---- many rows: the waves of a workgroup walk the same key tiles
//
// A workgroup has NW x 32 columns (dense: rows of one sequence and key/value head; 2-simplicial: NW (token, head) units) and walks the
// union of their keys; K and V tiles stream through an LDS ring of four buffers that all waves read, one tile and one barrier per step.  A step's
// fragments travel through windows of FW register sets, requested FW products before their use: V's along the logit chain, the next
// tile's K along the value chain (a scheduling fence behind every product keeps them there).  Steps that need a mask, two or three of a
// walk, take the plain form of PagedWave.
//
// Bound by instruction issue of two waves per SIMD.  Dense, 128 channels: 2048 tokens of 16 heads over 32768 keys 491 to 533 us by card (532 GFLOP, 1.0 to 1.07 PFLOP/s where a
// large product of the library reaches 1.27), the matrix unit busy 54 % of the time; a step issues 16 products, 62 other vector instructions and 16 exponentials, which with
// their issue times fill nine tenths of it.  2-simplicial: 4 x 1024 tokens, 8 heads, w1 512, w2 32 424 to 453 us (276 GFLOP, and its logits' 138 again for the second part of
// the operand); its windows are short, so of a wave's 3400 vector instructions 2000 stand in front of and behind the walk.
// Tried and taken back: the two waves of a SIMD half a step apart by a second barrier (499 -> 581 us).
template <int D, bool SIMP>
struct ManyCfg {
    using RT = DmaTile<D>;
    static constexpr int NW = D == 256 || SIMP ? 4 : 8;
    static constexpr int BUF = 2 * RT::BYTES;                       // a K tile and a V tile
    static constexpr int NBUF = D == 256 ? 2 : 4;
    static constexpr bool AHEAD = NBUF == 4;                        // the next tile has landed while a tile is used
    static constexpr int WPE = D == 256 ? 1 : D == 128 ? 2 : D == 64 ? 3 : 4;     // waves per SIMD that the registers allow
    static constexpr int WPE_PACKED = D == 64 ? 2 : WPE;
    static constexpr int FW = D == 128 ? 4 : 2;
    static constexpr int RING = NBUF * BUF;
    static_assert(RING - RT::CP < 65536, "the LDS address of a direct load travels in 16 bits of M0");
    static constexpr int SEG = SIMP ? 512 : 1024;                   // circular: places of 16 (32) tiles, refilled by halves
    static constexpr int HALF = SEG / 64;                           // tiles of a half
    static constexpr int LDS = RING + 2 * SEG * 8 + 16;
    static constexpr int LOADS = 2 * RT::NCH > NW ? 2 * RT::NCH / NW : 1;    // per wave and tile
};

// PACKED (2-simplicial, many units with second windows up to 16): a wave has 32 / width (token, head) units of `width` columns each, width the power of two that holds
// the window
template <class E, int D, bool SIMP, bool PACKED>
__global__ __launch_bounds__((ManyCfg<D, SIMP>::NW * 64)) __attribute__((amdgpu_waves_per_eu(PACKED ? ManyCfg<D, SIMP>::WPE_PACKED : ManyCfg<D, SIMP>::WPE, PACKED ? ManyCfg<D, SIMP>::WPE_PACKED : ManyCfg<D, SIMP>::WPE))) void
paged_many_kernel(PagedParams p) {
    using C = ManyCfg<D, SIMP>;
    using RT = DmaTile<D>;
    constexpr int NW = C::NW, DT = D / 32, KS = D / 16, NBUF = C::NBUF, FW = C::FW;
    __shared__ __attribute__((aligned(16))) char lds[C::LDS];
    // addresses of the walked positions' rows in the K and the V pool; a row of zeros where there is none
    const char **seg_k = reinterpret_cast<const char **>(lds + C::RING), **seg_v = seg_k + C::SEG;
    int *gaps = reinterpret_cast<int *>(lds + C::RING + 2 * C::SEG * 8);     // per half (of four): keys are missing in front of the last one
    const int tid = threadIdx.x, wave = wave_index(), lane = tid & 63, c = lane & 31, hf = lane >> 5;
    const int width = PACKED ? p.unit_columns : SIMP ? 32 : 1, units = 32 / width;      // columns of a row (t, g), rows of a wave
    const int PER_WG = NW * units;                      // ... of a workgroup
    constexpr bool ONE = SIMP && !PACKED;               // all columns of a wave attend to the same keys

    // grid: (row tile, sequence and key/value head with the heads next to each other: one XCD has all workgroups of a head where their number is a multiple
    // of eight), part; the longest rows first
    const int parts = p.splits * p.dblocks, part = blockIdx.y;
    const int row = uniform((int)p.seqs(blockIdx.x)), seq = blockIdx.x - row * (int)p.seqs.by, tile_r = p.row_tiles - 1 - row;
    const int grid_b = uniform((int)p.heads(seq)), hk = seq - grid_b * p.HK, place = SIMP ? 0 : part * p.B + grid_b;
    const int db = p.dblocks == 1 ? 0 : uniform(part / p.splits);
    int b = grid_b, split = part - db * p.splits, splits = p.splits;
    PagedSeq s;
    if (!SIMP && !p.even) {
        const PagedShares shares(p, lane);
        // (for the merge)
        if (blockIdx.x == 0 && part == 0 && tid < p.B) p.shares[tid] = make_int2(shares.behind - shares.count, shares.count);
        const uint64_t before = __builtin_amdgcn_ballot_w64(shares.behind <= place);
        b = __builtin_popcountll(before);                // (lanes beyond the sequences add no place)
        if (b >= p.B) return;
        splits = PagedShares::of(shares.count, b);
        split = place - (PagedShares::of(shares.behind, b) - splits);
        s = {p.tables + b * p.t_sb, PagedShares::of(shares.s.first, b), PagedShares::of(shares.s.count, b), shares.s.reach};
    } else {
        s = paged_seq(p, b);
    }

    const int R0 = tile_r * PER_WG, R = R0 + wave * units + (PACKED ? c / width : SIMP ? 0 : c);
    const int t = (int)p.group((uint32_t)R), g = R - t * p.G, h = hk * p.G + g;
    const int pos = s.first + t;
    const bool row_there = R < p.n * p.G;
    const bool on = row_there && t < s.count && pos >= 0;
    const int t_first = (int)p.group((uint32_t)R0), t_last = min((int)p.group((uint32_t)(R0 + PER_WG - 1)), s.count - 1);
    const int last = min(s.first + t_last, s.reach - 1);
    const int first_key = SIMP ? first_key_of(p, s.first + t_first) : 0;
    const int tiles = t_first < s.count && last >= first_key ? (last - first_key) / 32 + 1 : 0;
    const int tile_a = splits == 1 ? 0 : (int)((int64_t)tiles * split / splits), tile_z = splits == 1 ? tiles : (int)((int64_t)tiles * (split + 1) / splits);
    const int NT = tile_z - tile_a;

    const char *const k_head = p.k1.ptr + hk * p.k1.sh, *const v_head = p.v1.ptr + hk * p.v1.sh;
    const char *zero = reinterpret_cast<const char *>(g_paged_zero_row);
    asm volatile("" : "+s"(zero));                       // (formed once)
    const int st_col = RT::st_col(lane);
    const bool col_there = st_col < p.dp * 2;
    const int start = first_key + 32 * tile_a;          // position of step 0
    auto fill = [&](int half) {                          // places of the tiles half * HALF ..
        const int from = half * (C::SEG / 2);
        int missing = 0;
        for (int x = from + tid; x < from + C::SEG / 2; x += NW * 64) {
            const int at = start + x;
            const int page = at <= last && at >= 0 ? paged_page(p, s, at) : -1;
            const int row = at - (int)p.div((uint32_t)at) * (int)p.div.by;
            seg_k[x & (C::SEG - 1)] = page < 0 ? zero : k_head + (int64_t)page * p.k1.sp + (int64_t)row * p.k1.sr;
            seg_v[x & (C::SEG - 1)] = page < 0 ? zero : v_head + (int64_t)page * p.v1.sp + (int64_t)row * p.v1.sr;
            missing |= page < 0 && at <= last;
        }
        if (missing) gaps[half & 3] = 1;
        if (tid == 0) gaps[(half + 1) & 3] = 0;          // (the next one's, long unused)
    };
    // keys of a tile that are there (keys beyond the last one are masked as the columns' future)
    auto there_of = [&](int u, int any_gap) {
        return any_gap ? (uint32_t)__builtin_amdgcn_ballot_w64(seg_k[(32 * u + c) & (C::SEG - 1)] != zero || start + 32 * u + c > last) : 0xffffffffu;
    };
    auto request = [&](int u) {                          // this wave's share of the transfers of step u
        const uint32_t buf = (uint32_t)(uintptr_t)lds + (u & (NBUF - 1)) * C::BUF;
#pragma unroll
        for (int i = 0; i < C::LOADS; ++i) {
            const int x = wave + i * NW;                 // chunk x % NCH of K (x < NCH) or V
            if (2 * RT::NCH < NW && x >= 2 * RT::NCH) break;
            const bool is_v = RT::NCH >= NW ? i >= RT::NCH / NW : x >= RT::NCH;
            const int ch = is_v ? x - RT::NCH : x;
            const char *from = (is_v ? seg_v : seg_k)[(32 * u + RT::st_row(ch, lane)) & (C::SEG - 1)];
            asm volatile("" : "+v"(from));
            load_to_lds16_from(col_there ? from + st_col : zero, buf + (is_v ? RT::BYTES : 0) + ch * RT::CP);
        }
    };

    PagedWave<E, D, SIMP, (D == 64 || D == 128)> w;
    SimplicialColumns<E, D> cols;
    if (NT > 0) {
        if (tid < 4) gaps[tid] = 0;
        __syncthreads();
        fill(0);
        __syncthreads();
        fill(1);
        __syncthreads();
        for (int u = 0; u < NBUF - 1; ++u) request(u);
    }
    // (the columns are read behind the first transfers)
    const char *q_row = p.q + b * p.q_sb + (int64_t)(row_there ? t : 0) * p.q_sn + (int64_t)(row_there ? h : 0) * p.q_sh;
    w.clear();
    // keys that any column of the wave attends
    int lo, hi;
    const int t0 = max((int)p.group((uint32_t)(R0 + wave * units)), -s.first), t1 = min((int)p.group((uint32_t)(R0 + wave * units + units - 1)), s.count - 1);
    bool any = t0 <= t1 && last >= 0;
    if constexpr (SIMP) {
        cols.build(p, s, w, q_row, pos, 32 * db + (PACKED ? c & (width - 1) : c), hk, hf, on);
        any = any && wave_any(on && cols.page2 >= 0);
    } else {
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) w.A[kk] = paged_piece(q_row, 16 * kk + 8 * hf, p.dq, on);
    }
    lo = any ? (SIMP ? first_key_of(p, s.first + t0) : 0) : 0x7fffffff;
    hi = any ? min(s.first + t1, last) : -1;
    any = any && lo <= hi;
    w.limits(SIMP ? first_key_of(p, pos) : 0, min(pos, last), on && (!SIMP || cols.page2 >= 0), any, SIMP ? first_key_of(p, s.first + t1) : 0, min(s.first + t0, last));
    lo = uniform(lo);
    hi = uniform(hi);
    w.most_lo = uniform(w.most_lo);
    w.least_hi = uniform(w.least_hi);
    // (in registers from here on: a wait for them inside the walk would wait for the transfers too)
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
        asm volatile("" : "+v"(w.A[kk]));
        if constexpr (SIMP) asm volatile("" : "+v"(w.A2[kk]));
    }
    if (NT > 0) {
        // their steps
        const int u_a = lo > hi || hi < start ? NT : min(NT, max(0, lo - start) >> 5), u_z = lo > hi || hi < start ? NT : min(NT, ((hi - start) >> 5) + 1);
        const int k_lane = RT::row_lane(lane), v_lane = RT::BYTES + RT::tr_lane(lane);
        u32x4 kf[FW];
        u32x2 vf[FW][2];
        // start of step u: the tile of step u + 1 (of step u, where there are two buffers) has landed and every wave is done with step u - 1
        auto open_step = [&]() {
            wait_loads<C::AHEAD ? C::LOADS : 0>();
            __syncthreads();
        };
        if (C::AHEAD) wait_loads<0>();
        for (int u = 0; u < NT;) {
            // sixteen steps at a time: the places of the sixteen that follow go where those of the sixteen before were
            __syncthreads();
            const int half = u / C::HALF, any_gap = uniform(gaps[half & 3]);
            if (half > 0) {
                __syncthreads();
                fill(half + 1);
            }
            const int end = min(NT, u + C::HALF), z = min(end, u_z);
            // steps in front of it need no mask
            const int m_z = any_gap || w.wide ? u : min(z, ((w.least_hi - start - 31) >> 5) + 1);
            for (; u < min(end, u_a); ++u) {
                open_step();
                request(u + NBUF - 1);
            }
            while (u < z) {
                bool opened = false;      // the step is open already (its weights outgrew a reference)
                if (C::AHEAD && u < m_z && start + 32 * u >= w.most_lo && !w.no_near_reference()) {
                    const f32x16 from = splat16(-w.M);      // (2-simplicial: where the chains of products start)
                    const char *first = lds + (u & (NBUF - 1)) * C::BUF + k_lane;
#pragma unroll
                    for (int kk = 0; kk < FW; ++kk) kf[kk] = ld_lds16(first + RT::row_imm(kk));
                    do {
                        open_step();
                        const char *buf = lds + (u & (NBUF - 1)) * C::BUF;
                        f32x16 S = SIMP ? from : zero16();
                        auto read_vf = [&](int f) {
                            vf[f % FW][0] = lds_read_tr<D, 0>(buf + v_lane + RT::tr_imm(16 * (f / DT), 32 * (f % DT)), 0, 0);
                            vf[f % FW][1] = lds_read_tr<D, 0>(buf + v_lane + RT::tr_imm(16 * (f / DT) + 8, 32 * (f % DT)), 0, 0);
                        };
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int kk = 0; kk < KS; ++kk) {
                            S = w.logit(kf[kk % FW], kk, S);
                            if (kk == 0) request(u + NBUF - 1);
                            if (kk + FW < KS) kf[kk % FW] = ld_lds16(buf + k_lane + RT::row_imm(kk + FW));
                            if (kk >= KS - FW) read_vf(kk - (KS - FW));
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        u32x4 pb[2];
                        float sum;
                        if (__builtin_expect(!w.weights(S, p.scale_log2e, pb, sum), 0)) {
                            opened = true;
                            break;
                        }
                        w.l += sum;
                        const char *next = lds + ((u + 1) & (NBUF - 1)) * C::BUF + k_lane;
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int m = 0; m < 2 * DT; ++m) {
                            const u32x4 v = {vf[m % FW][0][0], vf[m % FW][0][1], vf[m % FW][1][0], vf[m % FW][1][1]};
                            w.add_product(m % DT, v, pb[m / DT]);
                            if (m + FW < 2 * DT) read_vf(m + FW);
                            if (m >= 2 * DT - FW) kf[m - (2 * DT - FW)] = ld_lds16(next + RT::row_imm(m - (2 * DT - FW)));
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        ++u;
                    } while (u < m_z);
                    w.settle();
                    if (!opened) continue;
                }
                // steps with a mask, and those that move a reference
                if (!opened) {
                    open_step();
                    request(u + NBUF - 1);
                }
                const char *buf = lds + (u & (NBUF - 1)) * C::BUF;
                const int tile = start + 32 * u;
                const uint32_t there = there_of(u, any_gap);
                const bool masked = w.needs_mask(tile, there);
                w.template step<ONE>(buf + k_lane, buf + v_lane, p.scale_log2e, masked, masked, tile, there, hf);
                ++u;
            }
            for (; u < end; ++u) {
                open_step();
                request(u + NBUF - 1);
            }
        }
        wait_loads<0>();
    }

    w.settle();
    const int64_t part_row = (SIMP ? (int64_t)part * p.B + grid_b : place) * p.n * p.H + (int64_t)t * p.H + h;
    if constexpr (SIMP) {
        float y[16 * DT], ref, sum;
        cols.template finish<PACKED>(p, w, hk, c, hf, width, y, ref, sum);
        if (!row_there) return;
        if constexpr (PACKED) {
            if ((c & (width - 1)) != 0) return;
            const bool something = sum > 0.f || sum != sum;
            const float inv = something ? 1.f / sum : 0.f;
#pragma unroll
            for (int x = 0; x < 2 * DT; ++x) {
                const int d0 = 32 * (x >> 1) + 16 * hf + 8 * (x & 1);
                float z[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = parts > 1 ? y[8 * x + e] : something ? y[8 * x + e] * inv : 0.f;
                if (parts == 1) {
                    paged_store8<E>(p, p.o + b * p.o_sb + t * p.o_sn + h * p.o_sh, d0, z);
                } else {
                    float *dst = p.part_o + part_row * D + d0;
                    *reinterpret_cast<float4 *>(dst) = make_float4(z[0], z[1], z[2], z[3]);
                    *reinterpret_cast<float4 *>(dst + 4) = make_float4(z[4], z[5], z[6], z[7]);
                }
            }
            if (parts > 1 && hf == 0) p.part_ml[part_row] = make_float2(ref, sum);
            return;
        }
        const int base = ColumnSum<16 * DT>::base(c);
        if (parts == 1) {
            const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
            char *orow = p.o + b * p.o_sb + t * p.o_sn + h * p.o_sh;
#pragma unroll
            for (int i = 0; i < ColumnSum<16 * DT>::LEFT; ++i) {
                const int d = 32 * ((base + i) >> 4) + 16 * hf + ((base + i) & 15);
                if (d < p.dq && (16 * DT >= 32 || (c & 1) == 0)) *reinterpret_cast<uint16_t *>(orow + d * 2) = (uint16_t)E::pack(y[i] * inv, 0.f);
            }
        } else {
            float *dst = p.part_o + part_row * D;
#pragma unroll
            for (int i = 0; i < ColumnSum<16 * DT>::LEFT; ++i)
                if (16 * DT >= 32 || (c & 1) == 0) dst[32 * ((base + i) >> 4) + 16 * hf + ((base + i) & 15)] = y[i];
            if (lane == 0) p.part_ml[part_row] = make_float2(ref, sum);
        }
    } else {
        if (!on) w.clear();
        const float sum = w.whole_sum();
        if (!row_there) return;
        if (parts == 1) {
            const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
            char *orow = p.o + b * p.o_sb + t * p.o_sn + h * p.o_sh;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float z[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[e] = w.O[dt][8 * half + e] * inv;
                    paged_store8<E>(p, orow, 32 * dt + 16 * hf + 8 * half, z);
                }
        } else {
            store_row_f32<DT>(p.part_o + part_row * D + 16 * hf, w.O, 1.f);
            if (hf == 0) p.part_ml[part_row] = make_float2(w.M, sum);
        }
    }
}

// ---- partial results of a row merged: D / 8 threads per part, PG parts at a time (few rows with many parts are a chain of
// dependent loads otherwise), the groups' sums added in order.  Measured with its walk, where eight parts of a thread were loaded one after the other and all at once: one token
// of 8 heads on one over 131072 rows of 128 channels in 256 parts 38 and 25 us, of 32768 rows in 128 parts 21 and 15
template <class E, int D, int PG>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p) {
    constexpr int TPR = D / 8, RPW = 256 / (TPR * PG);
    __shared__ float sums[PG > 1 ? 256 : 1][PG > 1 ? 11 : 1];
    const int64_t rows = (int64_t)p.B * p.n * p.H, row = (int64_t)blockIdx.x * RPW + threadIdx.x / (TPR * PG);
    const int d0 = 8 * (threadIdx.x % TPR), group = threadIdx.x / TPR % PG;
    // (rows are fewer than 2^26)
    const uint32_t bt = (uint32_t)row / p.H, b = bt / p.n;
    const int h = (int)((uint32_t)row - bt * p.H), t = (int)(bt - b * p.n);
    // the row's places: one in each of the parts, or those of its sequence's shares
    int parts = p.splits * p.dblocks;
    int64_t from = row, step = rows;
    if (!p.even) {
        const int2 of_b = p.shares[min((int)b, p.B - 1)];
        parts = of_b.y;
        step = (int64_t)p.n * p.H;
        from = of_b.x * step + (row - b * step);
    }
    float top = kNoRef, total = 0.f, z[8] = {};
    if (row < rows) {
        // (a part that attended to nothing has left no row: what is read in its place is set aside.  Eight parts in flight: one after the other
        // they are a chain of loads)
        constexpr int AHEAD = 8;
        for (int x0 = group; x0 < parts; x0 += AHEAD * PG) {
            float2 ml[AHEAD];
            float4 a[AHEAD], c[AHEAD];
#pragma unroll
            for (int y = 0; y < AHEAD; ++y) {
                const int64_t at = from + min(x0 + y * PG, parts - 1) * step;
                const float *src = p.part_o + at * D + d0;
                ml[y] = p.part_ml[at];
                a[y] = *reinterpret_cast<const float4 *>(src);
                c[y] = *reinterpret_cast<const float4 *>(src + 4);
            }
#pragma unroll
            for (int y = 0; y < AHEAD; ++y) {
                if (x0 + y * PG >= parts || ml[y].y == 0.f) continue;
                const float ref = fmaxf(top, ml[y].x), f = fast_exp2(ml[y].x - ref), old = fast_exp2(top - ref);
                top = ref;
                total = total * old + f * ml[y].y;
                z[0] = z[0] * old + f * a[y].x; z[1] = z[1] * old + f * a[y].y; z[2] = z[2] * old + f * a[y].z; z[3] = z[3] * old + f * a[y].w;
                z[4] = z[4] * old + f * c[y].x; z[5] = z[5] * old + f * c[y].y; z[6] = z[6] * old + f * c[y].z; z[7] = z[7] * old + f * c[y].w;
            }
        }
    }
    if constexpr (PG > 1) {
        float *mine = sums[threadIdx.x];
        mine[8] = top;
        mine[9] = total;
#pragma unroll
        for (int e = 0; e < 8; ++e) mine[e] = z[e];
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int y = 1; y < PG; ++y) top = fmaxf(top, mine[y * TPR * 11 + 8]);
        const float own = fast_exp2(mine[8] - top);
        total *= own;
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] *= own;
#pragma unroll
        for (int y = 1; y < PG; ++y) {
            const float *other = mine + y * TPR * 11;
            const float f = fast_exp2(other[8] - top);
            total += f * other[9];
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] += f * other[e];
        }
    }
    if (row >= rows) return;
    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] *= inv;
    paged_store8<E>(p, p.o + b * p.o_sb + t * p.o_sn + h * p.o_sh, d0, z);
}

}  // namespace sa2
