// Next tokens from logits: temperature, top-k, top-p, min-p, from given random numbers.
//
// Order the tokens of a row by (logit descending, index ascending) and let p = softmax(logit / T).  A token is kept if its rank is below
// top_k, the mass in front of it below top_p, and p at least min_p times the largest; every one of these keeps a prefix of the order, so
// the kept tokens are a prefix too.  The token is the kept one with the largest  logit / T - log(-log u),  which draws from p restricted to the
// prefix (compared as  p / -log u,  one logarithm and a reciprocal).  No sort: the best of ALL tokens is the answer if it is kept, and otherwise nothing behind it is, so the race is run again among the tokens
// in front of it.  Whether a token is kept takes two sums over the tokens in front of it, formed in the pass that runs the next race.
// Each race that fails leaves a uniformly drawn share of the mass, so their number grows with the logarithm of the vocabulary at most.
//
// Rows of up to 4096 tokens stay in the registers of one workgroup.  Longer ones are read once, 4096 tokens per workgroup, which leaves the chunk's sums, the best token
// of an unfiltered row, and the largest logit of every 16 tokens.  A second kernel merges them, one workgroup per row; the largest logits
// of the sixteens bound the kept prefix so closely that the races of a filtered row, and its random numbers, are looked up for few tokens.
// Measured: 8 rows of 256 tokens 6.3 us (one launch); 96 rows of 100000, half of them with min-p, all with top-k and top-p, 30 us: 12 for the reading (19 MB: the chip
// is filled by 600 workgroups that read once) and 18 for a chain of reductions over a workgroup (top, bound, races).  A flat row without top-k holds thousands of kept tokens,
// which its workgroup reads again in every race: 45 to 50 us.  Without filters the random numbers are read as well: 96 rows of 100000 in bf16 20 us (floor 12), 8 rows of 131072
// in fp32 9.
// Weights are exp2 of log2 units: exp2, log2 and reciprocals are single instructions, exact to an ulp.
#pragma once

#include "sa2_common.hpp"

namespace sa2 {

constexpr int kSampleEach = 16;            // tokens of a thread
constexpr int kSampleThreads = 256;
constexpr int kSampleChunk = kSampleEach * kSampleThreads;

struct SampleRecord {                      // what a workgroup leaves of a chunk
    float top, mass1, massT, score;        // largest logit; sums of exp(x - top) and exp((x - top) / T); the best token's score, relative to `top`
    int top_at, best_at;                   // (-1: no token)
    float best;                            // logit of the best
    int pad;
};

struct SampleParams {
    const char *logits;
    int64_t stride;               // elements
    const float *noise;
    int64_t noise_stride;
    const float *temperature, *top_p, *min_p;      // per row, or nullptr: the number below
    const int32_t *top_k;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int vocab, chunks;
    int64_t *tokens;
    float *logprobs;
    SampleRecord *records;        // [rows][chunks]
    float *tops;                  // [rows][chunks][kSampleThreads]: largest logit of a thread's tokens
};

constexpr float kMostFloat = 3.402823466e38f;
// (not a number: never drawn; infinity: the largest number)
__device__ __forceinline__ float clean_logit(float x) { return fminf(fmaxf(x, -INFINITY), kMostFloat); }

template <int TYPE>
struct Logits {
    static constexpr int SIZE = TYPE == 2 ? 4 : 2, PIECE = 16 / SIZE, PIECES = kSampleEach / PIECE;
    static __device__ __forceinline__ float one(uint16_t w) { return TYPE == 1 ? (float)__builtin_bit_cast(_Float16, w) : as_f32((uint32_t)w << 16); }
    static __device__ __forceinline__ float at(const char *row, int i) {
        if constexpr (TYPE == 2) return clean_logit(reinterpret_cast<const float *>(row)[i]);
        else return clean_logit(one(reinterpret_cast<const uint16_t *>(row)[i]));
    }
    // token of element e of thread t of a chunk: pieces of 16 bytes, neighbours in neighbouring threads
    static __device__ __forceinline__ int index(int chunk, int threads, int t, int e) {
        return chunk * threads * kSampleEach + ((e / PIECE) * threads + t) * PIECE + e % PIECE;
    }
    // a piece at any alignment; tokens beyond the vocabulary are -inf
    static __device__ __forceinline__ void piece(const char *row, int i, int vocab, float (&x)[PIECE]) {
        if (i + PIECE <= vocab) {
            u32x4 w;
            __builtin_memcpy(&w, row + (int64_t)i * SIZE, 16);
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                if constexpr (TYPE == 2) x[e] = clean_logit(as_f32(w[e]));
                else x[e] = clean_logit(one((uint16_t)(w[e >> 1] >> (16 * (e & 1)))));
            }
        } else {
#pragma unroll
            for (int e = 0; e < PIECE; ++e) x[e] = i + e < vocab ? at(row, i + e) : -INFINITY;
        }
    }
};

// 1 / -log2 u, u held inside (0, 1): a token's score is its weight times this
__device__ __forceinline__ float race_factor(float u) {
    return __builtin_amdgcn_rcpf(-__builtin_amdgcn_logf(fminf(fmaxf(u, 1.17549435e-38f), 0.99999994f)));
}

struct Best {
    float score, x;
    int index;                    // -1: none
};
__device__ __forceinline__ bool beats(const Best &a, const Best &b) {
    if (a.index < 0 || b.index < 0) return b.index < 0 && a.index >= 0;
    return a.score > b.score || (a.score == b.score && a.index < b.index);
}

// ---- reductions of a wave in the vector unit (lane 63 collects), then of the workgroup through LDS; orders are fixed
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t identity, uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)identity, (int)x, CTRL, ROWS, 0xf, false);
}
template <typename OP>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t x, uint32_t identity, OP op) {
    x = op(x, dpp<0x111, 0xf>(identity, x));          // the row's lanes 1, 2, 4 and 8 before this one
    x = op(x, dpp<0x112, 0xf>(identity, x));
    x = op(x, dpp<0x114, 0xf>(identity, x));
    x = op(x, dpp<0x118, 0xf>(identity, x));
    x = op(x, dpp<0x142, 0xa>(identity, x));          // lane 15 of a row into the next row
    x = op(x, dpp<0x143, 0xc>(identity, x));          // lane 31 into the upper half
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ float wave_sum(float x) {
    return as_f32(wave_reduce(as_u32(x), 0u, [](uint32_t a, uint32_t b) { return as_u32(as_f32(a) + as_f32(b)); }));
}
__device__ __forceinline__ float wave_max(float x) {
    return as_f32(wave_reduce(as_u32(x), 0xff800000u, [](uint32_t a, uint32_t b) { return as_u32(fmaxf(as_f32(a), as_f32(b))); }));
}
__device__ __forceinline__ uint32_t wave_min(uint32_t x) {
    return wave_reduce(x, 0xffffffffu, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
// the lane's bests' first (scores are numbers; index -1, as the largest unsigned number, loses)
__device__ __forceinline__ Best wave_first(const Best &v) {
    const float s = wave_max(v.index < 0 ? -INFINITY : v.score);
    const uint32_t i = wave_min(v.score == s ? (uint32_t)v.index : 0xffffffffu);
    const uint64_t owner = __builtin_amdgcn_ballot_w64((uint32_t)v.index == i);
    const int lane = (int)__builtin_ctzll(owner | (1ull << 63));
    return {s, as_f32((uint32_t)__builtin_amdgcn_readlane((int)as_u32(v.x), lane)), (int)i};
}

template <int THREADS>
struct RowReduce {
    static constexpr int NW = THREADS / 64;
    float a[NW], b[NW], s[NW], x[NW];
    int i[NW];
    uint32_t n[2][3][NW];
    // sums of two numbers and the first of the bests, for the whole workgroup
    __device__ __forceinline__ void all(float &p, float &q, Best &v) {
        p = wave_sum(p);
        q = wave_sum(q);
        v = wave_first(v);
        if (NW == 1) return;
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        __syncthreads();
        if (lane == 0) {
            a[w] = p;
            b[w] = q;
            s[w] = v.score;
            x[w] = v.x;
            i[w] = v.index;
        }
        __syncthreads();
        p = wave_sum(lane < NW ? a[lane % NW] : 0.f);
        q = wave_sum(lane < NW ? b[lane % NW] : 0.f);
        v = wave_first(lane < NW ? Best{s[lane % NW], x[lane % NW], i[lane % NW]} : Best{-INFINITY, 0.f, -1});
    }
    __device__ __forceinline__ Best first(Best v) {
        float p = 0.f, q = 0.f;
        all(p, q, v);
        return v;
    }
    // The largest number v (to 16 bits of its order) that at least k of the workgroup's numbers reach, -infinity if there are not k of them: two bits at a time,
    // the counts by ballots
    template <int N>
    __device__ __forceinline__ float reached_by(const float (&g)[N], uint32_t k) {
        uint32_t key[N], v = 0u;
#pragma unroll
        for (int e = 0; e < N; ++e) key[e] = as_u32(g[e]) & 0x80000000u ? ~as_u32(g[e]) : as_u32(g[e]) | 0x80000000u;
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        for (int shift = 30; shift >= 16; shift -= 2) {
            uint32_t count[3] = {0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < N; ++e)
#pragma unroll
                for (int j = 0; j < 3; ++j) count[j] += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[e] >= (v | ((uint32_t)(j + 1) << shift))));
            if (NW > 1) {
                uint32_t(&at)[3][NW] = n[(shift >> 1) & 1];
                if (lane < 3) at[lane][w] = lane == 0 ? count[0] : lane == 1 ? count[1] : count[2];
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    count[j] = 0u;
#pragma unroll
                    for (int y = 0; y < NW; ++y) count[j] += at[j][y];
                }
            }
            v |= (uint32_t)(count[2] >= k ? 3 : count[1] >= k ? 2 : count[0] >= k ? 1 : 0) << shift;
        }
        return v <= 0x007fffffu ? -INFINITY : as_f32(v & 0x80000000u ? v & 0x7fffffffu : ~v);
    }
};

struct RowRules {
    float inv, top_p, min_p;      // inv: log2(e) / T, above 0 (a logit of -inf times it has to weigh nothing) but for a greedy row
    int top_k;
    bool greedy;
    __device__ RowRules(const SampleParams &p, int64_t r) {
        const float T = p.temperature ? p.temperature[r] : p.temperature_all;
        greedy = !(T > 0.f);
        inv = greedy ? 0.f : fmaxf(fminf(kLog2e / T, kMostFloat), 1e-44f);
        top_p = p.top_p ? p.top_p[r] : p.top_p_all;
        min_p = p.min_p ? p.min_p[r] : p.min_p_all;
        top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    }
    __device__ bool filters() const { return top_k > 0 || !(top_p >= 1.f) || !(min_p <= 0.f); }
    // a token with `count` tokens and the mass `front` in front of it
    __device__ bool keeps(float count, float front, float mass, float weight) const {
        return (top_k <= 0 || count < (float)top_k) && (top_p >= 1.f || front < top_p * mass) && weight >= min_p;
    }
};

__device__ __forceinline__ void write_token(const SampleParams &p, int64_t r, const Best &best, float top, float mass1) {
    p.tokens[r] = best.index;
    p.logprobs[r] = best.index < 0 ? -INFINITY : best.x - top - kLn2 * __builtin_amdgcn_logf(mass1);
}

// a token in a race (tokens enter in ascending order: ties stay with the first)
__device__ __forceinline__ void enter(Best &mine, float x, int i, float score) {
    if (score > mine.score) mine = {score, x, i};
}
constexpr Best kNobody = {0.f, 0.f, -1};      // (a weight too small for fp32 loses to any other)

// EACH: tokens of a thread.  ONE: the row is one chunk, and this kernel finishes it; else a row with top_k runs no race here
template <int TYPE, int THREADS, int EACH, bool ONE>
__global__ __launch_bounds__(THREADS) void sample_chunk_kernel(SampleParams p) {
    using L = Logits<TYPE>;
    constexpr int PIECES = EACH / L::PIECE;
    __shared__ RowReduce<THREADS> red;
    const int64_t r = ONE ? blockIdx.x : blockIdx.x / p.chunks;
    const int chunk = ONE ? 0 : blockIdx.x - (int)r * p.chunks;
    const int tid = threadIdx.x, V = p.vocab;
    const char *row = p.logits + r * p.stride * L::SIZE;
    const float *noise = p.noise + r * p.noise_stride;
    const RowRules rules(p, r);
    const bool races = !rules.greedy && (ONE || rules.top_k <= 0);
    auto first_of = [&](int q) { return chunk * THREADS * EACH + (q * THREADS + tid) * L::PIECE; };
    float x[EACH], u[EACH];
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
        const int i = first_of(q);
        float y[L::PIECE];
        L::piece(row, i, V, y);
#pragma unroll
        for (int e = 0; e < L::PIECE; ++e) x[q * L::PIECE + e] = y[e];
    }
    if (races) {
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            const int i = first_of(q);
            if (i + L::PIECE <= V) {
                __builtin_memcpy(&u[q * L::PIECE], noise + i, 4 * L::PIECE);
            } else {
#pragma unroll
                for (int e = 0; e < L::PIECE; ++e) u[q * L::PIECE + e] = i + e < V ? noise[i + e] : 0.f;
            }
        }
    }
    auto index = [&](int e) { return first_of(e / L::PIECE) + e % L::PIECE; };
    float most = x[0];
#pragma unroll
    for (int e = 1; e < EACH; ++e) most = fmaxf(most, x[e]);
    if (!ONE) p.tops[(r * p.chunks + chunk) * THREADS + tid] = most;
    Best top = {most, most, -1};
    if (most > -INFINITY) {
#pragma unroll
        for (int e = EACH - 1; e >= 0; --e)    // (a thread's tokens ascend: the first that equals)
            top.index = x[e] == most ? index(e) : top.index;
    }
    top = red.first(top);
    if (ONE && top.index < 0) {                // nothing to draw from
        if (tid == 0) write_token(p, r, top, 0.f, 1.f);
        return;
    }
    float mass1 = 0.f, mass = 0.f;
    Best mine = kNobody;
    float w[EACH];                             // weights; then u: scores
    if (top.index >= 0) {
        // (-inf: a weight of zero; inv is finite, so 0 stays 0)
#pragma unroll
        for (int e = 0; e < EACH; ++e) mass1 += fast_exp2((x[e] - top.x) * kLog2e);
        if (!rules.greedy && (races || rules.top_p < 1.f)) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                w[e] = fast_exp2((x[e] - top.x) * rules.inv);
                mass += w[e];
            }
        }
        if (races) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                u[e] = w[e] * race_factor(u[e]);
                enter(mine, x[e], index(e), u[e]);
            }
        }
    }
    red.all(mass1, mass, mine);
    Best best = rules.greedy ? top : mine;
    if constexpr (!ONE) {
        if (tid == 0) p.records[r * p.chunks + chunk] = {top.x, mass1, mass, best.score, top.index, best.index, best.x, 0};
        return;
    }
    if (!rules.greedy && best.index != top.index && rules.filters()) {
        // (with top_k the race is run again in front of the bound, once the winner of all is behind it)
        const float cut = rules.top_k > 0 ? red.reached_by(x, (uint32_t)rules.top_k) : -INFINITY;
        if (best.x < cut) best = {0.f, cut, 0x7fffffff};
        while (best.index != top.index) {
            float front = 0.f, count = 0.f;
            mine = kNobody;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const bool in = x[e] > best.x || (x[e] == best.x && index(e) < best.index);
                front += in ? w[e] : 0.f;
                count += in ? 1.f : 0.f;
                enter(mine, x[e], index(e), in ? u[e] : 0.f);
            }
            red.all(front, count, mine);
            if (best.index != 0x7fffffff && rules.keeps(count, front, mass, fast_exp2((best.x - top.x) * rules.inv))) break;
            best = mine;
        }
    }
    if (tid == 0) write_token(p, r, best, top.x, mass1);
}

// The chunks of a row merged; rows with filters: their races (the first one is the chunks' where there is no top_k).  The threads' largest logits bound the
// kept prefix from behind: if k of them are at least v, no token below v has a rank below k.  Races then look at those sixteens alone whose largest logit is in front;
// a wave that finds few of them keeps their tokens in registers for the races that follow.
constexpr int kRowThreads = 1024, kRowBatch = 8;       // sixteens per thread that a pass looks at together
template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleParams p) {
    using L = Logits<TYPE>;
    constexpr int THREADS = kRowThreads;
    __shared__ RowReduce<THREADS> red;
    __shared__ uint16_t list[THREADS / 64][kRowBatch * 64];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(), V = p.vocab;
    const char *row = p.logits + r * p.stride * L::SIZE;
    const float *noise = p.noise + r * p.noise_stride;
    const RowRules rules(p, r);
    const SampleRecord *records = p.records + r * p.chunks;
    const float *tops = p.tops + r * p.chunks * kSampleThreads;
    const int groups = p.chunks * kSampleThreads;
    const bool races = !rules.greedy && rules.filters();
    float g[kRowBatch];
#pragma unroll
    for (int k = 0; k < kRowBatch; ++k) g[k] = races && k * THREADS + tid < groups ? tops[k * THREADS + tid] : -INFINITY;
    Best top = {-INFINITY, -INFINITY, -1};
    for (int c = tid; c < p.chunks; c += THREADS) {
        const Best o = {records[c].top, records[c].top, records[c].top_at};
        if (beats(o, top)) top = o;
    }
    top = red.first(top);
    if (top.index < 0) {
        if (tid == 0) write_token(p, r, top, 0.f, 1.f);
        return;
    }
    float mass1 = 0.f, mass = 0.f;
    Best best = kNobody;
    for (int c = tid; c < p.chunks; c += THREADS) {
        const SampleRecord o = records[c];
        if (o.top_at < 0) continue;
        const float d = o.top - top.x, y = d * rules.inv;
        mass1 += o.mass1 * fast_exp2(d * kLog2e);
        mass += o.massT * fast_exp2(y);
        enter(best, o.best, o.best_at, o.score * fast_exp2(y));
    }
    red.all(mass1, mass, best);
    if (rules.greedy) best = top;
    if (!races) {
        if (tid == 0) write_token(p, r, best, top.x, mass1);
        return;
    }
    constexpr int AT_ONCE = 64 / L::PIECES;     // sixteens that a wave looks at together: one lane per piece of 16 bytes
    float x[L::PIECE], w[L::PIECE], score[L::PIECE];
    int i = 0;
    bool kept = false;                          // (of the wave) x, w and score hold every token that can still be in front
    auto load_piece = [&](int at) {
        i = L::index(at / kSampleThreads, kSampleThreads, at % kSampleThreads, lane % L::PIECES * L::PIECE);
        float u[L::PIECE];
        L::piece(row, i, V, x);
        if (i + L::PIECE <= V) {
            __builtin_memcpy(u, noise + i, 4 * L::PIECE);
        } else {
#pragma unroll
            for (int e = 0; e < L::PIECE; ++e) u[e] = i + e < V ? noise[i + e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < L::PIECE; ++e) {
            w[e] = fast_exp2((x[e] - top.x) * rules.inv);
            score[e] = w[e] * race_factor(u[e]);
        }
    };
    // tokens in front of (x, i): a race among them, their number and mass
    auto race = [&](float cut_x, int cut_i, float &count, float &front) {
        Best mine = kNobody;
        count = front = 0.f;
        auto look = [&] {
#pragma unroll
            for (int e = 0; e < L::PIECE; ++e) {
                const bool in = (x[e] > cut_x || (x[e] == cut_x && i + e < cut_i)) && w[e] >= rules.min_p && x[e] > -INFINITY;
                front += in ? w[e] : 0.f;
                count += in ? 1.f : 0.f;
                // (the list is not in the order of the tokens)
                if (in && (score[e] > mine.score || (score[e] == mine.score && (unsigned)(i + e) < (unsigned)mine.index))) mine = {score[e], x[e], i + e};
            }
        };
        if (kept) {
            look();
        } else {
            for (int base = 0; base < groups; base += kRowBatch * THREADS) {
                int listed = 0;
#pragma unroll
                for (int k = 0; k < kRowBatch; ++k) {
                    const int at = base + k * THREADS + tid;
                    const float t = base == 0 ? g[k] : at < groups ? tops[at] : -INFINITY;
                    const bool in = t >= cut_x && t > -INFINITY;
                    const uint64_t who = __builtin_amdgcn_ballot_w64(in);
                    if (in) list[wave][listed + __builtin_popcountll(who & ((1ull << lane) - 1))] = (uint16_t)(k * THREADS + tid);
                    listed += __builtin_popcountll(who);
                }
                // (a wave reads what it wrote)
                kept = listed <= AT_ONCE && groups <= kRowBatch * THREADS;
                for (int k = 0; k < listed; k += AT_ONCE) {
                    const int which = k + lane / L::PIECES;
                    if (which < listed) {
                        load_piece(base + list[wave][which]);
                        look();
                    }
                }
                if (kept && lane / L::PIECES >= listed) {
#pragma unroll
                    for (int e = 0; e < L::PIECE; ++e) x[e] = -INFINITY;
                }
            }
        }
        red.all(front, count, mine);
        return mine;
    };
    float count, front;
    if (rules.top_k > 0) best = race(red.reached_by(g, (uint32_t)rules.top_k), 0x7fffffff, count, front);
    while (best.index != top.index && best.index >= 0) {
        const Best next = race(best.x, best.index, count, front);
        if (rules.keeps(count, front, mass, fast_exp2((best.x - top.x) * rules.inv))) break;
        best = next;
    }
    if (best.index < 0) best = top;            // (a min_p that nothing reaches)
    if (tid == 0) write_token(p, r, best, top.x, mass1);
}

}  // namespace sa2
