// Next tokens from logits: temperature, top-k, top-p, min-p, from given random numbers.
//
// Order the tokens of a row by (logit descending, index ascending) and let p = softmax(logit / T).  A token is kept if its rank is below
// top_k, the mass in front of it below top_p, and p at least min_p times the largest; every one of these keeps a prefix of the order, so
// the kept tokens are a prefix too.  The token is the kept one with the largest  logit / T - log(-log u),  which draws from p restricted to the
// prefix.  No sort: the best of ALL tokens is the answer if it is kept, and otherwise nothing behind it is, so the race is run again among the tokens
// in front of it.  Whether a token is kept takes two sums over the tokens in front of it, formed in the pass that runs the next race.
// Each race that fails leaves a uniformly drawn share of the mass, so their number grows with the logarithm of the vocabulary at most.
#pragma once

#include "sa2_common.hpp"

namespace sa2 {

struct SampleParams {
    const char *logits;
    int64_t stride;               // elements
    const float *noise;
    int64_t noise_stride;
    const float *temperature, *top_p, *min_p;      // per row, or nullptr: the number below
    const int32_t *top_k;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int vocab;
    int64_t *tokens;
    float *logprobs;
};

constexpr float kMostFloat = 3.402823466e38f;
template <int TYPE>
__device__ __forceinline__ float logit_at(const char *row, int i) {
    float x;
    if constexpr (TYPE == 2) x = reinterpret_cast<const float *>(row)[i];
    else {
        const uint16_t w = reinterpret_cast<const uint16_t *>(row)[i];
        x = TYPE == 1 ? (float)__builtin_bit_cast(_Float16, w) : as_f32((uint32_t)w << 16);
    }
    // (not a number: never drawn; infinity: the largest number)
    return x != x ? -INFINITY : fminf(x, kMostFloat);
}

// -log(-log u), u held inside (0, 1)
__device__ __forceinline__ float gumbel(float u) { return -logf(-logf(fminf(fmaxf(u, 1.17549435e-38f), 0.99999994f))); }

struct Best {
    float score, x;
    int index;                    // -1: none
};
__device__ __forceinline__ bool beats(const Best &a, const Best &b) {
    if (a.index < 0 || b.index < 0) return b.index < 0 && a.index >= 0;
    return a.score > b.score || (a.score == b.score && a.index < b.index);
}

template <int THREADS>
struct RowReduce {
    static constexpr int NW = THREADS / 64;
    float f[NW];
    Best best[NW];
    template <typename OP>
    __device__ float all(float v, OP op) {
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) v = op(v, __shfl_xor(v, m));
        if (NW == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) f[threadIdx.x >> 6] = v;
        __syncthreads();
        v = f[0];
        for (int w = 1; w < NW; ++w) v = op(v, f[w]);
        return v;
    }
    __device__ Best all(Best v) {
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) {
            const Best o = {__shfl_xor(v.score, m), __shfl_xor(v.x, m), __shfl_xor(v.index, m)};
            if (beats(o, v)) v = o;
        }
        if (NW == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = v;
        __syncthreads();
        v = best[0];
        for (int w = 1; w < NW; ++w)
            if (beats(best[w], v)) v = best[w];
        return v;
    }
};

template <int TYPE, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleParams p) {
    __shared__ RowReduce<THREADS> red;
    const int64_t r = blockIdx.x;
    const int V = p.vocab;
    const char *row = p.logits + r * p.stride * (TYPE == 2 ? 4 : 2);
    const float *noise = p.noise + r * p.noise_stride;
    const float T = p.temperature ? p.temperature[r] : p.temperature_all;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p_all, min_p = p.min_p ? p.min_p[r] : p.min_p_all;
    const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    const auto add = [](float a, float b) { return a + b; };

    // the largest logit, in front of all others in the order
    Best top = {-INFINITY, 0.f, -1};
    for (int i = threadIdx.x; i < V; i += THREADS) {
        const float x = logit_at<TYPE>(row, i);
        const Best o = {x, x, i};
        if (x > -INFINITY && beats(o, top)) top = o;
    }
    top = red.all(top);
    if (top.index < 0) {                      // nothing to draw from
        if (threadIdx.x == 0) {
            p.tokens[r] = -1;
            p.logprobs[r] = -INFINITY;
        }
        return;
    }
    const bool greedy = !(T > 0.f);
    const float inv = greedy ? 0.f : fminf(1.f / T, kMostFloat);
    Best best = top;
    float sum = 0.f, mass = 0.f;
    Best mine = {0.f, 0.f, -1};
    for (int i = threadIdx.x; i < V; i += THREADS) {
        const float x = logit_at<TYPE>(row, i);
        if (!(x > -INFINITY)) continue;
        sum += expf(x - top.x);
        if (greedy) continue;
        const float y = (x - top.x) * inv, e = expf(y);
        mass += e;
        if (e >= min_p || i == top.index) {
            const Best o = {y + gumbel(noise[i]), x, i};
            if (beats(o, mine)) mine = o;
        }
    }
    sum = red.all(sum, add);
    if (!greedy) {
        mass = red.all(mass, add);
        best = red.all(mine);
        while (best.index != top.index && (top_k > 0 || top_p < 1.f)) {
            float front = 0.f, count = 0.f;   // (counts up to 2^24 are exact)
            mine = {0.f, 0.f, -1};
            for (int i = threadIdx.x; i < V; i += THREADS) {
                const float x = logit_at<TYPE>(row, i);
                if (!(x > best.x || (x == best.x && i < best.index))) continue;
                const float y = (x - top.x) * inv, e = expf(y);
                front += e;
                count += 1.f;
                const Best o = {y + gumbel(noise[i]), x, i};
                if (beats(o, mine)) mine = o;
            }
            front = red.all(front, add);
            count = red.all(count, add);
            if ((top_k <= 0 || count < (float)top_k) && (top_p >= 1.f || front < top_p * mass)) break;
            best = red.all(mine);
        }
    }
    if (threadIdx.x == 0) {
        p.tokens[r] = best.index;
        p.logprobs[r] = best.x - top.x - logf(sum);
    }
}

}  // namespace sa2
