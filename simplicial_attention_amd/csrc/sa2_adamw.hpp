// One step of AdamW over many tensors in one launch, with states in 32 bits or in 8.
//
//   m' = b1 m + (1 - b1) g      v' = b2 v + (1 - b2) g^2      p' = (1 - lr wd) p - (lr / (1 - b1^n)) m' / (sqrt(v') / sqrt(1 - b2^n) + eps)
//
// States in 8 bits are e4m3 values with one fp32 scale per 256 consecutive elements, the largest magnitude being 448 times the scale; of v the
// root is kept, which halves the range that the exponent has to span.  An average that moves by a thousandth per step stands still
// if it is rounded to the nearest of values an eighth apart, so both are rounded stochastically: up with the probability that leaves
// the expectation as it is, from 16 random bits per state that are a hash of seed, step, tensor and element (nothing is kept for them, and a step
// can be repeated).  A root that is not zero never becomes zero: the quotient would have no bound.
//
// The list of tensors travels in the kernel's arguments; every workgroup takes one chunk of one tensor.  Bound by bytes: bf16
// parameters with fp32 masters move 28 bytes an element with states in 32 bits, 16 in 8 (12 layers of 512 channels, 37 M elements: 218 and 134 us, 4.8 and 4.5 TB/s).  States in 8 bits without
// masters move 10 and are bound by vector instructions, of which an element takes about 125, a third of them the correctly rounded root and quotient (118 us, 3.1 TB/s).  Every operation is rounded as written
// (no contraction), so results depend on neither the launch shape nor the order of the tensors' elements.
#pragma once

#include "sa2_elements.hpp"

namespace sa2 {

struct AdamTensor {
    char *p;
    const char *g;
    char *m, *v;                  // fp32, or e4m3
    float *ms, *vs;               // scales of 8-bit states
    float *master;                // or NULL
    int64_t n;
};

constexpr int kAdamTensors = 52;
struct AdamParams {
    AdamTensor tensor[kAdamTensors];
    int32_t first[kAdamTensors + 2];      // chunks in front of each tensor
    int count, chunk;                     // tensors, elements of a chunk (a multiple of 2048)
    uint32_t index[kAdamTensors];         // place of each in the caller's list
    uint32_t seed;
    // as numbers, or (step_at) read and formed on the device
    uint32_t step;
    float b1, c1, b2, c2, keep, rate, inv_root, eps;     // c = 1 - b, keep = 1 - lr wd, rate = lr / (1 - b1^n), inv_root = (1 - b2^n)^-1/2
    const int64_t *step_at;
    const float *lr_at, *grad_scale;
    double beta1, beta2, lr, decay;
};
static_assert(sizeof(AdamParams) <= 4096, "kernel arguments");

__device__ __forceinline__ uint32_t mixed_bits(uint32_t x) {      // the finalizer of MurmurHash3 (A. Appleby)
    x = (x ^ (x >> 16)) * 0x85ebca6bu;
    x = (x ^ (x >> 13)) * 0xc2b2ae35u;
    return x ^ (x >> 16);
}

// the magnitude t (0 .. 448) in e4m3, rounded up with the probability u / 2^16 where u is uniform
__device__ __forceinline__ uint32_t e4m3_code(float t, uint32_t u) {
#pragma clang fp contract(off)
    const uint32_t normal = ((as_u32(t) + (u << 4)) >> 20) - 960u;      // three bits behind the point, exponents from 2^-6 on
    const float part = (float)u * 0x1p-16f;
    const uint32_t small = (uint32_t)floorf(t * 512.f + part);          // below that in steps of 2^-9
    return min(t < 0x1p-6f ? small : normal, 126u);
}

template <int TP, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_kernel(AdamParams p) {
#pragma clang fp contract(off)
    __shared__ float made[3];
    const int lane = threadIdx.x & 63;
    // the tensor of this workgroup: the last one whose chunks begin at or in front of it
    const int blk = blockIdx.x;
    const bool le = lane < p.count && p.first[lane < p.count ? lane : 0] <= blk;
    const int which = uniform(__popcll(__ballot(le)) - 1);
    const AdamTensor &t = p.tensor[which];
    const int64_t begin = (int64_t)(blk - p.first[which]) * p.chunk, end = min(t.n, begin + p.chunk);

    float keep = p.keep, rate = p.rate, inv_root = p.inv_root;
    uint32_t step = p.step;
    if (p.step_at) {
        const int64_t n = *p.step_at;
        step = (uint32_t)n;
        if (threadIdx.x == 0) {
            const double lr = p.lr_at ? (double)*p.lr_at : p.lr;
            made[0] = (float)(1. - lr * p.decay);
            made[1] = (float)(lr / (1. - pow(p.beta1, (double)n)));
            made[2] = (float)(1. / sqrt(1. - pow(p.beta2, (double)n)));
        }
        __syncthreads();
        keep = made[0], rate = made[1], inv_root = made[2];
    } else if (p.lr_at) {
        const double lr = (double)*p.lr_at;
        keep = (float)(1. - lr * p.decay);
        rate = (float)(lr * (double)rate);          // (the host gave 1 / (1 - b1^n))
    }
    const float gs = p.grad_scale ? *p.grad_scale : 1.f;
    const uint32_t key = mixed_bits(mixed_bits(step + 0x9e3779b9u * (p.index[which] + 1u)) ^ p.seed);

    // (E consecutive elements a thread: four with fp32 states, whose accesses are whole lines of 16 bytes a lane then; eight of 8-bit ones)
    constexpr int E = EIGHT ? 8 : 4;
    for (int64_t at = begin + threadIdx.x * E; at - (int64_t)(threadIdx.x * E) < end; at += 256 * E) {
        const int count = (int)min((int64_t)E, end - at);          // (8-bit states: lanes behind the end go along in the reductions)
        float g[E], x[E], m[E], v[E], root[E];
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] = x[i] = m[i] = v[i] = 0.f;
        float ms = 0.f, vs = 0.f;
        if (count > 0) {
            ld_some<TP>(t.g + at * element_size<TP>, count, g);
            if (t.master) ld_some<kF32>(reinterpret_cast<const char *>(t.master + at), count, x);
            else ld_some<TP>(t.p + at * element_size<TP>, count, x);
            if constexpr (EIGHT) {
                ms = t.ms[at >> 8];
                vs = t.vs[at >> 8];
                u32x2 mw = {0, 0}, vw = {0, 0};
                if (count == 8) {
                    mw = *reinterpret_cast<const u32x2_any *>(t.m + at);
                    vw = *reinterpret_cast<const u32x2_any *>(t.v + at);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < count) {
                            mw[i >> 2] |= (uint32_t)(uint8_t)t.m[at + i] << (8 * (i & 3));
                            vw[i >> 2] |= (uint32_t)(uint8_t)t.v[at + i] << (8 * (i & 3));
                        }
                }
                unpack_e4m3(mw[0], m);
                unpack_e4m3(mw[1], m + 4);
                unpack_e4m3(vw[0], v);
                unpack_e4m3(vw[1], v + 4);
            } else {
                ld_some<kF32>(t.m + at * 4, count, m);
                ld_some<kF32>(t.v + at * 4, count, v);
            }
        }
        uint32_t m_most = 0, v_most = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (p.grad_scale) g[i] *= gs;
            if constexpr (EIGHT) {
                m[i] *= ms;
                v[i] *= vs;
                v[i] *= v[i];
            }
            m[i] = m[i] * p.b1 + g[i] * p.c1;
            v[i] = v[i] * p.b2 + g[i] * g[i] * p.c2;
            root[i] = sqrtf(v[i]);
            x[i] = x[i] * keep - m[i] / (root[i] * inv_root + p.eps) * rate;
            if constexpr (EIGHT) {
                m_most = max(m_most, i < count ? magnitude(m[i]) : 0u);
                v_most = max(v_most, i < count ? magnitude(root[i]) : 0u);
            }
        }
        if constexpr (EIGHT) {
            // the 32 lanes that hold a block of 256 elements
            m_most = lanes_max<32>(m_most);
            v_most = lanes_max<32>(v_most);
            const float mscale = m_most > 0x7f800000u ? as_f32(m_most) : fmaxf(as_f32(m_most) * (float)(1 / 448.), 0x1p-126f);
            const float vscale = v_most > 0x7f800000u ? as_f32(v_most) : fmaxf(as_f32(v_most) * (float)(1 / 448.), 0x1p-126f);
            const float minv = 1.f / mscale, vinv = 1.f / vscale;
            if (count > 0) {
                if ((lane & 31) == 0) {
                    t.ms[at >> 8] = mscale;
                    t.vs[at >> 8] = vscale;
                }
                u32x2 mw = {0, 0}, vw = {0, 0};
                const uint32_t k = key + (uint32_t)(at >> 32) * 0x9e3779b9u;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t random = mixed_bits(((uint32_t)at + i) ^ k);
                    const uint32_t mc = e4m3_code(fabsf(m[i]) * minv, random & 0xffffu) | (as_u32(m[i]) >> 31 << 7);
                    const uint32_t vc = max(e4m3_code(root[i] * vinv, random >> 16), root[i] > 0.f ? 1u : 0u);
                    mw[i >> 2] |= mc << (8 * (i & 3));
                    vw[i >> 2] |= vc << (8 * (i & 3));
                }
                if (count == 8) {
                    *reinterpret_cast<u32x2_any *>(t.m + at) = mw;
                    *reinterpret_cast<u32x2_any *>(t.v + at) = vw;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < count) {
                            t.m[at + i] = (char)(mw[i >> 2] >> (8 * (i & 3)));
                            t.v[at + i] = (char)(vw[i >> 2] >> (8 * (i & 3)));
                        }
                }
            }
        } else if (count > 0) {
            st_some<kF32>(t.m + at * 4, count, m);
            st_some<kF32>(t.v + at * 4, count, v);
        }
        if (count > 0) {
            if (t.master) st_some<kF32>(reinterpret_cast<char *>(t.master + at), count, x);
            st_some<TP>(t.p + at * element_size<TP>, count, x);
        }
    }
}

}  // namespace sa2
