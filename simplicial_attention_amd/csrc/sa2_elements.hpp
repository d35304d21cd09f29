// Eight consecutive elements of a bf16, fp16 or fp32 row as floats, and back, at any alignment (the ISA takes unaligned vector accesses).
#pragma once

#include "sa2_common.hpp"

namespace sa2 {

// element types as sa2_element names them
constexpr int kBf16 = 0, kF16 = 1, kF32 = 2;
template <int T>
constexpr int element_size = T == kF32 ? 4 : 2;

typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u32x4 ld_any16(const char *p) { return *reinterpret_cast<const u32x4_any *>(p); }
__device__ __forceinline__ void st_any16(char *p, u32x4 v) { *reinterpret_cast<u32x4_any *>(p) = v; }

template <int T>
__device__ __forceinline__ float element_f32(const char *p) {
    if constexpr (T == kF32) return *reinterpret_cast<const float *>(p);
    else if constexpr (T == kF16) return (float)*reinterpret_cast<const _Float16 *>(p);
    else return as_f32((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16);
}

// x rounded to the type (nearest even)
template <int T>
__device__ __forceinline__ float rounded(float x) {
    if constexpr (T == kF32) return x;
    else if constexpr (T == kF16) return (float)(_Float16)x;
    else return (float)(__bf16)x;
}

template <int T>
__device__ __forceinline__ void put_element(char *p, float x) {
    if constexpr (T == kF32) *reinterpret_cast<float *>(p) = x;
    else if constexpr (T == kF16) *reinterpret_cast<_Float16 *>(p) = (_Float16)x;
    else *reinterpret_cast<__bf16 *>(p) = (__bf16)x;
}

// eight elements as they lie in memory, and what they are (kept apart so that several loads can be under way)
template <int T>
struct Raw8 {
    u32x4 a, b;      // b: fp32 only
};

template <int T>
__device__ __forceinline__ Raw8<T> ld_raw8(const char *p) {
    Raw8<T> r;
    r.a = ld_any16(p);
    if constexpr (T == kF32) r.b = ld_any16(p + 16);
    return r;
}

template <int T>
__device__ __forceinline__ void widen8(const Raw8<T> &r, float (&v)[8]) {
    if constexpr (T == kF32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = as_f32(r.a[i]), v[4 + i] = as_f32(r.b[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kF16) {
                const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)r.a[i]);
                v[2 * i] = (float)h[0], v[2 * i + 1] = (float)h[1];
            } else {
                v[2 * i] = bf16_lo(r.a[i]), v[2 * i + 1] = bf16_hi(r.a[i]);
            }
        }
    }
}

// the first `count` (1 .. 8) of eight elements; the others read as zero
template <int T>
__device__ __forceinline__ void ld_some8(const char *p, int count, float (&v)[8]) {
    if (count >= 8) {
        widen8<T>(ld_raw8<T>(p), v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < count ? element_f32<T>(p + i * element_size<T>) : 0.f;
    }
}
__device__ __forceinline__ void ld_some8(int type, const char *p, int count, float (&v)[8]) {
    if (type == kBf16) ld_some8<kBf16>(p, count, v);
    else if (type == kF16) ld_some8<kF16>(p, count, v);
    else ld_some8<kF32>(p, count, v);
}

// eight floats as bf16 or fp16
template <int T>
__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (T == kF16) {
            const f16x2 h = {(_Float16)v[2 * i], (_Float16)v[2 * i + 1]};
            o[i] = __builtin_bit_cast(uint32_t, h);
        } else {
            o[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        }
    }
    return o;
}

// four
template <int T>
__device__ __forceinline__ u32x2 pack4(const float (&v)[4]) {
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (T == kF16) {
            const f16x2 h = {(_Float16)v[2 * i], (_Float16)v[2 * i + 1]};
            w[i] = __builtin_bit_cast(uint32_t, h);
        } else {
            w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        }
    }
    return w;
}

template <int T>
__device__ __forceinline__ void st_some8(char *p, int count, const float (&v)[8]) {
    if (count >= 8) {
        if constexpr (T == kF32) {
            st_any16(p, (u32x4){as_u32(v[0]), as_u32(v[1]), as_u32(v[2]), as_u32(v[3])});
            st_any16(p + 16, (u32x4){as_u32(v[4]), as_u32(v[5]), as_u32(v[6]), as_u32(v[7])});
        } else {
            st_any16(p, pack8<T>(v));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < count) put_element<T>(p + i * element_size<T>, v[i]);
    }
}

// the first `count` (1 .. N) of N = 4 or 8 elements
template <int T, int N>
__device__ __forceinline__ void ld_some(const char *p, int count, float (&v)[N]) {
    if constexpr (N == 8) {
        ld_some8<T>(p, count, v);
    } else {
        static_assert(N == 4, "pieces of four or eight");
        if (count >= 4) {
            if constexpr (T == kF32) {
                const u32x4 w = ld_any16(p);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = as_f32(w[i]);
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2_any *>(p);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (T == kF16) {
                        const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)w[i]);
                        v[2 * i] = (float)h[0], v[2 * i + 1] = (float)h[1];
                    } else {
                        v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = i < count ? element_f32<T>(p + i * element_size<T>) : 0.f;
        }
    }
}
template <int T, int N>
__device__ __forceinline__ void st_some(char *p, int count, const float (&v)[N]) {
    if constexpr (N == 8) {
        st_some8<T>(p, count, v);
    } else {
        if (count >= 4) {
            if constexpr (T == kF32) {
                st_any16(p, (u32x4){as_u32(v[0]), as_u32(v[1]), as_u32(v[2]), as_u32(v[3])});
            } else {
                *reinterpret_cast<u32x2_any *>(p) = pack4<T>(v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < count) put_element<T>(p + i * element_size<T>, v[i]);
        }
    }
}

// four floats in e4m3, round to nearest even (v_cvt_pk_fp8_f32)
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// four e4m3 values as floats
__device__ __forceinline__ void unpack_e4m3(uint32_t w, float *v) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
}

// The larger of two magnitudes given as bits: numbers that are not numbers count as larger than infinity, so a maximum keeps them.
__device__ __forceinline__ uint32_t magnitude(float x) { return as_u32(x) & 0x7fffffffu; }

// reductions over L consecutive lanes (a power of two up to 64), the result in all of them
template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
    for (int off = L / 2; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
    return x;
}
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
#pragma unroll
    for (int off = L / 2; off >= 1; off >>= 1) {
        const uint32_t y = (uint32_t)__shfl_xor((int)x, off, 64);
        x = x > y ? x : y;
    }
    return x;
}

}  // namespace sa2
