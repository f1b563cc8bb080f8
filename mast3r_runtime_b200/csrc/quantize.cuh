// Values to 8 bits with a scale for each row, shared by the row kernels and the 8-bit product.
#pragma once

#include "common.cuh"

namespace m3r {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) {
    return __bfloat162float(v);
}

// The integer nearest to 127 v / a, ties to even, decided by the two exact products 254 v and
// (2 m + 1) a on either side of a half.
static __device__ __noinline__ int quantize_exact(float v, float p, float a) {
    const float lo = floorf(p);
    const double d = 254.0 * static_cast<double>(v) - (2.0 * static_cast<double>(lo) + 1.0) * static_cast<double>(a);
    const int l = static_cast<int>(lo);
    return d > 0.0 ? l + 1 : d < 0.0 ? l : (l & 1) ? l + 1 : l;
}

// A row's scaling to 8 bits.  The row is first scaled by a power of two that keeps 127 v and 1 / a
// away from the ends of the 32-bit range; k = 127 times that power.
struct Quantizer {
    float a, top, k, inv;  // largest magnitude, the same scaled, 127 scaled, 1 / top
    __device__ __forceinline__ explicit Quantizer(float largest) : a(largest) {
        const float pre = a < 0x1p-60f ? 0x1p90f : a > 0x1p60f ? 0x1p-60f : 1.0f;
        top = a * pre;
        k = 127.0f * pre;
        inv = 1.0f / top;
    }
    // The quotient t / top for t = k v: for 16-bit v, t, the remainder and a quotient halfway between
    // two levels are exact in 32 bits, and any other quotient is 2^-19 away from half a level, so that
    // one correction makes its nearest integer the right one.
    __device__ __forceinline__ uint64_t quotient16(uint64_t v) const {  // two values
        const uint64_t t = mul2(v, pair(k, k)), i = pair(inv, inv), q = mul2(t, i);
        return fma2(fma2(q, pair(-top, -top), t), i, q);
    }
};

// Eight values in 8 bits: adding 1.5 * 2^23 rounds the quotient to the integer that then stands in
// the sum's low byte.  32-bit values: k v * inv lies within 3e-5 of 127 v / a (three roundings of a
// value up to 127), which decides unless it is that near to a half; one test for the eight, taken
// for about one value in 10^4, sends them to quantize_exact.
template <bool EXACT16>
__device__ __forceinline__ uint2 quantize8(const float* v, const Quantizer& z) {
    constexpr float kMagic = 12582912.0f;
    uint32_t b[8];
    if constexpr (EXACT16) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float2 t = unpair(add2(z.quotient16(pair(v[j], v[j + 1])), pair(kMagic, kMagic)));
            b[j] = __float_as_uint(t.x), b[j + 1] = __float_as_uint(t.y);
        }
    } else {
        float off = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint64_t p = mul2(mul2(pair(v[j], v[j + 1]), pair(z.k, z.k)), pair(z.inv, z.inv));
            const uint64_t t = add2(p, pair(kMagic, kMagic));
            const float2 d = unpair(fma2(add2(t, pair(-kMagic, -kMagic)), pair(-1.0f, -1.0f), p)), u = unpair(t);
            off = fmaxf(off, fmaxf(fabsf(d.x), fabsf(d.y)));
            b[j] = __float_as_uint(u.x), b[j + 1] = __float_as_uint(u.y);
        }
        if (off > 0.49996f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = v[j] * z.k * z.inv;
                if (fabsf(p - rintf(p)) > 0.49996f) b[j] = quantize_exact(v[j], p, z.a);
            }
        }
    }
    return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// The larger magnitude; NaN when either is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Largest magnitudes of a row as integers (NaN above infinity above every number): whether the row
// holds anything to quantise.  Rows without a finite, non-zero magnitude hold zeros: a zero scale
// gives zeros, an infinite or NaN one gives NaN in every product.
__device__ __forceinline__ bool live_magnitude(uint32_t top) { return top != 0 && top < 0x7F800000u; }

}  // namespace m3r
