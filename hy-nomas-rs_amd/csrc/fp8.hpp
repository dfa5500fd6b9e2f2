// 8-bit values (e4m3: 1 + 4 + 3 bits, largest 448) with an f32 scale for each block of
// 128: along a row (activations: 1 x 128) or a square (weights: 128 x 128).
//   scale = max(amax / 448, 2^-126), the nearest f32     q = e4m3(x / scale)
// A block that holds an infinity or a NaN has scale NaN and values NaN, so that
// every sum it enters says so.
#pragma once

#include "kernels.hpp"

namespace nomas {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

// From the largest magnitude's bits (those of infinities and NaN are above all others).
__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    return fmaxf(__uint_as_float(amax_bits) / 448.0f, 0x1p-126f);
}

// x / scale rounded to e4m3 once.  The quotient in f32 would be rounded twice, and
// quotients of 16-bit values are often next to the middle of two e4m3 (one of 1,000
// values of a bf16 tensor came out a step off).  So the f32 quotient is rounded to odd:
// where it is not exact it takes, of the two f32 next to the true one, the one whose last
// bit is set, which is on the true one's side of every middle.
struct Fp8Quot {
    float up, s, r;  // (blocks of tiny scales are taken times 2^64: the remainder is then no subnormal)
    __device__ __forceinline__ explicit Fp8Quot(float scale) {
        up = scale < 0x1p-60f ? 0x1p64f : 1.0f;
        s = scale * up;
        r = __builtin_amdgcn_rcpf(s);  // within 1 ulp
    }
    __device__ __forceinline__ float operator()(float v) const {
        const float x = v * up;
        float q = x * r;
        q = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);  // the true quotient or a neighbour of it
        const float e = __builtin_fmaf(-q, s, x);             // has the sign of (true - q) s
        const uint32_t b = __float_as_uint(q);
        // towards the true one, if the last bit is not set: away from zero or towards it
        const bool grow = ((__float_as_uint(e) ^ b) >> 31) == 0;
        const uint32_t odd = grow ? (b | 1u) : b - 1u + (b & 1u);
        return __uint_as_float(e == 0.0f || !(e == e) ? b : odd);
    }
};

// Four values as e4m3, the first in the lowest byte (round to nearest even).
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_maxu(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xf, 0xf, true));
}
// The largest over each 16 neighbouring lanes, in all of them.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = dpp_maxu<0xb1>(v);
    v = dpp_maxu<0x4e>(v);
    v = dpp_maxu<0x141>(v);
    return dpp_maxu<0x140>(v);
}

}  // namespace nomas
