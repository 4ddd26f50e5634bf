// cache8.hpp -- values held in 8 bits: int8 and e4m3 codes with one scale per row.
//
// A row x of one token and head is held as codes c and a scale s: x ~ c s with
//   int8: s = max|x| / 127, c = round(x / s)       e4m3: s = max|x| / 448, c = e4m3(x / s),
// both rounding half to even (the e4m3 conversion of the hardware does).  Rows whose largest
// magnitude is below 2^-100 (1 / s would overflow) are held as zeros with s = 0; a row that
// holds an Inf or NaN gets s = NaN and codes 0, so it reads back as NaN and no code is one.
#pragma once
#include "decode_kernels.hpp"

namespace kvc {
namespace {

constexpr int kCacheF16 = KVC_F16, kCacheI8 = KVC_I8, kCacheE4M3 = KVC_E4M3;

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <int CT> constexpr int kCodeBytes = CT == kCacheF16 ? 2 : 1;

// Four codes (one register) as two pairs of fp16, exactly: int8 is at most 127 in size, e4m3
// has three fraction bits and exponents within fp16's.
// int8: with the sign bit flipped a byte is c + 128, and 0x6400 | byte is the fp16 1024 + byte.
template <int CT>
__device__ __forceinline__ void codes_to_f16(unsigned x, f16x2& lo, f16x2& hi) {
    if constexpr (CT == kCacheI8) {
        const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
        x ^= 0x80808080u;
        lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - bias;
        hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - bias;
    } else {
        lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false));
        hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true));
    }
}

// Eight codes as eight fp16.
template <int CT>
__device__ __forceinline__ f16x8 codes_to_f16x8(u32x2 x) {
    f16x2 a, b, c, d;
    codes_to_f16<CT>(x[0], a, b);
    codes_to_f16<CT>(x[1], c, d);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Scale of a row from the bits of max|x| (as an integer, whose order is that of the
// magnitudes with NaN above Inf), and the factor that turns values into codes, as a sum of
// two floats: with one alone the quotient would be rounded twice.
template <int CT>
__device__ __forceinline__ void row_scale(unsigned amax_bits, float& s, f32x2& inv) {
    constexpr float kTop = CT == kCacheI8 ? 127.f : 448.f;
    const float a = __uint_as_float(amax_bits);
    s = a / kTop;
    inv[0] = kTop / a;
    inv[1] = __builtin_fmaf(-inv[0], a, kTop) * inv[0] * (1.f / kTop);
    if (amax_bits < 0x0D800000u) s = inv[0] = inv[1] = 0.f;  // 2^-100
    if (amax_bits >= 0x7F800000u) {
        s = __builtin_nanf("");
        inv[0] = inv[1] = 0.f;
    }
}

// Eight values times inv as codes.  (inv 0 with an Inf or NaN among x: codes 0.)
template <int CT>
__device__ __forceinline__ u32x2 values_to_codes(const float (&x)[8], f32x2 inv) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = inv[0] == 0.f ? 0.f : __builtin_fmaf(x[e], inv[0], x[e] * inv[1]);
    u32x2 c;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if constexpr (CT == kCacheI8) {
            unsigned r = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) r |= ((unsigned)(int)rintf(y[4 * w + e]) & 0xFFu) << (8 * e);
            c[w] = r;
        } else {
            int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w], y[4 * w + 1], 0, false);
            r = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w + 2], y[4 * w + 3], r, true);
            c[w] = (unsigned)r;
        }
    }
    return c;
}

__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ unsigned dpp_u(unsigned x) {
    return (unsigned)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true);
}
// Maximum over each aligned group of LPT (2 .. 16) consecutive lanes, in every lane.
template <int LPT>
__device__ __forceinline__ unsigned group_umax(unsigned x) {
    if constexpr (LPT >= 2) x = umax(x, dpp_u<0xB1>(x));
    if constexpr (LPT >= 4) x = umax(x, dpp_u<0x4E>(x));
    if constexpr (LPT >= 8) x = umax(x, dpp_u<0x141>(x));
    if constexpr (LPT >= 16) x = umax(x, dpp_u<0x140>(x));
    return x;
}
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

}  // namespace
}  // namespace kvc
