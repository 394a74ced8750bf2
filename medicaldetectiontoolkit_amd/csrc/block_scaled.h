// block_scaled.h -- the block-scaled number formats shared by block_scaled.hip, act8_backward.hip and mx4_linear.hip (gfx950).
//
// 32 consecutive values share one power of two 2^e.  With m the block's largest magnitude, e is the smallest exponent >= -127 for which
// m <= Q * 2^e, so that no value is clipped: Q = 255 (8-bit codes of a ReLU's output), 127 (signed 8-bit codes), 6 (4-bit codes, the
// magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6).  A value is rounded to the nearest code, ties to the even one; a positive ReLU output keeps at
// least the code 1, so code > 0 IS the ReLU's mask.  The scale byte is e + 127; 255 marks a block with an infinity or a NaN, all of whose
// values read back as NaN (its ReLU codes still hold the mask).
//
// Why a power of two: code * 2^e has at most 8 significant bits and is therefore exact in bf16 and fp32, so products of the kept values
// run on the bf16 (fp4) matrix units without a further rounding.
#ifndef MDT_BLOCK_SCALED_H
#define MDT_BLOCK_SCALED_H

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <type_traits>
#include "mdt_hip.h"

namespace mdt_bs {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));

constexpr int BLOCK = 32;
constexpr unsigned INF_BITS = 0x7f800000u;
constexpr float FLT_BIG = 3.402823466e38f;

// Q = significand * 2^shift with 1 <= significand < 2: m / Q in terms of m's bits is (exponent - shift), plus one where m's fraction is larger
// than the significand's.  Adding (fraction mask - Q's fraction) carries into the exponent exactly then.
struct Q255 { static constexpr unsigned frac = 0x7f0000u; static constexpr int shift = 7; };
struct Q127 { static constexpr unsigned frac = 0x7e0000u; static constexpr int shift = 6; };
struct Q6 { static constexpr unsigned frac = 0x400000u; static constexpr int shift = 2; };

// the scale byte of a block whose largest magnitude has the bits mb
template <class Q>
__device__ __forceinline__ int scale_byte(unsigned mb)
{
    const int b = (int)((mb + (0x7fffffu - Q::frac)) >> 23) - Q::shift;
    return mb >= INF_BITS ? 255 : (b > 0 ? b : 0);
}
// 2^-e and 2^e of a finite block's scale byte (b <= 253: 2^-e is normal; b = 0 gives the subnormal 2^-127)
__device__ __forceinline__ float inv_scale(int b) { return __uint_as_float((unsigned)(254 - b) << 23); }
__device__ __forceinline__ float scale_of(int b) { return __uint_as_float(b == 255 ? 0x7fc00000u : b == 0 ? 0x00400000u : (unsigned)b << 23); }

__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true); }
// the maximum over aligned groups of 4 (quad permutes) or 8 lanes (plus the mirror within half a row)
template <int LANES>
__device__ __forceinline__ unsigned group_max(unsigned v)
{
    v = umax(v, dpp<0xb1>(v));                  // lanes 1 0 3 2
    v = umax(v, dpp<0x4e>(v));                  // lanes 2 3 0 1
    if (LANES == 8) v = umax(v, dpp<0x141>(v)); // row_half_mirror
    return v;
}

// n / d for 0 <= n < 2^31 by a multiplication (d >= 1), Granlund and Montgomery's division by an invariant integer: m = floor(2^32 (2^s - d) / d) + 1 with s = ceil(log2 d)
struct FastDiv {
    unsigned d, mul, shift;
    __host__ explicit FastDiv(unsigned dd = 1) : d(dd)
    {
        unsigned s = 0;
        while (s < 32 && (1ull << s) < dd) ++s;
        shift = s;
        mul = (unsigned)((((1ull << s) - dd) << 32) / dd) + 1u;
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return (unsigned)(((unsigned long long)__umulhi(n, mul) + n) >> shift); }
};

// the three float types; loads and stores of GV = 16 / sizeof(T) values, at any alignment of T
template <typename T> struct Io;
template <> struct Io<float> {
    static constexpr int GV = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ float to_f(float v) { return v; }
    static __device__ __forceinline__ float from_f(float v) { return v; }
};
template <> struct Io<__bf16> {
    static constexpr int GV = 8;
    typedef __bf16 vec __attribute__((ext_vector_type(8), aligned(2)));
    static __device__ __forceinline__ float to_f(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 from_f(float v) { return (__bf16)v; }
};
template <> struct Io<_Float16> {
    static constexpr int GV = 8;
    typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
    static __device__ __forceinline__ float to_f(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 from_f(float v) { return (_Float16)v; }
};
// the largest finite value: reading back a code that was rounded up across it saturates (a block whose maximum is in the top half-step of the type)
template <typename T> struct Largest { static constexpr float v = FLT_BIG; };
template <> struct Largest<__bf16> { static constexpr float v = 3.3895314e38f; };
template <> struct Largest<_Float16> { static constexpr float v = 65504.0f; };

template <typename T>
__device__ __forceinline__ T read_back(float code, int b)
{
    float v = code * scale_of(b);
    const float big = Largest<T>::v;
    v = v > big ? big : v < -big ? -big : v;    // NaN stays
    return Io<T>::from_f(v);
}

// one lane's GV values of a 4-bit block held by 32 / GV lanes -> its GV / 2 bytes of codes (the conversion rounds to nearest even) and the block's scale byte
template <int GV>
__device__ __forceinline__ unsigned quantize4_group(const float (&v)[GV], int &b)
{
    unsigned mb = 0;
#pragma unroll
    for (int j = 0; j < GV; ++j) mb = umax(mb, __float_as_uint(v[j]) & 0x7fffffffu);
    mb = group_max<BLOCK / GV>(mb);
    b = scale_byte<Q6>(mb);
    const float s = scale_of(b == 255 ? 127 : b);
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    if (GV == 8) {
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[GV - 4], v[GV - 3], s, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[GV - 2], v[GV - 1], s, 3);
    }
    return b == 255 ? 0u : w;
}

inline int launch_check()
{
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return MDT_OK;
    if (getenv("MDT_VERBOSE")) fprintf(stderr, "libmdt_hip: HIP error %d (%s)\n", (int)e, hipGetErrorString(e));
    return MDT_ERR_LAUNCH_FAILED;
}

}  // namespace mdt_bs

#endif
