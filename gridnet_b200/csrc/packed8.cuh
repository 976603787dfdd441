// Activations held in 8 bits: groups of 32 values of a row share a power of two.
//
// For a group with the largest finite magnitude m, e is the smallest whole number >= -126 with m <= 125 * 2^e; a value x is held
// as the code round(x / 2^e), half to even, in [-125, 125]. x / 2^e is exact (up to values that round to 0 anyway), so the
// code depends on x alone, not on the order or kind of any arithmetic. Codes 127, -127 and -128 stand for +inf, -inf and NaN:
// what is not finite stays what it is and touches no neighbour. The group's scale byte is e + 127, the exponent field
// of the float 2^e, in [1, 249]. At the largest e, 122, codes end at 63: 64 * 2^122 is no float, and what is
// finite stays so. 33 bytes hold 32 values; a value is off by at most 2^(e-1) < m / 125 (m / 250 where m is just below 125 * 2^e), but for the two
// ends: at e = 122 a value beyond 63.5 * 2^122 is off by up to 2^122, and at e = -126 the bound 2^-127 may be all of a value.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include "common.cuh"

namespace gn {

constexpr int kPackGroup = 32;

// ---- values of the three types as floats, four at a time (vec: 4-element aligned, all four there)
template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void load4v(const float *p, float (&v)[4])
{
    const float4 q = *reinterpret_cast<const float4 *>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
}
__device__ __forceinline__ void load4v(const __nv_bfloat16 *p, float (&v)[4])
{
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    v[0] = __uint_as_float(q.x << 16); v[1] = __uint_as_float(q.x & 0xffff0000u);
    v[2] = __uint_as_float(q.y << 16); v[3] = __uint_as_float(q.y & 0xffff0000u);
}
__device__ __forceinline__ void load4v(const __half *p, float (&v)[4])
{
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&q.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&q.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ void store4v(float *p, const float (&v)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4v(__nv_bfloat16 *p, const float (&v)[4])
{
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    uint2 q;
    q.x = *reinterpret_cast<const unsigned *>(&a);
    q.y = *reinterpret_cast<const unsigned *>(&b);
    *reinterpret_cast<uint2 *>(p) = q;
}
__device__ __forceinline__ void store4v(__half *p, const float (&v)[4])
{
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    uint2 q;
    q.x = *reinterpret_cast<const unsigned *>(&a);
    q.y = *reinterpret_cast<const unsigned *>(&b);
    *reinterpret_cast<uint2 *>(p) = q;
}
// n: how many of the four are there (what is not reads as 0)
template <typename T>
__device__ __forceinline__ void load4(const T *p, bool vec, int n, float (&v)[4])
{
    if (vec && n == 4) {
        load4v(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? to_float<T>(p[i]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store4(T *p, bool vec, int n, const float (&v)[4])
{
    if (vec && n == 4) {
        store4v(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = from_float<T>(v[i]);
}

// ---- the format
__device__ __forceinline__ unsigned magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ bool bits_finite(unsigned m) { return m < 0x7f800000u; }

// scale byte of a group whose largest finite magnitude has these bits: 125 / 64 = 1.953125 = mantissa 0x7a0000
__device__ __forceinline__ unsigned pack_scale(unsigned m)
{
    const int b = (int)(m >> 23) - 6 + ((m & 0x7fffffu) > 0x7a0000u ? 1 : 0);
    return (unsigned)max(b, 1);
}
__device__ __forceinline__ float pack_inverse(unsigned scale) { return __uint_as_float((254u - scale) << 23); }
__device__ __forceinline__ float pack_step(unsigned scale) { return __uint_as_float(scale << 23); }

// the code of a finite x in the low byte: adding 1.5 * 2^23 rounds to a whole number, half to even
__device__ __forceinline__ unsigned pack_code(float x, float inverse) { return __float_as_uint(fmaf(x, inverse, 12582912.0f)); }
constexpr unsigned kPackLargest = 0x7f7a0000u;  // 125 * 2^121: beyond it a group's 2^e is 2^122, and 64 * 2^122 is no float
__device__ __forceinline__ unsigned pack_code_any(float x, unsigned scale)
{
    const unsigned m = magnitude_bits(x);
    if (bits_finite(m)) {
        const float most = scale == 249u ? 63.0f * pack_step(scale) : FLT_MAX;
        return pack_code(fminf(fmaxf(x, -most), most), pack_inverse(scale)) & 0xffu;
    }
    if (m > 0x7f800000u) return 0x80u;
    return x > 0.0f ? 0x7fu : 0x81u;
}
__device__ __forceinline__ unsigned pack_word(unsigned a, unsigned b, unsigned c, unsigned d)  // the low bytes
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// largest over the eight lanes 8k .. 8k+7 of a warp
__device__ __forceinline__ unsigned max_of_8_lanes(unsigned m)
{
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// Four values of a group that eight lanes hold together (all 32 lanes of the warp call) -> the four codes and the scale byte
__device__ __forceinline__ unsigned pack_group(const float (&x)[4], unsigned &scale)
{
    unsigned m = max(max(magnitude_bits(x[0]), magnitude_bits(x[1])), max(magnitude_bits(x[2]), magnitude_bits(x[3])));
    m = max_of_8_lanes(m);
    if (__any_sync(0xffffffffu, m > kPackLargest)) {  // rare: once more over what is finite
        m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned b = magnitude_bits(x[i]);
            if (bits_finite(b)) m = max(m, b);
        }
        m = max_of_8_lanes(m);
        scale = pack_scale(m);
        return pack_word(pack_code_any(x[0], scale), pack_code_any(x[1], scale), pack_code_any(x[2], scale), pack_code_any(x[3], scale));
    }
    scale = pack_scale(m);
    const float inv = pack_inverse(scale);
    return pack_word(pack_code(x[0], inv), pack_code(x[1], inv), pack_code(x[2], inv), pack_code(x[3], inv));
}

__device__ __forceinline__ float unpack_special(float v, unsigned code)
{
    return code == 0x7fu ? __uint_as_float(0x7f800000u) : code == 0x81u ? __uint_as_float(0xff800000u)
         : code == 0x80u ? __uint_as_float(0x7fc00000u) : v;
}
// four codes, all of them of finite values, as whole numbers
__device__ __forceinline__ void unpack4_finite(unsigned word, float (&v)[4])
{
    const unsigned w = word ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i)  // 2^23 + (code + 128), as a float, less 2^23 + 128: exact
        v[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)) - 8388736.0f;
}
// not 0 where one of the four stands for what is not finite
__device__ __forceinline__ unsigned unpack_odd(unsigned word)
{
    // code + 129 as a byte: 0, 1 and 2 stand for what is not finite, 4 .. 254 for the rest
    const unsigned w = word ^ 0x80808080u, up = (((w & 0x7f7f7f7fu) + 0x01010101u) ^ (w & 0x80808080u)) & 0xfcfcfcfcu;
    return (up - 0x01010101u) & ~up & 0x80808080u;  // a byte of 0
}
// four codes -> the values they stand for
__device__ __forceinline__ void unpack4(unsigned word, float step, float (&v)[4])
{
    unpack4_finite(word, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= step;
    if (unpack_odd(word)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = unpack_special(v[i], (word >> (8 * i)) & 0xffu);
    }
}
__device__ __forceinline__ float unpack1(unsigned code, float step) { return unpack_special((float)(int)(signed char)code * step, code & 0xffu); }

// The bytes of four codes at p, n of them there
__device__ __forceinline__ unsigned load_codes(const unsigned char *p, bool vec, int n)
{
    if (vec && n == 4) return *reinterpret_cast<const unsigned *>(p);
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) w |= (unsigned)p[i] << (8 * i);
    return w;
}
__device__ __forceinline__ void store_codes(unsigned char *p, bool vec, int n, unsigned w)
{
    if (vec && n == 4) {
        *reinterpret_cast<unsigned *>(p) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = (unsigned char)(w >> (8 * i));
}

}  // namespace gn
