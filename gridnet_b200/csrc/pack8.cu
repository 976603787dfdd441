// Packing of activations to 8 bits and back (packed8.cuh has the format), as calls of their own.
//
// Bytes: a float value is 4 read and 1.03 written, or the other way round; a few operations each, so HBM is what bounds both.
// Eight lanes hold a group, four values each.
#include "kernels.h"
#include "packed8.cuh"

namespace gn {

// rows x cols values; group j of a row: values 32 j .. of that row, the last one as many as there are
template <typename T>
__global__ void __launch_bounds__(256) pack8_k(const T *__restrict__ x, unsigned char *__restrict__ codes, unsigned char *__restrict__ scales,
                                               long long groups, long long per_row, long long cols, int vec)
{
    const int lane8 = threadIdx.x & 7;
    const long long stride = (long long)gridDim.x * 32;
    // whole warps stay together: the groups of a warp are four in a row
    for (long long g0 = (long long)blockIdx.x * 32 + (threadIdx.x >> 5) * 4; g0 < groups; g0 += stride) {
        const long long g = g0 + ((threadIdx.x & 31) >> 3);
        const long long row = g / per_row, col = (g - row * per_row) * kPackGroup + lane8 * 4;
        const int n = g < groups ? (int)min(4LL, max(0LL, cols - col)) : 0;
        const long long at = row * cols + col;
        float v[4];
        load4(x + at, vec, n, v);
        unsigned scale;
        const unsigned w = pack_group(v, scale);
        store_codes(codes + at, vec, n, w);
        if (lane8 == 0 && g < groups) scales[g] = (unsigned char)scale;
    }
}

// The largest halves have codes that stand for 65536, which is no half and would be rounded to an infinity: 65504 again. Codes for more than that are
// not of halves, and rounded like any float
template <typename T>
__device__ __forceinline__ float held_by(float v) { return v; }
template <>
__device__ __forceinline__ float held_by<__half>(float v) { return fabsf(v) == 65536.0f ? copysignf(65504.0f, v) : v; }

template <typename T>
__global__ void __launch_bounds__(256) unpack8_k(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales,
                                                 T *__restrict__ x, long long groups, long long per_row, long long cols, int vec)
{
    const long long stride = (long long)gridDim.x * 32;
    for (long long g = (long long)blockIdx.x * 32 + (threadIdx.x >> 3); g < groups; g += stride) {
        const long long row = g / per_row, col = (g - row * per_row) * kPackGroup + (threadIdx.x & 7) * 4;
        const int n = (int)min(4LL, max(0LL, cols - col));
        const long long at = row * cols + col;
        float v[4];
        unpack4(load_codes(codes + at, vec, n), pack_step(scales[g]), v);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = held_by<T>(v[i]);
        store4(x + at, vec, n, v);
    }
}

// Whole groups one after the other, everything on 16 bytes: a thread has 16 bytes of values four times, all loads ahead of the rest. us for
// 64 x 64^3 floats (84 MB, 13 at 6.5 TB/s), both directions, against the kernels above: 25.6 -> 14.9 and 20.3 -> 14.7
template <typename T>
struct Flat {
    static constexpr int kPer = 16 / sizeof(T), kLanes = kPackGroup / kPer, kTimes = 4;  // values of a thread, threads of a group
};
__device__ __forceinline__ void load16(const float *p, float (&v)[4]) { load4v(p, v); }
template <typename T>
__device__ __forceinline__ void load16(const T *p, float (&v)[8])
{
    const uint4 q = *reinterpret_cast<const uint4 *>(p);
    const uint2 h[2] = {{q.x, q.y}, {q.z, q.w}};
    float a[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        load4v(reinterpret_cast<const T *>(&h[i]), a);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * i + k] = a[k];
    }
}
__device__ __forceinline__ void store16(float *p, const float (&v)[4]) { store4v(p, v); }
template <typename T>
__device__ __forceinline__ void store16(T *p, const float (&v)[8])
{
    uint4 q;
    store4v(reinterpret_cast<T *>(&q.x), {v[0], v[1], v[2], v[3]});
    store4v(reinterpret_cast<T *>(&q.z), {v[4], v[5], v[6], v[7]});
    *reinterpret_cast<uint4 *>(p) = q;
}

template <typename T>
__global__ void __launch_bounds__(256) pack8_flat_k(const T *__restrict__ x, unsigned char *__restrict__ codes, unsigned char *__restrict__ scales,
                                                    long long values)
{
    using F = Flat<T>;
    const long long at0 = ((long long)blockIdx.x * F::kTimes * 256 + threadIdx.x) * F::kPer;
    float v[F::kTimes][F::kPer];
#pragma unroll
    for (int i = 0; i < F::kTimes; ++i) load16(x + min(at0 + (long long)i * 256 * F::kPer, values - F::kPer), v[i]);
#pragma unroll
    for (int i = 0; i < F::kTimes; ++i) {
        const long long at = at0 + (long long)i * 256 * F::kPer;
        const bool there = at < values;  // of a group all threads or none
        unsigned m = 0;
#pragma unroll
        for (int k = 0; k < F::kPer; ++k) m = max(m, magnitude_bits(v[i][k]));
#pragma unroll
        for (int o = F::kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const bool rare = __any_sync(0xffffffffu, m > kPackLargest);
        if (rare) {  // once more over what is finite
            m = 0;
#pragma unroll
            for (int k = 0; k < F::kPer; ++k) {
                const unsigned b = magnitude_bits(v[i][k]);
                if (bits_finite(b)) m = max(m, b);
            }
#pragma unroll
            for (int o = F::kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        }
        const unsigned scale = pack_scale(m);
        const float inverse = pack_inverse(scale);
        unsigned w[F::kPer / 4];
#pragma unroll
        for (int k = 0; k < F::kPer; k += 4) {
            if (rare)
                w[k / 4] = pack_word(pack_code_any(v[i][k], scale), pack_code_any(v[i][k + 1], scale), pack_code_any(v[i][k + 2], scale),
                                     pack_code_any(v[i][k + 3], scale));
            else
                w[k / 4] = pack_word(pack_code(v[i][k], inverse), pack_code(v[i][k + 1], inverse), pack_code(v[i][k + 2], inverse),
                                     pack_code(v[i][k + 3], inverse));
        }
        if (there) {
            if constexpr (F::kPer == 4)
                *reinterpret_cast<unsigned *>(codes + at) = w[0];
            else
                *reinterpret_cast<uint2 *>(codes + at) = make_uint2(w[0], w[1]);
            if (threadIdx.x % F::kLanes == 0) scales[at / kPackGroup] = (unsigned char)scale;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) unpack8_flat_k(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales,
                                                      T *__restrict__ x, long long values)
{
    using F = Flat<T>;
    const long long at0 = ((long long)blockIdx.x * F::kTimes * 256 + threadIdx.x) * F::kPer;
    unsigned w[F::kTimes][F::kPer / 4], scale[F::kTimes];
#pragma unroll
    for (int i = 0; i < F::kTimes; ++i) {
        const long long at = min(at0 + (long long)i * 256 * F::kPer, values - F::kPer);
        if constexpr (F::kPer == 4) {
            w[i][0] = *reinterpret_cast<const unsigned *>(codes + at);
        } else {
            const uint2 q = *reinterpret_cast<const uint2 *>(codes + at);
            w[i][0] = q.x;
            w[i][1] = q.y;
        }
        scale[i] = scales[at / kPackGroup];
    }
#pragma unroll
    for (int i = 0; i < F::kTimes; ++i) {
        const long long at = at0 + (long long)i * 256 * F::kPer;
        float v[F::kPer];
#pragma unroll
        for (int k = 0; k < F::kPer; k += 4) {
            float f[4];
            unpack4(w[i][k / 4], pack_step(scale[i]), f);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k + j] = held_by<T>(f[j]);
        }
        if (at < values) store16(x + at, v);
    }
}

static unsigned pack_blocks(long long groups)
{
    const long long want = (groups + 31) / 32, most = 16LL * sm_count();
    return (unsigned)(want < most ? want : most);
}

template <typename T>
static int launch_pack8(const void *x, void *codes, void *scales, long long rows, long long cols, bool unpack, cudaStream_t st)
{
    const long long per_row = (cols + kPackGroup - 1) / kPackGroup, groups = rows * per_row;
    if (cols % kPackGroup == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0) {
        const long long values = rows * cols, of_cta = 256LL * Flat<T>::kTimes * Flat<T>::kPer, blocks = (values + of_cta - 1) / of_cta;
        if (blocks <= 0x7fffffffLL) {
            if (unpack)
                unpack8_flat_k<T><<<(unsigned)blocks, 256, 0, st>>>((const unsigned char *)codes, (const unsigned char *)scales, (T *)x, values);
            else
                pack8_flat_k<T><<<(unsigned)blocks, 256, 0, st>>>((const T *)x, (unsigned char *)codes, (unsigned char *)scales, values);
            return check_launch(unpack ? "unpack8" : "pack8");
        }
    }
    const int vec = cols % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0;
    if (unpack)
        unpack8_k<T><<<pack_blocks(groups), 256, 0, st>>>((const unsigned char *)codes, (const unsigned char *)scales, (T *)x, groups, per_row,
                                                         cols, vec);
    else
        pack8_k<T><<<pack_blocks(groups), 256, 0, st>>>((const T *)x, (unsigned char *)codes, (unsigned char *)scales, groups, per_row, cols,
                                                       vec);
    return check_launch(unpack ? "unpack8" : "pack8");
}

static int pack8_call(const void *x, void *codes, void *scales, long long rows, long long cols, int dtype, bool unpack, void *stream)
{
    if (rows < 0 || cols < 0 || (cols > 0 && rows > (1LL << 48) / cols)) return GN_ERR_BAD_SHAPE;
    if (dtype < GN_F32 || dtype > GN_F16) return GN_ERR_UNSUPPORTED;
    if (rows == 0 || cols == 0) return GN_OK;
    if (!x || !codes || !scales) return GN_ERR_NULL_POINTER;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == GN_F32) return launch_pack8<float>(x, codes, scales, rows, cols, unpack, st);
    if (dtype == GN_BF16) return launch_pack8<__nv_bfloat16>(x, codes, scales, rows, cols, unpack, st);
    return launch_pack8<__half>(x, codes, scales, rows, cols, unpack, st);
}

// ---- IL4 tensors ([Q][P][4 samples], P a multiple of 32): a group is 32 neighbouring positions of one sample, so that no sample's scale
// depends on another's. A lane has a position, a word the codes of its four samples; behind the codes a word of four scales per 32 positions.
__global__ void __launch_bounds__(256) pack_il4_k(const float4 *x, unsigned *codes, unsigned *scales, long long groups)
{
    constexpr int kTimes = 4;
    const int lane = threadIdx.x & 31;
    const long long g0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * kTimes;
    float4 v[kTimes];
#pragma unroll
    for (int i = 0; i < kTimes; ++i) v[i] = x[min(g0 + i, groups - 1) * 32 + lane];
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        if (g0 + i >= groups) return;
        const float f[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        unsigned m[4], code[4], scale[4];
        bool rare = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            m[k] = __reduce_max_sync(0xffffffffu, magnitude_bits(f[k]));
            rare |= m[k] > kPackLargest;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (rare) {
                const unsigned b = magnitude_bits(f[k]);
                m[k] = __reduce_max_sync(0xffffffffu, bits_finite(b) ? b : 0u);
            }
            scale[k] = pack_scale(m[k]);
            code[k] = rare ? pack_code_any(f[k], scale[k]) : pack_code(f[k], pack_inverse(scale[k]));
        }
        codes[(g0 + i) * 32 + lane] = pack_word(code[0], code[1], code[2], code[3]);
        if (lane == 0) scales[g0 + i] = pack_word(scale[0], scale[1], scale[2], scale[3]);
    }
}

__global__ void __launch_bounds__(256) unpack_il4_k(const unsigned *__restrict__ codes, const unsigned *__restrict__ scales, float4 *__restrict__ x,
                                                    long long positions)
{
    constexpr int kTimes = 4;
    const long long at0 = (long long)blockIdx.x * kTimes * 256 + threadIdx.x;
    unsigned w[kTimes], sc[kTimes];
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const long long at = min(at0 + i * 256, positions - 1);
        w[i] = codes[at];
        sc[i] = scales[at / kPackGroup];
    }
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        float f[4];
        unpack4_finite(w[i], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] *= pack_step((sc[i] >> (8 * k)) & 0xffu);
        if (unpack_odd(w[i])) {
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = unpack_special(f[k], (w[i] >> (8 * k)) & 0xffu);
        }
        if (at0 + i * 256 < positions) x[at0 + i * 256] = make_float4(f[0], f[1], f[2], f[3]);
    }
}

size_t il4_packed_bytes(int Q, long long P) { return ((size_t)Q * P * 4 + (size_t)Q * (P / kPackGroup) * 4 + 255) / 256 * 256; }

int launch_pack_il4(const float *x, void *packed, int Q, long long P, cudaStream_t st)
{
    const long long groups = Q * (P / kPackGroup);
    unsigned *const codes = (unsigned *)packed;
    pack_il4_k<<<(unsigned)((groups + 31) / 32), 256, 0, st>>>((const float4 *)x, codes, codes + Q * P, groups);
    return check_launch("pack_il4");
}

int launch_unpack_il4(const void *packed, float *x, int Q, long long P, cudaStream_t st)
{
    const unsigned *const codes = (const unsigned *)packed;
    unpack_il4_k<<<(unsigned)((Q * P + 1023) / 1024), 256, 0, st>>>(codes, codes + Q * P, (float4 *)x, Q * P);
    return check_launch("unpack_il4");
}

}  // namespace gn

using namespace gn;

extern "C" {

GN_API int gn_pack8(const void *x, void *codes, void *scales, long long rows, long long cols, int dtype, void *stream)
{
    return pack8_call(x, codes, scales, rows, cols, dtype, false, stream);
}

GN_API int gn_unpack8(const void *codes, const void *scales, void *x, long long rows, long long cols, int dtype, void *stream)
{
    return pack8_call(x, const_cast<void *>(codes), const_cast<void *>(scales), rows, cols, dtype, true, stream);
}

}  // extern "C"
