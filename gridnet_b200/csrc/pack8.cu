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

// a half holds no more than 65504: what stands for 65536 next to it is not made an infinity
template <typename T>
__device__ __forceinline__ float held_by(float v) { return v; }
template <>
__device__ __forceinline__ float held_by<__half>(float v) { return magnitude_bits(v) < 0x7f800000u ? fminf(fmaxf(v, -65504.0f), 65504.0f) : v; }

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

static unsigned pack_blocks(long long groups)
{
    const long long want = (groups + 31) / 32, most = 16LL * sm_count();
    return (unsigned)(want < most ? want : most);
}

template <typename T>
static int launch_pack8(const void *x, void *codes, void *scales, long long rows, long long cols, bool unpack, cudaStream_t st)
{
    const long long per_row = (cols + kPackGroup - 1) / kPackGroup, groups = rows * per_row;
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
