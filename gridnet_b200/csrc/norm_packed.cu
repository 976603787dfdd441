// Whole-grid normalisation (norm.cu) whose backward pass reads its input from 8 bits (packed8.cuh) instead of 32.
//
//     y = (x - m) r gamma + beta,  m and r = 1 / sqrt(var + eps) per sample, of x itself
//     with p = (x~ - m) r from the packed copy x~ and q = gamma g:
//     gx = r (q - mean(q) - p mean(q p)),  ggamma = sum over the batch of g p,  gbeta = sum over the batch of g
//
// HBM-bound: forward 4 + 4 bytes for a value (and 4 more where a sample's second reading does not hit L2) and 1.03 for its packed
// copy, backward 5.03 twice and 4. Sums are in double, in a fixed order.
#include "kernels.h"
#include "packed8.cuh"

namespace gn {

// y and the packed copy, eight lanes a group
__global__ void __launch_bounds__(256) norm_apply_pack_k(const float *__restrict__ x, const float *__restrict__ gamma,
                                                         const float *__restrict__ beta, const float2 *__restrict__ stats, float *__restrict__ y,
                                                         unsigned char *__restrict__ codes, unsigned char *__restrict__ scales, long long groups,
                                                         long long per_row, long long P, int vec)
{
    const int lane8 = threadIdx.x & 7;
    const long long stride = (long long)gridDim.x * 32;
    for (long long g0 = (long long)blockIdx.x * 32 + (threadIdx.x >> 5) * 4; g0 < groups; g0 += stride) {
        const long long g = g0 + ((threadIdx.x & 31) >> 3);
        const long long row = g / per_row, col = (g - row * per_row) * kPackGroup + lane8 * 4;
        const int n = g < groups ? (int)min(4LL, max(0LL, P - col)) : 0;
        const long long at = row * P + col;
        float v[4], ga[4], be[4];
        load4(x + at, vec, n, v);
        load4(gamma + col, vec, n, ga);
        load4(beta + col, vec, n, be);
        unsigned scale;
        const unsigned w = pack_group(v, scale);
        store_codes(codes + at, vec, n, w);
        if (lane8 == 0 && g < groups) scales[g] = (unsigned char)scale;
        if (n > 0) {
            const float2 mr = stats[row];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = fmaf((v[i] - mr.x) * mr.y, ga[i], be[i]);
            store4(y + at, vec, n, v);
        }
    }
}

// grid B * parts: sums of q and q p over a slice (a multiple of 32 long) of a sample
__global__ void __launch_bounds__(256) norm_packed_sums_k(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales,
                                                          const float2 *__restrict__ stats, const float *__restrict__ gamma,
                                                          const float *__restrict__ gy, double2 *__restrict__ partials, long long P, long long slice,
                                                          long long per_row, int parts, int vec)
{
    __shared__ double red[33];
    const int b = blockIdx.x / parts, part = blockIdx.x - b * parts;
    const float2 mr = stats[b];
    const long long lo = part * slice, hi = min(P, lo + slice);
    double sq = 0.0, sp = 0.0;
    for (long long col = lo + 4 * threadIdx.x; col < hi; col += 4 * 256) {
        const int n = (int)min(4LL, hi - col);
        const long long at = b * P + col;
        float v[4], g[4], ga[4];
        load4(gy + at, vec, n, g);
        load4(gamma + col, vec, n, ga);
        unpack4(load_codes(codes + at, vec, n), pack_step(scales[b * per_row + col / kPackGroup]), v);
        float q = 0.0f, p = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) {
                const float t = g[i] * ga[i];
                q += t;
                p = fmaf(t, (v[i] - mr.x) * mr.y, p);
            }
        sq += (double)q;
        sp += (double)p;
    }
    sq = block_sum(sq, red);
    sp = block_sum(sp, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = make_double2(sq, sp);
}

// one CTA per sample: means of q and q p
__global__ void __launch_bounds__(64) norm_packed_means_k(const double2 *__restrict__ partials, int parts, float2 *__restrict__ ac, long long P)
{
    __shared__ double red[33];
    double q = 0.0, p = 0.0;
    for (int i = threadIdx.x; i < parts; i += blockDim.x) {
        q += partials[(size_t)blockIdx.x * parts + i].x;
        p += partials[(size_t)blockIdx.x * parts + i].y;
    }
    q = block_sum(q, red);
    p = block_sum(p, red);
    if (threadIdx.x == 0) ac[blockIdx.x] = make_float2((float)(q / (double)P), (float)(p / (double)P));
}

// a thread has four positions and walks the batch
__global__ void __launch_bounds__(256) norm_packed_apply_k(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales,
                                                           const float2 *__restrict__ stats, const float2 *__restrict__ ac,
                                                           const float *__restrict__ gamma, const float *__restrict__ gy, float *__restrict__ gx,
                                                           float *__restrict__ ggamma, float *__restrict__ gbeta, int B, long long P,
                                                           long long per_row, int vec)
{
    const long long col = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (col >= P) return;
    const int n = (int)min(4LL, P - col);
    float ga[4], sg[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sb[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    load4(gamma + col, vec, n, ga);
    for (int b = 0; b < B; ++b) {
        const long long at = b * P + col;
        const float2 mr = stats[b], m = ac[b];
        float v[4], g[4];
        load4(gy + at, vec, n, g);
        unpack4(load_codes(codes + at, vec, n), pack_step(scales[b * per_row + col / kPackGroup]), v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = (v[i] - mr.x) * mr.y;
            sg[i] = fmaf(g[i], p, sg[i]);
            sb[i] += g[i];
            v[i] = mr.y * (fmaf(-p, m.y, g[i] * ga[i]) - m.x);
        }
        store4(gx + at, vec, n, v);
    }
    store4(ggamma + col, vec, n, sg);
    store4(gbeta + col, vec, n, sb);
}

static bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

struct PackedNormWs {
    double2 *partials;
    float2 *ac;
    size_t bytes;
};
static PackedNormWs carve_packed_norm(void *base, int B)
{
    PackedNormWs w;
    const size_t partials = sizeof(double2) * (size_t)B * kNormMaxParts;
    w.partials = static_cast<double2 *>(base);
    w.ac = reinterpret_cast<float2 *>(static_cast<unsigned char *>(base) + partials);
    w.bytes = partials + sizeof(float2) * (size_t)B;
    return w;
}
static int packed_norm_check(int B, long long P, const void *workspace, size_t bytes)
{
    if (B < 0 || P <= 0 || P > (1LL << 40) || (long long)B * ((P + 1023) / 1024) > 0x7fffffffLL) return GN_ERR_BAD_SHAPE;
    if (B > 0 && (!workspace || !aligned(workspace, 16) || bytes < carve_packed_norm(nullptr, B).bytes)) return GN_ERR_WORKSPACE;
    return GN_OK;
}

}  // namespace gn

using namespace gn;

extern "C" {

GN_API size_t gn_norm_packed_workspace_bytes(int B, long long P)
{
    (void)P;
    return B > 0 ? carve_packed_norm(nullptr, B).bytes : 256;
}

GN_API int gn_norm_forward_packed_f32(const float *x, const float *gamma, const float *beta, float *y, float *mean_rstd, void *codes, void *scales,
                                      int B, long long P, float eps, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = packed_norm_check(B, P, workspace, workspace_bytes);
    if (rc != GN_OK) return rc;
    if (B == 0) return GN_OK;
    if (!x || !gamma || !beta || !y || !mean_rstd || !codes || !scales) return GN_ERR_NULL_POINTER;
    if (!aligned(mean_rstd, 8)) return GN_ERR_UNSUPPORTED;
    cudaStream_t st = (cudaStream_t)stream;
    const PackedNormWs ws = carve_packed_norm(workspace, B);
    float2 *const stats = reinterpret_cast<float2 *>(mean_rstd);
    const int parts = norm_pick_parts(P);
    rc = launch_norm_partial_stats(x, ws.partials, B, P, parts, st);
    if (rc == GN_OK) rc = launch_norm_finalize(ws.partials, parts, stats, B, P, eps, st);
    if (rc != GN_OK) return rc;
    const long long per_row = (P + kPackGroup - 1) / kPackGroup, groups = B * per_row, want = (groups + 31) / 32, most = 16LL * sm_count();
    const int vec = P % 4 == 0 && aligned(x, 16) && aligned(gamma, 16) && aligned(beta, 16) && aligned(y, 16) && aligned(codes, 4);
    norm_apply_pack_k<<<(unsigned)(want < most ? want : most), 256, 0, st>>>(x, gamma, beta, stats, y, (unsigned char *)codes,
                                                                             (unsigned char *)scales, groups, per_row, P, vec);
    return check_launch("norm_apply_pack");
}

GN_API int gn_norm_backward_packed_f32(const void *codes, const void *scales, const float *mean_rstd, const float *gamma, const float *gy, float *gx,
                                       float *ggamma, float *gbeta, int B, long long P, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = packed_norm_check(B, P, workspace, workspace_bytes);
    if (rc != GN_OK) return rc;
    if (!gamma || !ggamma || !gbeta) return GN_ERR_NULL_POINTER;
    cudaStream_t st = (cudaStream_t)stream;
    if (B > 0) {
        if (!codes || !scales || !mean_rstd || !gy || !gx) return GN_ERR_NULL_POINTER;
        if (!aligned(mean_rstd, 8)) return GN_ERR_UNSUPPORTED;
    }
    const PackedNormWs ws = carve_packed_norm(workspace, B);
    const float2 *const stats = reinterpret_cast<const float2 *>(mean_rstd);
    const unsigned char *const c = (const unsigned char *)codes, *const s = (const unsigned char *)scales;
    const long long per_row = (P + kPackGroup - 1) / kPackGroup;
    const int vec = P % 4 == 0 && aligned(gamma, 16) && aligned(gy, 16) && aligned(gx, 16) && aligned(ggamma, 16) && aligned(gbeta, 16) &&
                    aligned(codes, 4);
    if (B > 0) {
        const int parts = norm_pick_parts(P);
        const long long slice = ((P + parts - 1) / parts + kPackGroup - 1) / kPackGroup * kPackGroup;
        norm_packed_sums_k<<<(unsigned)B * parts, 256, 0, st>>>(c, s, stats, gamma, gy, ws.partials, P, slice, per_row, parts, vec);
        norm_packed_means_k<<<B, 64, 0, st>>>(ws.partials, parts, ws.ac, P);
    }
    norm_packed_apply_k<<<(unsigned)((P + 1023) / 1024), 256, 0, st>>>(c, s, stats, ws.ac, gamma, gy, gx, ggamma, gbeta, B, P, per_row, vec);
    return check_launch("norm_backward_packed");
}

}  // extern "C"
