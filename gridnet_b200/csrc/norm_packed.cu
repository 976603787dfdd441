// Whole-grid normalisation (norm.cu) whose backward pass reads its input from 8 bits (packed8.cuh) instead of 32.
//
//     y = (x - m) r gamma + beta,  m and r = 1 / sqrt(var + eps) per sample, of x itself
//     with p = (x~ - m) r from the packed copy x~ and q = gamma g:
//     gx = r (q - mean(q) - p mean(q p)),  ggamma = sum over the batch of g p,  gbeta = sum over the batch of g
//
// HBM-bound: forward 8 bytes for a value (and 4 more where its second reading does not hit L2) and 1.03 for its packed
// copy, backward 5.03 twice and 4. Sums over a sample are in double (backward of four products at a time, those added up as floats), sums over the
// batch, which ggamma and gbeta are, in float; all in a fixed order.
#include "kernels.h"
#include "packed8.cuh"

namespace gn {

constexpr int kTogether = 4;     // samples that a thread loads at a time
constexpr int kFoldParts = 128;  // partial sums that a CTA may add up itself (703, 40 x 56 x 72 x 37: 26 us instead of 16 + 3.5)

// Sum of up to 64 partial sums by a warp, in the order in which a block of threads adds them up (block_sum)
__device__ __forceinline__ double2 sum_of_parts(const double2 *partials, int parts)
{
    static_assert(kNormMaxParts == 64, "two to a lane");
    const int lane = threadIdx.x & 31;
    const double2 none = make_double2(0.0, 0.0), a = lane < parts ? partials[lane] : none, b = lane + 32 < parts ? partials[lane + 32] : none;
    return make_double2(warp_sum(a.x) + warp_sum(b.x), warp_sum(a.y) + warp_sum(b.y));
}

// y and the packed copy. With partial sums a CTA finishes the statistics of its four samples itself, a launch
// less; without them stats has them. A thread has four positions of four samples, with gamma and beta read once for them; eight lanes have a group. Later
// samples first: of them, what the sums were taken from is still in L2.
__global__ void __launch_bounds__(256) norm_apply_pack_k(const float *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta,
                                                         const double2 *partials, int parts, float eps, float2 *stats, float *__restrict__ y,
                                                         unsigned char *__restrict__ codes, unsigned char *__restrict__ scales, int B, int slices,
                                                         long long per_row, long long P, int vec)
{
    __shared__ float2 of_sample[kTogether];
    const int chunk = blockIdx.x / slices, last = B - 1 - chunk * kTogether;
    const long long col = ((long long)(blockIdx.x - chunk * slices) * 256 + threadIdx.x) * 4;
    const int n = (int)min(4LL, max(0LL, P - col));
    float v[kTogether][4], ga[4], be[4];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) load4(x + (long long)max(last - i, 0) * P + col, vec, n, v[i]);
    load4(gamma + col, vec, n, ga);
    load4(beta + col, vec, n, be);
    previous_done();
    const int warp = threadIdx.x >> 5;
    if (!partials) {
        if (threadIdx.x < kTogether && last - (int)threadIdx.x >= 0) of_sample[threadIdx.x] = stats[last - threadIdx.x];
    } else if (warp < kTogether && last - warp >= 0) {
        const double2 sums = sum_of_parts(partials + (size_t)(last - warp) * parts, parts);
        const double mean = sums.x / (double)P;
        double var = sums.y / (double)P - mean * mean;
        if (var < 0.0) var = 0.0;
        const float2 mr = make_float2((float)mean, (float)(1.0 / sqrt(var + (double)eps)));
        if ((threadIdx.x & 31) == 0) {
            of_sample[warp] = mr;
            if (blockIdx.x == chunk * slices) stats[last - warp] = mr;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
        const int b = last - i;
        if (b < 0) return;
        unsigned scale;
        const unsigned w = pack_group(v[i], scale);
        if (n > 0) {
            const long long at = b * P + col;
            store_codes(codes + at, vec, n, w);
            if ((threadIdx.x & 7) == 0) scales[b * per_row + col / kPackGroup] = (unsigned char)scale;
            const float2 mr = of_sample[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][k] = fmaf((v[i][k] - mr.x) * mr.y, ga[k], be[k]);
            store4(y + at, vec, n, v[i]);
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
    const float *const gs = gy + b * P;
    const unsigned char *const cs = codes + b * P, *const ss = scales + b * per_row;
    auto add = [&](const float (&g)[4], const float (&ga)[4], unsigned w, unsigned scale, int n) {
        float v[4], q = 0.0f, p = 0.0f;
        unpack4(w, pack_step(scale), v);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < n) {
                const float t = g[k] * ga[k];
                q += t;
                p = fmaf(t, (v[k] - mr.x) * mr.y, p);
            }
        sq += (double)q;
        sp += (double)p;
    };
    long long col = lo + 4 * threadIdx.x;
    constexpr int kStride = 4 * 256;
    if (vec) {
        constexpr int kAtOnce = 4;
        for (; col + (kAtOnce - 1) * kStride < hi; col += kAtOnce * kStride) {  // loads first
            float g[kAtOnce][4], ga[kAtOnce][4];
            unsigned w[kAtOnce], sc[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                load4v(gs + col + i * kStride, g[i]);
                load4v(gamma + col + i * kStride, ga[i]);
                w[i] = *reinterpret_cast<const unsigned *>(cs + col + i * kStride);
                sc[i] = ss[(col + i * kStride) / kPackGroup];
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) add(g[i], ga[i], w[i], sc[i], 4);
        }
    }
    for (; col < hi; col += kStride) {
        const int n = (int)min(4LL, hi - col);
        float g[4], ga[4];
        load4(gs + col, vec, n, g);
        load4(gamma + col, vec, n, ga);
        add(g, ga, load_codes(cs + col, vec, n), ss[col / kPackGroup], n);
    }
    sq = block_sum(sq, red);
    sp = block_sum(sp, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = make_double2(sq, sp);
}

// one warp per sample: means of q and q p
__device__ __forceinline__ float2 means_of(const double2 *partials, int parts, long long P)
{
    const double2 sums = sum_of_parts(partials, parts);
    return make_float2((float)(sums.x / (double)P), (float)(sums.y / (double)P));
}
__global__ void __launch_bounds__(32) norm_packed_means_k(const double2 *partials, int parts, float2 *ac, long long P)
{
    previous_done();
    const float2 m = means_of(partials + (size_t)blockIdx.x * parts, parts, P);
    if (threadIdx.x == 0) ac[blockIdx.x] = m;
}

// A thread has four positions and every PARTS-th sample, 256 / PARTS threads side by side; the parts' sums are added up in a fixed order. Four
// samples' loads ahead of the rest. One part where that leaves CTAs enough (rows of 4 KB: 128^3 x 32 127 us, with eight parts 146), else
// eight (40 x 56 x 72 x 37 37 -> 19 us, 32^3 x 8 10.6 -> 4.5).
template <int PARTS>
__global__ void __launch_bounds__(256) norm_packed_apply_k(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales,
                                                           const float2 *stats, const float2 *ac, const double2 *partials, int parts,
                                                           const float *__restrict__ gamma,
                                                           const float *__restrict__ gy, float *__restrict__ gx, float *__restrict__ ggamma,
                                                           float *__restrict__ gbeta, int B, long long P, long long per_row, int vec)
{
    constexpr int kSide = 256 / PARTS;
    __shared__ float4 sums[2][PARTS][PARTS > 1 ? kSide : 1];
    __shared__ float2 means[kFoldParts];
    const int place = threadIdx.x % kSide, part = threadIdx.x / kSide;
    const long long col = ((long long)blockIdx.x * kSide + place) * 4;
    const int n = (int)min(4LL, max(0LL, P - col));
    float ga[4], sg[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sb[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    load4(gamma + col, vec, n, ga);
    previous_done();
    if (!ac) {  // few enough: every CTA adds them up itself, a launch less
        for (int b = threadIdx.x >> 5; b < B; b += 8) {
            const float2 m = means_of(partials + (size_t)b * parts, parts, P);
            if ((threadIdx.x & 31) == 0) means[b] = m;
        }
        __syncthreads();
        ac = means;
    }
    if (n > 0) {
        for (int b0 = part; b0 < B; b0 += PARTS * kTogether) {
            float g[kTogether][4];
            unsigned w[kTogether], sc[kTogether];
#pragma unroll
            for (int i = 0; i < kTogether; ++i) {
                const int b = min(b0 + PARTS * i, B - 1);
                const long long at = b * P + col;
                load4(gy + at, vec, n, g[i]);
                w[i] = load_codes(codes + at, vec, n);
                sc[i] = scales[b * per_row + col / kPackGroup];
            }
#pragma unroll
            for (int i = 0; i < kTogether; ++i) {
                const int b = b0 + PARTS * i;
                if (b >= B) break;
                const float2 mr = stats[b], m = ac[b];
                float v[4];
                unpack4(w[i], pack_step(sc[i]), v);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float p = (v[k] - mr.x) * mr.y;
                    sg[k] = fmaf(g[i][k], p, sg[k]);
                    sb[k] += g[i][k];
                    v[k] = mr.y * (fmaf(-p, m.y, g[i][k] * ga[k]) - m.x);
                }
                store4(gx + b * P + col, vec, n, v);
            }
        }
    }
    if constexpr (PARTS > 1) {
        sums[0][part][place] = make_float4(sg[0], sg[1], sg[2], sg[3]);
        sums[1][part][place] = make_float4(sb[0], sb[1], sb[2], sb[3]);
        __syncthreads();
        if (part < 2) {
            float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int i = 0; i < PARTS; ++i) {
                const float4 s = sums[part][i][place];
                t[0] += s.x; t[1] += s.y; t[2] += s.z; t[3] += s.w;
            }
            store4((part ? gbeta : ggamma) + col, vec, n, t);
        }
    } else {
        store4(ggamma + col, vec, n, sg);
        store4(gbeta + col, vec, n, sb);
    }
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
    if (B < 0 || P <= 0 || P > (1LL << 37) || (long long)B * ((P + 1023) / 1024) > 0x7fffffffLL) return GN_ERR_BAD_SHAPE;
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
    if (rc != GN_OK) return rc;
    const long long per_row = (P + kPackGroup - 1) / kPackGroup, slices = (P + 1023) / 1024, ctas = slices * ((B + kTogether - 1) / kTogether);
    // two rounds of CTAs: 40 x 56 x 72 x 37 13.2 us instead of 10.9 + 3.6; 128^3 x 32, seven rounds, 113 instead of 103 + 3.8
    const bool fold = ctas <= 16LL * sm_count();
    if (!fold) rc = launch_norm_finalize(ws.partials, parts, stats, B, P, eps, st);
    if (rc != GN_OK) return rc;
    const int vec = P % 4 == 0 && aligned(x, 16) && aligned(gamma, 16) && aligned(beta, 16) && aligned(y, 16) && aligned(codes, 4);
    launch_after(norm_apply_pack_k, dim3((unsigned)ctas), dim3(256), 0, st, x, gamma, beta, fold ? ws.partials : nullptr, parts,
                 eps, stats, y, (unsigned char *)codes, (unsigned char *)scales, B, (int)slices, per_row, P, vec);
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
    const int parts = norm_pick_parts(P);
    const bool fold = (long long)B * parts <= kFoldParts;
    const float2 *const ac = fold ? nullptr : ws.ac;
    if (B > 0) {
        const long long slice = ((P + parts - 1) / parts + kPackGroup - 1) / kPackGroup * kPackGroup;
        norm_packed_sums_k<<<(unsigned)B * parts, 256, 0, st>>>(c, s, stats, gamma, gy, ws.partials, P, slice, per_row, parts, vec);
        if (!fold) launch_after(norm_packed_means_k, dim3(B), dim3(32), 0, st, ws.partials, parts, ws.ac, P);
    }
    if (P >= 2048LL * sm_count())
        launch_after(norm_packed_apply_k<1>, dim3((unsigned)((P + 1023) / 1024)), dim3(256), 0, st, c, s, stats, ac, ws.partials, parts, gamma, gy, gx,
                     ggamma, gbeta, B, P, per_row, vec);
    else
        launch_after(norm_packed_apply_k<8>, dim3((unsigned)((P + 127) / 128)), dim3(256), 0, st, c, s, stats, ac, ws.partials, parts, gamma, gy, gx,
                     ggamma, gbeta, B, P, per_row, vec);
    return check_launch("norm_backward_packed");
}

}  // extern "C"
