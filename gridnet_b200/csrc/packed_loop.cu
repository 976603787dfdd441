// The loops with gradients, 8-bit copies between the passes: entry points. What packs an IL4 tensor is in pack8.cu, the loops are in quad_loop.cu.
#include "common.cuh"
#include "kernels.h"

using namespace gn;

static LoopPacked packed_by(void *const *of) { return {of, launch_pack_il4, launch_unpack_il4}; }

extern "C" {

GN_API size_t gn_loop_packed_bytes(int B, int M, int N, int K)
{
    if (B <= 0 || M <= 0 || N <= 0 || K <= 0 || (long long)M * N * K % 32) return 0;
    return il4_packed_bytes((B + 3) / 4, (long long)M * N * K);
}

GN_API size_t gn_loop_packed_workspace_bytes(int B, int M, int N, int K, int inner, int outer, int block, int residual, int gated, int backward)
{
    return loop_packed_workspace(B, M, N, K, inner, outer, gated ? 8 : block, residual, gated != 0, backward != 0);
}

GN_API int gn_loop_forward_packed_f32(const float *const *weights, const float *const *biases, const float *const *scales, int nparams,
                                      const float *gamma, const float *beta, const float *x, float *y, void *const *packed, float *stats,
                                      int B, int M, int N, int K, int inner, int outer, int block, float ln_eps, int activation,
                                      int residual, void *workspace, size_t workspace_bytes, void *stream)
{
    return loop_forward_packed(packed_by(packed), weights, biases, scales, nparams, gamma, beta, x, y, stats, B, M, N, K, inner, outer,
        block, ln_eps, activation, residual, workspace, workspace_bytes, (cudaStream_t)stream);
}

GN_API int gn_loop_backward_packed_f32(const float *const *weights, const float *const *biases, const float *const *scales, int nparams,
                                       const float *gamma, const float *beta, void *const *packed, const float *stats, const float *gy,
                                       float *const *gw, float *const *gb, float *const *gs, float *ggamma, float *gbeta, float *gx, int B,
                                       int M, int N, int K, int inner, int outer, int block, int activation, int residual, void *workspace,
                                       size_t workspace_bytes, void *stream)
{
    return loop_backward_packed(packed_by(packed), weights, biases, scales, nparams, gamma, beta, stats, gy, gw, gb, gs, ggamma, gbeta,
        gx, B, M, N, K, inner, outer, block, activation, residual, workspace, workspace_bytes, (cudaStream_t)stream);
}

GN_API int gn_gated_loop_forward_packed_f32(const float *weight, const float *bias, const float *gamma, const float *beta, const float *x,
                                            float *y, void *const *packed, float *stats, int B, int M, int N, int K, int inner, int outer,
                                            float ln_eps, int act, void *workspace, size_t workspace_bytes, void *stream)
{
    return gated_loop_forward_packed(packed_by(packed), weight, bias, gamma, beta, x, y, stats, B, M, N, K, inner, outer, ln_eps, act,
        workspace, workspace_bytes, (cudaStream_t)stream);
}

GN_API int gn_gated_loop_backward_packed_f32(const float *weight, const float *bias, const float *gamma, const float *beta,
                                             void *const *packed, const float *stats, const float *gy, float *gw, float *gb, float *ggamma,
                                             float *gbeta, float *gx, int B, int M, int N, int K, int inner, int outer, int act,
                                             void *workspace, size_t workspace_bytes, void *stream)
{
    return gated_loop_backward_packed(packed_by(packed), weight, bias, gamma, beta, stats, gy, gw, gb, ggamma, gbeta, gx, B, M, N, K,
        inner, outer, act, workspace, workspace_bytes, (cudaStream_t)stream);
}

}  // extern "C"
