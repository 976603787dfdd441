// Gated linear recurrence over sequences: h_t = a_t h_{t-1} + n_t u_t with a_t = s(z_t), n_t = s(-z_t) = 1 - a_t, s the logistic
// function - the update of the gated grid's cell (gridnet/backend_torch.py:241-265) with gate z and value u given.
//
// Every step is an affine map of the state, and so is every run of steps: (A, H) stands for h -> A h + H, and
// (A2, H2) after (A1, H1) is (A1 A2, A2 H1 + H2). A thread composes the steps it holds in registers, lanes compose by shuffles,
// warps through shared memory, the CTAs of a cluster through each other's shared memory; then each thread knows the state ahead of its first step
// and runs its steps again from registers. So gate and value are read once and h is written once, however long the sequence.
//
// Backward: c_t = gradient of h_{t-1} = a_t (g_t + c_{t+1}) is affine in c_{t+1}, from the end to the start, with the same A;
//     dh_t = g_t + c_{t+1},  du_t = n_t dh_t,  dz_t = a_t n_t (h_{t-1} - u_t) dh_t.
// h is not kept but run again: both directions are composed in the same exchange, from one reading of gate, value and g. Where a
// sequence is longer than what a CTA or cluster holds at a time, the forward pass has left the state at each such boundary.
//
// Steps whose n_t is 0 (gates from about 104 up, and +inf) do not look at their value, which may be NaN; steps whose a_t is 0 do not look
// at the state. Anything else that is not finite stays in the state.
// A product of many a_t must not become 0 by underflow, or it would hide such a state: it ends at the smallest normal number.
#include <cooperative_groups.h>

#include "kernels.h"
#include "packed8.cuh"

namespace gn {

namespace cg = cooperative_groups;

constexpr int kScanThreads = 256, kScanWarps = 8, kMaxCluster = 16;
constexpr int kFwdSteps = 8, kBwdSteps = 4;  // steps that a thread holds

// A row of a tile is 128 bytes: 8 lanes x 4 floats, 16 lanes x 4 values of 16 bits
template <typename T>
struct Lay {
    static constexpr int kLanes = sizeof(T) == 4 ? 8 : 16;
    static constexpr int kWidth = 4 * kLanes;        // channels of a slab
    static constexpr int kRuns = 32 / kLanes;        // runs of steps side by side in a warp
    static constexpr int kFwd = kScanWarps * kRuns * kFwdSteps, kBwd = kScanWarps * kRuns * kBwdSteps;  // steps of a CTA's tile
};

struct Scan {
    const void *gate, *value;  // or codes
    const unsigned char *gate_scales, *value_scales;
    long long gate_seq, gate_step, value_seq, value_step;  // strides in elements
    const float *state;         // [n][width] or nullptr
    const long long *offsets;   // [n + 1] or nullptr
    void *h;
    float *last;
    unsigned char *pack_gate, *pack_value, *pack_gate_scales, *pack_value_scales;
    float *bounds;  // state ahead of every interval-th step
    int interval;
    const void *gh;
    const float *glast;
    void *dgate, *dvalue;
    float *dstate;
    int n, width, slabs, cluster, vec;
    long long steps, total;  // steps of a sequence; rows of everything
};

struct Place {  // of a sequence
    long long first, len;
};
__device__ __forceinline__ Place sequence(const Scan &p, int seq)
{
    Place s;
    if (!p.offsets) {
        s.first = seq * p.steps;
        s.len = p.steps;
    } else {  // whatever stands in the offsets, nothing outside the rows is touched
        s.first = min(max(p.offsets[seq], 0LL), p.total);
        s.len = min(max(p.offsets[seq + 1], s.first), p.total) - s.first;
    }
    return s;
}
// row of p.bounds that holds the state ahead of step interval * k of a sequence, k >= 1
__device__ __forceinline__ long long bound_row(const Scan &p, int seq, const Place &s, long long k)
{
    if (!p.offsets) return seq * ((p.steps + p.interval - 1) / p.interval) + k;
    return s.first / p.interval + seq + k;  // a sequence has at most one boundary more than its rows have multiples of the interval
}

// logistic function of z and of -z, both to a few units in the last place
__device__ __forceinline__ void gates(float z, float &a, float &n)
{
    const float e = expf(-fabsf(z));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    const float q = e * r;
    a = z < 0.0f ? q : r;
    n = z < 0.0f ? r : q;
}
__device__ __forceinline__ float through(float a, float h, float b) { return a == 0.0f ? b : fmaf(a, h, b); }
__device__ __forceinline__ float product(float a, float b)
{
    const float p = a * b;
    return a == 0.0f || b == 0.0f ? 0.0f : (p < FLT_MIN ? FLT_MIN : p);  // NaN stays
}

// Rows outside of every sequence of a ragged call: zeros
template <typename T>
__device__ void clear_rows(const Scan &p, T *x, int slab, int rank)
{
    using L = Lay<T>;
    const long long lo = min(max(p.offsets[0], 0LL), p.total), hi = min(max(p.offsets[p.n], lo), p.total);
    const int lr = threadIdx.x % L::kLanes, ch = slab * L::kWidth + lr * 4, nch = min(4, max(0, p.width - ch));
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int rows = kScanThreads / L::kLanes;
    for (long long i = (long long)rank * rows + threadIdx.x / L::kLanes; i < lo + p.total - hi; i += (long long)rows * p.cluster) {
        const long long row = i < lo ? i : i - lo + hi;
        store4(x + row * p.width + ch, p.vec, nch, zero);
    }
}

template <typename T, int S>
__device__ __forceinline__ void load_rows(const T *x, long long step, bool vec, int cnt, int nch, float (&v)[S][4])
{
    if (vec && nch == 4) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (s < cnt)
                load4v(x + s * step, v[s]);
            else
                v[s][0] = v[s][1] = v[s][2] = v[s][3] = 0.0f;
        }
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s) load4(x + s * step, false, s < cnt ? nch : 0, v[s]);
    }
}

template <int S>
__device__ __forceinline__ void load_packed(const unsigned char *codes, const unsigned char *scales, long long row, int width, int ch, bool vec,
                                            int cnt, int nch, float (&v)[S][4])
{
    const int per_row = (width + kPackGroup - 1) / kPackGroup;
    unsigned w[S], sc[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const bool there = s < cnt && nch > 0;
        w[s] = there ? load_codes(codes + (row + s) * width + ch, vec, nch) : 0u;
        sc[s] = there ? scales[(row + s) * per_row + ch / kPackGroup] : 127u;
    }
#pragma unroll
    for (int s = 0; s < S; ++s) unpack4(w[s], pack_step(sc[s]), v[s]);
}

// What a warp's, a CTA's steps amount to, per channel; two copies, so that one barrier lies between writing and writing again
template <typename T, int VALUES>
struct Exchange {
    float warp[2][kScanWarps][VALUES][Lay<T>::kWidth];
    float rank[2][kMaxCluster][VALUES][Lay<T>::kWidth];
};

__device__ __forceinline__ void get4(const float *p, float (&v)[4]) { load4v(p, v); }

// ------------------------------------------------------------------ forward
// PACKED: gate and value are codes, and only the states at the boundaries are wanted. KEEP: packs gate and value.
template <typename T, bool PACKED, bool KEEP>
__global__ void __launch_bounds__(kScanThreads, 2) scan_forward_k(const Scan p)
{
    using L = Lay<T>;
    constexpr int S = kFwdSteps;
    __shared__ __align__(16) Exchange<T, 2> ex;
    const int rank = blockIdx.x % p.cluster, id = blockIdx.x / p.cluster;
    const int slab = id % p.slabs, seq = id / p.slabs;
    if (seq >= p.n) {
        if (!PACKED) clear_rows<T>(p, (T *)p.h, slab, rank);
        return;
    }
    const Place q = sequence(p, seq);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lr = lane % L::kLanes, run = lane / L::kLanes;
    const int ch = slab * L::kWidth + lr * 4, nch = min(4, max(0, p.width - ch));
    const bool vec = p.vec;
    float carry[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.state) load4(p.state + (long long)seq * p.width + ch, vec, nch, carry);
    if (q.len == 0) {
        if (!PACKED && p.last && rank == 0 && threadIdx.x < L::kLanes) store4(p.last + (long long)seq * p.width + ch, vec, nch, carry);
        return;
    }
    if (PACKED && q.len <= p.interval) return;  // the whole cluster
    const long long gate_at = p.offsets ? q.first * p.gate_step : seq * p.gate_seq;
    const long long value_at = p.offsets ? q.first * p.value_step : seq * p.value_seq;
    // a CTA's shared memory may be written to by others once it runs: waited for ahead of the first such store
    if (p.cluster > 1) cg::this_cluster().sync();
    int par = 0;
    for (long long base = 0; base < q.len; base += (long long)L::kFwd * p.cluster, par ^= 1) {
        const long long t0 = base + (long long)rank * L::kFwd + (warp * L::kRuns + run) * S;
        const int cnt = (int)min((long long)S, max(0LL, q.len - t0));
        float a[S][4], b[S][4];
        if (PACKED) {
            load_packed<S>((const unsigned char *)p.gate, p.gate_scales, q.first + t0, p.width, ch, vec, cnt, nch, a);
            load_packed<S>((const unsigned char *)p.value, p.value_scales, q.first + t0, p.width, ch, vec, cnt, nch, b);
        } else {
            load_rows<T, S>((const T *)p.gate + gate_at + t0 * p.gate_step + ch, p.gate_step, vec, cnt, nch, a);
            load_rows<T, S>((const T *)p.value + value_at + t0 * p.value_step + ch, p.value_step, vec, cnt, nch, b);
        }
        if (KEEP) {
            const int per_row = (p.width + kPackGroup - 1) / kPackGroup;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                unsigned sg, sv;
                const unsigned wg = pack_group(a[s], sg), wv = pack_group(b[s], sv);
                if (s < cnt) {
                    const long long row = q.first + t0 + s, at = row * p.width + ch;
                    store_codes(p.pack_gate + at, vec, nch, wg);
                    store_codes(p.pack_value + at, vec, nch, wv);
                    if ((lr & 7) == 0 && nch > 0) {
                        p.pack_gate_scales[row * per_row + ch / kPackGroup] = (unsigned char)sg;
                        p.pack_value_scales[row * per_row + ch / kPackGroup] = (unsigned char)sv;
                    }
                }
            }
        }
        float A[4], H[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            A[i] = 1.0f;
            H[i] = 0.0f;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                float w, n;
                gates(a[s][i], w, n);
                a[s][i] = s < cnt ? w : 1.0f;
                b[s][i] = s < cnt && n != 0.0f ? n * b[s][i] : 0.0f;
                H[i] = through(a[s][i], H[i], b[s][i]);
                A[i] = product(A[i], a[s][i]);
            }
        }
        // runs before this one in the warp
#pragma unroll
        for (int d = 1; d < L::kRuns; d *= 2)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float pa = __shfl_up_sync(0xffffffffu, A[i], d * L::kLanes), ph = __shfl_up_sync(0xffffffffu, H[i], d * L::kLanes);
                if (run >= d) {
                    H[i] = through(A[i], ph, H[i]);
                    A[i] = product(pa, A[i]);
                }
            }
        if (run == L::kRuns - 1) {
            store4v(&ex.warp[par][warp][0][lr * 4], A);
            store4v(&ex.warp[par][warp][1][lr * 4], H);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            A[i] = __shfl_up_sync(0xffffffffu, A[i], L::kLanes);
            H[i] = __shfl_up_sync(0xffffffffu, H[i], L::kLanes);
            if (run == 0) {
                A[i] = 1.0f;
                H[i] = 0.0f;
            }
        }
        __syncthreads();
        float h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = carry[i];
        if (p.cluster > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (warp < 1 && run == 0) {
                float ta[4] = {1.0f, 1.0f, 1.0f, 1.0f}, th[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int w = 0; w < kScanWarps; ++w) {
                    float wa[4], wh[4];
                    get4(&ex.warp[par][w][0][lr * 4], wa);
                    get4(&ex.warp[par][w][1][lr * 4], wh);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        th[i] = through(wa[i], th[i], wh[i]);
                        ta[i] = product(ta[i], wa[i]);
                    }
                }
                for (int r = 0; r < p.cluster; ++r) {
                    store4v(cluster.map_shared_rank(&ex.rank[par][rank][0][lr * 4], r), ta);
                    store4v(cluster.map_shared_rank(&ex.rank[par][rank][1][lr * 4], r), th);
                }
            }
            cluster.sync();
            for (int r = 0; r < p.cluster; ++r) {
                float ra[4], rh[4];
                get4(&ex.rank[par][r][0][lr * 4], ra);
                get4(&ex.rank[par][r][1][lr * 4], rh);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (r == rank) h[i] = carry[i];
                    carry[i] = through(ra[i], carry[i], rh[i]);
                }
            }
        }
        for (int w = 0; w < kScanWarps; ++w) {
            float wa[4], wh[4];
            if (p.cluster > 1 && w >= warp) break;
            get4(&ex.warp[par][w][0][lr * 4], wa);
            get4(&ex.warp[par][w][1][lr * 4], wh);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (w < warp) h[i] = through(wa[i], h[i], wh[i]);
                if (p.cluster == 1) carry[i] = through(wa[i], carry[i], wh[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = through(A[i], h[i], H[i]);
        if (p.bounds && cnt > 0 && t0 > 0 && t0 % p.interval == 0)
            store4(p.bounds + bound_row(p, seq, q, t0 / p.interval) * p.width + ch, vec, nch, h);
        if (!PACKED) {
            T *out = (T *)p.h + (q.first + t0) * p.width + ch;
#pragma unroll
            for (int s = 0; s < S; ++s) {
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = through(a[s][i], h[i], b[s][i]);
                if (s < cnt) store4(out + (long long)s * p.width, vec, nch, h);
            }
            if (p.last && cnt > 0 && t0 + cnt == q.len) store4(p.last + (long long)seq * p.width + ch, vec, nch, h);
        }
    }
}

// ------------------------------------------------------------------ backward
template <typename T, bool PACKED>
__global__ void __launch_bounds__(kScanThreads, 2) scan_backward_k(const Scan p)
{
    using L = Lay<T>;
    constexpr int S = kBwdSteps;
    __shared__ __align__(16) Exchange<T, 3> ex;
    const int rank = blockIdx.x % p.cluster, id = blockIdx.x / p.cluster;
    const int slab = id % p.slabs, seq = id / p.slabs;
    if (seq >= p.n) {
        clear_rows<T>(p, (T *)p.dgate, slab, rank);
        clear_rows<T>(p, (T *)p.dvalue, slab, rank);
        return;
    }
    const Place q = sequence(p, seq);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lr = lane % L::kLanes, run = lane / L::kLanes;
    const int ch = slab * L::kWidth + lr * 4, nch = min(4, max(0, p.width - ch));
    const bool vec = p.vec;
    const long long state_at = (long long)seq * p.width + ch;
    float carry[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // gradient of the state behind the steps in hand
    if (p.glast) load4(p.glast + state_at, vec, nch, carry);
    const long long gate_at = p.offsets ? q.first * p.gate_step : seq * p.gate_seq;
    const long long value_at = p.offsets ? q.first * p.value_step : seq * p.value_seq;
    const long long held = (long long)L::kBwd * p.cluster;  // == p.interval
    // a CTA's shared memory may be written to by others once it runs: waited for ahead of the first such store
    if (p.cluster > 1) cg::this_cluster().sync();
    int par = 0;
    for (long long k = (q.len + held - 1) / held - 1; k >= 0; --k, par ^= 1) {
        const long long t0 = k * held + (long long)rank * L::kBwd + (warp * L::kRuns + run) * S;
        const int cnt = (int)min((long long)S, max(0LL, q.len - t0));
        float z[S][4], u[S][4], g[S][4], h[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (PACKED) {
            load_packed<S>((const unsigned char *)p.gate, p.gate_scales, q.first + t0, p.width, ch, vec, cnt, nch, z);
            load_packed<S>((const unsigned char *)p.value, p.value_scales, q.first + t0, p.width, ch, vec, cnt, nch, u);
        } else {
            load_rows<T, S>((const T *)p.gate + gate_at + t0 * p.gate_step + ch, p.gate_step, vec, cnt, nch, z);
            load_rows<T, S>((const T *)p.value + value_at + t0 * p.value_step + ch, p.value_step, vec, cnt, nch, u);
        }
        load_rows<T, S>((const T *)p.gh + (q.first + t0) * p.width + ch, p.width, vec, cnt, nch, g);
        if (k > 0)
            load4(p.bounds + bound_row(p, seq, q, k) * p.width + ch, vec, nch, h);
        else if (p.state)
            load4(p.state + state_at, vec, nch, h);
        float A[4], H[4], C[4], a[S][4], n[S][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            A[i] = 1.0f;
            H[i] = C[i] = 0.0f;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                gates(z[s][i], a[s][i], n[s][i]);
                if (s >= cnt) {
                    a[s][i] = 1.0f;
                    n[s][i] = 0.0f;
                }
                H[i] = through(a[s][i], H[i], n[s][i] == 0.0f ? 0.0f : n[s][i] * u[s][i]);
                A[i] = product(A[i], a[s][i]);
            }
#pragma unroll
            for (int s = S - 1; s >= 0; --s) C[i] = a[s][i] == 0.0f ? 0.0f : a[s][i] * (g[s][i] + C[i]);
        }
        // exclusive, before (A, H) and behind (B, C) this run in the warp
        float B[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) B[i] = A[i];
#pragma unroll
        for (int d = 1; d < L::kRuns; d *= 2)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float pa = __shfl_up_sync(0xffffffffu, A[i], d * L::kLanes), ph = __shfl_up_sync(0xffffffffu, H[i], d * L::kLanes);
                const float nb = __shfl_down_sync(0xffffffffu, B[i], d * L::kLanes), nc = __shfl_down_sync(0xffffffffu, C[i], d * L::kLanes);
                if (run >= d) {
                    H[i] = through(A[i], ph, H[i]);
                    A[i] = product(pa, A[i]);
                }
                if (run + d < L::kRuns) {
                    C[i] = through(B[i], nc, C[i]);
                    B[i] = product(nb, B[i]);
                }
            }
        if (run == L::kRuns - 1) {
            store4v(&ex.warp[par][warp][0][lr * 4], A);
            store4v(&ex.warp[par][warp][1][lr * 4], H);
        }
        if (run == 0) store4v(&ex.warp[par][warp][2][lr * 4], C);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            A[i] = __shfl_up_sync(0xffffffffu, A[i], L::kLanes);
            H[i] = __shfl_up_sync(0xffffffffu, H[i], L::kLanes);
            B[i] = __shfl_down_sync(0xffffffffu, B[i], L::kLanes);
            C[i] = __shfl_down_sync(0xffffffffu, C[i], L::kLanes);
            if (run == 0) {
                A[i] = 1.0f;
                H[i] = 0.0f;
            }
            if (run == L::kRuns - 1) {
                B[i] = 1.0f;
                C[i] = 0.0f;
            }
        }
        __syncthreads();
        float c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = carry[i];
        if (p.cluster > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (warp == 0 && run == 0) {
                float ta[4] = {1.0f, 1.0f, 1.0f, 1.0f}, th[4] = {0.0f, 0.0f, 0.0f, 0.0f}, tc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int w = 0; w < kScanWarps; ++w) {
                    float wa[4], wh[4], wc[4], va[4];
                    get4(&ex.warp[par][w][0][lr * 4], wa);
                    get4(&ex.warp[par][w][1][lr * 4], wh);
                    get4(&ex.warp[par][kScanWarps - 1 - w][0][lr * 4], va);
                    get4(&ex.warp[par][kScanWarps - 1 - w][2][lr * 4], wc);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        th[i] = through(wa[i], th[i], wh[i]);
                        ta[i] = product(ta[i], wa[i]);
                        tc[i] = through(va[i], tc[i], wc[i]);
                    }
                }
                for (int r = 0; r < p.cluster; ++r) {
                    store4v(cluster.map_shared_rank(&ex.rank[par][rank][0][lr * 4], r), ta);
                    store4v(cluster.map_shared_rank(&ex.rank[par][rank][1][lr * 4], r), th);
                    store4v(cluster.map_shared_rank(&ex.rank[par][rank][2][lr * 4], r), tc);
                }
            }
            cluster.sync();
            for (int r = 0; r < rank; ++r) {
                float ra[4], rh[4];
                get4(&ex.rank[par][r][0][lr * 4], ra);
                get4(&ex.rank[par][r][1][lr * 4], rh);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = through(ra[i], h[i], rh[i]);
            }
            for (int r = p.cluster - 1; r >= 0; --r) {
                float ra[4], rc[4];
                get4(&ex.rank[par][r][0][lr * 4], ra);
                get4(&ex.rank[par][r][2][lr * 4], rc);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (r == rank) c[i] = carry[i];
                    carry[i] = through(ra[i], carry[i], rc[i]);
                }
            }
        }
        for (int w = 0; w < warp; ++w) {
            float wa[4], wh[4];
            get4(&ex.warp[par][w][0][lr * 4], wa);
            get4(&ex.warp[par][w][1][lr * 4], wh);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = through(wa[i], h[i], wh[i]);
        }
        for (int w = kScanWarps - 1; w >= 0; --w) {
            float wa[4], wc[4];
            if (p.cluster > 1 && w <= warp) break;
            get4(&ex.warp[par][w][0][lr * 4], wa);
            get4(&ex.warp[par][w][2][lr * 4], wc);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (w > warp) c[i] = through(wa[i], c[i], wc[i]);
                if (p.cluster == 1) carry[i] = through(wa[i], carry[i], wc[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[i] = through(A[i], h[i], H[i]);
            c[i] = through(B[i], c[i], C[i]);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const float w = a[s][i] * n[s][i], d = h[i] - u[s][i];
                h[i] = through(a[s][i], h[i], n[s][i] == 0.0f ? 0.0f : n[s][i] * u[s][i]);
                z[s][i] = w == 0.0f ? 0.0f : w * d;
            }
        }
        const long long at = (q.first + t0) * p.width + ch;
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            float dz[4], du[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float dh = g[s][i] + c[i];
                du[i] = n[s][i] * dh;
                dz[i] = z[s][i] * dh;
                // a step behind the end has a = 1 and g = 0
                c[i] = a[s][i] == 0.0f ? 0.0f : a[s][i] * dh;
            }
            if (s < cnt) {
                store4((T *)p.dgate + at + (long long)s * p.width, vec, nch, dz);
                store4((T *)p.dvalue + at + (long long)s * p.width, vec, nch, du);
            }
        }
    }
    if (p.dstate && rank == 0 && threadIdx.x < L::kLanes) store4(p.dstate + state_at, vec, nch, carry);
}

// ------------------------------------------------------------------ one step
template <typename T>
__global__ void __launch_bounds__(256) scan_step_k(const T *__restrict__ gate, const T *__restrict__ value, const float *state, T *__restrict__ h,
                                                   float *out_state, long long rows, int width, long long gate_row, long long value_row, int vec)
{
    const int quads = (width + 3) / 4;
    const long long stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < rows * quads; i += stride) {
        const long long row = i / quads;
        const int ch = (int)(i - row * quads) * 4, nch = min(4, width - ch);
        float z[4], u[4], s[4];
        load4(gate + row * gate_row + ch, vec, nch, z);
        load4(value + row * value_row + ch, vec, nch, u);
        load4(state + row * width + ch, vec, nch, s);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float a, n;
            gates(z[k], a, n);
            s[k] = through(a, s[k], n == 0.0f ? 0.0f : n * u[k]);
        }
        store4(h + row * width + ch, vec, nch, s);
        store4(out_state + row * width + ch, vec, nch, s);
    }
}

// ------------------------------------------------------------------ host side
static bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// CTAs that share a sequence's steps
static int scan_cluster(int n, long long steps, int width, int size, bool backward)
{
    (void)n; (void)steps; (void)width; (void)size; (void)backward;
    return 1;
}
static int slab_width(int dtype) { return dtype == GN_F32 ? Lay<float>::kWidth : Lay<__half>::kWidth; }
static int held_steps(int dtype) { return dtype == GN_F32 ? Lay<float>::kBwd : Lay<__half>::kBwd; }

static int scan_check(int n, long long steps, long long total, int width, int dtype, bool ragged)
{
    if (n < 0 || steps < 0 || total < 0 || width <= 0) return GN_ERR_BAD_SHAPE;
    if (!ragged && total != n * steps) return GN_ERR_BAD_SHAPE;
    if (dtype < GN_F32 || dtype > GN_F16) return GN_ERR_UNSUPPORTED;
    if (total > (1LL << 48) / width) return GN_ERR_TOO_LARGE;
    const long long slabs = (width + slab_width(dtype) - 1) / slab_width(dtype);
    if ((n + 1LL) * slabs * kMaxCluster > 0x7fffffffLL) return GN_ERR_TOO_LARGE;
    return GN_OK;
}

static int scan_interval(int n, long long steps, long long total, int width, int dtype, bool ragged)
{
    const long long mean = ragged ? total / (n > 0 ? n : 1) : steps;
    return held_steps(dtype) * scan_cluster(n, mean, width, dtype == GN_F32 ? 4 : 2, true);
}

static int launch_scan(void (*kern)(const Scan), const Scan &p, const char *what, cudaStream_t st)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.n + (p.offsets ? 1LL : 0LL)) * p.slabs * p.cluster));
    cfg.blockDim = dim3(kScanThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) {
        record_cuda_error(e, what);
        (void)cudaGetLastError();
        return GN_ERR_CUDA;
    }
    return check_launch(what);
}

template <typename T>
static int scan_forward(Scan &p, cudaStream_t st)
{
    p.slabs = (p.width + Lay<T>::kWidth - 1) / Lay<T>::kWidth;
    return launch_scan(p.pack_gate ? scan_forward_k<T, false, true> : scan_forward_k<T, false, false>, p, "gated_scan", st);
}

template <typename T>
static int scan_backward(Scan &p, bool packed, bool long_sequences, cudaStream_t st)
{
    p.slabs = (p.width + Lay<T>::kWidth - 1) / Lay<T>::kWidth;
    if (packed && long_sequences) {  // the states that the codes lead to
        const int rc = launch_scan(scan_forward_k<T, true, false>, p, "gated_scan states", st);
        if (rc != GN_OK) return rc;
    }
    return launch_scan(packed ? scan_backward_k<T, true> : scan_backward_k<T, false>, p, "gated_scan backward", st);
}

}  // namespace gn

using namespace gn;

extern "C" {

GN_API size_t gn_gated_scan_bounds_bytes(int n, long long steps, long long total, int width, int dtype, int ragged)
{
    if (scan_check(n, steps, total, width, dtype, ragged != 0) != GN_OK || n == 0 || total == 0) return 0;
    const int interval = scan_interval(n, steps, total, width, dtype, ragged != 0);
    if ((ragged ? total : steps) <= interval) return 0;
    const long long rows = ragged ? total / interval + n + 1 : n * ((steps + interval - 1) / interval);
    return sizeof(float) * (size_t)rows * width;
}

GN_API int gn_gated_scan_forward(const void *gate, const void *value, const float *state, const long long *offsets, void *h, float *last,
                                 void *gate_codes, void *gate_scales, void *value_codes, void *value_scales, float *bounds, int n,
                                 long long steps, long long total, int width, long long gate_seq, long long gate_step, long long value_seq,
                                 long long value_step, int dtype, void *stream)
{
    const int rc = scan_check(n, steps, total, width, dtype, offsets != nullptr);
    if (rc != GN_OK) return rc;
    if (gate_codes && (!gate_scales || !value_codes || !value_scales)) return GN_ERR_NULL_POINTER;
    if (total > 0 && (!gate || !value || !h)) return GN_ERR_NULL_POINTER;
    if (n == 0 && !(offsets && total > 0)) return GN_OK;
    Scan p{};
    p.gate = gate; p.value = value; p.state = state; p.offsets = offsets; p.h = h; p.last = last;
    p.pack_gate = (unsigned char *)gate_codes; p.pack_gate_scales = (unsigned char *)gate_scales;
    p.pack_value = (unsigned char *)value_codes; p.pack_value_scales = (unsigned char *)value_scales;
    p.bounds = gate_codes ? nullptr : bounds;  // those of the codes are found when they are wanted
    p.interval = scan_interval(n, steps, total, width, dtype, offsets != nullptr);
    p.gate_seq = gate_seq; p.gate_step = gate_step; p.value_seq = value_seq; p.value_step = value_step;
    p.n = n; p.steps = steps; p.total = total; p.width = width;
    const int size = dtype == GN_F32 ? 4 : 2;
    p.cluster = scan_cluster(n, offsets ? total / (n > 0 ? n : 1) : steps, width, size, false);
    p.vec = width % 4 == 0 && gate_seq % 4 == 0 && gate_step % 4 == 0 && value_seq % 4 == 0 && value_step % 4 == 0 && aligned(gate, 4 * size) &&
            aligned(value, 4 * size) && aligned(h, 4 * size) && aligned(state, 16) && aligned(last, 16) && aligned(bounds, 16) &&
            aligned(gate_codes, 4) && aligned(value_codes, 4);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == GN_F32) return scan_forward<float>(p, st);
    if (dtype == GN_BF16) return scan_forward<__nv_bfloat16>(p, st);
    return scan_forward<__half>(p, st);
}

GN_API int gn_gated_scan_backward(const void *gate, const void *value, const void *gate_scales, const void *value_scales, const float *state,
                                  const long long *offsets, float *bounds, const void *grad_h, const float *grad_last, void *grad_gate,
                                  void *grad_value, float *grad_state, int n, long long steps, long long total, int width, long long gate_seq,
                                  long long gate_step, long long value_seq, long long value_step, int dtype, void *stream)
{
    const int rc = scan_check(n, steps, total, width, dtype, offsets != nullptr);
    if (rc != GN_OK) return rc;
    if (!gate_scales != !value_scales) return GN_ERR_NULL_POINTER;
    if (total > 0 && (!gate || !value || !grad_h || !grad_gate || !grad_value)) return GN_ERR_NULL_POINTER;
    if (n == 0 && !(offsets && total > 0)) return GN_OK;
    const bool long_sequences = gn_gated_scan_bounds_bytes(n, steps, total, width, dtype, offsets != nullptr) > 0;
    if (long_sequences && !bounds) return GN_ERR_WORKSPACE;
    Scan p{};
    p.gate = gate; p.value = value; p.state = state; p.offsets = offsets; p.bounds = bounds;
    p.gate_scales = (const unsigned char *)gate_scales; p.value_scales = (const unsigned char *)value_scales;
    p.gh = grad_h; p.glast = grad_last; p.dgate = grad_gate; p.dvalue = grad_value; p.dstate = grad_state;
    p.interval = scan_interval(n, steps, total, width, dtype, offsets != nullptr);
    p.gate_seq = gate_seq; p.gate_step = gate_step; p.value_seq = value_seq; p.value_step = value_step;
    p.n = n; p.steps = steps; p.total = total; p.width = width;
    p.cluster = p.interval / held_steps(dtype);
    const int size = dtype == GN_F32 ? 4 : 2, in = gate_scales ? 1 : size;
    p.vec = width % 4 == 0 && gate_seq % 4 == 0 && gate_step % 4 == 0 && value_seq % 4 == 0 && value_step % 4 == 0 && aligned(gate, 4 * in) &&
            aligned(value, 4 * in) && aligned(grad_h, 4 * size) && aligned(grad_gate, 4 * size) && aligned(grad_value, 4 * size) &&
            aligned(state, 16) && aligned(grad_last, 16) && aligned(grad_state, 16) && aligned(bounds, 16);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == GN_F32) return scan_backward<float>(p, gate_scales != nullptr, long_sequences, st);
    if (dtype == GN_BF16) return scan_backward<__nv_bfloat16>(p, gate_scales != nullptr, long_sequences, st);
    return scan_backward<__half>(p, gate_scales != nullptr, long_sequences, st);
}

GN_API int gn_gated_scan_step(const void *gate, const void *value, const float *state, void *h, float *out_state, long long rows, int width,
                              long long gate_row, long long value_row, int dtype, void *stream)
{
    if (rows < 0 || width <= 0 || rows > (1LL << 48) / width) return GN_ERR_BAD_SHAPE;
    if (dtype < GN_F32 || dtype > GN_F16) return GN_ERR_UNSUPPORTED;
    if (rows == 0) return GN_OK;
    if (!gate || !value || !state || !h || !out_state) return GN_ERR_NULL_POINTER;
    const int size = dtype == GN_F32 ? 4 : 2;
    const int vec = width % 4 == 0 && gate_row % 4 == 0 && value_row % 4 == 0 && aligned(gate, 4 * size) && aligned(value, 4 * size) &&
                    aligned(h, 4 * size) && aligned(state, 16) && aligned(out_state, 16);
    const long long want = (rows * ((width + 3) / 4) + 255) / 256, most = 16LL * sm_count();
    const unsigned blocks = (unsigned)(want < most ? want : most);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == GN_F32)
        scan_step_k<float><<<blocks, 256, 0, st>>>((const float *)gate, (const float *)value, state, (float *)h, out_state, rows, width, gate_row,
                                                   value_row, vec);
    else if (dtype == GN_BF16)
        scan_step_k<__nv_bfloat16><<<blocks, 256, 0, st>>>((const __nv_bfloat16 *)gate, (const __nv_bfloat16 *)value, state, (__nv_bfloat16 *)h,
                                                           out_state, rows, width, gate_row, value_row, vec);
    else
        scan_step_k<__half><<<blocks, 256, 0, st>>>((const __half *)gate, (const __half *)value, state, (__half *)h, out_state, rows, width,
                                                    gate_row, value_row, vec);
    return check_launch("gated_scan_step");
}

}  // extern "C"
