// Gated linear recurrence over sequences: h_t = a_t h_{t-1} + n_t u_t with a_t = s(z_t), n_t = s(-z_t) = 1 - a_t, s the logistic
// function - the update of the gated grid's cell (gridnet/backend_torch.py:241-265) with gate z and value u given.
//
// Every step is an affine map of the state, and so is every run of steps: (A, H) stands for h -> A h + H, and
// (A2, H2) after (A1, H1) is (A1 A2, A2 H1 + H2). A thread composes the steps it holds in registers, warps compose through shared memory;
// then each thread knows the state ahead of its first step and runs its steps again from registers.
//
// Backward: c_t = gradient of h_{t-1} = a_t (g_t + c_{t+1}) is affine in c_{t+1}, from the end to the start, with the same A;
//     dh_t = g_t + c_{t+1},  du_t = n_t dh_t,  dz_t = a_t n_t (h_{t-1} - u_t) dh_t.
// h is not kept but run again: both directions are composed in the same exchange, from one reading of gate, value and g.
//
// Two ways along a sequence:
//   walk     a CTA has 64 channels of a sequence and goes from tile to tile, everything read once. Backward it needs the state ahead
//            of each tile, which the forward pass has left. For many sequences or channels.
//   chunks   every tile is a CTA of its own: one kernel composes each tile's steps, one goes over the tiles and says where
//            each starts, one does the work. gate and value (and g) are read twice, the second time from L2 where they fit.
//            For few and long sequences, and for the backward pass from packed copies, where there is no state that could have been left.
// A cluster of CTAs that walks together and exchanges maps through distributed shared memory was measured as a third way: 1.5 us more for
// a round of tiles, slower than the chunks (4 x 4097 x 1024 float32, backward from packed copies, 157 us).
//
// Steps whose n_t is 0 (gates from about 104 up, and +inf) do not look at their value, which may be NaN; steps whose a_t is 0 do not look
// at the state. Anything else that is not finite stays in the state. Threads that hold a gate beyond 80 select while they compute the gates,
// those that hold a reset (a_t = 0) also while they go through the steps; all others have products and sums alone. A run with a reset has the
// sign bit in A (-0). One without, whose factors' product is too small for a float, has the smallest one there is: off by less
// than that, as a product of that size is once it is rounded, and a state that is infinite stays so, where 0 * inf would be no number.
//
// A thread has two channels, so that a row is read 64 channels at a time and arithmetic is on pairs (f32x2); a warp has a run of steps
// of its own, no lane has to know another lane's.
#include <type_traits>

#include "kernels.h"
#include "packed8.cuh"

namespace gn {

constexpr int kScanThreads = 128, kScanWarps = 4;
constexpr int kSlab = 64;                     // channels of a CTA
constexpr int kFwdSteps = 16, kBwdSteps = 8;  // steps that a thread holds
constexpr int kFwdLog2 = 6, kBwdLog2 = 5;     // of a tile's steps
constexpr int kFwdTile = 1 << kFwdLog2, kBwdTile = 1 << kBwdLog2;
static_assert(kFwdTile == kScanWarps * kFwdSteps && kBwdTile == kScanWarps * kBwdSteps, "a tile is what a CTA holds");
constexpr int kSumSteps = 8;                  // steps that a thread composes at a time when a warp has a tile to itself
constexpr int kStartRuns = 64;                // at most

struct Scan {
    const void *gate, *value;  // or codes
    const unsigned char *gate_scales, *value_scales;
    long long gate_seq, gate_step, value_seq, value_step;  // strides in elements
    const float *state;         // [n][width] or nullptr
    const long long *offsets;   // [n + 1] or nullptr
    void *h;
    float *last;
    unsigned char *pack_gate, *pack_value, *pack_gate_scales, *pack_value_scales;
    float *bounds;  // walk: state ahead of each backward tile of a sequence but the first
    float *maps;    // chunks: A, H and (backward) C of each tile, planes of map_rows x padded; H and C give way to where the tile starts
    long long map_rows;
    int tiles_per_cta;  // chunks
    const void *gh;
    const float *glast;
    void *dgate, *dvalue;
    float *dstate;
    int n, width, slabs, padded;  // padded: slabs * kSlab
    int vec;   // pairs of channels lie on whole pairs' addresses
    int wide;  // 16 bytes of a row on multiples of 16
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
// Row of p.bounds or p.maps that belongs to tile k of a sequence, tiles of 2^LOG2 steps
template <int LOG2>
__device__ __forceinline__ long long tile_row(const Scan &p, int seq, const Place &s, long long k)
{
    if (!p.offsets) return seq * ((p.steps + (1 << LOG2) - 1) >> LOG2) + k;
    return (s.first >> LOG2) + seq + k;  // a sequence has at most one tile more than its rows have multiples of a tile
}
// and the other way round; false where the row belongs to no tile. All lanes of a warp call with the same row
template <int LOG2>
__device__ __forceinline__ bool tile_of_row(const Scan &p, long long row, int &seq, Place &s, long long &k)
{
    if (!p.offsets) {
        const long long tiles = (p.steps + (1 << LOG2) - 1) >> LOG2;
        seq = (int)(row / tiles);
        s = sequence(p, seq);
        k = row - seq * tiles;
        return true;
    }
    // the last sequence that starts at this row or before: 32 places at a time, a lane each (n <= 1024: two loads one after the other)
    const int lane = threadIdx.x & 31;
    int lo = 0;
    for (int left = p.n; left > 1;) {
        const int step = (left + 31) / 32, at = lo + lane * step;
        const bool before = lane * step < left && (min(max(p.offsets[min(at, p.n)], 0LL), p.total) >> LOG2) + at <= row;
        const int found = max(__popc(__ballot_sync(0xffffffffu, before)) - 1, 0);
        lo += found * step;
        left = min(step, left - found * step);
    }
    seq = lo;
    s = sequence(p, seq);
    k = row - ((s.first >> LOG2) + seq);
    return k >= 0 && k << LOG2 < s.len;
}

// ---- pairs
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 two(float v) { return make_float2(v, v); }

__device__ __forceinline__ float2 load2v(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 load2v(const __nv_bfloat16 *p)
{
    const unsigned q = *reinterpret_cast<const unsigned *>(p);
    return make_float2(__uint_as_float(q << 16), __uint_as_float(q & 0xffff0000u));
}
__device__ __forceinline__ float2 load2v(const __half *p) { return __half22float2(*reinterpret_cast<const __half2 *>(p)); }
__device__ __forceinline__ void store2v(float *p, float2 v) { *reinterpret_cast<float2 *>(p) = v; }
__device__ __forceinline__ void store2v(__nv_bfloat16 *p, float2 v) { *reinterpret_cast<__nv_bfloat162 *>(p) = __float22bfloat162_rn(v); }
__device__ __forceinline__ void store2v(__half *p, float2 v) { *reinterpret_cast<__half2 *>(p) = __float22half2_rn(v); }
// n: how many of the two are there (what is not reads as 0); vec: pairs lie on whole pairs' addresses
template <typename T>
__device__ __forceinline__ float2 load2(const T *p, bool vec, int n)
{
    if (vec && n == 2) return load2v(p);
    return make_float2(n > 0 ? to_float<T>(p[0]) : 0.0f, n > 1 ? to_float<T>(p[1]) : 0.0f);
}
template <typename T>
__device__ __forceinline__ void store2(T *p, bool vec, int n, float2 v)
{
    if (vec && n == 2) {
        store2v(p, v);
        return;
    }
    if (n > 0) p[0] = from_float<T>(v.x);
    if (n > 1) p[1] = from_float<T>(v.y);
}

// s(z) and s(-z) for |z| < kFar; everything else, and what is behind the end, goes through gates_any.
// e = exp(-z) as 2^t: t is rounded, which is as if z were another number 1.3 half steps of float32 away, about as far as z has been rounded
// to begin with. Where s(z) is the larger of the two it is 1 less the other, so that its error is its own rounding: memories of thousands of
// steps add it up (8 x 2048 x 4096, gradient of the state, off in the 2-norm: 1.8e-7; as 1 / (1 + e) with a Newton step 2.3e-6, because of
// the rounding of 1 + e; without that step 1.4e-6).
constexpr float kFar = 80.0f;
__device__ __forceinline__ void gates(float2 z, float2 &a, float2 &n)
{
    const float2 t = mul2(z, two(-1.4426950408889634f));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    const float2 one = two(1.0f), w = add2(e, one);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(w.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(w.y));
    n = mul2(e, r);
    const float2 p = fma2(n, two(-1.0f), one);
    a = make_float2(z.x < 0.0f ? r.x : p.x, z.y < 0.0f ? r.y : p.y);
}
// For every z. From kFar on 1 + e is 1 and the smaller of the two is e itself, 0 from |z| = 104 on
__device__ __forceinline__ void gates_any(float2 z, float2 &a, float2 &n)
{
    const float dx = fabsf(z.x), dy = fabsf(z.y);
    const bool fx = !(dx < kFar), fy = !(dy < kFar);
    gates(make_float2(fx ? 0.0f : z.x, fy ? 0.0f : z.y), a, n);
    float ex, ey;
    asm("ex2.approx.f32 %0, %1;" : "=f"(ex) : "f"(-1.4426950408889634f * dx));
    asm("ex2.approx.f32 %0, %1;" : "=f"(ey) : "f"(-1.4426950408889634f * dy));
    if (fx) {
        const float one = dx == dx ? 1.0f : dx;  // NaN: both
        a.x = z.x < 0.0f ? ex : one;
        n.x = z.x < 0.0f ? one : ex;
    }
    if (fy) {
        const float one = dy == dy ? 1.0f : dy;
        a.y = z.y < 0.0f ? ey : one;
        n.y = z.y < 0.0f ? one : ey;
    }
}

// ---- maps of runs. The sign bit of A: the run has a reset, what was before it does not show
__device__ __forceinline__ bool resets(float a) { return __float_as_int(a) < 0; }
__device__ __forceinline__ float through(float a, float h, float b) { return resets(a) ? b : fmaf(a, h, b); }
__device__ __forceinline__ float2 through(float2 a, float2 h, float2 b) { return make_float2(through(a.x, h.x, b.x), through(a.y, h.y, b.y)); }
__device__ __forceinline__ float product(float a, float b)
{
    return __uint_as_float(__float_as_uint(a * b) | ((__float_as_uint(a) | __float_as_uint(b)) & 0x80000000u));
}
__device__ __forceinline__ float2 product(float2 a, float2 b) { return make_float2(product(a.x, b.x), product(a.y, b.y)); }
__device__ __forceinline__ float at_least(float a)  // a >= 0 or NaN
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(__uint_as_float(1u)));
    return m;
}
__device__ __forceinline__ float2 at_least(float2 a) { return make_float2(at_least(a.x), at_least(a.y)); }
__device__ __forceinline__ float2 kept(float2 a) { return make_float2(resets(a.x) ? a.x : at_least(a.x), resets(a.y) ? a.y : at_least(a.y)); }
// one step with a_t = 0 or n_t = 0 among those of the thread
__device__ __forceinline__ float after(float a, float h, float b) { return a == 0.0f ? b : fmaf(a, h, b); }
__device__ __forceinline__ float2 after(float2 a, float2 h, float2 b) { return make_float2(after(a.x, h.x, b.x), after(a.y, h.y, b.y)); }
__device__ __forceinline__ float2 more(float2 A, float2 a)
{
    return make_float2(a.x == 0.0f ? -0.0f : product(A.x, a.x), a.y == 0.0f ? -0.0f : product(A.y, a.y));
}
__device__ __forceinline__ float2 looked_at(float2 n, float2 v) { return make_float2(n.x == 0.0f ? 0.0f : v.x, n.y == 0.0f ? 0.0f : v.y); }

// Gradient term of a run with another step (or run) behind it: A of all of them, g of that one; nothing passes a reset
__device__ __forceinline__ float behind(float A, float g, float c) { return resets(A) ? c : fmaf(A, g, c); }
__device__ __forceinline__ float2 behind(float2 A, float2 g, float2 c) { return make_float2(behind(A.x, g.x, c.x), behind(A.y, g.y, c.y)); }
__device__ __forceinline__ bool not_a_number(float2 v) { return v.x != v.x || v.y != v.y; }

// Rows outside of every sequence of a ragged call: zeros
template <typename T>
__device__ void clear_rows(const Scan &p, T *x, int slab)
{
    const long long lo = min(max(p.offsets[0], 0LL), p.total), hi = min(max(p.offsets[p.n], lo), p.total);
    const int ch = slab * kSlab + (threadIdx.x & 31) * 2, nch = min(2, max(0, p.width - ch));
    for (long long i = threadIdx.x >> 5; i < lo + p.total - hi; i += blockDim.x >> 5) {
        const long long row = i < lo ? i : i - lo + hi;
        store2(x + row * p.width + ch, p.vec, nch, two(0.0f));
    }
}

// Rows behind the end have `end`. Every load stands without a condition of its own (rows behind the end read the last one again): loads under
// conditions are waited for one by one, 600 cycles each.
template <typename T, int S>
__device__ __forceinline__ void load_rows(const T *x, long long step, bool vec, int cnt, int nch, float end, float2 (&v)[S])
{
    if (cnt == S && vec && nch == 2) {
#pragma unroll
        for (int s = 0; s < S; ++s) v[s] = load2v(x + s * step);
        return;
    }
    if (cnt > 0 && nch > 0) {
        T one[S], other[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const T *const at = x + min(s, cnt - 1) * step;
            one[s] = at[0];
            other[s] = at[nch - 1];
        }
#pragma unroll
        for (int s = 0; s < S; ++s) v[s] = s < cnt ? make_float2(to_float<T>(one[s]), nch > 1 ? to_float<T>(other[s]) : 0.0f) : two(end);
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s) v[s] = s < cnt ? two(0.0f) : two(end);
    }
}

// the codes of two channels of each row; rows behind the end have the last one's
template <int S>
__device__ __forceinline__ void load_codes(const unsigned char *c, long long width, bool vec, int cnt, int nch, unsigned (&w)[S])
{
    if (cnt <= 0 || nch <= 0) {
#pragma unroll
        for (int s = 0; s < S; ++s) w[s] = 0u;
    } else if (vec && nch == 2) {
#pragma unroll
        for (int s = 0; s < S; ++s) w[s] = *reinterpret_cast<const unsigned short *>(c + min(s, cnt - 1) * width);
    } else {
        unsigned other[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const unsigned char *const at = c + min(s, cnt - 1) * width;
            w[s] = at[0];
            other[s] = at[nch - 1];
        }
#pragma unroll
        for (int s = 0; s < S; ++s) w[s] |= nch > 1 ? other[s] << 8 : 0u;
    }
}

// ---- packing of the rows that a warp holds, 16 of gate and of value, 64 channels each: two groups a row, half of the warp's lanes a group.
// The scale of a group follows from the upper 16 bits of its largest magnitude, rounded up (125 / 64 has no more), so that of gate and value are
// looked for together, as two 16-bit numbers; and for all rows at a time, halving the rows that a lane still looks at: lane l of a
// half ends up with row l. What is not finite is above kLargestKey, and so is a group that would need 2^122.
constexpr unsigned kLargestKey = kPackLargest >> 16;
__device__ __forceinline__ float larger(float2 v)  // magnitude; NaN where one of the two is
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(v.x)), "f"(fabsf(v.y)));
    return m;
}
__device__ __forceinline__ unsigned keys_of(float gate, float value)
{
    return __byte_perm(__float_as_uint(gate) + 0xffffu, __float_as_uint(value) + 0xffffu, 0x7632);
}
__device__ __forceinline__ unsigned scale_of_key(unsigned key)
{
    return (unsigned)max((int)(key >> 7) - 6 + ((key & 0x7fu) > 0x7au ? 1 : 0), 1);
}
// the largest of 16 lanes, row by row
__device__ __forceinline__ unsigned rows_to_lanes(unsigned (&m)[kFwdSteps])
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = kFwdSteps / 2; h > 0; h >>= 1) {
        const bool upper = lane & h;
#pragma unroll
        for (int s = 0; s < h; ++s) {
            const unsigned give = upper ? m[s] : m[s + h], keep = upper ? m[s + h] : m[s];
            m[s] = __vmaxu2(keep, __shfl_xor_sync(0xffffffffu, give, h));
        }
    }
    return m[0];
}
struct PackTo {
    unsigned char *gate, *value, *gate_scales, *value_scales;
};
// whole: all rows are there, and pairs of codes lie on even addresses (a lane has two channels or none)
__device__ __forceinline__ void pack_rows(const float2 (&z)[kFwdSteps], const float2 (&u)[kFwdSteps], const PackTo &to, long long row, int width, int ch,
                                          bool whole, int cnt, int nch)
{
    const int lane = threadIdx.x & 31, per_row = (width + kPackGroup - 1) / kPackGroup, group = ch / kPackGroup;
    if (cnt <= 0) return;  // the whole warp
    unsigned m[kFwdSteps];
#pragma unroll
    for (int s = 0; s < kFwdSteps; ++s) m[s] = keys_of(larger(z[s]), larger(u[s]));
    if (!whole)
#pragma unroll
        for (int s = 0; s < kFwdSteps; ++s)
            if (s >= cnt) m[s] = 0u;
    unsigned key = rows_to_lanes(m);
    const bool rare = __any_sync(0xffffffffu, (key & 0xffffu) > kLargestKey || key >> 16 > kLargestKey);
    if (rare) {  // once more over what is finite
#pragma unroll
        for (int s = 0; s < kFwdSteps; ++s) {
            float2 f = z[s], g = u[s];
            f.x = bits_finite(magnitude_bits(f.x)) ? f.x : 0.0f;
            f.y = bits_finite(magnitude_bits(f.y)) ? f.y : 0.0f;
            g.x = bits_finite(magnitude_bits(g.x)) ? g.x : 0.0f;
            g.y = bits_finite(magnitude_bits(g.y)) ? g.y : 0.0f;
            m[s] = s < cnt ? keys_of(larger(f), larger(g)) : 0u;
        }
        key = rows_to_lanes(m);
    }
    const unsigned zs = scale_of_key(key & 0xffffu), us = scale_of_key(key >> 16);
    if ((lane & 15) < cnt && group < per_row) {
        const long long at = (row + (lane & 15)) * per_row + group;
        to.gate_scales[at] = (unsigned char)zs;
        to.value_scales[at] = (unsigned char)us;
    }
    unsigned char *zc = to.gate + row * width + ch, *uc = to.value + row * width + ch;
    // the last rows and odd widths byte by byte, in a loop of their own: 4 x 4097 x 1023 float32 122 us code by code -> 100, 16 x 1024 x 1001 148 -> 98
    auto code_rows = [&](auto store) {
        // the upper halves of both 2^-e (the lower ones are 0)
        const unsigned inverses = __byte_perm(__float_as_uint(pack_inverse(zs)), __float_as_uint(pack_inverse(us)), 0x7632);
        const float2 magic = two(12582912.0f);
#pragma unroll
        for (int s = 0; s < kFwdSteps; ++s, zc += width, uc += width) {
            const unsigned both = __shfl_sync(0xffffffffu, inverses, (lane & 16) | s);
            const float2 c = fma2(z[s], two(__uint_as_float(both << 16)), magic), d = fma2(u[s], two(__uint_as_float(both & 0xffff0000u)), magic);
            store(s, __byte_perm(__float_as_uint(c.x), __float_as_uint(c.y), 0x0040), __byte_perm(__float_as_uint(d.x), __float_as_uint(d.y), 0x0040));
        }
    };
    if (whole && !rare) {
        code_rows([&](int, unsigned z2, unsigned u2) {
            if (nch == 2) {
                *reinterpret_cast<unsigned short *>(zc) = (unsigned short)z2;
                *reinterpret_cast<unsigned short *>(uc) = (unsigned short)u2;
            }
        });
        return;
    }
    if (!rare) {
        code_rows([&](int s, unsigned z2, unsigned u2) {
            if (s < cnt && nch > 0) {
                zc[0] = (unsigned char)z2;
                uc[0] = (unsigned char)u2;
            }
            if (s < cnt && nch > 1) {
                zc[1] = (unsigned char)(z2 >> 8);
                uc[1] = (unsigned char)(u2 >> 8);
            }
        });
        return;
    }
#pragma unroll
    for (int s = 0; s < kFwdSteps; ++s, zc += width, uc += width) {
        const unsigned both = __shfl_sync(0xffffffffu, zs | us << 16, (lane & 16) | s);
        if (s < cnt && nch > 0) {
            zc[0] = (unsigned char)pack_code_any(z[s].x, both & 0xffffu);
            uc[0] = (unsigned char)pack_code_any(u[s].x, both >> 16);
            if (nch > 1) {
                zc[1] = (unsigned char)pack_code_any(z[s].y, both & 0xffffu);
                uc[1] = (unsigned char)pack_code_any(u[s].y, both >> 16);
            }
        }
    }
}

template <int S>
__device__ __forceinline__ float farthest(const float2 (&z)[S])  // |z|; NaN does not count
{
    float m = 0.0f;
#pragma unroll
    for (int s = 0; s < S; ++s) m = fmaxf(m, fmaxf(fabsf(z[s].x), fabsf(z[s].y)));
    return m;
}

// ---- a warp's next steps on their way to shared memory while the ones in hand are worked on: S rows of 64 values each
__device__ __forceinline__ void copy16(void *to, const void *from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_on_their_way() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_there()  // all lanes' of the warp
{
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
}
template <typename V, int S>
struct Rows {
    V v[S][kSlab];
    static constexpr int kPer = 16 / sizeof(V), kChunks = kSlab / kPer, kAtOnce = 32 / kChunks;  // values of a copy, copies of a row, rows of a round
};
// Where a lane's first copy of a tile starts; from: first value of the slab in the first row
template <typename V, int S>
__device__ __forceinline__ const V *asks_from(const V *from, long long step)
{
    using R = Rows<V, S>;
    const int lane = threadIdx.x & 31;
    return from + lane / R::kChunks * step + lane % R::kChunks * R::kPer;
}
// left: values of a row from the slab's first on
template <typename V, int S>
__device__ __forceinline__ void ask(Rows<V, S> &to, const V *from, long long step, int cnt, int left)
{
    using R = Rows<V, S>;
    const int lane = threadIdx.x & 31;
    V *const place = &to.v[0][0] + lane * R::kPer;
    if (cnt == S && left >= kSlab) {
#pragma unroll
        for (int i = 0; i < S / R::kAtOnce; ++i, from += R::kAtOnce * step) copy16(place + i * 32 * R::kPer, from);
    } else {
        const int row = lane / R::kChunks, col = lane % R::kChunks * R::kPer;
        for (int i = 0; i < S / R::kAtOnce; ++i, from += R::kAtOnce * step)
            if (row + i * R::kAtOnce < cnt && col < left) copy16(place + i * 32 * R::kPer, from);
    }
}
// What has been asked for, as load_rows gives it
template <typename T, int S>
__device__ __forceinline__ void take(const Rows<T, S> &from, int cnt, int nch, float end, float2 (&v)[S])
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int s = 0; s < S; ++s) v[s] = load2v(&from.v[s][lane * 2]);
    if (cnt < S || nch == 0)
#pragma unroll
        for (int s = 0; s < S; ++s) v[s] = s >= cnt ? two(end) : nch == 0 ? two(0.0f) : v[s];
}
// The scale bytes of gate and of value for a warp's steps: lane 2 r + g has row r, group g of the slab. Put together only where they are used:
// whoever combines them waits for them.
struct Scales {
    unsigned char gate, value;
};
__device__ __forceinline__ Scales ask_scales(const Scan &p, long long row, int slab, int cnt)
{
    const int lane = threadIdx.x & 31, r = lane >> 1, g = slab * (kSlab / kPackGroup) + (lane & 1), per_row = (p.width + kPackGroup - 1) / kPackGroup;
    const bool there = r < cnt && g < per_row;
    const long long at = there ? (row + r) * per_row + g : 0;
    return {p.gate_scales[at], p.value_scales[at]};
}
// gate and value as their codes give them; word(value, s): the codes of steps s and s + 1
template <int S, typename Word>
__device__ __forceinline__ void take_packed(Word word, Scales scales, int cnt, int nch, float end, float2 (&z)[S], float2 (&u)[S])
{
    const int lane = threadIdx.x & 31;
    unsigned wz[S / 2], wu[S / 2];
    float far = 0.0f;
    auto whole = [&](unsigned w, float2 &a, float2 &b) {
        float f[4];
        unpack4_finite(w, f);
        far = fmaxf(fmaxf(far, fmaxf(fabsf(f[0]), fabsf(f[1]))), fmaxf(fabsf(f[2]), fabsf(f[3])));
        a = make_float2(f[0], f[1]);
        b = make_float2(f[2], f[3]);
    };
#pragma unroll
    for (int s = 0; s < S; s += 2) {
        whole(wz[s / 2] = word(false, s), z[s], z[s + 1]);
        whole(wu[s / 2] = word(true, s), u[s], u[s + 1]);
    }
    const unsigned steps = (scales.gate | (unsigned)scales.value << 16) << 7;  // the upper halves of both 2^e (the lower ones are 0)
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const unsigned both = __shfl_sync(0xffffffffu, steps, 2 * s + (lane >> 4));
        z[s] = mul2(z[s], two(__uint_as_float(both << 16)));
        u[s] = mul2(u[s], two(__uint_as_float(both & 0xffff0000u)));
    }
    if (far > 125.0f) {  // some code stands for what is not finite
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const unsigned c = wz[s / 2] >> (s % 2 * 16), d = wu[s / 2] >> (s % 2 * 16);
            z[s] = make_float2(unpack_special(z[s].x, c & 0xffu), unpack_special(z[s].y, (c >> 8) & 0xffu));
            u[s] = make_float2(unpack_special(u[s].x, d & 0xffu), unpack_special(u[s].y, (d >> 8) & 0xffu));
        }
    }
    if (cnt < S || nch == 0)
#pragma unroll
        for (int s = 0; s < S; ++s) {
            z[s] = s >= cnt ? two(end) : nch == 0 ? two(0.0f) : z[s];
            u[s] = s >= cnt || nch == 0 ? two(0.0f) : u[s];
        }
}

// All gates of a thread's steps: z becomes s(z), and a value that is not looked at 0. Returns what there is
enum { kNear, kFarGates, kResets };
template <int S>
__device__ __forceinline__ int gates_of(float2 (&z)[S], float2 (&n)[S], float2 (&u)[S])
{
    if (farthest(z) < kFar) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float2 a;
            gates(z[s], a, n[s]);
            z[s] = a;
        }
        return kNear;
    }
    float least = 1.0f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        float2 a;
        gates_any(z[s], a, n[s]);
        z[s] = a;
        u[s] = looked_at(n[s], u[s]);
        least = fminf(least, fminf(a.x, a.y));
    }
    return least == 0.0f ? kResets : kFarGates;
}

// What a warp's, a CTA's steps amount to: (A, H) and, backward, (A, C) of a channel pair; two copies, so that one barrier lies between
// writing and writing again
__device__ __forceinline__ float4 map_of(float2 A, float2 H) { return make_float4(A.x, A.y, H.x, H.y); }
__device__ __forceinline__ float2 factor(float4 m) { return make_float2(m.x, m.y); }
__device__ __forceinline__ float2 term(float4 m) { return make_float2(m.z, m.w); }
__device__ __forceinline__ float2 through(float4 m, float2 h) { return through(factor(m), h, term(m)); }
__device__ __forceinline__ float2 straight(float4 m, float2 h) { return fma2(factor(m), h, term(m)); }  // no resets
template <int WAYS>
struct Exchange {
    float4 warp[2][WAYS][kScanWarps][32];
};
__device__ __forceinline__ float2 *plane(const Scan &p, int way, long long row, int slab)
{
    return reinterpret_cast<float2 *>(p.maps + (way * p.map_rows + row) * p.padded + slab * kSlab) + (threadIdx.x & 31);
}

// Where a warp's rows of gate and value (and g) come from; S rows at a time
template <typename T, bool PACKED, bool GRAD, int S>
struct Source {
    using V = std::conditional_t<PACKED, unsigned char, T>;
    static constexpr size_t kBytes = sizeof(Rows<V, S>) * 2 + (GRAD ? sizeof(Rows<T, S>) : 0);  // shared memory of a warp
    static_assert(kScanWarps * kBytes + 8192 <= 48 * 1024, "what a kernel may have without being asked for, with an Exchange");
    const Scan &p;
    const int slab, ch, nch, left;
    const long long gate_step, value_step;
    long long first;
    const V *gate, *value;
    const T *grad;
    Rows<V, S> *zs, *us;
    Rows<T, S> *gs;
    Scales scales;

    __device__ __forceinline__ Source(const Scan &p, int slab, unsigned char *shared)
        : p(p), slab(slab), ch(slab * kSlab + (threadIdx.x & 31) * 2), nch(min(2, max(0, p.width - ch))), left(p.width - slab * kSlab),
          // codes lie in rows of width, one after the other
          gate_step(PACKED ? p.width : p.gate_step), value_step(PACKED ? p.width : p.value_step)
    {
        zs = reinterpret_cast<Rows<V, S> *>(shared);
        us = zs + 1;
        gs = reinterpret_cast<Rows<T, S> *>(us + 1);
    }
    __device__ __forceinline__ void turn_to(int seq, const Place &q)
    {
        first = q.first;
        gate = (const V *)p.gate + (PACKED || p.offsets ? first * gate_step : seq * p.gate_seq) + slab * kSlab;
        value = (const V *)p.value + (PACKED || p.offsets ? first * value_step : seq * p.value_seq) + slab * kSlab;
        grad = GRAD ? (const T *)p.gh + first * p.width + slab * kSlab : nullptr;
    }
    // cnt rows from step t of the sequence on (none: nothing)
    __device__ __forceinline__ void ask_for(long long t, int cnt)
    {
        if (cnt <= 0) return;
        if constexpr (PACKED) scales = ask_scales(p, first + t, slab, cnt);
        if (!p.wide) return;
        ask(*zs, asks_from<V, S>(gate + t * gate_step, gate_step), gate_step, cnt, left);
        ask(*us, asks_from<V, S>(value + t * value_step, value_step), value_step, cnt, left);
        if constexpr (GRAD) ask(*gs, asks_from<T, S>(grad + t * p.width, p.width), (long long)p.width, cnt, left);
        copies_on_their_way();
    }
    // What was asked for; a step behind the end holds the state and has no gradient of its own. Then `ask_for` may ask for other rows
    __device__ __forceinline__ void take_from(long long t, int cnt, float2 (&z)[S], float2 (&u)[S], float2 (&g)[GRAD ? S : 1])
    {
        const float inf = __uint_as_float(0x7f800000u);
        if (p.wide) {
            copies_there();
            if constexpr (PACKED) {
                auto word = [&](bool value, int s) {
                    const unsigned char *const at = &(value ? us : zs)->v[s][(threadIdx.x & 31) * 2];
                    return __byte_perm(*reinterpret_cast<const unsigned short *>(at), *reinterpret_cast<const unsigned short *>(at + kSlab), 0x5410);
                };
                take_packed<S>(word, scales, cnt, nch, inf, z, u);
            } else {
                take(*zs, cnt, nch, inf, z);
                take(*us, cnt, nch, 0.0f, u);
            }
            if constexpr (GRAD) take(*gs, cnt, nch, 0.0f, g);
            __syncwarp();
        } else {
            const int lane = threadIdx.x & 31;
            if constexpr (PACKED) {
                unsigned wz[S], wu[S];
                load_codes<S>(gate + lane * 2 + t * p.width, p.width, p.vec, cnt, nch, wz);
                load_codes<S>(value + lane * 2 + t * p.width, p.width, p.vec, cnt, nch, wu);
                take_packed<S>([&](bool value, int s) { return value ? wu[s] | wu[s + 1] << 16 : wz[s] | wz[s + 1] << 16; }, scales, cnt, nch, inf, z, u);
            } else {
                load_rows<T, S>(gate + lane * 2 + t * gate_step, gate_step, p.vec, cnt, nch, inf, z);
                load_rows<T, S>(value + lane * 2 + t * value_step, value_step, p.vec, cnt, nch, 0.0f, u);
            }
            if constexpr (GRAD) load_rows<T, S>(grad + lane * 2 + t * p.width, p.width, p.vec, cnt, nch, 0.0f, g);
        }
    }
};

// A tile of a sequence, and what comes after it: walk - the next one of the sequence (backward: the one before); chunks - the next
// row of p.maps that belongs to a tile, up to the CTA's last one
template <int LOG2, bool CHUNK, bool BACKWARD>
struct Cursor {
    Place q;
    long long tile, row, end;
    int seq;

    __device__ __forceinline__ bool find(const Scan &p)
    {
        while (row < end && !tile_of_row<LOG2>(p, row, seq, q, tile)) ++row;
        return row < end;
    }
    __device__ __forceinline__ bool start(const Scan &p, int place)
    {
        if (CHUNK) {
            row = (long long)place * p.tiles_per_cta;
            end = min(row + p.tiles_per_cta, p.map_rows);
            return find(p);
        }
        seq = place;
        q = sequence(p, seq);
        tile = BACKWARD ? ((q.len + (1 << LOG2) - 1) >> LOG2) - 1 : 0;
        return q.len > 0;
    }
    __device__ __forceinline__ bool next(const Scan &p)
    {
        if (CHUNK) {
            ++row;
            ++tile;
            if (row < end && tile << LOG2 < q.len) return true;  // of the same sequence
            return find(p);
        }
        if (BACKWARD) return --tile >= 0;
        return ++tile << LOG2 < q.len;
    }
};

// ------------------------------------------------------------------ chunks: what each tile amounts to, a warp per tile
// C of a tile as products and sums do not give it, where a gradient that is infinite has met a product of 0: step by step, from memory. Threads come here
// by themselves, so the search is another; and from the row alone, so that the kernel holds nothing more for it (selections in the loop above,
// with what they start from held: 4 x 4097 x 1024 float32 backward 105.7 -> 110.8 us, this way 106.7)
template <typename T, bool PACKED>
__device__ float2 once_more(const Scan &p, long long row, int slab)
{
    int seq = 0, end = p.n;
    if (!p.offsets)
        seq = (int)(row / ((p.steps + kBwdTile - 1) >> kBwdLog2));
    else
        while (end - seq > 1) {
            const int middle = seq + (end - seq) / 2;
            (tile_row<kBwdLog2>(p, middle, sequence(p, middle), 0) <= row ? seq : end) = middle;
        }
    const Place q = sequence(p, seq);
    const long long t0 = (row - tile_row<kBwdLog2>(p, seq, q, 0)) << kBwdLog2;
    const int ch = slab * kSlab + (threadIdx.x & 31) * 2, per_row = (p.width + kPackGroup - 1) / kPackGroup;
    float2 A = two(1.0f), C = two(0.0f);
    for (long long t = max(t0, 0LL); t < min(t0 + kBwdTile, q.len); ++t) {  // whatever stands in the offsets, rows of the sequence
        const long long r = q.first + t;
        float z[2] = {0.0f, 0.0f}, g[2] = {0.0f, 0.0f};
        for (int k = 0; k < 2 && ch + k < p.width; ++k) {
            if constexpr (PACKED)
                z[k] = unpack1(((const unsigned char *)p.gate)[r * p.width + ch + k], pack_step(p.gate_scales[r * per_row + (ch + k) / kPackGroup]));
            else
                z[k] = to_float<T>(((const T *)p.gate)[(p.offsets ? r * p.gate_step : seq * p.gate_seq + t * p.gate_step) + ch + k]);
            g[k] = to_float<T>(((const T *)p.gh)[r * p.width + ch + k]);
        }
        float2 a, n;
        gates_any(make_float2(z[0], z[1]), a, n);
        A = kept(more(A, a));
        C = behind(A, make_float2(g[0], g[1]), C);
    }
    return C;
}

template <typename T, bool PACKED, bool BACKWARD>
__global__ void __launch_bounds__(kScanThreads, 7) scan_maps_k(const Scan p)
{
    constexpr int S = kSumSteps, kLog2 = BACKWARD ? kBwdLog2 : kFwdLog2;
    using From = Source<T, PACKED, BACKWARD, S>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int warp = threadIdx.x >> 5;
    const long long id = (long long)blockIdx.x * kScanWarps + warp, row = id / p.slabs;
    const int slab = (int)(id - row * p.slabs);
    if (row >= p.map_rows) return;
    int seq;
    Place q;
    long long k;
    if (!tile_of_row<kLog2>(p, row, seq, q, k)) return;
    From from(p, slab, dynamic + warp * From::kBytes);
    from.turn_to(seq, q);
    long long t = k << kLog2;
    int rows = (int)min(1LL << kLog2, q.len - t);
    from.ask_for(t, min(S, rows));
    float2 A = two(1.0f), H = two(0.0f), C = two(0.0f);
    for (; rows > 0; t += S, rows -= S) {
        float2 z[S], u[S], g[BACKWARD ? S : 1];
        from.take_from(t, min(S, rows), z, u, g);
        from.ask_for(t + S, min(S, rows - S));
        float2 n[S];
        if (gates_of(z, n, u) != kResets && !resets(A.x) && !resets(A.y)) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                H = fma2(z[s], H, mul2(n[s], u[s]));
                A = mul2(A, z[s]);
                if constexpr (BACKWARD) C = fma2(A, g[s], C);
            }
            A = at_least(A);
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                H = after(z[s], H, mul2(n[s], u[s]));
                A = kept(more(A, z[s]));
                if constexpr (BACKWARD) C = behind(A, g[s], C);
            }
        }
    }
    *plane(p, 0, row, slab) = A;
    *plane(p, 1, row, slab) = H;
    if (BACKWARD) {
        if (not_a_number(C)) C = once_more<T, PACKED>(p, row, slab);
        *plane(p, 2, row, slab) = C;
    }
}

// ------------------------------------------------------------------ chunks: where each tile starts. A CTA has 16 channels of a sequence; 8 lanes, two
// channels each, have a run of its tiles; there are up to 64 runs. Channels of the last slab that are not there are computed along
template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(8 * kStartRuns) scan_starts_k(const Scan p)
{
    constexpr int kLog2 = BACKWARD ? kBwdLog2 : kFwdLog2, kBatch = 8;
    __shared__ float4 runs[BACKWARD ? 2 : 1][kStartRuns][8];
    const int all_runs = blockDim.x >> 3;
    const int parts = p.padded / 16, part = blockIdx.x % parts, seq = blockIdx.x / parts;
    previous_done();
    if (seq >= p.n) {
        if (part % 4 == 0) {
            if (BACKWARD) {
                clear_rows<T>(p, (T *)p.dgate, part / 4);
                clear_rows<T>(p, (T *)p.dvalue, part / 4);
            } else {
                clear_rows<T>(p, (T *)p.h, part / 4);
            }
        }
        return;
    }
    const Place q = sequence(p, seq);
    const int lane = threadIdx.x & 7, run = threadIdx.x >> 3, ch = part * 16 + lane * 2, nch = min(2, max(0, p.width - ch));
    const long long state_at = (long long)seq * p.width + ch, tiles = (q.len + (1 << kLog2) - 1) >> kLog2, row = tile_row<kLog2>(p, seq, q, 0);
    const long long per = (tiles + all_runs - 1) / all_runs, lo = min(tiles, run * per);
    const int count = (int)(min(tiles, lo + per) - lo);
    const long long step = p.padded / 2, plane_step = p.map_rows * step;  // of pairs
    float2 *const map = reinterpret_cast<float2 *>(p.maps + (row + lo) * p.padded + ch);
    float2 a[kBatch], b[kBatch], c[kBatch];  // maps of eight tiles at a time
    auto load = [&](int k) {                 // whether none of them has a reset
        int signs = 0;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const float2 *const at = map + min(k + i, count - 1) * step;
            a[i] = at[0];
            b[i] = at[plane_step];
            if (BACKWARD) c[i] = at[2 * plane_step];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) signs |= __float_as_int(a[i].x) | __float_as_int(a[i].y);
        return signs >= 0;
    };
    const bool one_batch = per <= kBatch;  // loaded once
    bool plain = true, all_plain = true;
    float2 A = two(1.0f), H = two(0.0f), C = two(0.0f);
    for (int k = 0; k < count; k += kBatch) {
        all_plain &= plain = load(k);
        if (all_plain && k + kBatch <= count) {  // no selections: 37 ragged sequences of mean 300 x 1000 bfloat16 backward 64 -> 61 us
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (BACKWARD) C = fma2(A, c[i], C);
                H = fma2(a[i], H, b[i]);
                A = at_least(mul2(A, a[i]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (k + i < count) {
                    if (BACKWARD) C = behind(A, c[i], C);
                    H = through(a[i], H, b[i]);
                    A = kept(product(A, a[i]));
                }
        }
    }
    runs[0][run][lane] = map_of(A, H);
    if (BACKWARD) runs[BACKWARD][run][lane] = map_of(A, C);
    const bool straight_on = !__syncthreads_or(!all_plain);
    float2 h = two(0.0f), g = two(0.0f);  // the state ahead of the run, the gradient behind it
    if (p.state) h = load2(p.state + state_at, p.vec, nch);
    if (!BACKWARD && tiles == 0 && run == 0 && p.last) store2(p.last + state_at, p.vec, nch, h);
    const int used = per > 0 ? (int)((tiles + per - 1) / per) : 0;  // runs that have tiles
    if (BACKWARD && p.glast) g = load2(p.glast + state_at, p.vec, nch);
    if (straight_on) {
#pragma unroll 4
        for (int r = 0; r < min(run, used); ++r) h = straight(runs[0][r][lane], h);
        if (BACKWARD)
#pragma unroll 4
            for (int r = used - 1; r > run; --r) g = straight(runs[BACKWARD][r][lane], g);
    } else {
        for (int r = 0; r < min(run, used); ++r) h = through(runs[0][r][lane], h);
        if (BACKWARD)
            for (int r = used - 1; r > run; --r) g = through(runs[BACKWARD][r][lane], g);
    }
    for (int k = 0; k < count; k += kBatch) {
        if (!one_batch) plain = load(k);
        if (plain && k + kBatch <= count) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                map[(k + i) * step + plane_step] = h;
                h = fma2(a[i], h, b[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (k + i < count) {
                    map[(k + i) * step + plane_step] = h;
                    h = through(a[i], h, b[i]);
                }
        }
    }
    if (BACKWARD) {
        for (int k = (count - 1) / kBatch * kBatch; k >= 0 && count > 0; k -= kBatch) {
            if (!one_batch) plain = load(k);  // the states have gone into plane 1 by now, and b is not looked at any more
            if (plain && k + kBatch <= count) {
#pragma unroll
                for (int i = kBatch - 1; i >= 0; --i) {
                    map[(k + i) * step + 2 * plane_step] = g;
                    g = fma2(a[i], g, c[i]);
                }
            } else {
#pragma unroll
                for (int i = kBatch - 1; i >= 0; --i)
                    if (k + i < count) {
                        map[(k + i) * step + 2 * plane_step] = g;
                        g = through(a[i], g, c[i]);
                    }
            }
        }
        if (p.dstate && run == 0) store2(p.dstate + state_at, p.vec, nch, g);
    }
}

// ------------------------------------------------------------------ forward. KEEP: packs gate and value. CHUNK: a tile, else a sequence
template <typename T, bool KEEP, bool CHUNK>
__global__ void __launch_bounds__(kScanThreads, 4) scan_forward_k(const Scan p)
{
    constexpr int S = kFwdSteps;
    using From = Source<T, false, false, S>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ __align__(16) Exchange<1> ex;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slab = blockIdx.x % p.slabs;
    Cursor<kFwdLog2, CHUNK, false> now;
    if (!CHUNK && (int)(blockIdx.x / p.slabs) >= p.n) {
        clear_rows<T>(p, (T *)p.h, slab);
        return;
    }
    bool more_to_come = now.start(p, blockIdx.x / p.slabs);
    From from(p, slab, dynamic + warp * From::kBytes);
    const int ch = from.ch, nch = from.nch;
    const bool vec = p.vec;
    auto rows_at = [&](long long t) { return (int)min((long long)S, max(0LL, now.q.len - t)); };
    auto ask_now = [&] {
        if (CHUNK) from.turn_to(now.seq, now.q);
        from.ask_for((now.tile << kFwdLog2) + warp * S, rows_at((now.tile << kFwdLog2) + warp * S));
    };
    if (!CHUNK) from.turn_to(now.seq, now.q);
    if (more_to_come) ask_now();
    float2 carry = two(0.0f);
    if constexpr (CHUNK) {
        previous_done();
    } else {
        const long long state_at = (long long)now.seq * p.width + ch;
        if (p.state) carry = load2(p.state + state_at, vec, nch);
        if (!more_to_come && p.last && warp == 0) store2(p.last + state_at, vec, nch, carry);
    }
    for (int par = 0; more_to_come; par ^= 1) {
        const long long t0 = (now.tile << kFwdLog2) + warp * S, len = now.q.len, first = now.q.first, state_at = (long long)now.seq * p.width + ch;
        const int cnt = rows_at(t0);
        if constexpr (CHUNK) carry = *plane(p, 1, now.row, slab);
        float2 a[S], b[S], none[1];
        from.take_from(t0, cnt, a, b, none);
        const long long bound_at = !CHUNK && p.bounds ? tile_row<kBwdLog2>(p, now.seq, now.q, t0 >> kBwdLog2) * p.width + ch : 0;
        more_to_come = now.next(p);
        if (more_to_come) ask_now();
        if constexpr (KEEP) {
            const PackTo to = {p.pack_gate, p.pack_value, p.pack_gate_scales, p.pack_value_scales};
            pack_rows(a, b, to, first + t0, p.width, ch, vec && cnt == S, cnt, nch);
        }
        float2 A = two(1.0f), H = two(0.0f);
        bool special;
        {
            float2 n[S];
            special = gates_of(a, n, b) == kResets;
#pragma unroll
            for (int s = 0; s < S; ++s) b[s] = mul2(n[s], b[s]);
        }
        if (!special) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                H = fma2(a[s], H, b[s]);
                A = mul2(A, a[s]);
            }
            A = at_least(A);
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                H = after(a[s], H, b[s]);
                A = more(A, a[s]);
            }
            A = kept(A);
        }
        ex.warp[par][0][warp][lane] = map_of(A, H);
        const bool any = __syncthreads_or(special);
        float2 h = carry;
        if (!any) {
#pragma unroll
            for (int w = 0; w < kScanWarps; ++w) {
                if (w == warp) h = carry;
                carry = straight(ex.warp[par][0][w][lane], carry);
            }
        } else {
#pragma unroll
            for (int w = 0; w < kScanWarps; ++w) {
                if (w == warp) h = carry;
                carry = through(ex.warp[par][0][w][lane], carry);
            }
        }
        // a backward tile is a multiple of a thread's steps: boundaries lie at the start of a thread's steps
        if (!CHUNK && p.bounds && cnt > 0 && t0 > 0 && (t0 & (kBwdTile - 1)) == 0)
            store2(p.bounds + bound_at, vec, nch, h);
        T *out = (T *)p.h + (first + t0) * p.width + ch;
        if (!special) {
#pragma unroll
            for (int s = 0; s < S; ++s) a[s] = h = fma2(a[s], h, b[s]);
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) a[s] = h = after(a[s], h, b[s]);
        }
        if (vec && nch == 2 && cnt == S) {
#pragma unroll
            for (int s = 0; s < S; ++s, out += p.width) store2v(out, a[s]);
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (s < cnt) store2(out + (long long)s * p.width, vec, nch, a[s]);
        }
        if (p.last && cnt > 0 && t0 + cnt == len) store2(p.last + state_at, vec, nch, h);
    }
}

// ------------------------------------------------------------------ backward
template <typename T, bool PACKED, bool CHUNK>
__global__ void __launch_bounds__(kScanThreads, 4) scan_backward_k(const Scan p)
{
    constexpr int S = kBwdSteps;
    using From = Source<T, PACKED, true, S>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ __align__(16) Exchange<2> ex;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slab = blockIdx.x % p.slabs;
    Cursor<kBwdLog2, CHUNK, true> now;
    if (!CHUNK && (int)(blockIdx.x / p.slabs) >= p.n) {
        clear_rows<T>(p, (T *)p.dgate, slab);
        clear_rows<T>(p, (T *)p.dvalue, slab);
        return;
    }
    bool more_to_come = now.start(p, blockIdx.x / p.slabs);
    From from(p, slab, dynamic + warp * From::kBytes);
    const int ch = from.ch, nch = from.nch;
    const bool vec = p.vec;
    auto rows_at = [&](long long t) { return (int)min((long long)S, max(0LL, now.q.len - t)); };
    auto ask_now = [&] {
        if (CHUNK) from.turn_to(now.seq, now.q);
        from.ask_for((now.tile << kBwdLog2) + warp * S, rows_at((now.tile << kBwdLog2) + warp * S));
    };
    if (!CHUNK) from.turn_to(now.seq, now.q);
    if (more_to_come) ask_now();
    float2 carry = two(0.0f);  // gradient of the state behind the steps in hand
    if constexpr (CHUNK) {
        previous_done();
    } else if (p.glast) {
        carry = load2(p.glast + (long long)now.seq * p.width + ch, vec, nch);
    }
    for (int par = 0; more_to_come; par ^= 1) {
        const long long t0 = (now.tile << kBwdLog2) + warp * S, at = (now.q.first + t0) * p.width + ch;
        const int cnt = rows_at(t0);
        float2 a[S], n[S], u[S], g[S], h = two(0.0f);
        from.take_from(t0, cnt, a, u, g);
        const Cursor<kBwdLog2, CHUNK, true> here = now;
        more_to_come = now.next(p);
        if (more_to_come) ask_now();
        if constexpr (CHUNK) {
            h = *plane(p, 1, here.row, slab);
            carry = *plane(p, 2, here.row, slab);
        } else {
            if (here.tile > 0)
                h = load2(p.bounds + tile_row<kBwdLog2>(p, here.seq, here.q, here.tile) * p.width + ch, vec, nch);
            else if (p.state)
                h = load2(p.state + (long long)here.seq * p.width + ch, vec, nch);
        }
        float2 A = two(1.0f), H = two(0.0f), C = two(0.0f);
        const int kind = gates_of(a, n, u);
        const bool special = kind == kResets;
        if (!special) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                H = fma2(a[s], H, mul2(n[s], u[s]));
                A = mul2(A, a[s]);
                C = fma2(A, g[s], C);
            }
            A = at_least(A);
        }
        if (special || not_a_number(C)) {  // or where a gradient that is infinite has met a product of 0
            A = two(1.0f);
            H = C = two(0.0f);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                H = after(a[s], H, mul2(n[s], u[s]));
                A = kept(more(A, a[s]));
                C = behind(A, g[s], C);
            }
        }
        ex.warp[par][0][warp][lane] = map_of(A, H);
        ex.warp[par][1][warp][lane] = map_of(A, C);
        const bool any = __syncthreads_or(special);
        float2 c = carry;
        if (!any) {
#pragma unroll
            for (int w = kScanWarps - 1; w >= 0; --w) {
                if (w == warp) c = carry;
                carry = straight(ex.warp[par][1][w][lane], carry);
            }
            for (int w = 0; w < warp; ++w) h = straight(ex.warp[par][0][w][lane], h);
        } else {
#pragma unroll
            for (int w = kScanWarps - 1; w >= 0; --w) {
                if (w == warp) c = carry;
                carry = through(ex.warp[par][1][w][lane], carry);
            }
            for (int w = 0; w < warp; ++w) h = through(ex.warp[par][0][w][lane], h);
        }
        // u becomes a n (h before the step - u), then both gradients in place of g and u
        if (kind == kNear) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const float2 d = fma2(u[s], two(-1.0f), h);
                h = fma2(a[s], h, mul2(n[s], u[s]));
                u[s] = mul2(mul2(a[s], n[s]), d);
            }
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                const float2 dh = add2(g[s], c);
                u[s] = mul2(u[s], dh);
                g[s] = mul2(n[s], dh);
                c = mul2(a[s], dh);
            }
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const float2 d = fma2(u[s], two(-1.0f), h), w = mul2(a[s], n[s]);
                h = after(a[s], h, mul2(n[s], u[s]));
                u[s] = looked_at(w, mul2(w, d));
            }
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                const float2 dh = add2(g[s], c);
                u[s] = mul2(u[s], dh);
                g[s] = mul2(n[s], dh);
                c = looked_at(a[s], mul2(a[s], dh));
            }
        }
        T *dz = (T *)p.dgate + at, *du = (T *)p.dvalue + at;
        if (vec && nch == 2 && cnt == S) {
#pragma unroll
            for (int s = 0; s < S; ++s, dz += p.width, du += p.width) {
                store2v(dz, u[s]);
                store2v(du, g[s]);
            }
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (s < cnt) {
                    store2(dz + (long long)s * p.width, vec, nch, u[s]);
                    store2(du + (long long)s * p.width, vec, nch, g[s]);
                }
        }
    }
    if (!CHUNK && p.dstate && warp == 0) store2(p.dstate + (long long)now.seq * p.width + ch, vec, nch, carry);
}

// ------------------------------------------------------------------ one step
// Four channels of a thread; quads: vectors of four lie on whole vectors' addresses
template <typename T>
__global__ void __launch_bounds__(256) scan_step_k(const T *__restrict__ gate, const T *__restrict__ value, const float *state, T *__restrict__ h,
                                                   float *out_state, long long rows, int width, long long gate_row, long long value_row, int quads)
{
    const int of_row = (width + 3) / 4;
    const long long stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < rows * of_row; i += stride) {
        const long long row = rows * of_row <= 0xffffffffLL ? (long long)((unsigned)i / (unsigned)of_row) : i / of_row;
        const int ch = (int)(i - row * of_row) * 4, nch = min(4, width - ch);
        float z[4], u[4], s[4];
        load4(gate + row * gate_row + ch, quads, nch, z);
        load4(value + row * value_row + ch, quads, nch, u);
        load4(state + row * width + ch, quads, nch, s);
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            float2 a, n;
            gates_any(make_float2(z[k], z[k + 1]), a, n);
            const float2 r = after(a, make_float2(s[k], s[k + 1]), mul2(n, looked_at(n, make_float2(u[k], u[k + 1]))));
            s[k] = r.x;
            s[k + 1] = r.y;
        }
        store4(h + row * width + ch, quads, nch, s);
        store4(out_state + row * width + ch, quads, nch, s);
    }
}

// ------------------------------------------------------------------ host side
static bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
static long long slabs_of(int width) { return (width + kSlab - 1) / kSlab; }

struct ScanDims {
    int n;
    long long steps, total;
    int width, dtype;
    bool ragged;
    int size() const { return dtype == GN_F32 ? 4 : 2; }
    long long tiles(int log2) const { return (steps + (1LL << log2) - 1) >> log2; }
    long long tile_rows(int log2) const { return ragged ? (total >> log2) + n + 1 : n * tiles(log2); }
};

static int scan_check(const ScanDims &d)
{
    if (d.n < 0 || d.steps < 0 || d.total < 0 || d.width <= 0) return GN_ERR_BAD_SHAPE;
    if (d.steps > 0 && d.n > (1LL << 48) / d.steps) return GN_ERR_TOO_LARGE;
    if (!d.ragged && d.total != d.n * d.steps) return GN_ERR_BAD_SHAPE;
    if (d.dtype < GN_F32 || d.dtype > GN_F16) return GN_ERR_UNSUPPORTED;
    if (d.total > (1LL << 48) / d.width) return GN_ERR_TOO_LARGE;
    if ((d.n + 1LL) * slabs_of(d.width) > 0x7fffffffLL / 4 || d.tile_rows(kBwdLog2) > 0x7fffffffLL / slabs_of(d.width)) return GN_ERR_TOO_LARGE;
    return GN_OK;
}

// Whether the forward pass (backward: the backward pass) walks or goes by chunks. A walk's tile takes 1.2 to 1.8 us however few CTAs there
// are, chunks cost two more kernels (8 to 10 us) and a second reading. us, walk / chunks, forward and backward: 64 CTAs, 8 x 1024 x 512 float32
// 24 / 18 and 58 / 31, 4 x 4097 x 1024 95 / 58 and 236 / 106; 256 CTAs, 16 x 1024 x 1000 float32 45 / 59 and 93 / 109, 16 x 512 x 1024
// bfloat16 14 / 25 and 26 / 40; 16 CTAs, 1 x 300 x 1024 float32 10 / 13 and 15 / 13. So: a CTA per SM, or few tiles one after the other.
// How long the longest of ragged sequences is is not known here: eight rounds of CTAs, so that one of eight times the mean takes no longer
// than all (37 of mean 300, the longest 2380, x 1000 bfloat16: a walk takes 118 and 183 us, chunks 41 and 61).
static bool scan_walks(const ScanDims &d, bool backward, bool packed)
{
    const int log2 = backward ? kBwdLog2 : kFwdLog2;
    const long long longest = d.ragged ? d.total : d.steps;
    if (d.n == 0 || longest <= 1LL << log2) return true;  // nothing, or a single tile
    if (backward && packed) return false;
    return longest <= 8LL << log2 || d.n * slabs_of(d.width) >= (d.ragged ? 32LL : 1LL) * sm_count();
}

static size_t bounds_bytes(const ScanDims &d)
{
    if (d.n == 0 || d.total == 0 || (d.ragged ? d.total : d.steps) <= kBwdTile || !scan_walks(d, true, false)) return 0;
    return sizeof(float) * (size_t)d.tile_rows(kBwdLog2) * d.width;
}
static size_t maps_bytes(const ScanDims &d, bool backward, bool packed)
{
    if ((d.n == 0 && !d.ragged) || d.total == 0 || scan_walks(d, backward, packed)) return 0;
    return sizeof(float) * (backward ? 3 : 2) * (size_t)d.tile_rows(backward ? kBwdLog2 : kFwdLog2) * slabs_of(d.width) * kSlab;
}

// the three kernels of the way by chunks
template <typename T, bool PACKED, bool BACKWARD, void (*WORK)(const Scan)>
static int launch_chunks(Scan &p, const ScanDims &d, size_t work_smem, const char *what, cudaStream_t st)
{
    constexpr int kLog2 = BACKWARD ? kBwdLog2 : kFwdLog2;
    p.map_rows = d.tile_rows(kLog2);
    const size_t smem = p.wide ? kScanWarps * Source<T, PACKED, BACKWARD, kSumSteps>::kBytes : 0;
    const long long warps = p.map_rows * p.slabs;
    // More than one tile to a CTA, the next asked for while one is worked on: 2 x 20000 x 2048 bfloat16 forward 191 -> 174 us, backward 356 ->
    // 298. Forward where six rounds of CTAs are left (four fit an SM), with fewer the last one costs as much (4 x 4097 x 1024 float32 58.1 -> 58.4
    // us, and 71.2 -> 73.9 with packing); backward, whose tiles are half as long, where two are (one to four tiles: 6 x 3000 x 640 bfloat16 55.4 ->
    // 51.4 us, 37 ragged sequences of mean 300 x 1000 69 -> 64; 8 x 1024 x 512 float32, one round, stays at one tile: 31)
    p.tiles_per_cta = 1;
    while (p.tiles_per_cta < 8 && warps / (2 * p.tiles_per_cta) >= (BACKWARD ? 8LL : 24LL) * sm_count()) p.tiles_per_cta *= 2;
    const long long ctas = (p.map_rows + p.tiles_per_cta - 1) / p.tiles_per_cta * p.slabs;
    scan_maps_k<T, PACKED, BACKWARD><<<(unsigned)((warps + kScanWarps - 1) / kScanWarps), kScanThreads, smem, st>>>(p);
    // eight tiles to a run (they are read together), 64 runs at most and four at least, a warp; ragged: for twice the mean sequence
    const long long tiles = d.ragged ? 2 * (d.total >> kLog2) / (p.n > 0 ? p.n : 1) : d.tiles(kLog2);
    int runs = 4;
    while (runs < kStartRuns && 8 * runs < tiles) runs *= 2;
    launch_after(scan_starts_k<T, BACKWARD>, dim3((unsigned)((p.n + (d.ragged ? 1LL : 0LL)) * p.slabs * (kSlab / 16))), dim3(8 * runs), 0, st, p);
    launch_after(WORK, dim3((unsigned)ctas), dim3(kScanThreads), work_smem, st, p);
    return check_launch(what);
}

template <void (*KERN)(const Scan)>
static int launch_walk(const Scan &p, const ScanDims &d, size_t smem, const char *what, cudaStream_t st)
{
    KERN<<<(unsigned)((p.n + (d.ragged ? 1LL : 0LL)) * p.slabs), kScanThreads, smem, st>>>(p);
    return check_launch(what);
}

template <typename T, bool KEEP>
static int launch_forward(Scan &p, const ScanDims &d, cudaStream_t st)
{
    const size_t smem = p.wide ? kScanWarps * Source<T, false, false, kFwdSteps>::kBytes : 0;
    if (scan_walks(d, false, false)) return launch_walk<scan_forward_k<T, KEEP, false>>(p, d, smem, "gated_scan", st);
    return launch_chunks<T, false, false, scan_forward_k<T, KEEP, true>>(p, d, smem, "gated_scan", st);
}
template <typename T>
static int launch_forward(Scan &p, const ScanDims &d, cudaStream_t st)
{
    return p.pack_gate ? launch_forward<T, true>(p, d, st) : launch_forward<T, false>(p, d, st);
}

template <typename T, bool PACKED>
static int launch_backward(Scan &p, const ScanDims &d, cudaStream_t st)
{
    const size_t smem = p.wide ? kScanWarps * Source<T, PACKED, true, kBwdSteps>::kBytes : 0;
    if (scan_walks(d, true, PACKED)) return launch_walk<scan_backward_k<T, PACKED, false>>(p, d, smem, "gated_scan backward", st);
    return launch_chunks<T, PACKED, true, scan_backward_k<T, PACKED, true>>(p, d, smem, "gated_scan backward", st);
}
template <typename T>
static int launch_backward(Scan &p, const ScanDims &d, bool packed, cudaStream_t st)
{
    return packed ? launch_backward<T, true>(p, d, st) : launch_backward<T, false>(p, d, st);
}

}  // namespace gn

using namespace gn;

extern "C" {

GN_API size_t gn_gated_scan_bounds_bytes(int n, long long steps, long long total, int width, int dtype, int ragged)
{
    const ScanDims d{n, ragged ? 0 : steps, total, width, dtype, ragged != 0};
    return scan_check(d) == GN_OK ? bounds_bytes(d) : 0;
}

GN_API size_t gn_gated_scan_workspace_bytes(int n, long long steps, long long total, int width, int dtype, int ragged, int backward, int packed)
{
    const ScanDims d{n, ragged ? 0 : steps, total, width, dtype, ragged != 0};
    return scan_check(d) == GN_OK ? maps_bytes(d, backward != 0, packed != 0) : 0;
}

GN_API int gn_gated_scan_forward(const void *gate, const void *value, const float *state, const long long *offsets, void *h, float *last,
                                 void *gate_codes, void *gate_scales, void *value_codes, void *value_scales, float *bounds, int n,
                                 long long steps, long long total, int width, long long gate_seq, long long gate_step, long long value_seq,
                                 long long value_step, int dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    const ScanDims d{n, offsets ? 0 : steps, total, width, dtype, offsets != nullptr};
    const int rc = scan_check(d);
    if (rc != GN_OK) return rc;
    if (gate_codes && (!gate_scales || !value_codes || !value_scales)) return GN_ERR_NULL_POINTER;
    if (total > 0 && (!gate || !value || !h)) return GN_ERR_NULL_POINTER;
    if (n == 0 && !(offsets && total > 0)) return GN_OK;
    const size_t need = maps_bytes(d, false, false);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return GN_ERR_WORKSPACE;
    Scan p{};
    p.gate = gate; p.value = value; p.state = state; p.offsets = offsets; p.h = h; p.last = last;
    p.pack_gate = (unsigned char *)gate_codes; p.pack_gate_scales = (unsigned char *)gate_scales;
    p.pack_value = (unsigned char *)value_codes; p.pack_value_scales = (unsigned char *)value_scales;
    p.bounds = gate_codes || bounds_bytes(d) == 0 ? nullptr : bounds;
    p.maps = static_cast<float *>(workspace);
    p.gate_seq = gate_seq; p.gate_step = gate_step; p.value_seq = value_seq; p.value_step = value_step;
    p.n = n; p.steps = d.steps; p.total = total; p.width = width;
    p.slabs = (int)slabs_of(width);
    p.padded = p.slabs * kSlab;
    const int size = d.size();
    p.vec = width % 2 == 0 && gate_seq % 2 == 0 && gate_step % 2 == 0 && value_seq % 2 == 0 && value_step % 2 == 0 && aligned(gate, 2 * size) &&
            aligned(value, 2 * size) && aligned(h, 2 * size) && aligned(state, 8) && aligned(last, 8) && aligned(bounds, 8) &&
            aligned(gate_codes, 2) && aligned(value_codes, 2);
    p.wide = (long long)width * size % 16 == 0 && gate_seq * size % 16 == 0 && gate_step * size % 16 == 0 && value_seq * size % 16 == 0 &&
             value_step * size % 16 == 0 && aligned(gate, 16) && aligned(value, 16);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == GN_F32) return launch_forward<float>(p, d, st);
    if (dtype == GN_BF16) return launch_forward<__nv_bfloat16>(p, d, st);
    return launch_forward<__half>(p, d, st);
}

GN_API int gn_gated_scan_backward(const void *gate, const void *value, const void *gate_scales, const void *value_scales, const float *state,
                                  const long long *offsets, const float *bounds, const void *grad_h, const float *grad_last, void *grad_gate,
                                  void *grad_value, float *grad_state, int n, long long steps, long long total, int width, long long gate_seq,
                                  long long gate_step, long long value_seq, long long value_step, int dtype, void *workspace,
                                  size_t workspace_bytes, void *stream)
{
    const ScanDims d{n, offsets ? 0 : steps, total, width, dtype, offsets != nullptr};
    const int rc = scan_check(d);
    if (rc != GN_OK) return rc;
    if (!gate_scales != !value_scales) return GN_ERR_NULL_POINTER;
    const bool packed = gate_scales != nullptr;
    if (total > 0 && (!gate || !value || !grad_h || !grad_gate || !grad_value)) return GN_ERR_NULL_POINTER;
    if (n == 0 && !(offsets && total > 0)) return GN_OK;
    if (!packed && bounds_bytes(d) > 0 && !bounds) return GN_ERR_WORKSPACE;
    const size_t need = maps_bytes(d, true, packed);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return GN_ERR_WORKSPACE;
    Scan p{};
    p.gate = gate; p.value = value; p.state = state; p.offsets = offsets; p.bounds = const_cast<float *>(bounds);
    p.maps = static_cast<float *>(workspace);
    p.gate_scales = (const unsigned char *)gate_scales; p.value_scales = (const unsigned char *)value_scales;
    p.gh = grad_h; p.glast = grad_last; p.dgate = grad_gate; p.dvalue = grad_value; p.dstate = grad_state;
    if (!packed) {
        p.gate_seq = gate_seq; p.gate_step = gate_step; p.value_seq = value_seq; p.value_step = value_step;
    }
    p.n = n; p.steps = d.steps; p.total = total; p.width = width;
    p.slabs = (int)slabs_of(width);
    p.padded = p.slabs * kSlab;
    const int size = d.size(), in = packed ? 1 : size;
    p.vec = width % 2 == 0 && p.gate_seq % 2 == 0 && p.gate_step % 2 == 0 && p.value_seq % 2 == 0 && p.value_step % 2 == 0 && aligned(gate, 2 * in) &&
            aligned(value, 2 * in) && aligned(grad_h, 2 * size) && aligned(grad_gate, 2 * size) && aligned(grad_value, 2 * size) &&
            aligned(state, 8) && aligned(grad_last, 8) && aligned(grad_state, 8) && aligned(bounds, 8);
    p.wide = (long long)width * in % 16 == 0 && (long long)width * size % 16 == 0 && p.gate_seq * in % 16 == 0 && p.gate_step * in % 16 == 0 &&
             p.value_seq * in % 16 == 0 && p.value_step * in % 16 == 0 && aligned(gate, 16) && aligned(value, 16) && aligned(grad_h, 16);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == GN_F32) return launch_backward<float>(p, d, packed, st);
    if (dtype == GN_BF16) return launch_backward<__nv_bfloat16>(p, d, packed, st);
    return launch_backward<__half>(p, d, packed, st);
}

GN_API int gn_gated_scan_step(const void *gate, const void *value, const float *state, void *h, float *out_state, long long rows, int width,
                              long long gate_row, long long value_row, int dtype, void *stream)
{
    if (rows < 0 || width <= 0 || rows > (1LL << 48) / width) return GN_ERR_BAD_SHAPE;
    if (dtype < GN_F32 || dtype > GN_F16) return GN_ERR_UNSUPPORTED;
    if (rows == 0) return GN_OK;
    if (!gate || !value || !state || !h || !out_state) return GN_ERR_NULL_POINTER;
    const int size = dtype == GN_F32 ? 4 : 2;
    const int quads = width % 4 == 0 && gate_row % 4 == 0 && value_row % 4 == 0 && aligned(gate, 4 * size) && aligned(value, 4 * size) &&
                      aligned(h, 4 * size) && aligned(state, 16) && aligned(out_state, 16);
    const long long want = (rows * ((width + 3) / 4) + 255) / 256, most = 32LL * sm_count();
    const unsigned blocks = (unsigned)(want < most ? want : most);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == GN_F32)
        scan_step_k<float><<<blocks, 256, 0, st>>>((const float *)gate, (const float *)value, state, (float *)h, out_state, rows, width, gate_row,
                                                   value_row, quads);
    else if (dtype == GN_BF16)
        scan_step_k<__nv_bfloat16><<<blocks, 256, 0, st>>>((const __nv_bfloat16 *)gate, (const __nv_bfloat16 *)value, state, (__nv_bfloat16 *)h,
                                                           out_state, rows, width, gate_row, value_row, quads);
    else
        scan_step_k<__half><<<blocks, 256, 0, st>>>((const __half *)gate, (const __half *)value, state, (__half *)h, out_state, rows, width,
                                                    gate_row, value_row, quads);
    return check_launch("gated_scan_step");
}

}  // extern "C"
