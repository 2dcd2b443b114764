// rope.hip -- rotary positions by a plan (gfx950): either pair layout, part of the head, scaled
// frequencies, f32 / f16 / bf16 rows at their own strides.
//
// Pair (x0, x1) of channel pair i turns by a = pos f_i: y0 = m (x0 cos a - x1 sin a), y1 = m (x0 sin a +
// x1 cos a).  In f32 the angle of position 10^6 is off by 0.06 rad; here pos f_i / 2 pi is formed and
// reduced to a half turn in f64 and only the remainder goes to f32 (sincospi, error below 2 ulp).
// The rotation is f32, rounded once to the rows' type.
//
// Bound by memory: a row is read and written once (4096 tokens of 32 + 8 heads, D 128, bf16: 14 us, 84 MB at 5.9 TB/s;
// 1000 tokens of 16 + 2 heads, D 256, f32, a quarter of it rotated: 8.7 us, 37 MB at 4.2; one token: 2.6 us, a launch).  A workgroup takes one token (its angles are computed
// once, into LDS) and its threads 8 pairs each: two 16-byte chunks half a rotation apart (halves), or one
// chunk (pairs); the rest of the head is copied when the output is another tensor.
#include "pi_device.hpp"
#include "q4_launch.hpp"

#include <algorithm>

namespace pi {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;

// cos and sin of pair i at a position, times m.
__device__ __forceinline__ float2 angle_f32(double pos, double turns, float m) {
    double t = pos * turns;
    t -= rint(t);
    float s, c;
    sincospif((float)(2.0 * t), &s, &c);
    return float2{m * c, m * s};
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
    typedef T t8 __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8 / W; ++j) {
        const t8 r = *reinterpret_cast<const t8*>(p + W * j);
#pragma unroll
        for (int i = 0; i < W; ++i) x[W * j + i] = to_f32(r[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
    typedef T t8 __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8 / W; ++j) {
        t8 r;
#pragma unroll
        for (int i = 0; i < W; ++i) r[i] = from_f32<T>(x[W * j + i]);
        *reinterpret_cast<t8*>(p + W * j) = r;
    }
}

// Rows whose chunks of 8 channels are 16-byte aligned and wholly in one half, or wholly past the rotation.
template <typename T, int LAYOUT>
__global__ __launch_bounds__(kThreads) void rope_vec_kernel(RopeArgs a, int copy_q, int copy_k) {
    __shared__ float2 s_cs[kMaxHalf];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int half = a.plan.half;
    const int rot = LAYOUT == 1 ? half / 8 : half / 4;        // rotating units of a head
    const int rest = (a.head_dim - 2 * half) / 8;             // chunks past the rotation
    const int per_q = rot + (copy_q ? rest : 0), per_k = rot + (copy_k ? rest : 0);
    const int nq = a.in[0].n * per_q, units = nq + a.in[1].n * per_k;
    const double pos = a.pos[t];
    if (tid < half) s_cs[tid] = angle_f32(pos, a.plan.turns[tid], (float)a.plan.mscale);
    __syncthreads();
    for (int u = blockIdx.y * kThreads + tid; u < units; u += gridDim.y * kThreads) {
        const int w = u >= nq;
        const int per = w ? per_k : per_q, v = w ? u - nq : u;
        const int h = v / per, c = v - h * per;
        const T* in = static_cast<const T*>(a.in[w].p) + t * a.in[w].tok + h * a.in[w].head;
        T* out = static_cast<T*>(a.out[w].p) + t * a.out[w].tok + h * a.out[w].head;
        float x[8], y[8];
        if (c >= rot) {
            const int d = 2 * half + 8 * (c - rot);
            load8(in + d, x);
            store8(out + d, x);
        } else if (LAYOUT == 1) {
            float x1[8], y1[8];
            load8(in + 8 * c, x);
            load8(in + half + 8 * c, x1);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 cs = s_cs[8 * c + i];
                y[i] = x[i] * cs.x - x1[i] * cs.y;
                y1[i] = x[i] * cs.y + x1[i] * cs.x;
            }
            store8(out + 8 * c, y);
            store8(out + half + 8 * c, y1);
        } else {
            load8(in + 8 * c, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 cs = s_cs[4 * c + i];
                y[2 * i] = x[2 * i] * cs.x - x[2 * i + 1] * cs.y;
                y[2 * i + 1] = x[2 * i] * cs.y + x[2 * i + 1] * cs.x;
            }
            store8(out + 8 * c, y);
        }
    }
}

// n (1 .. 8) elements at any alignment of T: eight by one wide access, which the memory takes at any address.
template <typename T>
__device__ __forceinline__ void load_n(const T* p, int n, float* x) {
    typedef T t8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (n == 8) {
        const t8 r = *reinterpret_cast<const t8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(r[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? to_f32(p[i]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_n(T* p, int n, const float* x) {
    typedef T t8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (n == 8) {
        t8 r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = from_f32<T>(x[i]);
        *reinterpret_cast<t8*>(p) = r;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = from_f32<T>(x[i]);
}

// Any widths, strides and alignment: the chunks above where they lie, the last of a part with fewer channels.  (4096 tokens of
// 32 + 8 heads, D 128, 34 channels rotated, f16: pairs 17 us, halves 35; a pair or a channel a thread took 56 and 53.)
template <typename T, int LAYOUT>
__global__ __launch_bounds__(kThreads) void rope_any_kernel(RopeArgs a, int copy_q, int copy_k) {
    __shared__ float2 s_cs[kMaxHalf];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int half = a.plan.half, D = a.head_dim;
    const int rot = LAYOUT == 1 ? (half + 7) / 8 : (half + 3) / 4;  // rotating units of a head
    const int past = LAYOUT == 1 ? 2 * half : min(8 * rot, D);      // first channel of the units past them
    const int rest = (D - past + 7) / 8;
    const int per_q = rot + (copy_q ? rest : 0), per_k = rot + (copy_k ? rest : 0);
    const int nq = a.in[0].n * per_q, units = nq + a.in[1].n * per_k;
    const double pos = a.pos[t];
    if (tid < half) s_cs[tid] = angle_f32(pos, a.plan.turns[tid], (float)a.plan.mscale);
    __syncthreads();
    for (int u = blockIdx.y * kThreads + tid; u < units; u += gridDim.y * kThreads) {
        const int w = u >= nq;
        const int per = w ? per_k : per_q, v = w ? u - nq : u;
        const int h = v / per, c = v - h * per;
        const T* in = static_cast<const T*>(a.in[w].p) + t * a.in[w].tok + h * a.in[w].head;
        T* out = static_cast<T*>(a.out[w].p) + t * a.out[w].tok + h * a.out[w].head;
        float x[8], y[8];
        if (c >= rot) {
            const int d = past + 8 * (c - rot), n = min(8, D - d);
            load_n(in + d, n, x);
            store_n(out + d, n, x);
        } else if (LAYOUT == 1) {
            const int n = min(8, half - 8 * c);
            float x1[8], y1[8];
            load_n(in + 8 * c, n, x);
            load_n(in + half + 8 * c, n, x1);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 cs = s_cs[min(8 * c + i, half - 1)];
                y[i] = x[i] * cs.x - x1[i] * cs.y;
                y1[i] = x[i] * cs.y + x1[i] * cs.x;
            }
            store_n(out + 8 * c, n, y);
            store_n(out + half + 8 * c, n, y1);
        } else {
            const int n = min(8, D - 8 * c);
            load_n(in + 8 * c, n, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool on = 4 * c + i < half;  // else channels past the rotation
                const float2 cs = s_cs[min(4 * c + i, half - 1)];
                y[2 * i] = on ? x[2 * i] * cs.x - x[2 * i + 1] * cs.y : x[2 * i];
                y[2 * i + 1] = on ? x[2 * i] * cs.y + x[2 * i + 1] * cs.x : x[2 * i + 1];
            }
            store_n(out + 8 * c, n, y);
        }
    }
}

template <typename T>
hipError_t launch_t(const RopeArgs& a, hipStream_t s) {
    const int half = a.plan.half, e = (int)sizeof(T);
    bool vec = a.head_dim % 8 == 0 && half % 8 == 0;
    for (int w = 0; w < 2; ++w) {
        if (!a.in[w].n) continue;
        for (const HeadRows* r : {&a.in[w], &a.out[w]})
            vec = vec && reinterpret_cast<uintptr_t>(r->p) % 16 == 0 && r->tok * e % 16 == 0 && r->head * e % 16 == 0;
    }
    const int copy_q = a.out[0].p != a.in[0].p, copy_k = a.out[1].p != a.in[1].p;
    const int per = a.plan.layout == 1 ? (half + 7) / 8 + (a.head_dim - 2 * half + 7) / 8 : (a.head_dim + 7) / 8;
    const int blocks = std::max(1, (per * (a.in[0].n + a.in[1].n) + kThreads - 1) / kThreads);
    // One pass of a token's rows a workgroup while that does not fill the chip, else a workgroup a token.
    const int y = (long long)a.n_tok * blocks <= 2048 ? std::min(blocks, 65535) : 1;
    const dim3 grid(a.n_tok, y);
    if (vec && a.plan.layout == 1)
        hipLaunchKernelGGL((rope_vec_kernel<T, 1>), grid, dim3(kThreads), 0, s, a, copy_q, copy_k);
    else if (vec)
        hipLaunchKernelGGL((rope_vec_kernel<T, 0>), grid, dim3(kThreads), 0, s, a, copy_q, copy_k);
    else if (a.plan.layout == 1)
        hipLaunchKernelGGL((rope_any_kernel<T, 1>), grid, dim3(kThreads), 0, s, a, copy_q, copy_k);
    else
        hipLaunchKernelGGL((rope_any_kernel<T, 0>), grid, dim3(kThreads), 0, s, a, copy_q, copy_k);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope_apply(const RopeArgs& a, hipStream_t s) {
    return a.dtype == 0 ? launch_t<float>(a, s) : a.dtype == 1 ? launch_t<f16>(a, s) : launch_t<bf16>(a, s);
}

}  // namespace pi
