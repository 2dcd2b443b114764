// q4.hip -- appending to the 4-bit paged KV cache with norm and rotation on the way, and moving its
// records in and out (gfx950).  The format is q4.hpp's.
//
// Per new token: q and k heads normed (optional), rotated by a plan (optional), q written in its own
// type, k and v quantised into the token's slot of its page and, when asked, the values that the
// cache now stands for written back in f16.
//
// K is normed and rotated in f64.  Which code a value gets depends on the side of a border it falls on,
// and the borders are where f32 results of different instruction orders disagree (a few codes of a
// million values); in f64 the codes are those of the formulas.  It costs nothing that shows: K is a fifth
// of the rows or less, and the launch is bound by memory.  V is not rotated and its quotients are
// exact comparisons already in f32 for 16-bit rows (f64 for f32 rows).
//
// A row's 8 channels are one lane's: a K word is one lane's 8 codes, a group of 32 channels 4 lanes.
#include "pi_device.hpp"
#include "q4_launch.hpp"

#include <algorithm>
#include <type_traits>

namespace pi {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 256;  // (token, pair) angles of a workgroup

__device__ __forceinline__ double shfl_xor(double v, int m) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl_xor((uint32_t)b, m, 64), hi = __shfl_xor((uint32_t)(b >> 32), m, 64);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ float shfl_xor(float v, int m) { return __shfl_xor(v, m, 64); }

template <typename R> struct Real;
template <> struct Real<float> {
    static __device__ __forceinline__ float inv_sqrt(float x) { return 1.0f / sqrtf(x); }
    static __device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
    static __device__ __forceinline__ float rint_(float x) { return rintf(x); }
    static __device__ __forceinline__ float max_(float a, float b) { return fmaxf(a, b); }
    static __device__ __forceinline__ float min_(float a, float b) { return fminf(a, b); }
};
template <> struct Real<double> {
    static __device__ __forceinline__ double inv_sqrt(double x) { return 1.0 / sqrt(x); }
    static __device__ __forceinline__ double fma_(double a, double b, double c) { return fma(a, b, c); }
    static __device__ __forceinline__ double rint_(double x) { return rint(x); }
    static __device__ __forceinline__ double max_(double a, double b) { return fmax(a, b); }
    static __device__ __forceinline__ double min_(double a, double b) { return fmin(a, b); }
};

// The group scale: -m / 8 to 7 significant bits, nearest even (multiples of 2^-20 below 2^-14), at most 904.
__device__ __forceinline__ float group_scale(double m) {
    const double x = m * -0.125, a = fabs(x);
    double r;
    if (a >= 904.0)
        r = 904.0;
    else if (a < 0x1p-14)
        r = (a + 0x1p32) - 0x1p32;  // an ulp of 2^32 .. 2^33 is 2^-20
    else {
        uint64_t b = __builtin_bit_cast(uint64_t, a);
        b += ((1ull << 45) - 1) + ((b >> 46) & 1);  // 6 stored mantissa bits of 52
        r = __builtin_bit_cast(double, b & ~((1ull << 46) - 1));
    }
    return (float)(x < 0 ? -r : r);
}

// Quantises 8 consecutive channels of a row: every lane of the group's 4 holds 8.  Packed codes (nibble e:
// channel e) and the group's scale.  NaN counts as 0; values past 8192 (and infinities) as 8192,
// over the largest that the format holds.
template <typename R>
__device__ __forceinline__ uint32_t quantise8(const R* xin, float* scale) {
    typedef Real<R> F;
    R x[8], hi = 0, lo = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = xin[e] > (R)8192 ? (R)8192 : xin[e] < (R)-8192 ? (R)-8192 : xin[e];
        hi = F::max_(hi, x[e]);
        lo = F::min_(lo, x[e]);
    }
#pragma unroll
    for (int m = 1; m <= 2; m <<= 1) {
        hi = F::max_(hi, shfl_xor(hi, m));
        lo = F::min_(lo, shfl_xor(lo, m));
    }
    const float s = group_scale(hi >= -lo ? (double)hi : (double)lo);
    *scale = s;
    const R sr = (R)s, inv = s == 0.f ? (R)0 : (R)1 / sr;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // x / s to the last bit that matters: a quotient that is a tie (k + 1/2) is exact after the correction
        R t = x[e] * inv;
        t = F::fma_(F::fma_(-t, sr, x[e]), inv, t);
        t = F::rint_(t);
        const int c = t == t ? (int)F::min_(F::max_(t, (R)-8), (R)7) : 0;
        w |= (uint32_t)(c + 8) << (4 * e);
    }
    return w;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T* p, T* x) {
    if (VEC) {
        constexpr int W = 16 / sizeof(T);
        typedef T tv __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int j = 0; j < 8 / W; ++j) {
            const tv r = *reinterpret_cast<const tv*>(p + W * j);
#pragma unroll
            for (int i = 0; i < W; ++i) x[W * j + i] = r[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}

// Where a token goes.
struct Place {
    long long pos;  // < 0: the row belongs to no sequence
    int page;       // < 0: no page holds the position
    int slot;
};

// Norm and rotation of channels d0 .. d0 + 7 of a row (LPR lanes hold the row).
template <typename T, typename R, bool VEC>
__device__ __forceinline__ void norm_rotate(const T* row, int d0, int D, int lpr, const float* w, float eps, int half, int layout,
                                            const double2* cs, R* y) {
    typedef Real<R> F;
    T xt[8], pt[8];
    load_row8<T, VEC>(row + d0, xt);
    const bool turn = layout == 1 && d0 < 2 * half;
    // halves: the partners sit half a rotation away
    if (turn) {
        if (VEC)
            load_row8<T, true>(row + (d0 < half ? d0 + half : d0 - half), pt);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = d0 + e;
                pt[e] = row[d < half ? d + half : d < 2 * half ? d - half : d];
            }
    }
    R x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (R)to_f32(xt[e]);
    R rs = 1;
    if (w) {
        R ss = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
        for (int m = 1; m < lpr; m <<= 1) ss += shfl_xor(ss, m);
        rs = F::inv_sqrt(ss / (R)D + (R)eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * rs * (R)w[d0 + e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e];
    if (layout == 0) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            if (d0 + e >= 2 * half) break;
            const double2 a = cs[(d0 + e) >> 1];
            y[e] = x[e] * (R)a.x - x[e + 1] * (R)a.y;
            y[e + 1] = x[e] * (R)a.y + x[e + 1] * (R)a.x;
        }
    } else if (turn) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = d0 + e;
            if (d >= 2 * half) break;
            const bool first = d < half;
            const int pd = first ? d + half : d - half;
            R p = (R)to_f32(pt[e]);
            if (w) p = p * rs * (R)w[pd];
            const double2 a = cs[first ? d : pd];
            y[e] = first ? x[e] * (R)a.x - p * (R)a.y : p * (R)a.y + x[e] * (R)a.x;
        }
    }
}

// The sequence and page of each of a workgroup's tokens, found by one wavefront: a sample of 64 of the
// sequences' starts, then the 64 between two samples.  The tables are read, not trusted: a row is placed only
// where its sequence's range holds it, as the attentions read it.
__device__ __forceinline__ void find_places(const Q4AppendArgs& a, int row0, int n, Place* out) {
    const int lane = threadIdx.x;
    const int per = (a.n_seq + 63) / 64;
    const int top = a.tok_start ? a.tok_start[min((lane + 1) * per, a.n_seq)] : 0;
    for (int i = 0; i < n; ++i) {
        const int row = row0 + i;
        int s = row, first = row;
        bool in = row < a.n_rows;
        if (a.tok_start) {
            const int blk = min((int)__popcll(__ballot((lane + 1) * per <= a.n_seq && top <= row)) * per, a.n_seq);
            const int j = blk + 1 + lane;
            s = blk;
            if (per > 1) s += __popcll(__ballot(lane < per && j <= a.n_seq && a.tok_start[min(j, a.n_seq)] <= row));
            in = in && s < a.n_seq;
            s = min(s, a.n_seq - 1);
            first = max(a.tok_start[s], 0);
            in = in && row >= first && row < a.tok_start[s + 1];
        }
        const long long pos = (long long)max(a.start_pos[s], 0) + (row - first);
        const long long lp = pos / sched::kPage;
        int page = -1;
        if (in && lp < a.max_pages) page = a.page_table[(size_t)s * a.max_pages + lp];
        if (lane == 0) {
            out[i].pos = in ? pos : -1;
            out[i].page = page < a.g.n_pages ? page : -1;
            out[i].slot = (int)(pos % sched::kPage);
        }
    }
}

// A workgroup: `toks` tokens (their angles fit the table), blockIdx.y: a share of their head rows.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void q4_append_kernel(Q4AppendArgs a, int toks) {
    __shared__ double2 s_cs[kTable];
    __shared__ Place s_place[4];
    const int tid = threadIdx.x, D = a.g.head_dim, half = a.plan.half;
    const int row0 = blockIdx.x * toks, n = min(toks, a.n_rows - row0);
    if (tid < 64) find_places(a, row0, n, s_place);
    __syncthreads();
    for (int i = tid; i < n * half; i += kThreads) {
        const int t = i / half;
        double turns = (double)s_place[t].pos * a.plan.turns[i - t * half];
        turns -= rint(turns);
        double sn, cn;
        sincospi(2.0 * turns, &sn, &cn);
        s_cs[i] = double2{cn * a.plan.mscale, sn * a.plan.mscale};
    }
    __syncthreads();
    const int lpr = D / 8, rpi = kThreads / lpr;       // lanes a row, rows at a time
    const int rl = tid / lpr, c = tid - rl * lpr, d0 = 8 * c;
    const int hkv = a.g.n_kv_heads, heads = a.q.n + 2 * hkv;
    for (int u = blockIdx.y * rpi + rl; u < n * heads; u += gridDim.y * rpi) {
        const int t = u / heads, h = u - t * heads, row = row0 + t;
        const Place pl = s_place[t];
        if (pl.pos < 0) continue;  // uniform over a row's lanes
        const double2* cs = s_cs + t * half;
        if (h < a.q.n) {
            const T* in = static_cast<const T*>(a.q.p) + row * a.q.tok + h * a.q.head;
            T* out = static_cast<T*>(a.q_out.p) + row * a.q_out.tok + h * a.q_out.head;
            float y[8];
            norm_rotate<T, float, VEC>(in, d0, D, lpr, a.q_norm, a.eps, half, a.plan.layout, cs, y);
            if (VEC) {
                constexpr int W = 16 / sizeof(T);
                typedef T tv __attribute__((ext_vector_type(W)));
#pragma unroll
                for (int j = 0; j < 8 / W; ++j) {
                    tv r;
#pragma unroll
                    for (int i = 0; i < W; ++i) r[i] = from_f32<T>(y[W * j + i]);
                    *reinterpret_cast<tv*>(out + d0 + W * j) = r;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) out[d0 + e] = from_f32<T>(y[e]);
            }
            continue;
        }
        const bool is_v = h >= a.q.n + hkv;
        const int kh = h - a.q.n - (is_v ? hkv : 0);
        float s;
        uint32_t w;
        if (!is_v) {
            double y[8];
            norm_rotate<T, double, VEC>(static_cast<const T*>(a.k.p) + row * a.k.tok + kh * a.k.head, d0, D, lpr, a.k_norm, a.eps,
                                        half, a.plan.layout, cs, y);
            w = quantise8<double>(y, &s);
        } else {
            typedef typename std::conditional<sizeof(T) == 4, double, float>::type R;
            T xt[8];
            R x[8];
            load_row8<T, VEC>(static_cast<const T*>(a.v.p) + row * a.v.tok + kh * a.v.head + d0, xt);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (R)to_f32(xt[e]);
            w = quantise8<R>(x, &s);
        }
        uint16_t* val = is_v ? a.v_val : a.k_val;
        if (val) {
            typedef f16 h8 __attribute__((ext_vector_type(8)));
            h8 r;
#pragma unroll
            for (int e = 0; e < 8; ++e) r[e] = (f16)(s * (float)((int)((w >> (4 * e)) & 15u) - 8));
            *reinterpret_cast<h8*>(val + ((size_t)row * hkv + kh) * D + d0) = r;
        }
        const uint32_t other = __shfl_xor(w, 2, 64);  // the channels 16 further on, or 16 before
        if (pl.page < 0) continue;
        char* blk = a.g.base + ((size_t)pl.page * hkv + kh) * q4_block_bytes(D);
        const uint16_t sb = __builtin_bit_cast(uint16_t, (f16)s);
        const int j = c >> 2, i4 = c & 3;
        if (!is_v) {
            uint32_t k = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) k |= ((w >> (4 * e)) & 15u) << (4 * ((e >> 1) + 4 * (e & 1)));
            *reinterpret_cast<uint32_t*>(blk + q4_k_off(D, pl.slot, c)) = k;
            if (i4 == 0) *reinterpret_cast<uint16_t*>(blk + q4_ks_off(D, pl.slot, j)) = sb;
        } else {
            const uint32_t lo = i4 < 2 ? w : other, hi = i4 < 2 ? other : w;
            const int m0 = 8 * (i4 & 1), e0 = i4 < 2 ? 0 : 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t b = ((lo >> (4 * (e0 + e))) & 15u) | (((hi >> (4 * (e0 + e))) & 15u) << 4);
                *reinterpret_cast<uint8_t*>(blk + q4_v_off(D, pl.slot, j, m0 + e0 + e)) = (uint8_t)b;
            }
            if (i4 == 0) *reinterpret_cast<uint16_t*>(blk + q4_vs_off(D, pl.slot, j)) = sb;
        }
    }
}

template <typename T>
hipError_t launch_append_t(const Q4AppendArgs& a, hipStream_t s) {
    const int e = (int)sizeof(T), D = a.g.head_dim;
    bool vec = a.plan.half % 8 == 0;
    for (const HeadRows* r : {&a.q, &a.q_out, &a.k, &a.v})
        if (r->p) vec = vec && reinterpret_cast<uintptr_t>(r->p) % 16 == 0 && r->tok * e % 16 == 0 && r->head * e % 16 == 0;
    // Tokens of a workgroup: their angles fill the table in one pass; one token while the launch is small.
    const int fit = a.plan.half ? std::max(1, kTable / a.plan.half) : 4;
    const int toks = a.n_rows >= 1024 ? std::min(fit, 4) : 1;
    const int rpi = kThreads * 8 / D, rows = toks * (a.q.n + 2 * a.g.n_kv_heads);
    const long long wgs = (a.n_rows + toks - 1) / toks;
    const int blocks = (rows + rpi - 1) / rpi;
    const int y = wgs * blocks <= 2048 ? std::min(blocks, 65535) : 1;
    const dim3 grid((unsigned)wgs, y);
    if (vec)
        hipLaunchKernelGGL((q4_append_kernel<T, true>), grid, dim3(kThreads), 0, s, a, toks);
    else
        hipLaunchKernelGGL((q4_append_kernel<T, false>), grid, dim3(kThreads), 0, s, a, toks);
    return hipGetLastError();
}

// One byte of codes a thread (two channels of a token), the group's scale with its first.
__global__ __launch_bounds__(kThreads) void q4_records_kernel(Q4Geom g, int write, const int32_t* row, int max_pages, int start,
                                                              int n_tok, uint8_t* kc, uint16_t* ks, uint8_t* vc, uint16_t* vs) {
    const int D = g.head_dim, hb = D / 2, nj = D / kQ4Group;
    const size_t total = (size_t)n_tok * g.n_kv_heads * hb;
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (size_t)gridDim.x * kThreads) {
        const int b = (int)(i % hb);
        const size_t th = i / hb;
        const int h = (int)(th % g.n_kv_heads);
        const long long pos = start + (long long)(th / g.n_kv_heads);
        const long long lp = pos / sched::kPage;
        const int t = (int)(pos % sched::kPage);
        int page = lp < max_pages ? row[lp] : -1;
        if (page >= g.n_pages) page = -1;
        const int d = 2 * b, word = d / 8, e = d & 7;  // channels d, d + 1
        const size_t si = th * nj + d / kQ4Group;
        const bool head = d % kQ4Group == 0;
        char* blk = g.base + ((size_t)max(page, 0) * g.n_kv_heads + h) * q4_block_bytes(D);
        // K: nibbles e / 2 and e / 2 + 4 of the word; byte i of the word holds nibbles 2 i, 2 i + 1
        uint8_t* kb = reinterpret_cast<uint8_t*>(blk + q4_k_off(D, t, word)) + (e >> 2);
        const int sh = 4 * ((e >> 1) & 1);
        const int j = d / kQ4Group, m = d & 15, vsh = 4 * ((d >> 4) & 1);
        uint8_t* v0 = reinterpret_cast<uint8_t*>(blk + q4_v_off(D, t, j, m));
        uint8_t* v1 = reinterpret_cast<uint8_t*>(blk + q4_v_off(D, t, j, m + 1));
        if (!write) {
            const bool ok = page >= 0;
            kc[i] = ok ? (uint8_t)(((kb[0] >> sh) & 15) | (((kb[2] >> sh) & 15) << 4)) : 0x88;
            vc[i] = ok ? (uint8_t)(((v0[0] >> vsh) & 15) | (((v1[0] >> vsh) & 15) << 4)) : 0x88;
            if (head) {
                ks[si] = ok ? *reinterpret_cast<uint16_t*>(blk + q4_ks_off(D, t, j)) : 0;
                vs[si] = ok ? *reinterpret_cast<uint16_t*>(blk + q4_vs_off(D, t, j)) : 0;
            }
        } else if (page >= 0) {
            // every byte of the block by one thread: the K byte of channels d .. d + 3 comes from d % 4 == 0
            // (its other record byte is the next one), the V byte of channels 32 j + m and + 16 from the lower
            if ((b & 1) == 0) {
                const uint32_t r = kc[i] | ((uint32_t)kc[i + 1] << 8);  // channels d .. d + 3
                kb[0] = (uint8_t)((r & 15u) | (((r >> 8) & 15u) << 4));
                kb[2] = (uint8_t)(((r >> 4) & 15u) | (((r >> 12) & 15u) << 4));
            }
            if (!(d & 16)) {
                const uint32_t lo = vc[i], hi = vc[i + 8];
                v0[0] = (uint8_t)((lo & 15u) | ((hi & 15u) << 4));
                v1[0] = (uint8_t)((lo >> 4) | (hi & 0xf0u));
            }
            if (head) {
                *reinterpret_cast<uint16_t*>(blk + q4_ks_off(D, t, j)) = q4_clean_scale(ks[si]);
                *reinterpret_cast<uint16_t*>(blk + q4_vs_off(D, t, j)) = q4_clean_scale(vs[si]);
            }
        }
    }
}

}  // namespace

hipError_t launch_q4_append(const Q4AppendArgs& a, hipStream_t s) {
    return a.dtype == 0 ? launch_append_t<float>(a, s) : a.dtype == 1 ? launch_append_t<f16>(a, s) : launch_append_t<bf16>(a, s);
}

hipError_t launch_q4_records(const Q4Geom& g, bool write, const int32_t* row, int32_t max_pages, int32_t start, int32_t n_tok,
                             uint8_t* kc, uint16_t* ks, uint8_t* vc, uint16_t* vs, hipStream_t s) {
    const size_t total = (size_t)n_tok * g.n_kv_heads * (g.head_dim / 2);
    const unsigned grid = (unsigned)std::min<size_t>((total + kThreads - 1) / kThreads, 8192);
    hipLaunchKernelGGL(q4_records_kernel, dim3(grid), dim3(kThreads), 0, s, g, write ? 1 : 0, row, max_pages, start, n_tok, kc, ks,
                       vc, vs);
    return hipGetLastError();
}

}  // namespace pi
