// q4.hip -- appending to the 4-bit paged KV cache with norm and rotation on the way, and moving its
// records in and out (gfx950).  The format is q4.hpp's.
//
// Per new token: q and k heads normed (optional), rotated by a plan (optional), q written in its own
// type, k and v quantised into the token's slot of its page and, when asked, the values that the
// cache now stands for written back in f16.
//
// K is normed and rotated in f64.  Which code a value gets depends on the side of a border it falls on,
// and the borders are where f32 results of different instruction orders disagree (a few codes of a
// million values); in f64 the codes are those of the formulas.  V is not rotated and its quotients are
// exact comparisons already in f32 for 16-bit rows (f64 for f32 rows).  Queries are f32, rounded once to their type.
//
// A lane holds 16 channels of a row as two chunks of 8, with the halves layout a chunk and its rotation partners: a row is
// read once, in 16-byte loads, and a group of 32 channels is 4 neighbouring lanes (rows of other strides, widths or
// alignment: 8 channels a lane, partners read again).  Keys and values have workgroups of their own, so that their f64
// arithmetic runs beside the queries' bytes.
//
// Bound: memory for a prompt, with the f64 of the keys next to it: 4096 tokens of 32 / 8 / 8 heads, D 128, bf16, with norm:
// 29.7 us a call back to back (105 MB, 3.5 TB/s; 20.6 at a large copy's rate); the key and value rows alone 20.7, the query
// rows alone 16.6.  f32 rows of D 256, 7 ragged sequences: 23 us (114 MB, 4.9 TB/s, the copy's rate 22.3).  32 sequences of one
// token: 6 us, three trips to memory one after the other (place, angles' frequencies, stores).
#include "pi_device.hpp"
#include "q4_launch.hpp"

#include <algorithm>
#include <type_traits>

namespace pi {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 512;     // (token, pair) angles of a workgroup
constexpr int kMaxToks = 8;     // tokens of a workgroup
constexpr int kManyRows = 1024; // rows from which a workgroup takes several tokens

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
// channel e) and the group's scale.  NaN counts as 0; infinities, and what lies past the largest value that the format
// holds, saturate.
template <typename R>
__device__ __forceinline__ uint32_t quantise8(const R* x, float* scale) {
    typedef Real<R> F;
    R hi = 0, lo = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
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
        R t = F::min_(F::max_(x[e] * inv, (R)-9), (R)8);
        t = F::rint_(F::fma_(F::fma_(-t, sr, x[e]), inv, t));
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

// A lane's 16 channels of a row: two chunks of 8, at a and b.  With the halves layout a rotating chunk's partners are the
// other chunk; in either layout four neighbouring lanes hold a group of 32 channels in each chunk.  (VEC: the widths divide
// so, rows of 16-byte chunks.  Otherwise a lane has one chunk, and reads its partners for itself.)
struct Chunks {
    int a, b;
    bool turn;  // halves: the two chunks rotate together
};
template <bool VEC, int D>
__device__ __forceinline__ Chunks chunks_of(int c, int half, int layout) {
    if (!VEC) return {8 * c, 8 * c, false};
    if (layout != 1 || half == 0) return {8 * c, 8 * c + D / 2, false};
    if (8 * c < half) return {8 * c, 8 * c + half, true};
    const int o = half + 8 * c;  // 2 half + 8 (c - half / 8)
    return {o, o + (D - 2 * half) / 2, false};
}

template <typename T, bool VEC>
struct Raw {
    T x[8], y[8];  // the chunks at a and b (VEC); the chunk and its partners
    __device__ __forceinline__ void load(const T* row, const Chunks& ch, int half, int layout) {
        load_row8<T, VEC>(row + ch.a, x);
        if (VEC)
            load_row8<T, true>(row + ch.b, y);
        else if (layout == 1 && ch.a < 2 * half)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = ch.a + e;
                y[e] = row[d < half ? d + half : d < 2 * half ? d - half : d];
            }
    }
};

// The norm's weights of a lane's channels, the same for all of its rows: in registers, so that the loop over the rows waits for
// nothing but the rows.
struct Weights {
    float x[8], y[8];
    bool on;
    template <bool VEC>
    __device__ __forceinline__ void load(const float* w, const Chunks& ch, int half, int layout) {
        on = w != nullptr;
        if (!on) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = ch.a + e;
            x[e] = w[d];
            y[e] = VEC ? w[ch.b + e] : layout == 1 && d < 2 * half ? w[d < half ? d + half : d - half] : 0.f;
        }
    }
};

// Norm and rotation of a lane's channels.  cs: cos and sin of the token's pairs.  u, v: the chunks
// (v: VEC only).
// CUT: the pairs layout's rotation may end inside a chunk (a test of every pair: 39 us for 33 for a prompt of 4096, but 34 for the
// 42 of one chunk a lane).
template <typename T, typename R, typename R2, bool VEC, int D, bool CUT>
__device__ __forceinline__ void norm_rotate(const Raw<T, VEC>& raw, const Chunks& ch, const Weights& w, float eps, int half, int layout,
                                            const R2* cs, R* u, R* v) {
    typedef Real<R> F;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        u[e] = (R)to_f32(raw.x[e]);
        v[e] = (R)to_f32(raw.y[e]);
    }
    if (w.on) {
        R ss = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += VEC ? u[e] * u[e] + v[e] * v[e] : u[e] * u[e];
#pragma unroll
        for (int m = 1; m < D / (VEC ? 16 : 8); m <<= 1) ss += shfl_xor(ss, m);
        const R rs = F::inv_sqrt(ss / (R)D + (R)eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            u[e] = u[e] * rs * (R)w.x[e];
            v[e] = v[e] * rs * (R)w.y[e];
        }
    }
    if (layout == 0) {
        auto pairs = [&](R* z, int d0) {
            if (d0 >= 2 * half) return;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                if (CUT && d0 + e >= 2 * half) break;
                const R2 a = cs[(d0 + e) >> 1];
                const R x0 = z[e], x1 = z[e + 1];
                z[e] = x0 * a.x - x1 * a.y;
                z[e + 1] = x0 * a.y + x1 * a.x;
            }
        };
        pairs(u, ch.a);
        if (VEC) pairs(v, ch.b);
    } else if (VEC) {
        if (!ch.turn) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const R2 a = cs[ch.a + e];
            const R x0 = u[e], x1 = v[e];
            u[e] = x0 * a.x - x1 * a.y;
            v[e] = x0 * a.y + x1 * a.x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = ch.a + e;
            if (d >= 2 * half) break;
            const bool first = d < half;
            const R2 a = cs[first ? d : d - half];
            u[e] = first ? u[e] * a.x - v[e] * a.y : v[e] * a.y + u[e] * a.x;
        }
    }
}

// The sequence and page of each of a workgroup's tokens, found by one wavefront: the token's place among a sample of 64 of
// the sequences' starts, then among the 64 between two samples; the rest a lane a token.  The tables are read, not
// trusted: a row is placed only where its sequence's range holds it, as the attentions read it.
__device__ __forceinline__ void find_places(const Q4AppendArgs& a, int row0, int n, Place* out, bool pages) {
    const int lane = threadIdx.x, row = row0 + lane;
    int s = row;
    if (a.tok_start) {
        const int per = (a.n_seq + 63) / 64;
        const int top = a.tok_start[min((lane + 1) * per, a.n_seq)];
        for (int i = 0; i < n; ++i) {
            int k = min((int)__popcll(__ballot((lane + 1) * per <= a.n_seq && top <= row0 + i)) * per, a.n_seq);
            if (per > 1) {
                const int j = k + 1 + lane;
                k += __popcll(__ballot(lane < per && j <= a.n_seq && a.tok_start[min(j, a.n_seq)] <= row0 + i));
            }
            if (lane == i) s = k;
        }
    }
    if (lane >= n) return;
    bool in = s < a.n_seq;
    s = min(s, a.n_seq - 1);
    const int start = a.start_pos[s];
    int first = row;
    if (a.tok_start) {
        first = max(a.tok_start[s], 0);
        in = in && row >= first && row < a.tok_start[s + 1];
    }
    const long long pos = (long long)max(start, 0) + (row - first);
    const long long lp = pos / sched::kPage;
    int page = -1;
    if (pages && in && lp < a.max_pages) page = a.page_table[(size_t)s * a.max_pages + lp];
    out[lane].pos = in ? pos : -1;
    out[lane].page = page < a.g.n_pages ? page : -1;
    out[lane].slot = (int)(pos % sched::kPage);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* out, const float* y) {
    if (VEC) {
        constexpr int W = 16 / sizeof(T);
        typedef T tv __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int j = 0; j < 8 / W; ++j) {
            tv r;
#pragma unroll
            for (int i = 0; i < W; ++i) r[i] = from_f32<T>(y[W * j + i]);
            *reinterpret_cast<tv*>(out + W * j) = r;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = from_f32<T>(y[e]);
    }
}

// A lane's channels of a query row: normed, rotated, written in the rows' type.
template <typename T, bool VEC, int D, bool CUT>
__device__ __forceinline__ void put_q(const Q4AppendArgs& a, const Raw<T, VEC>& raw, const Weights& w, int row, int h, const Chunks& ch,
                                      const float2* cs) {
    float u[8], v[8];
    norm_rotate<T, float, float2, VEC, D, CUT>(raw, ch, w, a.eps, a.plan.half, a.plan.layout, cs, u, v);
    T* out = static_cast<T*>(a.q_out.p) + row * a.q_out.tok + h * a.q_out.head;
    store8<T, VEC>(out + ch.a, u);
    if (VEC) store8<T, VEC>(out + ch.b, v);
}

// A chunk's codes w and scale s to its page, and its values to where the caller wants them.
template <int D>
__device__ __forceinline__ void put_codes(const Q4AppendArgs& a, uint32_t w, float s, bool is_v, int row, int kh, int d0, const Place& pl) {
    const int hkv = a.g.n_kv_heads, c = d0 >> 3;
    uint16_t* val = is_v ? a.v_val : a.k_val;
    if (val) {
        typedef f16 h8 __attribute__((ext_vector_type(8)));
        h8 r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (f16)(s * (float)((int)((w >> (4 * e)) & 15u) - 8));
        *reinterpret_cast<h8*>(val + ((size_t)row * hkv + kh) * D + d0) = r;
    }
    const uint32_t other = __shfl_xor(w, 2, 64);  // the channels 16 further on, or 16 before
    if (pl.page < 0) return;
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

// A lane's channels of a key or value row: normed and rotated (keys), quantised, stored.
template <typename T, bool VEC, int D, bool CUT>
__device__ __forceinline__ void put_kv(const Q4AppendArgs& a, const Raw<T, VEC>& raw, const Weights& nw, bool is_v, int row, int kh,
                                       const Chunks& ch, const Place& pl, const double2* cs) {
    float s0, s1 = 0.f;
    uint32_t w0, w1 = 0;
    if (!is_v) {
        double u[8], v[8];
        norm_rotate<T, double, double2, VEC, D, CUT>(raw, ch, nw, a.eps, a.plan.half, a.plan.layout, cs, u, v);
        w0 = quantise8<double>(u, &s0);
        if (VEC) w1 = quantise8<double>(v, &s1);
    } else {
        typedef typename std::conditional<sizeof(T) == 4, double, float>::type R;
        R u[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            u[e] = (R)to_f32(raw.x[e]);
            v[e] = (R)to_f32(raw.y[e]);
        }
        w0 = quantise8<R>(u, &s0);
        if (VEC) w1 = quantise8<R>(v, &s1);
    }
    put_codes<D>(a, w0, s0, is_v, row, kh, ch.a, pl);
    if (VEC) put_codes<D>(a, w1, s1, is_v, row, kh, ch.b, pl);
}

// Workgroups 0 .. kv_wgs - 1 take the keys and values of `toks` tokens each (f64 angles, quantiser), the others the
// queries of `toks` tokens (f32): in one launch, so that the heavier arithmetic runs beside the larger share
// of the bytes.  blockIdx.y: a share of the tokens' rows.  A workgroup's first rows are requested before it looks
// up its tokens' places and computes their angles.
template <typename T, bool VEC, int D, bool CUT>
__global__ __launch_bounds__(kThreads, 3) void q4_append_kernel(Q4AppendArgs a, int toks, int kv_wgs) {
    __shared__ double2 s_cs[kTable];
    __shared__ Place s_place[kMaxToks];
    const int tid = threadIdx.x, half = a.plan.half;
    const bool kv = (int)blockIdx.x < kv_wgs;
    const int row0 = (kv ? blockIdx.x : blockIdx.x - kv_wgs) * toks, n = min(toks, a.n_rows - row0);
    const int hkv = a.g.n_kv_heads, heads = kv ? hkv : a.q.n, n_keys = kv ? n * hkv : 0;
    constexpr int lpr = D / (VEC ? 16 : 8), rpi = kThreads / lpr;  // lanes a row, rows at a time
    const int rl = tid / lpr;
    const Chunks ch = chunks_of<VEC, D>(tid - rl * lpr, half, a.plan.layout);
    const int step = gridDim.y * rpi;
    // Row u: all tokens' key rows, then all their value rows (the key rows' f64 work then falls to all wavefronts alike);
    // or the query rows.  t, h: its token and head, is_v: a value row.
    int u = blockIdx.y * rpi + rl, t, h;
    bool is_v;
    auto place = [&] {
        is_v = kv && u >= n_keys;
        const int r = is_v ? u - n_keys : u;
        t = r / heads;
        h = r - t * heads;
    };
    place();
    const T* const p0 = static_cast<const T*>(kv ? a.k.p : a.q.p);
    const T* const p1 = static_cast<const T*>(a.v.p);
    const int64_t tok0 = kv ? a.k.tok : a.q.tok, head0 = kv ? a.k.head : a.q.head, tok1 = a.v.tok, head1 = a.v.head;
    const int rows = kv ? 2 * n_keys : n * heads;
    Raw<T, VEC> raw;
    auto load = [&] {
        if (u >= rows) return;
        const T* row = is_v ? p1 + (row0 + t) * tok1 + h * head1 : p0 + (row0 + t) * tok0 + h * head0;
        raw.load(row, ch, is_v ? 0 : half, a.plan.layout);
    };
    load();
    Weights w;
    w.template load<VEC>(kv ? a.k_norm : a.q_norm, ch, half, a.plan.layout);
    if (tid < 64) find_places(a, row0, n, s_place, kv);
    __syncthreads();
    if (kv) {
        for (int i = tid; i < n * half; i += kThreads) {
            const int tt = i / half;
            double turns = (double)s_place[tt].pos * a.plan.turns[i - tt * half];
            turns -= rint(turns);
            double sn, cn;
            sincospi(2.0 * turns, &sn, &cn);
            s_cs[i] = double2{cn * a.plan.mscale, sn * a.plan.mscale};
        }
    } else {
        float2* f_cs = reinterpret_cast<float2*>(s_cs);
        for (int i = tid; i < n * half; i += kThreads) {
            const int tt = i / half;
            double turns = (double)s_place[tt].pos * a.plan.turns[i - tt * half];
            turns -= rint(turns);
            float sn, cn;
            sincospif((float)(2.0 * turns), &sn, &cn);
            f_cs[i] = float2{cn * (float)a.plan.mscale, sn * (float)a.plan.mscale};
        }
    }
    __syncthreads();
    while (u < rows) {
        const Raw<T, VEC> now = raw;
        const int tn = t, hn = h;
        const bool vn = is_v;
        u += step;
        place();
        load();
        const Place pl = s_place[tn];
        if (pl.pos < 0) continue;  // a row of no sequence; uniform over a row's lanes
        if (kv)
            put_kv<T, VEC, D, CUT>(a, now, w, vn, row0 + tn, hn, ch, pl, s_cs + tn * half);
        else
            put_q<T, VEC, D, CUT>(a, now, w, row0 + tn, hn, ch, reinterpret_cast<const float2*>(s_cs) + tn * half);
    }
}

template <typename T, int D>
hipError_t launch_append_d(const Q4AppendArgs& a, hipStream_t s) {
    const int e = (int)sizeof(T);
    const int half = a.plan.half;
    bool vec = a.plan.layout == 1 && half ? half % 32 == 0 && (D - 2 * half) % 64 == 0 : true;
    for (const HeadRows* r : {&a.q, &a.q_out, &a.k, &a.v})
        if (r->p) vec = vec && reinterpret_cast<uintptr_t>(r->p) % 16 == 0 && r->tok * e % 16 == 0 && r->head * e % 16 == 0;
    // Tokens of a workgroup: as many as fill the angles' table in one pass of its threads; one while the launch is small.
    const int fit = half ? std::max(1, kTable / half) : kMaxToks;
    const int toks = a.n_rows >= kManyRows ? std::min(fit, kMaxToks) : 1;
    const int rpi = kThreads * (vec ? 16 : 8) / D;
    const long long wgs = (a.n_rows + toks - 1) / toks, all = wgs * (a.q.n ? 2 : 1);
    const int blocks = (toks * std::max(a.q.n, 2 * a.g.n_kv_heads) + rpi - 1) / rpi;
    const int y = all * blocks <= 2048 ? std::min(blocks, 65535) : 1;
    const dim3 grid((unsigned)all, y);
    if (vec && a.plan.layout == 0 && half % 4)
        hipLaunchKernelGGL((q4_append_kernel<T, true, D, true>), grid, dim3(kThreads), 0, s, a, toks, (int)wgs);
    else if (vec)
        hipLaunchKernelGGL((q4_append_kernel<T, true, D, false>), grid, dim3(kThreads), 0, s, a, toks, (int)wgs);
    else
        hipLaunchKernelGGL((q4_append_kernel<T, false, D, true>), grid, dim3(kThreads), 0, s, a, toks, (int)wgs);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_append_t(const Q4AppendArgs& a, hipStream_t s) {
    switch (a.g.head_dim) {
        case 64: return launch_append_d<T, 64>(a, s);
        case 128: return launch_append_d<T, 128>(a, s);
        default: return launch_append_d<T, 256>(a, s);
    }
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
