// q4.hpp -- the paged KV cache held in 4 bits: where its bytes lie and how a lane turns them
// into matrix operands.  Host and device share the arithmetic; the device part needs hipcc.
//
// A group is 32 channels of one token's key or value head: a scale s and 32 codes c of
// 0..15, value s (c - 8).  s is an f16 of at most 7 significant bits (its 4 low mantissa
// bits are zero) with |s| <= 904, never an infinity or NaN, so that s (c - 8) is exact in f16
// and one packed f16 fma forms it: (64 + c) s - 72 s, with 72 s exact too (see deq_pair).
//
// Block of one (page, KV head), 18 D bytes, D = head_dim, NJ = D / 32 groups:
//   K codes   8 D bytes  word (g, t, j), g < 4, t < 16, j < NJ at ((g * 16 + t) * NJ + j) * 4:
//                        channels 32 j + 8 g .. + 7 of token t; channel 2 s + h of them in nibble s + 4 h
//   V codes   8 D bytes  word (q, m, j), q < 4, m < 16, j < NJ at ((q * 16 + m) * NJ + j) * 4:
//                        byte i: token 4 q + i, channel 32 j + m in the low nibble, 32 j + 16 + m in the high one
//   K scales  D bytes    f16 (t, j) at (t * NJ + j) * 2
//   V scales  D bytes    f16 (q, j, i) at ((q * NJ + j) * 4 + i) * 2, i-th of tokens 4 q + {0, 2, 1, 3}
// Lane l of a wavefront holds K words (g = l / 16, t = l mod 16, all j) and V words (q = l / 16,
// m = l mod 16, all j): both are one linear run of 4 NJ bytes a lane, and after deq_* the
// A operands of a 16-row MFMA.  A token owns whole bytes, so tokens are appended without
// reading their neighbours.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "decode_sched.hpp"

namespace pi {

constexpr int kQ4Group = 32;
constexpr float kQ4MaxScale = 904.0f;  // 72 * 904 = 65088: the largest grid scale whose 72-fold is finite in f16

PI_HD size_t q4_block_bytes(int d) { return (size_t)18 * d; }
PI_HD int q4_k_off(int d, int t, int word) {  // byte offset of K word `word` (channels 8 word ..) of token t
    const int nj = d / kQ4Group, j = word / 4, g = word % 4;
    return ((g * 16 + t) * nj + j) * 4;
}
PI_HD int q4_v_off(int d, int t, int j, int m) {  // byte offset of token t's channels 32 j + m and 32 j + 16 + m
    const int nj = d / kQ4Group;
    return 8 * d + (((t >> 2) * 16 + m) * nj + j) * 4 + (t & 3);
}
PI_HD int q4_ks_off(int d, int t, int j) { return 16 * d + (t * (d / kQ4Group) + j) * 2; }
PI_HD int q4_vs_off(int d, int t, int j) {
    const int i = t & 3, p = ((i & 1) << 1) | (i >> 1);  // 0, 2, 1, 3
    return 17 * d + (((t >> 2) * (d / kQ4Group) + j) * 4 + p) * 2;
}

// One (page, KV head) block per page and head, page-major.
struct Q4Geom {
    char* base;
    int32_t n_pages;
    int32_t n_kv_heads;
    int32_t head_dim;  // 64, 128 or 256
};

// Rows [first, first + n) of the launch's packed tokens belong to the sequence; its cache holds
// `len` tokens with them.  Clamped so that malformed tables name rows and keys that exist.
struct Q4Rows {
    int first, n, start, len;
};
PI_HD Q4Rows q4_rows(const int32_t* tok_start, const int32_t* pos, int b, int n_rows, int max_tok, int max_pages) {
    Q4Rows r;
    if (!tok_start) {  // one row a sequence; pos holds context lengths
        r.first = b;
        r.n = 1;
        r.len = sched::seq_tokens(pos[b], max_pages);
        r.start = r.len - 1;
        return r;
    }
    const int a = sched::imin(sched::imax(tok_start[b], 0), n_rows);
    const int e = sched::imin(sched::imax(tok_start[b + 1], a), n_rows);
    r.first = a;
    r.n = sched::imin(e - a, max_tok);
    r.start = sched::imax(pos[b], 0);
    const long long len = r.n ? (long long)r.start + r.n : 0, cap = (long long)sched::kPage * max_pages;
    r.len = (int)(len < cap ? len : cap);
    return r;
}

}  // namespace pi

#if defined(__HIPCC__)
#include "pi_device.hpp"

namespace pi {

// The two constants of deq_pair in registers: and_or takes no literals, and with literals the
// compiler emits an AND and an OR (16 instead of 12 instructions for 8 codes).
struct Q4Magic {
    uint32_t mask, one;
    __device__ __forceinline__ Q4Magic() {
        mask = 0x00f000f0u;
        one = 0x54005400u;
        asm volatile("" : "+s"(mask));
        asm volatile("" : "+v"(one));
    }
};

// Codes at bits 4..7 and 20..23 of x as f16: the mantissa of 64 + c, then (64 + c) s - 72 s.
__device__ __forceinline__ f16x2 deq_pair(uint32_t x, f16x2 s, f16x2 off, const Q4Magic& mg) {
    return __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (x & mg.mask) | mg.one), s, off);
}

__device__ __forceinline__ f16x8 join4(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A K word: 8 consecutive channels of a token.
__device__ __forceinline__ f16x8 deq_k(uint32_t w, f16 s, const Q4Magic& mg) {
    const f16x2 s2 = {s, s}, off = s2 * (f16)-72.0f;
    return join4(deq_pair(w << 4, s2, off, mg), deq_pair(w, s2, off, mg), deq_pair(w >> 4, s2, off, mg),
                 deq_pair(w >> 8, s2, off, mg));
}

// N words of a lane by its widest loads.
template <int N> struct Words {
    uint32_t w[N];
    __device__ __forceinline__ void load(const char* p) {
        if (N == 2) {
            const u32x2 r = *reinterpret_cast<const u32x2*>(p);
            w[0] = r[0];
            w[1] = r[1];
        } else {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const u32x4 r = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * i + e] = r[e];
            }
        }
    }
};
template <> struct Words<1> {
    uint32_t w[1];
    __device__ __forceinline__ void load(const char* p) { w[0] = *reinterpret_cast<const uint32_t*>(p); }
};

// One of a word's two f16. By a shift: an element of the word taken as a vector sends the words through scratch memory.
__device__ __forceinline__ f16 half_of(uint32_t w, int i) { return __builtin_bit_cast(f16, (uint16_t)(w >> (16 * i))); }

// Scale words: an exact f16 on the format's grid whatever the bits were (records come from callers).
__device__ __forceinline__ uint16_t q4_clean_scale(uint16_t bits) {
    const uint16_t mag = bits & 0x7ff0u, sign = bits & 0x8000u;
    if (mag > 0x7c00u || (bits & 0x7fffu) > 0x7c00u) return 0;  // NaN
    return sign | (mag > 0x6310u ? 0x6310u : mag);              // 0x6310 = 904
}

}  // namespace pi
#endif
