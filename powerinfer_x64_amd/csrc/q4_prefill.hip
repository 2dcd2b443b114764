// q4_prefill.hip -- attention of many rows a KV head over the 4-bit paged cache (gfx950): prompts and chunks.
//
// Work: the rows (token, query head) of one sequence and KV head, token by token, 32 to a wavefront. A workgroup walks
// the keys its rows see in tiles of 64 (four pages); each tile's codes are dequantised once, into LDS, by all of its
// wavefronts, so a code is unpacked once for 256 rows (128 where a wavefront needs a SIMD's registers alone).  Per tile and
// wavefront, on v_mfma_f32_32x32x16_f16:
//   S^T[64 x 32] = K . Q^T,   O^T[D x 32] += V^T . P^T
// A lane owns one row's scores (half of them; lane + 32 has the rest), so a row's sum needs one cross-lane step at
// the end, and its P values are the operand of the second product in place: the k index of a 16-key step is the order
// in which a lane's scores and the dequantised V words come (q4.hpp).
//
// LDS: K tile [D / 8 chunks][64 keys] of 16 bytes, V tile [4 pages][2][D] of 16 bytes (8 keys of a channel), each doubled;
// odd chunks / halves are shifted by 256 bytes so that a dequantising wavefront's stores and the operand reads both
// cover all banks.
//
// Schedule of 8 wavefronts, two a SIMD (16-bit rows at D 64 and 128, f32 at 64): in step t wavefronts 0..3 run the products
// (PV of tile t - 1, QK of tile t) and then the softmax of tile t and the unpacking of K tile t + 1; wavefronts 4..7 run
// the softmax of tile t - 1 and the unpacking of V tile t first and the products after: on each SIMD one wavefront's
// matrix instructions run beside the other's vector instructions.  One barrier a step.
// Schedule of 4, one a SIMD with all its registers (D 256, f32 at 128): in step t the exps of tile t are written between
// the matrix instructions of QK t + 1, and the unpacking of K t + 2 and V t + 1 between those of PV t, in fixed order.
// (Against QK, softmax, PV and unpacking one after the other: 16-bit D 256 581 -> 714 TFLOP/s, f32 D 128 400 -> 470, f32
// D 256 349 -> 414.  Two such workgroups a CU at 16-bit D 128 reach 683 where 8 wavefronts reach 838: every code is unpacked
// for 128 rows, not 256.)
//
// Bound: the matrix cores' rate under load (a matrix product of 8192 cubed reaches 1230 TFLOP/s) and, at D 256, LDS reads, which
// take as long as the products.  One sequence, 1000 rows over 8200 keys, 32 / 8 heads, back to back: D 64 115 us
// (618 TFLOP/s: exps weigh twice), D 128 163-171 us (830-875), f32 D 128 303 us (470, each product twice);
// 16 / 2 heads, D 256: 200 us (714), f32 344 us (414).  An 8 us merge is in them (two key splits).
//
// Softmax: exps against the running max as it stands; only where a row's sum of a tile passes 2^13 (the first
// tile, or a score outgrew the max) is the tile's max taken, O and l rescaled and the tile done again.
//
// f32 rows: q and P in two f16 parts (22 bits), each product twice, f32 accumulation.
#include "pi_device.hpp"
#include "q4_launch.hpp"

#include <algorithm>
#include <type_traits>

namespace pi {
namespace {

constexpr int kTile = 64;                    // keys
constexpr int kTilePages = kTile / sched::kPage;
constexpr float kRedo = 8192.0f;

__device__ __forceinline__ float sigmoidf_(float x) { return 1.0f / (1.0f + expf(-x)); }

__device__ __forceinline__ void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int D> __device__ __forceinline__ int k_addr(int chunk, int key) { return (chunk * kTile + (key ^ (16 * (chunk & 1)))) * 16; }
template <int D> __device__ __forceinline__ int v_addr(int page, int hh, int ch) { return ((page * 2 + hh) * D + (ch ^ (16 * hh))) * 16; }

// One page's K codes of a lane (token lane % 16, chunks 4 j + lane / 16), or its V codes (tokens 4 (lane / 16) ..).
template <int D>
struct KPart {
    static constexpr int NJ = D / kQ4Group;
    Words<NJ> w;
    Words<NJ / 2> s;
    __device__ __forceinline__ void load(const char* blk, int lane) {
        w.load(blk + lane * (4 * NJ));
        s.load(blk + 16 * D + (lane & 15) * (2 * NJ));
    }
    // word j to p = tile + at(page, lane)
    static __device__ __forceinline__ int at(int page, int lane) { return k_addr<D>(lane >> 4, page * 16 + (lane & 15)); }
    __device__ __forceinline__ void put1(int j, char* p, const Q4Magic& mg) const {
        *reinterpret_cast<f16x8*>(p + j * (4 * kTile * 16)) = deq_k(w.w[j], half_of(s.w[j / 2], j & 1), mg);
    }
    __device__ __forceinline__ void put(char* tile, int page, int lane, const Q4Magic& mg) const {
#pragma unroll
        for (int j = 0; j < NJ; ++j) put1(j, tile + at(page, lane), mg);
    }
};
template <int D>
struct VPart {
    static constexpr int NJ = D / kQ4Group;
    Words<NJ> w;
    Words<2 * NJ> s;
    __device__ __forceinline__ void load(const char* blk, int lane) {
        w.load(blk + 8 * D + lane * (4 * NJ));
        s.load(blk + 17 * D + (lane >> 4) * (8 * NJ));
    }
    static __device__ __forceinline__ int at(int page, int lane) {
        return v_addr<D>(page, (lane >> 4) & 1, lane & 15) + (lane >> 5) * 8;
    }
    __device__ __forceinline__ void put1(int j, char* p0, char* p1, const Q4Magic& mg) const {  // p1: 16 channels on
        const f16 off = (f16)-72.0f;
        const f16x2 a = __builtin_bit_cast(f16x2, s.w[2 * j]), b = __builtin_bit_cast(f16x2, s.w[2 * j + 1]);
        const f16x2 oa = a * off, ob = b * off;
        const uint32_t x = w.w[j];
        const f16x2 l0 = deq_pair(x << 4, a, oa, mg), l1 = deq_pair(x >> 4, b, ob, mg);
        const f16x2 h0 = deq_pair(x, a, oa, mg), h1 = deq_pair(x >> 8, b, ob, mg);
        *reinterpret_cast<f16x4*>(p0 + j * 512) = f16x4{l0[0], l0[1], l1[0], l1[1]};
        *reinterpret_cast<f16x4*>(p1 + j * 512) = f16x4{h0[0], h0[1], h1[0], h1[1]};
    }
    __device__ __forceinline__ void put(char* tile, int page, int lane, const Q4Magic& mg) const {
#pragma unroll
        for (int j = 0; j < NJ; ++j) put1(j, tile + at(page, lane), tile + (at(page, lane) ^ 256), mg);
    }
};

struct TileArgs {
    float* o;   // partial O [split][row][D], row = packed token * n_q_heads + head
    float* ml;  // partial (max, sum) [split][row][2]
    int n_blk, splits;
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, NW / 4) void q4_tile_kernel(Q4AttnArgs a, TileArgs ta) {
    constexpr int KS = D / 16, NB = D / 32, PREC = std::is_same<T, float>::value ? 2 : 1;
    constexpr int kRows = NW * 32, kBuf = kTile * D * 2;
    extern __shared__ __attribute__((aligned(16))) char lds[];  // K tiles 0, 1, V tiles 0, 1
    const int n_kv = a.g.n_kv_heads;
    // KV heads fastest: with 8 of them each XCD's L2 sees one.  The last row blocks see most keys: first.
    int id = blockIdx.x;
    const int kvh = id % n_kv;
    id /= n_kv;
    const int split = id % ta.splits;
    id /= ta.splits;
    const int b = id % a.batch;
    const int blk = ta.n_blk - 1 - id / a.batch;
    const Q4Rows rw = q4_rows(a.tok_start, a.pos, b, a.n_rows, a.max_tok, a.use_pages);
    const int row0 = blk * kRows, n_rows = rw.n * a.group;
    if (row0 >= n_rows) return;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hh = lane >> 5;
    const Q4Magic mg;
    // keys that the workgroup's last row sees, and its share of their tiles
    const int last_tok = (min(row0 + kRows, n_rows) - 1) / a.group;
    const int keys = (int)min((long long)rw.start + last_tok + 1, (long long)rw.len);
    const int all_tiles = (keys + kTile - 1) / kTile;
    const int t0 = (int)((long long)all_tiles * split / ta.splits), t1 = (int)((long long)all_tiles * (split + 1) / ta.splits);

    // the lane's row
    const int r = row0 + wave * 32 + col, tok = r / a.group, c = r - tok * a.group;
    const int head = a.gqa_mode == 0 ? kvh + c * n_kv : kvh * a.group + c;
    const bool on = tok < rw.n && head < a.n_q_heads;
    const size_t row = on ? (size_t)(rw.first + tok) * a.n_q_heads + head : 0;
    const int lim = on ? (int)min((long long)rw.start + tok + 1, (long long)rw.len) : 0;
    // the wavefront's: keys that all rows see, and that any sees
    const int w_tok0 = (row0 + wave * 32) / a.group, w_tok1 = (row0 + wave * 32 + 31) / a.group;
    const int lim_all = (int)min((long long)rw.start + w_tok0 + 1, (long long)rw.len);
    const int lim_any = w_tok0 < rw.n ? (int)min((long long)rw.start + min(w_tok1, rw.n - 1) + 1, (long long)rw.len) : 0;

    // Q^T operand: channels 16 ks + 8 hh + e of the row
    f16x8 q[PREC][KS];
    float back = a.scale * kLog2e;
    {
        const T* p = static_cast<const T*>(a.q) + row * D + 8 * hh;
        float x[8 * KS];
        constexpr int W = 16 / sizeof(T);
        typedef T tv __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < 8 / W; ++j) {
                const tv v = *reinterpret_cast<const tv*>(p + 16 * k + W * j);
#pragma unroll
                for (int i = 0; i < W; ++i) x[8 * k + W * j + i] = on ? to_f32(v[i]) : 0.f;
            }
        float f = 1.f;
        if (!std::is_same<T, f16>::value) {  // the row's largest magnitude to [1, 2)
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < 8 * KS; ++i) mx = fmaxf(mx, fabsf(x[i]));
            mx = wave_max_xor(mx, 32);
            const int ex = (int)((__builtin_bit_cast(uint32_t, mx) >> 23) & 255u) - 127;
            const int e1 = mx > 0.f && ex > -127 && ex < 127 ? ex : 0;
            f = __builtin_bit_cast(float, (uint32_t)(127 - e1) << 23);
            back = ldexpf(back, e1);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = x[8 * k + e] * f;
                const f16 h = to_f16(y);
                q[0][k][e] = h;
                if (PREC == 2) q[PREC - 1][k][e] = to_f16(y - (float)h);
            }
    }
    if (fabsf(back) < 1e-30f) back = copysignf(1e-30f, back);  // a scale of 0: all scores as good as equal, masks stay -inf
    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -1e30f, l = 0.f;
    f32x16 s[2];
    f16x8 pf[PREC][4];  // P of the tile's four 16-key steps

    const int32_t* pt = a.page_table + (size_t)b * a.max_pages;
    const int seq_pages = (rw.len + sched::kPage - 1) / sched::kPage;
    // page ids of a tile in lanes 0..3 (a page past the sequence: none)
    auto ids_of = [&](int t) {
        const int p = t * kTilePages + (lane & 3);
        return p < seq_pages ? pt[p] : -1;
    };
    auto bad_of = [&](int ids) { return (uint32_t)(__ballot(!sched::page_ok(ids, a.g.n_pages)) & 15u); };
    auto block_of = [&](int ids, int page) {
        const int id1 = __builtin_amdgcn_readlane(ids, page);
        const int pid = sched::page_ok(id1, a.g.n_pages) ? id1 : 0;
        return a.g.base + ((size_t)pid * n_kv + kvh) * q4_block_bytes(D);
    };

    // Both products read their LDS operands kAhead ahead, one read beside each matrix instruction (left alone, the
    // compiler requests them all first and spills).
    constexpr int kAhead = 4;
    auto plain = [](int n) {
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int i = 0; i < 64; ++i)
            if (i < n - kAhead) {
                __builtin_amdgcn_sched_group_barrier(0x008, PREC, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        __builtin_amdgcn_sched_group_barrier(0x008, kAhead * PREC, 0);
    };
    auto none = [](auto&&...) {};
    auto qk = [&](int t, f32x16 (&s)[2], auto&& also, auto&& pace) {
        const char* tile = lds + (t & 1) * kBuf + k_addr<D>(hh, col);
        auto frag = [&](int i) {  // chunk 2 (i / 2) + hh, keys 32 (i % 2) + col
            return *reinterpret_cast<const f16x8*>(tile + (i >> 1) * (2 * kTile * 16) + (i & 1) * 512);
        };
        s[0] = f32x16{};
        s[1] = f32x16{};
        f16x8 f[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) f[i] = frag(i);
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
            const f16x8 kf = f[i % kAhead];
            if (i + kAhead < 2 * KS) f[i % kAhead] = frag(i + kAhead);
#pragma unroll
            for (int h = 0; h < PREC; ++h) s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, q[h][i >> 1], s[i & 1], 0, 0, 0);
            also(i);
        }
        pace(2 * KS);
    };
    auto pv = [&](int t, auto&& also, auto&& pace) {
        // page i / NB, half hh, channel (32 (i % NB) + col) ^ 16 hh
        const char* tile = lds + (2 + (t & 1)) * kBuf + v_addr<D>(0, hh, col);
        auto frag = [&](int i) { return *reinterpret_cast<const f16x8*>(tile + (i / NB) * (2 * D * 16) + (i % NB) * 512); };
        f16x8 f[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) f[i] = frag(i);
#pragma unroll
        for (int i = 0; i < 4 * NB; ++i) {
            const f16x8 vf = f[i % kAhead];
            if (i + kAhead < 4 * NB) f[i % kAhead] = frag(i + kAhead);
#pragma unroll
            for (int h = 0; h < PREC; ++h)
                o[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[h][i / NB], o[i % NB], 0, 0, 0);
            also(i);
        }
        pace(4 * NB);
    };
    // P of the tile against m, its sum over the lane's 32 keys.
    auto exps = [&] {
        float part[4];
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = fast_exp2(fmaf(s[st >> 1][8 * (st & 1) + i], back, -m));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = p[(i & 4) | ((i & 1) << 1) | ((i >> 1) & 1)];  // 0, 2, 1, 3 of each four: the V words' order
                const f16 h = to_f16(x);
                pf[0][st][i] = h;
                if (PREC == 2) pf[PREC - 1][st][i] = to_f16(x - (float)h);
            }
            part[st] = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        }
        return (part[0] + part[1]) + (part[2] + part[3]);
    };
    auto mask = [&](int t, uint32_t bad) {
        if (bad != 0 || (t + 1) * kTile > lim_all) {  // scores that do not count: -inf after the factor, which is not 0
            const int left = lim - t * kTile - 4 * hh;
            const float none = back < 0.f ? INFINITY : -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * kb + 8 * (e >> 2) + (e & 3) >= left || ((bad >> (2 * kb + (e >> 3))) & 1)) s[kb][e] = none;
        }
    };
    auto add = [&](float sum) {
        if (__any(sum > kRedo)) {  // no P is above 1 after it
            float mx = -1e30f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e] * back);
            mx = wave_max_xor(mx, 32);
            const float m_new = fmaxf(m, mx), alpha = fast_exp2(m - m_new);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; ++i) o[i] *= alpha;
            m = m_new;
            sum = exps();
        }
        l += sum;
    };
    auto softmax = [&](int t, uint32_t bad) {
        mask(t, bad);
        add(exps());
    };

    auto finish = [&] {
        l = wave_sum_xor(l, 32);
        if (!on) return;
        // O^T: channel 32 nb + 8 (e / 4) + 4 hh + e % 4 of the lane's row
        if (ta.splits > 1) {
            const size_t prow = (size_t)split * a.n_rows * a.n_q_heads + row;
            float* po = ta.o + prow * D + 4 * hh;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4*>(po + 32 * nb + 8 * i) =
                        f32x4{o[nb][4 * i], o[nb][4 * i + 1], o[nb][4 * i + 2], o[nb][4 * i + 3]};
            if (hh == 0) {
                ta.ml[2 * prow] = m;
                ta.ml[2 * prow + 1] = l;
            }
            return;
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        typedef T t4 __attribute__((ext_vector_type(4)));
        T* out = static_cast<T*>(a.out) + row * D + 4 * hh;
        if (a.gate) {
            const T* gate = static_cast<const T*>(a.gate) + row * D + 4 * hh;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const t4 g = *reinterpret_cast<const t4*>(gate + 32 * nb + 8 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nb][4 * i + e] *= sigmoidf_(to_f32(g[e]));
                }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t4 y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(o[nb][4 * i + e] * inv);
                *reinterpret_cast<t4*>(out + 32 * nb + 8 * i) = y;
            }
    };

    if (t0 >= t1) {
        finish();
        return;
    }
    // The wavefront's own last tile: its rows see none of the later ones, it only unpacks them.
    const int n = max(t0, min(t1, (lim_any + kTile - 1) / kTile));
    // ids of tiles t + 1 and t + 2 and the unusable pages of tile t, one step at a time
    int i1 = ids_of(t0), i2 = ids_of(t0 + 1);
    uint32_t bad = 0;
    auto step_ids = [&](int t) {  // to step t
        bad = bad_of(i1);
        i1 = i2;
        i2 = ids_of(t + 2);
    };
    if constexpr (NW == 8) {
        const int page = wave & 3;
        if (wave < 4) {
            KPart<D> kp;
            kp.load(block_of(i1, page), lane);
            kp.put(lds + (t0 & 1) * kBuf, page, lane, mg);
            kp.load(block_of(i2, page), lane);
            barrier_lds();
            auto unpack = [&](int t) {
                if (t + 1 < t1) {
                    kp.put(lds + ((t + 1) & 1) * kBuf, page, lane, mg);
                    kp.load(block_of(i2, page), lane);
                }
                barrier_lds();
            };
            step_ids(t0);
            if (n > t0) {
                qk(t0, s, none, plain);
                softmax(t0, bad);
            }
            unpack(t0);
            for (int t = t0 + 1; t < n; ++t) {
                step_ids(t);
                __builtin_amdgcn_s_setprio(2);
                pv(t - 1, none, plain);
                qk(t, s, none, plain);
                __builtin_amdgcn_s_setprio(0);
                softmax(t, bad);
                unpack(t);
            }
            if (n > t0) pv(n - 1, none, plain);
            for (int t = max(n, t0 + 1); t <= t1; ++t) {
                step_ids(t);
                unpack(t);
            }
            finish();
        } else {
            VPart<D> vp;
            vp.load(block_of(i1, page), lane);
            barrier_lds();
            auto unpack = [&](int t) {
                if (t < t1) {
                    vp.put(lds + (2 + (t & 1)) * kBuf, page, lane, mg);
                    vp.load(block_of(i1, page), lane);
                }
            };
            step_ids(t0);
            unpack(t0);
            if (n > t0) qk(t0, s, none, plain);
            barrier_lds();
            uint32_t was = bad;
            for (int t = t0 + 1; t < n; ++t) {
                step_ids(t);
                unpack(t);
                softmax(t - 1, was);
                was = bad;
                __builtin_amdgcn_s_setprio(2);
                pv(t - 1, none, plain);
                qk(t, s, none, plain);
                __builtin_amdgcn_s_setprio(0);
                barrier_lds();
            }
            int t = t0 + 1;
            if (n > t0) {
                step_ids(n);
                unpack(n);
                softmax(n - 1, was);
                pv(n - 1, none, plain);
                barrier_lds();
                t = n + 1;
            }
            for (; t <= t1; ++t) {
                step_ids(t);
                unpack(t);
                barrier_lds();
            }
            finish();
        }
    } else {
        KPart<D> kp;
        VPart<D> vp;
        int i3 = ids_of(t0 + 2), i4 = ids_of(t0 + 3);  // of tiles t + 2, t + 3 (i1, i2: t, t + 1)
        auto put_k = [&](int t) { kp.put(lds + (t & 1) * kBuf, wave, lane, mg); };
        auto put_v = [&](int t) { vp.put(lds + (2 + (t & 1)) * kBuf, wave, lane, mg); };
        auto next = [&](int t) {  // pages of step t + 1
            kp.load(block_of(i4, wave), lane);
            vp.load(block_of(i3, wave), lane);
            i1 = i2;
            i2 = i3;
            i3 = i4;
            i4 = ids_of(t + 4);
        };
        // beside the second product: every second step a word of the next K or V codes
        auto put_some = [&](int t) {
            // opaque: left alone, the compiler keeps an address for every word, in scratch memory
            int ko = (t & 1) * kBuf + KPart<D>::at(wave, lane), vo = (2 + ((t + 1) & 1)) * kBuf + VPart<D>::at(wave, lane), vx = vo ^ 256;
            asm volatile("" : "+v"(ko), "+v"(vo), "+v"(vx));
            return [&, ko, vo, vx](int i) {
                constexpr int NJ = D / kQ4Group;
                const int j = i / 2;
                if (i & 1) {
                } else if (j < NJ) kp.put1(j, lds + ko, mg);
                else vp.put1(j - NJ, lds + vo, lds + vx, mg);
                __builtin_amdgcn_sched_barrier(0);
            };
        };
        kp.load(block_of(i1, wave), lane);
        vp.load(block_of(i1, wave), lane);
        put_k(t0);
        put_v(t0);
        kp.load(block_of(i2, wave), lane);
        vp.load(block_of(i2, wave), lane);
        put_k(t0 + 1);
        kp.load(block_of(i3, wave), lane);
        barrier_lds();
        if (n > t0) qk(t0, s, none, plain);
        barrier_lds();
        int t = t0;
        for (; t < n - 1; ++t) {
            mask(t, bad_of(i1));
            f32x16 sn[2];
            float sum = 0.f, even = 0.f;
            qk(t + 1, sn, [&](int i) {
                constexpr int E = 16 / KS;  // scores a step
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const int k = E * i + j, st = k >> 3, e = k & 7;
                    const float x = fast_exp2(fmaf(s[st >> 1][8 * (st & 1) + ((e & 4) | ((e & 1) << 1) | ((e >> 1) & 1))], back, -m));
                    sum += x;
                    if (!(e & 1)) {
                        even = x;
                        continue;
                    }
                    const f16 h0 = to_f16(even), h1 = to_f16(x);
                    pf[0][st][e - 1] = h0;
                    pf[0][st][e] = h1;
                    if (PREC == 2) {
                        pf[PREC - 1][st][e - 1] = to_f16(even - (float)h0);
                        pf[PREC - 1][st][e] = to_f16(x - (float)h1);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }, none);
            add(sum);
            pv(t, put_some(t), none);
            next(t);
            s[0] = sn[0];
            s[1] = sn[1];
            barrier_lds();
        }
        if (n > t0) {
            softmax(t, bad_of(i1));
            pv(t, put_some(t), none);
            next(t);
            ++t;
            barrier_lds();
        }
        for (; t < t1; ++t) {
            put_k(t + 2);
            put_v(t + 1);
            next(t);
            barrier_lds();
        }
        finish();
    }
}

// Joins the splits of each row: D / 4 threads a row.  Bound by memory: two splits of 1000 tokens, 32 heads, D 128, 33 MB of
// f32 partials read and 8 MB written in 9.2 us (4.5 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void q4_tile_merge_kernel(Q4AttnArgs a, TileArgs ta, int D) {
    const int per = 256 / (D / 4), rl = threadIdx.x / (D / 4), d = 4 * (threadIdx.x - rl * (D / 4));
    const size_t rows = (size_t)a.n_rows * a.n_q_heads;
    const size_t row = (size_t)blockIdx.x * per + rl;
    if (row >= rows) return;
    // Rows of no sequence, and rows past max_tok, hold no partials: they are read (the
    // workspace covers them) and not stored. The D / 4 lanes of a row look at as many
    // sequences at once; one after the other each costs a trip to the L2.
    const int tok = (int)(row / a.n_q_heads);
    bool in_seq = false;
    for (int b0 = d / 4; b0 < a.batch; b0 += D / 4) {
        const Q4Rows rw = q4_rows(a.tok_start, a.pos, b0, a.n_rows, a.max_tok, a.use_pages);
        in_seq |= tok >= rw.first && tok < rw.first + rw.n;
    }
    const int lane = threadIdx.x & 63;
    const uint64_t lanes = (D == 256 ? ~0ull : (1ull << (D / 4)) - 1) << (lane & ~(D / 4 - 1));
    const bool mine = (__ballot(in_seq) & lanes) != 0;
    // four splits' loads in flight at a time, joined against the running maximum
    float mx = -1e30f, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < ta.splits; s0 += 4) {
        float mm[4], ll[4];
        f32x4 oo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = s0 + i < ta.splits;
            const size_t p = (in ? s0 + i : s0) * rows + row;
            mm[i] = ta.ml[2 * p];
            ll[i] = in ? ta.ml[2 * p + 1] : 0.f;
            oo[i] = *reinterpret_cast<const f32x4*>(ta.o + p * D + d);
        }
        const float was = mx;
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, mm[i]);
        const float f = fast_exp2(was - mx);
        o *= f;
        l *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float w = s0 + i < ta.splits ? fast_exp2(mm[i] - mx) : 0.f;
            o += w * oo[i];
            l += w * ll[i];
        }
    }
    if (!mine) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float v = o[e] * inv;
        if (a.gate) v *= sigmoidf_(to_f32(static_cast<const T*>(a.gate)[row * D + d + e]));
        y[e] = from_f32<T>(v);
    }
    *reinterpret_cast<t4*>(static_cast<T*>(a.out) + row * D + d) = y;
}

template <typename T, int D, int NW>
hipError_t launch_t(const Q4AttnArgs& a, const Q4Plan& p, const TileArgs& ta, hipStream_t s) {
    const size_t lds = (size_t)4 * kTile * D * 2;
    if (lds > (64 << 10)) {
        static std::atomic<uint64_t> on{0};
        const hipError_t e = allow_lds(reinterpret_cast<const void*>(&q4_tile_kernel<T, D, NW>), lds, on);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((q4_tile_kernel<T, D, NW>), dim3((unsigned)p.grid), dim3(NW * 64), lds, s, a, ta);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || ta.splits == 1) return e;
    const int per = 256 / (D / 4);
    const size_t rows = (size_t)a.n_rows * a.n_q_heads;
    hipLaunchKernelGGL((q4_tile_merge_kernel<T>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a, ta, D);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_d(const Q4AttnArgs& a, const Q4Plan& p, const TileArgs& ta, hipStream_t s) {
    constexpr int kWide = sizeof(T) == 2 ? 8 : 4;
    switch (a.g.head_dim) {
        case 64: return launch_t<T, 64, 8>(a, p, ta, s);
        case 128: return launch_t<T, 128, kWide>(a, p, ta, s);
        default: return launch_t<T, 256, 4>(a, p, ta, s);
    }
}

}  // namespace

int q4_tile_rows(int head_dim, int dtype) { return head_dim == 64 || (head_dim == 128 && dtype != 0) ? 256 : 128; }

hipError_t launch_q4_tiles(const Q4AttnArgs& a, const Q4Plan& p, void* ws, hipStream_t s) {
    TileArgs ta{};
    ta.n_blk = p.n_blk;
    ta.splits = p.splits;
    if (p.splits > 1) {
        ta.o = static_cast<float*>(ws);
        ta.ml = ta.o + (size_t)p.splits * a.n_rows * a.n_q_heads * a.g.head_dim;
    }
    return a.dtype == 0 ? launch_d<float>(a, p, ta, s) : a.dtype == 1 ? launch_d<f16>(a, p, ta, s) : launch_d<bf16>(a, p, ta, s);
}

}  // namespace pi
