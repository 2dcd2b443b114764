// q4_attn.hip -- attention over the 4-bit paged cache for few rows a KV head (gfx950): one token a sequence
// (decode), or a short chunk.  Split over the keys, balanced over a ragged batch.
//
// Work: rows = (token, query head) of one KV head ride in the MFMA columns, 16 to a column block and
// up to 4 blocks to a wavefront, so a K / V code is dequantised once for up to 64 rows.  Per pair of 16-token pages
//   S^T[16 tok x 16 rows] = K[16 x D] . Q^T[D x 16]           (v_mfma_f32_16x16x32_f16, a page each)
//   O^T[D x 16]          += V^T[D x 32 tok] . P^T[32 x 16]    (the same instruction, both pages at once)
// A lane's scores are tokens 4 (lane / 16) + r of its column, and the V words are laid out so that exactly
// these tokens are the lane's share of V^T (q4.hpp): P never crosses lanes.
//
// Rounding: K and V values are exact in f16, f16 / bf16 queries too (bf16 and f32 rows are first scaled by a power
// of two, so that no exponent leaves f16).  P goes to f16 (2^-12 relative, below the rounding of a
// 16-bit output).  f32 queries and their P are split into two f16 (22 bits) and multiplied twice.  The scale is
// applied to the f32 scores.
//
// Bound: a long context by HBM (18 D bytes a page and KV head) with the dequantisation, about 1.5 VALU instructions
// a code, beside it: 32 ragged sequences of 1k to 32k tokens, 32 / 8 heads, D 128, f16 102-106 us (523 MB, 5.0 TB/s, what a
// large copy reaches; the loads alone 97-99, the arithmetic alone on pages in the L2 90); 8 of 64k, 16 / 2 heads, D 256, bf16
// 59-60 (302 MB, 5.1 TB/s).  A few drafted tokens a sequence by the VALU, half of the SIMDs' cycles, at two wavefronts a
// SIMD: 8 sequences of 1 to 8 rows over 2k to 16k tokens, 32 / 8 heads 36 us (97 MB, 2.7 TB/s).  A short context by a launch
// and round trips: 512 tokens, 32 heads, f32 8.9 us.  The merge: 4 to 6 us.
//
// Schedule: decode_sched.hpp's items (pages of one (sequence, KV head, row block) segment), an equal contiguous range
// to each of a persistent grid's workgroups; a segment inside one workgroup is written at once,
// others leave (max, sum, O) for q4_merge_kernel.  Short segments are a workgroup each instead, and no merge follows (q4_plan).
#include "pi_device.hpp"
#include "q4_launch.hpp"

#include <algorithm>
#include <type_traits>

namespace pi {
namespace {

constexpr int kWaves = sched::kWaves;
constexpr int kThreads = 64 * kWaves;
constexpr float kLazy = 8.0f;     // log2 headroom before the running max moves
constexpr int kMaxRuns = 1024;    // runs of one segment the merge stages
constexpr int kStage = 1024;      // most floats a wavefront stages at a time for the merge in LDS
constexpr int kMaxSplits = 32;    // key splits of a tiled row block
// Rows of a KV head past which the tiled kernel runs.  8 sequences over 8000 tokens, 32 / 8 heads, this kernel against the
// tiled one, us: 32 rows, D 128, f16 37, 53, f32 52, 88; 64 rows 67, 56 and 70, 91; 80 rows 87, 59 and 102, 93.
constexpr int kTileRows = 64;
// Grid workgroups a segment from which segments are cut into pieces of their own.  (From 2: pieces of ragged segments
// differ by up to twice; 32 sequences of 1k to 32k tokens, 8 KV heads, 158 us against 110.)
constexpr int kAlign = 8;
constexpr int kItemPages = 16;    // pages of a work item

// Pages on their way: each wavefront keeps a ring of whole (page, KV head) blocks in LDS, filled by direct loads
// (no registers, no LDS stores) several pages ahead of the pair it works on.
template <int D>
struct Ring {
    static constexpr int kBytes = 18 * D;                       // a block, copied as it lies
    static constexpr int kWide = kBytes / 1024, kNarrow = (kBytes % 1024 + 255) / 256;  // 16- and 4-byte loads of 64 lanes
    static constexpr int kSlot = kWide * 1024 + kNarrow * 256;  // D 64: the last load reads half a load past the block
    static constexpr int kLoads = kWide + kNarrow;
    // Slots: a pair at work, the others in flight.  The LDS then holds two (D 256) or three workgroups a CU, as the registers do.
    static constexpr int kPages = D == 256 ? 4 : D == 128 ? 5 : 8;
};

static_assert(kStage * 4 <= Ring<64>::kPages * Ring<64>::kSlot && kStage * 4 <= Ring<256>::kPages * Ring<256>::kSlot, "O is staged in the rings");

// A block into a slot: its bytes in order, 16 (the rest: 4) a lane and load.  An instruction's offset counts for
// both addresses.  From assembly so that the compiler adds no waits before LDS reads of other slots; M0 (the
// destination) is saved, blk and dst are wave-uniform, and the wavefront's reads of the slot are done first.
template <int D>
__device__ __forceinline__ void load_block(const char* blk, uint32_t dst, uint32_t lane16, uint32_t lane4) {
    uint32_t saved;
    if constexpr (D == 64)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\t"
                     "global_load_lds_dwordx4 %1, %3\n\t"
                     "global_load_lds_dword %2, %3 offset:0x400\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(saved) : "v"(lane16), "v"(lane4), "s"(blk), "s"(dst) : "memory");
    else if constexpr (D == 128)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\t"
                     "global_load_lds_dwordx4 %1, %3\n\t"
                     "global_load_lds_dwordx4 %1, %3 offset:0x400\n\t"
                     "global_load_lds_dword %2, %3 offset:0x800\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(saved) : "v"(lane16), "v"(lane4), "s"(blk), "s"(dst) : "memory");
    else
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\t"
                     "global_load_lds_dwordx4 %1, %3\n\t"
                     "global_load_lds_dwordx4 %1, %3 offset:0x400\n\t"
                     "global_load_lds_dwordx4 %1, %3 offset:0x800\n\t"
                     "global_load_lds_dwordx4 %1, %3 offset:0xc00\n\t"
                     "s_mov_b32 m0, %5\n\t"
                     "global_load_lds_dword %2, %6\n\t"
                     "global_load_lds_dword %2, %6 offset:0x100\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(saved) : "v"(lane16), "v"(lane4), "s"(blk), "s"(dst), "s"(dst + 4096), "s"(blk + 4096) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// A page of one KV head as a lane holds it.
template <int D>
struct Page {
    static constexpr int NJ = D / kQ4Group;
    Words<NJ> k, v;
    Words<NJ / 2> ks;   // K scales of token lane % 16, group j in half j % 2 of word j / 2
    Words<2 * NJ> vs;   // V scales of the lane's four tokens: (t0, t2), (t1, t3) of group j
    __device__ __forceinline__ void load(const char* blk, int lane) {
        k.load(blk + lane * (4 * NJ));
        v.load(blk + 8 * D + lane * (4 * NJ));
        ks.load(blk + 16 * D + (lane & 15) * (2 * NJ));
        vs.load(blk + 17 * D + (lane >> 4) * (8 * NJ));
    }
};

__device__ __forceinline__ int head_of(int kvh, int c, int n_kv, int group, int mode) {
    return mode == 0 ? kvh + c * n_kv : kvh * group + c;
}

// Row r of a KV head's rows: token r / group, head r % group; the element offset of its first channel
// in q / gate / out, or -1.
__device__ __forceinline__ long long row_offset(const Q4AttnArgs& a, const Q4Rows& rw, int kvh, int r, int D) {
    const int t = r / a.group, c = r - t * a.group;
    if (t >= rw.n) return -1;
    const int h = head_of(kvh, c, a.g.n_kv_heads, a.group, a.gqa_mode);
    if (h >= a.n_q_heads) return -1;
    return ((long long)(rw.first + t) * a.n_q_heads + h) * D;
}

__device__ __forceinline__ float sigmoidf_(float x) { return 1.0f / (1.0f + expf(-x)); }

__device__ __forceinline__ Q4Rows rows_of(const Q4AttnArgs& a, int b) {
    Q4Rows r = q4_rows(a.tok_start, a.pos, b, a.n_rows, a.max_tok, a.use_pages);
    return r;
}

template <typename T>
__device__ __forceinline__ void load8f(const T* p, float* x) {
    constexpr int W = 16 / sizeof(T);
    typedef T tv __attribute__((ext_vector_type(W)));
#pragma unroll
    for (int j = 0; j < 8 / W; ++j) {
        const tv r = *reinterpret_cast<const tv*>(p + W * j);
#pragma unroll
        for (int i = 0; i < W; ++i) x[W * j + i] = to_f32(r[i]);
    }
}

// Query operand of one 16-row block: channels 32 j + 8 grp + e of the lane's row, scaled by 2^-ex.
template <typename T, int D>
struct Query {
    static constexpr int NJ = D / kQ4Group, PREC = std::is_same<T, float>::value ? 2 : 1;
    f16x8 r[PREC][NJ];
    // returns the factor from a raw product to log2 units, above 0
    __device__ __forceinline__ float load(const T* q, long long off, int grp, float scale) {
        float x[8 * NJ];
        const T* p = q + (off < 0 ? 0 : off) + 8 * grp;
#pragma unroll
        for (int j = 0; j < NJ; ++j) load8f(p + 32 * j, x + 8 * j);
        float f = 1.f, back = scale * kLog2e;
        if (!std::is_same<T, f16>::value) {
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < 8 * NJ; ++i) mx = fmaxf(mx, fabsf(x[i]));
            mx = wave_max_xor(mx, 16);
            mx = wave_max_xor(mx, 32);
            // the row's largest magnitude to [1, 2)
            const int ex = (int)((__builtin_bit_cast(uint32_t, mx) >> 23) & 255u) - 127;
            const int e1 = mx > 0.f && ex > -127 && ex < 127 ? ex : 0;
            f = __builtin_bit_cast(float, (uint32_t)(127 - e1) << 23);
            back = ldexpf(back, e1);
        }
        // A negative scale turns the row instead, and one of 0 stays above it (all scores as good as equal, masks -inf): the
        // largest raw product is the largest score.
        if (back < 0.f) {
            f = -f;
            back = -back;
        }
        if (back < 1e-30f) back = 1e-30f;
        if (off < 0) f = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = off < 0 ? 0.f : x[8 * j + e] * f;
                const f16 h = to_f16(y);
                r[0][j][e] = h;
                if (PREC == 2) r[PREC - 1][j][e] = to_f16(y - (float)h);
            }
        return back;
    }
};

template <int D, int NCB>
struct Acc {
    f32x4 o[NCB][D / 16];
    float m[NCB], l[NCB];
};

// Two pages: scores, softmax, values.  lim[cb]: keys below it are seen by the lane's row; tok0[u]: first token
// of page u; edge: some row's limit may fall inside (then tokens are compared).
// N: the row blocks that hold rows, of NCB.
template <typename T, int D, int NCB, int N>
__device__ __forceinline__ void process(Acc<D, NCB>& acc, const Page<D>* pg, const Query<T, D>* q, const float* back, const int* lim,
                                        const int* tok0, bool edge, int grp, const Q4Magic& mg) {
    constexpr int NJ = D / kQ4Group, PREC = Query<T, D>::PREC;
    f32x4 s[2][N];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int cb = 0; cb < N; ++cb) s[u][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const f16x2 sc = __builtin_bit_cast(f16x2, pg[u].ks.w[j / 2]);
            const f16x8 kf = deq_k(pg[u].k.w[j], sc[j & 1], mg);
#pragma unroll
            for (int cb = 0; cb < N; ++cb)
#pragma unroll
                for (int h = 0; h < PREC; ++h)
                    s[u][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[cb].r[h][j], s[u][cb], 0, 0, 0);
        }
    }
    f16x8 pb[N][PREC];
#pragma unroll
    for (int cb = 0; cb < N; ++cb) {
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (edge) {
                const int left = lim[cb] - tok0[u] - 4 * grp;  // tokens of the lane's four that count
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (r >= left) s[u][cb][r] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[u][cb][r]);
        }
        mx *= back[cb];
        if (__any(mx > acc.m[cb] + kLazy)) {
            mx = wave_max_xor(mx, 16);
            mx = wave_max_xor(mx, 32);
            const float m_new = fmaxf(acc.m[cb], mx);
            const float alpha = fast_exp2(acc.m[cb] - m_new);
            acc.l[cb] *= alpha;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) acc.o[cb][t] *= alpha;
            acc.m[cb] = m_new;
        }
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) p[r] = fast_exp2(fmaf(s[u][cb][r], back[cb], -acc.m[cb]));
            sum += (p[0] + p[1]) + (p[2] + p[3]);
            const float pv[4] = {p[0], p[2], p[1], p[3]};  // the order of the V codes
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f16 h = to_f16(pv[r]);
                pb[cb][0][4 * u + r] = h;
                if (PREC == 2) pb[cb][PREC - 1][4 * u + r] = to_f16(pv[r] - (float)h);
            }
        }
        acc.l[cb] += sum;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const f16x2 a0 = __builtin_bit_cast(f16x2, pg[0].vs.w[2 * j]), b0 = __builtin_bit_cast(f16x2, pg[0].vs.w[2 * j + 1]);
        const f16x2 a1 = __builtin_bit_cast(f16x2, pg[1].vs.w[2 * j]), b1 = __builtin_bit_cast(f16x2, pg[1].vs.w[2 * j + 1]);
        const f16 off = (f16)-72.0f;
        const f16x2 oa0 = a0 * off, ob0 = b0 * off, oa1 = a1 * off, ob1 = b1 * off;
        const uint32_t w0 = pg[0].v.w[j], w1 = pg[1].v.w[j];
        const f16x8 lo = join4(deq_pair(w0 << 4, a0, oa0, mg), deq_pair(w0 >> 4, b0, ob0, mg), deq_pair(w1 << 4, a1, oa1, mg),
                               deq_pair(w1 >> 4, b1, ob1, mg));
        const f16x8 hi = join4(deq_pair(w0, a0, oa0, mg), deq_pair(w0 >> 8, b0, ob0, mg), deq_pair(w1, a1, oa1, mg),
                               deq_pair(w1 >> 8, b1, ob1, mg));
#pragma unroll
        for (int cb = 0; cb < N; ++cb)
#pragma unroll
            for (int h = 0; h < PREC; ++h) {
                acc.o[cb][2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pb[cb][h], acc.o[cb][2 * j], 0, 0, 0);
                acc.o[cb][2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pb[cb][h], acc.o[cb][2 * j + 1], 0, 0, 0);
            }
    }
}

struct Q4Ws {
    float* o;       // [slot][cols][D]
    float* ml;      // [slot][cols][2]
    int32_t* runs;  // [segment][2]
};

// Prefix sums of the sequences' items into s_cum; returns their total.
// (of each count divided by `per`, rounded up, where per > 1).
__device__ __forceinline__ int scan_items(const Q4AttnArgs& a, int* s_cum, int* s_red, int per) {
    const int tid = threadIdx.x;
    int carry = 0;
    for (int base = 0; base < a.batch; base += kThreads) {
        const int b = base + tid;
        const int n = b < a.batch ? (sched::items_of(rows_of(a, b).len, a.item_pages) + per - 1) / per : 0;
        int x = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o, 64);
            if ((tid & 63) >= o) x += y;
        }
        if ((tid & 63) == 63) s_red[tid >> 6] = x;
        __syncthreads();
        int wsum = 0;
        for (int w = 0; w < (tid >> 6); ++w) wsum += s_red[w];
        const int incl = carry + wsum + x;
        if (b < a.batch) s_cum[b] = incl - n;
        carry += s_red[0] + s_red[1] + s_red[2] + s_red[3];
        __syncthreads();
    }
    if (tid == 0) s_cum[a.batch] = carry;
    __syncthreads();
    return carry;
}

struct LenOf {
    const Q4AttnArgs& a;
    __device__ __forceinline__ int operator()(int b) const { return rows_of(a, b).len; }
};

// Two wavefronts a SIMD where the rows' registers allow it.
template <typename T, int D, int NCB>
constexpr int min_waves() { return NCB * D * (sizeof(T) == 4 ? 3 : 2) <= 512 ? 2 : 1; }

// WHOLE: no merge follows.  Workgroup i takes segments i, i + grid, .. whole, and the schedule's scan of the batch (three trips to
// memory and back before a first page is asked for) is not needed.
template <typename T, int D, int NCB, bool WHOLE>
__global__ __launch_bounds__(kThreads, (min_waves<T, D, NCB>())) void q4_attn_kernel(Q4AttnArgs a, Q4Ws ws, int stage) {
    typedef Ring<D> R;
    // the wavefronts' rings, then s_cum[batch + 1]; the rings' space also stages O: [4][stage] floats
    extern __shared__ __attribute__((aligned(16))) char s_dyn[];
    __shared__ int s_red[4];
    __shared__ float s_m[kWaves][16 * NCB];
    __shared__ float s_l[kWaves][16 * NCB];
    float* s_o = reinterpret_cast<float*>(s_dyn);
    int* s_cum = reinterpret_cast<int*>(s_dyn + kWaves * R::kPages * R::kSlot);

    const Q4Magic mg;
    const int n_kv = a.g.n_kv_heads, n_seg = n_kv * a.n_cb, tid = threadIdx.x;
    const int segs = a.batch * n_seg;
    int chunk = 1, piece = 0, cur = blockIdx.x, end = segs;
    if constexpr (!WHOLE) {
        int n_items = n_seg * scan_items(a, s_cum, s_red, 1);
        chunk = (n_items + gridDim.x - 1) / gridDim.x;
        // Few segments for the grid: each is cut into pieces of its own instead, a piece a workgroup, so that none pays the
        // start and the end of two runs.  Pieces of `piece` items number at most the grid.
        if (segs * kAlign <= (int)gridDim.x) {
            piece = max(1, (n_items + (int)gridDim.x - segs - 1) / ((int)gridDim.x - segs));
            __syncthreads();
            n_items = n_seg * scan_items(a, s_cum, s_red, piece);
            chunk = 1;  // s_cum counts pieces now
        }
        cur = blockIdx.x * chunk;
        end = min(n_items, cur + chunk);
    }
    if (cur >= end) return;

    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const size_t blk_bytes = q4_block_bytes(D);
    const char* ring = s_dyn + wave * (R::kPages * R::kSlot);
    const uint32_t lane16 = lane * 16, lane4 = lane * 4;
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)ring);

    int b = WHOLE ? 0 : sched::find_seq(s_cum, a.batch, n_seg, cur);
    while (cur < end) {
        sched::Run run;
        int pid_first = 0;  // WHOLE: the wavefront's page ids, asked for together with the length
        if constexpr (WHOLE) {
            b = cur / n_seg;
            pid_first = a.page_table[(size_t)b * a.max_pages + min(wave + kWaves * lane, a.use_pages - 1)];
            run.b = b;
            run.kvh = cur - b * n_seg;
            run.seg0 = cur;
            run.run_end = cur + gridDim.x;
            run.len = rows_of(a, b).len;
            run.pg0 = 0;
            run.pg1 = (run.len + sched::kPage - 1) / sched::kPage;
            run.whole = true;
        } else {
            run = sched::run_of(s_cum, LenOf{a}, n_seg, a.item_pages, b, cur, end);
            b = run.b;
        }
        if (piece) {  // the segment's pages in equal pieces
            const int k = s_cum[b + 1] - s_cum[b], pages = (run.len + sched::kPage - 1) / sched::kPage;
            const int i = cur - run.seg0, each = (pages + k - 1) / k;
            run.pg0 = min(pages, i * each);
            run.pg1 = min(pages, run.pg0 + each);
        }
        const int sidx = run.kvh, kvh = sidx / a.n_cb, row0 = (sidx % a.n_cb) * a.cols;
        const Q4Rows rw = rows_of(a, b);
        const size_t seg = (size_t)b * n_seg + sidx;
        if (cur == run.seg0 && !WHOLE && tid == 0) {
            int wg1;
            const int n_runs = sched::merge_runs(s_cum, n_seg, chunk, b, sidx, &wg1);
            ws.runs[2 * seg] = wg1;
            ws.runs[2 * seg + 1] = n_runs;
        }
        if (row0 >= rw.n * a.group) {  // a row block past the sequence's rows
            cur = run.run_end;
            continue;
        }
        const int first_lim = rw.start + row0 / a.group + 1;  // keys that every row of the block sees
        const int32_t* pt = a.page_table + (size_t)b * a.max_pages;
        Query<T, D> q[NCB];
        Acc<D, NCB> acc;
        float back[NCB];
        int lim[NCB];
        bool have_q = false;
        // 16-row blocks with rows of this sequence (a ragged batch's shorter chunks fill fewer)
        const int live = __builtin_amdgcn_readfirstlane(min(NCB, (rw.n * a.group - row0 + 15) / 16));
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) acc.o[cb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            acc.m[cb] = -1e30f;
            acc.l[cb] = 0.f;
        }
        auto walk = [&](auto blocks) {  // the run's pages for the first N row blocks
            constexpr int N = decltype(blocks)::value;
            for (int sub = run.pg0; sub < run.pg1; sub += sched::kSubPages) {
                int first, n_my;
                sched::sub_pages(sub, run.pg1, wave, &first, &n_my);
                // A page id outside the pool holds no tokens: page 0 is read in its place, all of it masked.
                const int pid_raw = lane >= n_my ? 0 : WHOLE && sub == 0 ? pid_first : pt[first + kWaves * lane];
                const bool bad = !sched::page_ok(pid_raw, a.g.n_pages);
                const int pid_v = bad ? 0 : pid_raw;
                const uint64_t bad_pages = __ballot(bad);
                constexpr int kNone = 0x7fffffc0;  // a page whose tokens are past every limit
                auto issue = [&](int j) {  // page j of the wavefront's into its slot
                    const int pid = __builtin_amdgcn_readlane(pid_v, j);
                    load_block<D>(a.g.base + ((size_t)pid * n_kv + kvh) * blk_bytes, ring_at + (j % R::kPages) * R::kSlot, lane16, lane4);
                };
                for (int j = 0; j < min(n_my, R::kPages); ++j) issue(j);
                if (!have_q) {  // the rows, while the first pages are on their way
                    have_q = true;
#pragma unroll
                    for (int cb = 0; cb < NCB; ++cb) {
                        const int r = cb * 16 + col;
                        const long long off = r < a.cols ? row_offset(a, rw, kvh, row0 + r, D) : -1;
                        back[cb] = q[cb].load(static_cast<const T*>(a.q), off, grp, a.scale);
                        lim[cb] = min(rw.start + (row0 + r) / a.group + 1, rw.len);
                    }
                }
                // pages 2 i and 2 i + 1 have landed; the younger ones may still be under way
                auto landed = [&](int i) {
                    constexpr int kAhead = R::kPages - 2;
                    const int ahead = n_my - 2 * i - 2;  // pages behind the pair
                    if (kAhead >= 6 && ahead >= 6)
                        wait_loads<(kAhead >= 6 ? 6 : 0) * R::kLoads>();
                    else if (kAhead >= 4 && ahead >= 4)
                        wait_loads<(kAhead >= 4 ? 4 : 0) * R::kLoads>();
                    else if (ahead >= 2)
                        wait_loads<2 * R::kLoads>();
                    else
                        wait_loads<0>();
                };
                auto fetch = [&](Page<D>* pg, int i) {  // the pair to registers; a second page that does not exist: the first, masked
#pragma unroll
                    for (int u = 0; u < 2; ++u) pg[u].load(ring + ((2 * i + u < n_my ? 2 * i + u : 2 * i) % R::kPages) * R::kSlot, lane);
                };
                auto run_pair = [&](const Page<D>* pg, int i) {
                    int tok0[2];
                    bool edge = false;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int j = 2 * i + u;
                        const int t = (first + kWaves * j) * sched::kPage;
                        const bool on = j < n_my && !((bad_pages >> j) & 1);
                        tok0[u] = on ? t : kNone;
                        edge = edge || !on || t + sched::kPage > first_lim;
                    }
                    process<T, D, NCB, N>(acc, pg, q, back, lim, tok0, edge, grp, mg);
                };
                auto refill = [&](int i) {  // the pair's slots, once it is in registers
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        if (2 * i + u + R::kPages < n_my) issue(2 * i + u + R::kPages);
                };
                const int n_iter = (n_my + 1) / 2;
                for (int i = 0; i < n_iter; ++i) {
                    Page<D> x[2];
                    landed(i);
                    fetch(x, i);
                    run_pair(x, i);
                    refill(i);
                }
            }
        };
        if (NCB == 2 && D <= 128 && live == 1)  // (a copy of the loop; in one loop the accumulators would be copied)
            walk(std::integral_constant<int, 1>{});
        else
            walk(std::integral_constant<int, NCB>{});
        // ---- the 4 wavefronts' shares meet in LDS, `stage` floats of rows at a time ----
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            acc.l[cb] = wave_sum_xor(acc.l[cb], 16);
            acc.l[cb] = wave_sum_xor(acc.l[cb], 32);
            if (grp == 0) {
                s_m[wave][16 * cb + col] = acc.m[cb];
                s_l[wave][16 * cb + col] = acc.l[cb];
            }
        }
        const size_t slot = (size_t)sched::run_slot(cur == run.seg0, b, sidx, n_seg, a.batch, blockIdx.x);
        __syncthreads();  // (the rings are read no more, either)
        const int rows = min(a.cols, rw.n * a.group - row0);  // of the block that exist in this sequence
        if (tid < rows) {  // each wavefront's weight, and the row's max and sum
            float M = s_m[0][tid], lsum = 0.f;
#pragma unroll
            for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_m[w][tid]);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = fast_exp2(s_m[w][tid] - M);
                lsum += f * s_l[w][tid];
                s_m[w][tid] = f;
            }
            if (!run.whole) {
                ws.ml[(slot * a.cols + tid) * 2] = M;
                ws.ml[(slot * a.cols + tid) * 2 + 1] = lsum;
            }
            s_l[0][tid] = run.whole ? (lsum == 0.f ? 0.f : 1.0f / lsum) : 1.0f;  // every key masked: zeros (a NaN stays)
        }
        const int per = stage / D;  // rows staged at a time: a power of two up to 16
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            for (int c0 = 0; c0 < 16; c0 += per) {
                const int r0 = 16 * cb + c0;  // rows r0 .. r0 + per - 1 of the block
                if (r0 >= rows) break;
                if (col >= c0 && col < c0 + per) {
#pragma unroll
                    for (int t = 0; t < D / 16; ++t)
                        *reinterpret_cast<f32x4*>(&s_o[wave * stage + (col - c0) * D + 16 * t + 4 * grp]) = acc.o[cb][t];
                }
                __syncthreads();
                for (int idx = 4 * tid; idx < per * D; idx += 4 * kThreads) {
                    const int c = idx / D, d = idx - c * D, r = r0 + c;
                    if (r >= rows) break;
                    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) o += s_m[w][r] * *reinterpret_cast<const f32x4*>(&s_o[w * stage + idx]);
                    o *= s_l[0][r];
                    if (!run.whole) {
                        *reinterpret_cast<f32x4*>(&ws.o[(slot * a.cols + r) * D + d]) = o;
                        continue;
                    }
                    const long long off = row_offset(a, rw, kvh, row0 + r, D);
                    if (off < 0) continue;
                    typedef T t4 __attribute__((ext_vector_type(4)));
                    t4 y;
                    if (a.gate && run.len) {  // (rows without keys get zeros)
                        const t4 g = *reinterpret_cast<const t4*>(static_cast<const T*>(a.gate) + off + d);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] *= sigmoidf_(to_f32(g[e]));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(o[e]);
                    *reinterpret_cast<t4*>(static_cast<T*>(a.out) + off + d) = y;
                }
                __syncthreads();
            }
        }
        cur = run.run_end;
    }
}

// Joins the runs of the segments that span several workgroups' ranges and writes zeros for the rows of
// sequences without keys.  A workgroup: 64 V values of one segment; its 4 wavefronts take every 4th run each.  A launch and two
// trips to memory: 4 to 6 us whatever the shape, so short segments go without it.
template <typename T, int V>
__global__ __launch_bounds__(256) void q4_merge_kernel(Q4AttnArgs a, Q4Ws ws, int D) {
    typedef typename std::conditional<V == 4, f32x4, float>::type VT;
    __shared__ float s_w[4][kMaxRuns];
    __shared__ int s_slot[kMaxRuns];
    __shared__ float s_inv[4];
    __shared__ __attribute__((aligned(16))) VT s_acc[4][64];
    const int sidx = blockIdx.y, b = blockIdx.z, n_seg = gridDim.y;
    const int kvh = sidx / a.n_cb, row0 = (sidx % a.n_cb) * a.cols;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int cols = a.cols, GD = cols * D, e0 = blockIdx.x * 64 * V;
    const size_t seg = (size_t)b * n_seg + sidx;
    const Q4Rows rw = rows_of(a, b);
    const int wg1 = ws.runs ? ws.runs[2 * seg] : 0, n_runs = ws.runs ? ws.runs[2 * seg + 1] : 0;
    T* out = static_cast<T*>(a.out);
    const int e = e0 + V * lane;
    const int c = e / D, d = e - c * D;
    const long long off = e < GD ? row_offset(a, rw, kvh, row0 + c, D) : -1;
    if (rw.len == 0) {  // a softmax over nothing leaves zeros (and the run table was not written)
        if (wave == 0 && off >= 0)
            for (int i = 0; i < V; ++i) out[off + d + i] = from_f32<T>(0.f);
        return;
    }
    if (row0 >= rw.n * a.group || n_runs <= 1) return;
    for (int r = tid; r < n_runs; r += 256) s_slot[r] = (int)sched::run_slot(r == 0, b, sidx, n_seg, a.batch, wg1 + r - 1);
    __syncthreads();
    const int c_lo = e0 / D, c_hi = min(cols - 1, (e0 + 64 * V - 1) / D);
    constexpr int kPre = 4;
    const bool on = off >= 0;  // partials of rows that do not exist were not written
    const float* po = ws.o + (on ? e : 0);
    auto part = [&](int r) { return *reinterpret_cast<const VT*>(po + (size_t)s_slot[r] * GD); };
    const VT zero = VT{};
    VT pre[kPre];
#pragma unroll
    for (int j = 0; j < kPre; ++j) {
        const int r = wave + 4 * j;
        pre[j] = r < n_runs ? part(r) : zero;
    }
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2* pml = reinterpret_cast<const f2*>(ws.ml);
    if (wave <= c_hi - c_lo) {  // a wavefront a row of this block
        const int cc = c_lo + wave;
        const f2 ml0 = lane < n_runs ? pml[(size_t)s_slot[lane] * cols + cc] : f2{-1e30f, 0.f};
        float M = ml0[0];
        for (int r = lane + 64; r < n_runs; r += 64) M = fmaxf(M, pml[(size_t)s_slot[r] * cols + cc][0]);
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) M = wave_max_xor(M, m);
        float lsum = 0.f;
        if (lane < n_runs) {
            const float w = fast_exp2(ml0[0] - M);
            s_w[wave][lane] = w;
            lsum = w * ml0[1];
        }
        for (int r = lane + 64; r < n_runs; r += 64) {
            const f2 ml = pml[(size_t)s_slot[r] * cols + cc];
            const float w = fast_exp2(ml[0] - M);
            s_w[wave][r] = w;
            lsum += w * ml[1];
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) lsum = wave_sum_xor(lsum, m);
        if (lane == 0) s_inv[wave] = lsum == 0.f ? 0.f : 1.0f / lsum;
    }
    __syncthreads();
    const int cw = (on ? c : c_lo) - c_lo;
    const float* w = s_w[cw];
    VT sum = zero;
#pragma unroll
    for (int j = 0; j < kPre; ++j) {
        const int r = wave + 4 * j;
        if (r < n_runs) sum += w[r] * pre[j];
    }
    for (int r = wave + 4 * kPre; r < n_runs; r += 4) sum += w[r] * part(r);
    s_acc[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || off < 0) return;
    VT res = ((s_acc[0][lane] + s_acc[1][lane]) + (s_acc[2][lane] + s_acc[3][lane])) * s_inv[cw];
    const float* rp = reinterpret_cast<const float*>(&res);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float y = rp[i];
        if (a.gate) y *= sigmoidf_(to_f32(static_cast<const T*>(a.gate)[off + d + i]));
        out[off + d + i] = from_f32<T>(y);
    }
}

template <typename T, int D, int NCB>
int vgpr_wgs() {  // resident workgroups a CU by registers alone
    static const int n = [] {
        int v = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, q4_attn_kernel<T, D, NCB, false>, kThreads, 0) != hipSuccess || v <= 0) v = 1;
        return v;
    }();
    return n;
}
// Row blocks of a wavefront, at most: what fits the registers of one wavefront a SIMD.
template <typename T>
constexpr int max_ncb(int d) { return (d == 256 ? 2 : 4) / (sizeof(T) == 4 && d != 64 ? 2 : 1); }

template <typename T>
int wgs_of(int d, int ncb) {
    constexpr int M256 = max_ncb<T>(256), M128 = max_ncb<T>(128);
    if (d == 256) return ncb == 1 ? vgpr_wgs<T, 256, 1>() : vgpr_wgs<T, 256, M256>();
    if (d == 128) return ncb == 1 ? vgpr_wgs<T, 128, 1>() : ncb == 2 ? vgpr_wgs<T, 128, 2>() : vgpr_wgs<T, 128, M128>();
    return ncb == 1 ? vgpr_wgs<T, 64, 1>() : ncb == 2 ? vgpr_wgs<T, 64, 2>() : vgpr_wgs<T, 64, 4>();
}

size_t ring_bytes(int d) {
    return kWaves * (d == 64 ? (size_t)Ring<64>::kPages * Ring<64>::kSlot
                             : d == 128 ? (size_t)Ring<128>::kPages * Ring<128>::kSlot : (size_t)Ring<256>::kPages * Ring<256>::kSlot);
}
int stage_floats(int cols, int d) {  // rows staged at a time: a power of two, at most 16
    int per = std::min(16, kStage / d);
    while (per > 1 && per / 2 >= cols) per /= 2;
    return per * d;
}

template <typename T, int D, int NCB, bool WHOLE>
hipError_t launch_w(const Q4AttnArgs& a, const Q4Plan& plan, void* wsp, hipStream_t s) {
    Q4Ws ws{};
    if (plan.merge) {
        ws.o = static_cast<float*>(wsp);
        ws.ml = ws.o + (size_t)plan.n_slots * a.cols * D;
        ws.runs = reinterpret_cast<int32_t*>(ws.ml + (size_t)plan.n_slots * a.cols * 2);
    }
    const int stage = stage_floats(a.cols, D);
    const size_t lds = ring_bytes(D) + (plan.merge ? (size_t)(a.batch + 1) * 4 : 0);
    if (lds > (64 << 10)) {
        static std::atomic<uint64_t> on{0};
        const hipError_t e =
            allow_lds(reinterpret_cast<const void*>(&q4_attn_kernel<T, D, NCB, WHOLE>), ring_bytes(D) + (kQ4MaxBatch + 1) * 4, on);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((q4_attn_kernel<T, D, NCB, WHOLE>), dim3(plan.grid), dim3(kThreads), lds, s, a, ws, stage);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (plan.merge) {
        const int n_seg = a.g.n_kv_heads * a.n_cb;
        // 256 values a workgroup, or 64 where that leaves few workgroups (8 sequences of 64k, 2 KV heads, D 256: the
        // whole step 78.2, 77.5 us; with many 64 lose: 64 sequences of 4000, 8 KV heads, D 128 73.4, 77.4)
        const long long wg4 = (long long)((a.cols * D + 255) / 256) * n_seg * a.batch;
        if (wg4 >= 256)
            hipLaunchKernelGGL((q4_merge_kernel<T, 4>), dim3((a.cols * D + 255) / 256, n_seg, a.batch), dim3(256), 0, s, a, ws, D);
        else
            hipLaunchKernelGGL((q4_merge_kernel<T, 1>), dim3((a.cols * D + 63) / 64, n_seg, a.batch), dim3(256), 0, s, a, ws, D);
    }
    return hipGetLastError();
}

template <typename T, int D, int NCB>
hipError_t launch_t(const Q4AttnArgs& a, const Q4Plan& p, void* ws, hipStream_t s) {
    return p.merge ? launch_w<T, D, NCB, false>(a, p, ws, s) : launch_w<T, D, NCB, true>(a, p, ws, s);
}

template <typename T>
hipError_t launch_d(const Q4AttnArgs& a, const Q4Plan& p, void* ws, hipStream_t s) {
    constexpr int M256 = max_ncb<T>(256), M128 = max_ncb<T>(128);
    const int d = a.g.head_dim;
    if (d == 256) return p.ncb == 1 ? launch_t<T, 256, 1>(a, p, ws, s) : launch_t<T, 256, M256>(a, p, ws, s);
    if (d == 128)
        return p.ncb == 1   ? launch_t<T, 128, 1>(a, p, ws, s)
               : p.ncb == 2 ? launch_t<T, 128, 2>(a, p, ws, s)
                            : launch_t<T, 128, M128>(a, p, ws, s);
    return p.ncb == 1 ? launch_t<T, 64, 1>(a, p, ws, s) : p.ncb == 2 ? launch_t<T, 64, 2>(a, p, ws, s) : launch_t<T, 64, 4>(a, p, ws, s);
}

}  // namespace

Q4Plan q4_plan(Q4AttnArgs& a, int device) {
    Q4Plan p{};
    const int d = a.g.head_dim, n_kv = a.g.n_kv_heads;
    a.group = a.gqa_mode == 0 ? (a.n_q_heads + n_kv - 1) / n_kv : a.n_q_heads / n_kv;
    const long long rows = (long long)a.group * std::max(a.max_tok, 1);  // of a KV head, at most
    int cus = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || cus <= 0) cus = 256;
    if (rows > kTileRows) {
        const int per = q4_tile_rows(d, a.dtype);
        const long long n_blk = (rows + per - 1) / per, wgs = n_blk * n_kv * a.batch;
        p.tiles = true;
        // Few row blocks: their keys are split while that fills idle CUs and each part keeps 4 tiles.  (40 rows over 16000 keys,
        // 32 / 8 heads, D 128: 8 parts 67 us, 32 35.  Parts of 2 tiles: a prompt of 512 at D 64 16.2, 17.5 us, at D 128 29.2,
        // 29.5, at D 256 34.0, 32.0; more parts than CUs: three prompts of 300 to 1200 at D 64 24.1, 29.0.)
        // Of a ragged batch's row blocks no more exist than its rows fill, and one more a sequence.  (7 chunks of up to 349 tokens
        // over up to 6900, f32 D 256, 5 / 1 heads: 264 us with the grid's count, 148 with this.)
        const long long blocks = n_kv * std::min<long long>(n_blk * a.batch, (long long)a.n_rows * a.group / per + a.batch);
        long long splits = std::min<long long>({kMaxSplits, cus / blocks, a.use_pages / 16});
        splits = std::max<long long>(splits, 1);
        // (a merge of mostly rows of no sequence may be more threads than a launch takes)
        if ((long long)a.n_rows * a.n_q_heads * (d / 4) >= 1ll << 32) splits = 1;
        p.splits = (int)splits;
        p.n_blk = (int)n_blk;
        p.grid = wgs * splits * 512 >= 1ll << 32 ? 0 : (int)(wgs * splits);  // a launch's most threads; 0: the caller refuses
        p.merge = splits > 1;
        p.ws_bytes = p.merge ? (size_t)splits * a.n_rows * a.n_q_heads * (d + 2) * 4 : 0;
        return p;
    }
    const int most = a.dtype == 0 ? max_ncb<float>(d) : max_ncb<f16>(d);
    const long long blocks = (rows + 15) / 16;
    p.ncb = blocks >= most ? most : blocks == 3 ? 4 : (int)blocks;
    a.n_cb = (int)((rows + 16 * p.ncb - 1) / (16 * p.ncb));
    a.cols = (int)std::min<long long>(rows, 16 * p.ncb);
    const int n_seg = n_kv * a.n_cb;
    const int regs = a.dtype == 0 ? wgs_of<float>(d, p.ncb) : a.dtype == 1 ? wgs_of<f16>(d, p.ncb) : wgs_of<bf16>(d, p.ncb);
    const size_t lds = ring_bytes(d) + (size_t)(a.batch + 1) * 4 + 2048;
    const int per_cu = std::max(1, std::min<int>(regs, (int)((160 << 10) / lds)));
    p.grid = std::min(cus * per_cu, kMaxRuns - 1);
    // Items of 16 pages, four for each wavefront: in smaller ones the wavefronts work on half pairs and the merge joins
    // more runs (one sequence of 4000 tokens, D 256, 2 KV heads: 36 us with single pages, 16 with 16).  With 2 to 8
    // items a workgroup the last one weighs, and 8 pages are better (16 sequences of 2000, 32 KV heads: 40 against
    // 41.6 us); below, 8 lose to 16 (one of 32k, 8 KV heads: 25.8 against 22.9).
    const long long items = (long long)a.batch * n_seg * a.use_pages / kItemPages;
    int ip = items >= 2LL * p.grid && items < 8LL * p.grid ? kItemPages / 2 : kItemPages;
    // A short segment is read whole by one workgroup in less time than the runs of several and their merge take, a longer
    // one too where segments fill the chip by themselves.  Cut against whole, 16-bit rows, us:
    //   8 KV heads, D 128:  1 sequence of 992 tokens (140 KB) 15.9, 11.6; of 2128 (300 KB) 16.4, 18.7
    //                       32 of 3264 (460 KB) 34.5, 29.4, the shortest a quarter as long 28.6, 28.1; of 6400 (900 KB) 39, 49
    //                       256 of 6400 369, 335 and 248, 243; of 12800 (1800 KB) 464, 477
    //   2 KV heads, D 256:  128 of 770 (217 KB) 32, 17; of 1632 (460 KB) 42, 27; 1024 of 3200 (900 KB) 361, 339 and 262, 242
    const long long segs = (long long)a.batch * n_seg;
    const long long whole = segs >= 8LL * cus ? 960 << 10 : segs >= cus ? 480 << 10 : 224 << 10;  // of a segment's pages, at most
    if ((long long)a.use_pages * q4_block_bytes(d) <= whole) ip = std::max(ip, a.use_pages);
    a.item_pages = ip;
    p.merge = a.use_pages > ip;
    p.n_slots = (long long)a.batch * n_seg + p.grid;
    if (!p.merge) p.grid = (int)std::min<long long>(std::max(segs, 1ll), 1 << 20);  // as many workgroups as segments
    if ((long long)a.batch * n_seg * ((a.use_pages + ip - 1) / ip) > 0x7fffffffll || n_seg > 65535) p.grid = 0;  // the caller refuses
    p.ws_bytes = p.merge ? ((size_t)p.n_slots * a.cols * (d + 2) + (size_t)2 * a.batch * n_seg) * 4 : 0;
    return p;
}

hipError_t launch_q4_attn(const Q4AttnArgs& a, const Q4Plan& p, void* ws, hipStream_t s) {
    if (p.tiles) return launch_q4_tiles(a, p, ws, s);
    return a.dtype == 0 ? launch_d<float>(a, p, ws, s) : a.dtype == 1 ? launch_d<f16>(a, p, ws, s) : launch_d<bf16>(a, p, ws, s);
}

}  // namespace pi
