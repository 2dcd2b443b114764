// q4_launch.hpp -- host-side launchers of the rotary plan and the 4-bit cache (rope.hip, q4.hip,
// q4_attn.hip, q4_prefill.hip).  Arguments are validated by the caller (api.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "q4.hpp"

namespace pi {

// Frequencies in turns a position (f / 2 pi, f64) and the factor of cos and sin.
struct RopePlan {
    double* turns;  // device, [half]
    int32_t half;   // rotary pairs
    int32_t layout; // PI_ROPE_PAIRS / PI_ROPE_HALVES
    double mscale;
};

// Element (t, h, d) of a tensor of head rows at p + t * tok + h * head + d.
struct HeadRows {
    void* p;
    int64_t tok, head;
    int32_t n;  // heads
};

struct RopeArgs {
    RopePlan plan;
    HeadRows in[2], out[2];  // q, k (n = 0: absent)
    const int32_t* pos;
    int32_t n_tok, head_dim, dtype;
};
hipError_t launch_rope_apply(const RopeArgs& a, hipStream_t s);

struct Q4AppendArgs {
    Q4Geom g;
    RopePlan plan;            // half = 0: no rotation
    HeadRows q, k, v, q_out;  // q.n = 0: no q
    const float *q_norm, *k_norm;
    float eps;
    const int32_t* tok_start; // null: one row a sequence
    const int32_t* start_pos;
    const int32_t* page_table;
    int32_t max_pages, n_seq, n_rows, dtype;
    uint16_t *k_val, *v_val;  // f16 values [n_rows][Hkv][D], or null
};
hipError_t launch_q4_append(const Q4AppendArgs& a, hipStream_t s);

// Records of positions start .. start + n - 1 of one page-table row: codes [n][Hkv][D / 2] (even
// channel low), scales [n][Hkv][D / 32] f16 bits.
hipError_t launch_q4_records(const Q4Geom& g, bool write, const int32_t* row, int32_t max_pages, int32_t start, int32_t n_tok,
                             uint8_t* kc, uint16_t* ks, uint8_t* vc, uint16_t* vs, hipStream_t s);

constexpr int kQ4MaxBatch = 4096;

struct Q4AttnArgs {
    Q4Geom g;
    const void *q, *gate;
    void* out;
    int32_t dtype;
    const int32_t* page_table;
    const int32_t* tok_start;  // null: decode (one row a sequence, pos holds context lengths)
    const int32_t* pos;        // start positions, or context lengths
    int32_t max_pages;         // columns of the page table
    int32_t use_pages;         // pages that any sequence uses at most (<= max_pages)
    int32_t batch, n_rows, max_tok, n_q_heads, gqa_mode;
    float scale;
    // set by q4_plan:
    int32_t group;       // query heads of a KV head (columns past n_q_heads are off)
    int32_t cols;        // rows (token, head) of a segment
    int32_t n_cb;        // segments a KV head
    int32_t item_pages;  // pages a work item
};

struct Q4Plan {
    bool tiles;          // the LDS-tiled kernel (many rows), else the column kernel
    int32_t grid, ncb;   // column kernel: workgroups, 16-row column blocks a segment
    int32_t splits;      // tiled kernel: key splits of a row block,
    int32_t n_blk;       // and row blocks of a sequence and KV head, at most
    bool merge;          // a second launch joins partials
    long long n_slots;
    size_t ws_bytes;
};
// Lets a kernel ask for more than 64 KB of LDS, on every device it runs on: `on` has a bit for each where it may.
inline hipError_t allow_lds(const void* kernel, size_t bytes, std::atomic<uint64_t>& on) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e != hipSuccess || (on.load(std::memory_order_relaxed) & bit)) return e;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess) on.fetch_or(bit, std::memory_order_relaxed);
    return e;
}
// Fills a's planned fields.
Q4Plan q4_plan(Q4AttnArgs& a, int device);
hipError_t launch_q4_attn(const Q4AttnArgs& a, const Q4Plan& plan, void* ws, hipStream_t s);
// Rows of a tiled workgroup.
int q4_tile_rows(int head_dim, int dtype);
hipError_t launch_q4_tiles(const Q4AttnArgs& a, const Q4Plan& plan, void* ws, hipStream_t s);

}  // namespace pi
