// Host walk of the 4-bit cache's layout (csrc/q4.hpp): every byte of a (page, KV head) block belongs to
// exactly one token's code byte or scale, every offset lies inside the block, and the rows of a ragged batch
// stay inside the launch's rows and the page-table row whatever the tables hold.  Needs no GPU.
#include "q4.hpp"

#include <climits>
#include <cstdio>
#include <random>
#include <vector>

static int g_fail = 0;
#define CHECK(c, ...)                       \
    do {                                    \
        if (!(c)) {                         \
            if (++g_fail < 20) {            \
                std::printf(__VA_ARGS__);   \
                std::printf("\n");          \
            }                               \
        }                                   \
    } while (0)

int main() {
    using namespace pi;
    for (int d : {64, 128, 256}) {
        const int nj = d / 32, bytes = (int)q4_block_bytes(d);
        std::vector<int> hit(bytes, 0);
        auto touch = [&](int off, int n, const char* what) {
            CHECK(off >= 0 && off + n <= bytes && off % n == 0, "%s: offset %d of %d bytes, D %d", what, off, n, d);
            if (off < 0 || off + n > bytes) return;
            for (int i = 0; i < n; ++i) ++hit[off + i];
        };
        for (int t = 0; t < 16; ++t) {
            for (int w = 0; w < d / 8; ++w) touch(q4_k_off(d, t, w), 4, "K word");
            for (int j = 0; j < nj; ++j) {
                for (int m = 0; m < 16; ++m) touch(q4_v_off(d, t, j, m), 1, "V byte");
                touch(q4_ks_off(d, t, j), 2, "K scale");
                touch(q4_vs_off(d, t, j), 2, "V scale");
            }
        }
        for (int i = 0; i < bytes; ++i) CHECK(hit[i] == 1, "byte %d of D %d is owned %d times", i, d, hit[i]);
        // what a lane loads: K words (g = lane / 16, t = lane % 16), V words (q, m), scales of its token / its four tokens
        for (int lane = 0; lane < 64; ++lane) {
            const int g = lane >> 4, c = lane & 15;
            for (int j = 0; j < nj; ++j) {
                CHECK(q4_k_off(d, c, 4 * j + g) == lane * 4 * nj + 4 * j, "K word of lane %d", lane);
                CHECK(q4_ks_off(d, c, j) == 16 * d + c * 2 * nj + 2 * j, "K scale of lane %d", lane);
                const int order[4] = {0, 2, 1, 3};
                for (int i = 0; i < 4; ++i) {
                    CHECK(q4_v_off(d, 4 * g + i, j, c) == 8 * d + lane * 4 * nj + 4 * j + i, "V byte of lane %d", lane);
                    CHECK(q4_vs_off(d, 4 * g + order[i], j) == 17 * d + g * 8 * nj + 8 * j + 2 * i, "V scale of lane %d", lane);
                }
            }
        }
    }
    std::mt19937 rng(5);
    const int32_t odd[] = {INT_MIN, INT_MIN + 1, -17, -1, 0, 1, 5, 16, 17, 100, 4096, INT_MAX - 1, INT_MAX};
    auto any = [&] { return odd[rng() % (sizeof odd / sizeof *odd)]; };
    for (int it = 0; it < 200000; ++it) {
        int32_t ts[4], pos[3];
        for (auto& x : ts) x = any();
        for (auto& x : pos) x = any();
        const int n_rows = rng() % 40, max_tok = rng() % 40, max_pages = 1 + rng() % 300;
        for (int b = 0; b < 3; ++b) {
            const Q4Rows r = q4_rows(ts, pos, b, n_rows, max_tok, max_pages);
            CHECK(r.first >= 0 && r.n >= 0 && r.n <= max_tok && r.first + r.n <= n_rows, "rows %d + %d of %d", r.first, r.n, n_rows);
            CHECK(r.start >= 0 && r.len >= 0 && r.len <= 16 * max_pages, "length %d of %d pages", r.len, max_pages);
            CHECK((r.len == 0) == (r.n == 0), "%d rows over %d keys", r.n, r.len);
            const Q4Rows o = q4_rows(nullptr, pos, b, 3, 1, max_pages);
            CHECK(o.first == b && o.n == 1 && o.len >= 0 && o.len <= 16 * max_pages && o.start == o.len - 1, "decode row %d", b);
        }
    }
    std::printf("test_q4_layout: %d failures\n", g_fail);
    return g_fail ? 1 : 0;
}
