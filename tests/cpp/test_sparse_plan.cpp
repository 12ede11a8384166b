// CPU tests of the launch plans of the selection and of the attention over listed blocks
// (rllm_amd/csrc/sparse_plan.h): whatever the sizes, launches are within a device's limit of
// threads, scratch within what was asked for, and what the kernel keeps in LDS fits.
//
// usage: test_sparse_plan      (exit status 0 = all passed)
#include "../../rllm_amd/csrc/sparse_plan.h"

#include <cstdio>
#include <initializer_list>

using namespace rllm;

static int g_failures = 0;
static void check(bool ok, const char* what, const SparseShape& s, const SparsePlan& p) {
    if (ok) return;
    if (++g_failures <= 10)
        std::fprintf(stderr, "FAILED %s: rows %lld hq %lld hkv %lld d %d bs %d maxb %lld k %lld: tile %d list %d waves %d splits %d\n",
                     what, (long long)s.rows, (long long)s.hq, (long long)s.hkv, s.d, 1 << s.bs_log2, (long long)s.maxb,
                     (long long)s.k, p.tile, p.list, p.waves, p.splits);
}

static void selection() {
    const int64_t widths[] = {0, 1, 2, 15, 16, 17, 63, 64, 65, 511, 512, 513, 2048, 2049, 8192, 16384, 100000, 1 << 20, (1 << 27) - 1};
    const int64_t rows[] = {1, 2, 63, 64, 65, 704, 4096, 99999, (1 << 21) + 1, (1 << 23) + 3, (1 << 24) - 1, 1 << 24};
    const int64_t heads[][2] = {{1, 1}, {8, 8}, {1024, 1024}, {4, 1}, {32, 8}, {24, 8}, {1024, 64}, {16, 1}, {17, 1}, {1024, 1}};
    const int64_t threads = (int64_t(1) << 32) - 1;      // of a launch
    long long total = 0, slabs = 0, tiles = 0;
    for (int64_t w : widths)
        for (int64_t r : rows)
            for (auto& h : heads)
                for (int64_t d : {int64_t(32), int64_t(128), int64_t(160), int64_t(256)})
                    for (int64_t k : {int64_t(1), int64_t(64), int64_t(4096)})
                        for (int64_t seqs : {int64_t(1), r / 3 + 1, r}) {
                            const int64_t hkv = h[1];
                            const SelectPlan p = select_plan(r, seqs, h[0], hkv, d, w, k, seqs < r);
                            bool ok = p.slab >= 1 && p.slab <= r && p.chunks * hkv >= 0;
                            ok = ok && p.slab * hkv * 256 <= threads;                                       // lists
                            if (p.tiles && p.chunks)
                                ok = ok && select_tiles(r, seqs, d, p.group_log2) * hkv * p.chunks * 256 <= threads;
                            else
                                ok = ok && p.slab * p.chunks * 256 <= threads;                              // scores
                            int64_t pitch;
                            const int64_t row = select_row_bytes(hkv, w, pitch);
                            if (w > k)
                                ok = ok && p.need == select_bytes(r, row) && p.slab * row <= p.need && p.pitch == pitch && pitch >= w &&
                                     p.chunk * p.chunks >= w && p.chunks <= pitch / SELECT_CHUNK_MIN && p.chunk >= SELECT_CHUNK_MIN;
                            else
                                ok = ok && p.need == 0 && p.chunks == 0;
                            if (p.tiles) ok = ok && h[0] / hkv <= 16 && (64 * select_m_tiles(d) >> p.group_log2) >= 1;
                            ++total;
                            slabs += p.slab < r;
                            tiles += p.tiles && p.chunks;
                            if (!ok && ++g_failures <= 10)
                                std::fprintf(stderr, "FAILED selection: rows %lld seqs %lld hq %lld hkv %lld d %lld maxb %lld k %lld: "
                                             "slab %lld chunk %lld chunks %lld tiles %d\n", (long long)r, (long long)seqs,
                                             (long long)h[0], (long long)hkv, (long long)d, (long long)w, (long long)k,
                                             (long long)p.slab, (long long)p.chunk, (long long)p.chunks, p.tiles);
                        }
    if (slabs == 0 || tiles == 0) ++g_failures;
    std::printf("selection: %lld plans, %lld in slabs, %lld in tiles\n", total, slabs, tiles);
}

int main() {
    selection();
    const int64_t ks[] = {1, 2, 3, 7, 16, 63, 64, 65, 128, 200, 201, 225, 255, 256, 257, 321, 400, 401, 409, 512, 513, 700, 801,
                          1000, 1024, 1025, 1600, 1601, 2000, 2047, 2048, 2049, 3000, 3200, 3201, 3300, 4000, 4095, 4096};
    const int64_t widths[] = {0, 1, 2, 31, 64, 100, 1000, 2047, 4095, 4096, 4097, 8000, 8192, 10000, 16000, 16510, 32000, 32768, 32893,
                              32894, 32895, 32896, 32897, 40000, 53375, 53376, 65535, 65536, 65788, 65789, 65790, 65791, 65800, 100000,
                              1 << 20, 1 << 24};
    const int64_t heads[][2] = {{1, 1}, {2, 2}, {8, 8}, {64, 64}, {2, 1}, {16, 2}, {3, 1}, {24, 8}, {4, 1}, {32, 8}, {5, 1}, {8, 1},
                                {64, 8}, {9, 1}, {16, 1}, {20, 1}, {48, 1}};
    const int64_t rows[] = {1, 2, 8, 64, 128, 129, 256, 512, 1024, 2048, 4096, 100000};
    long long tiles = 0, few_waves = 0, total = 0;
    for (int d = 32; d <= 256; d += 32)
        for (int bs_log2 = 4; bs_log2 <= 7; ++bs_log2)
            for (auto& h : heads)
                for (int64_t k : ks)
                    for (int64_t w : widths)
                        for (int64_t r : rows)
                            for (int mode = 0; mode < 4; ++mode) {
                                const SparseShape s = {r, mode & 1 ? 1 : r, h[0], h[1], w, k, d, bs_log2, (mode & 1) != 0};
                                if (w > INT32_MAX >> bs_log2) continue;
                                const SparsePlan p = sparse_plan(s, (mode & 2) != 0);
                                const int64_t windows = int64_t(p.waves) * sa_stage_bytes(d);
                                ++total;
                                tiles += p.tile > 1;
                                few_waves += p.tile > 1 && p.waves < 4;
                                check(p.waves == 1 || p.waves == 2 || p.waves == 4 || p.waves == 8, "waves", s, p);
                                check(p.waves <= sa_max_waves(d), "waves of a workgroup", s, p);
                                check(windows + int64_t(p.list) * SA_ENTRY <= SA_LDS, "LDS", s, p);
                                check(p.list % 4 == 0 && p.list >= k, "a row's list", s, p);
                                check(p.splits >= 1 && p.splits <= SA_MAX_SPLITS, "splits", s, p);
                                check(p.splits == 1 || sparse_units(s) * p.splits <= 256, "parts", s, p);
                                if (p.tile == 1) continue;
                                check(s.chunk && p.splits == 1 && p.tile * (h[0] / h[1]) <= 16, "a tile's rows", s, p);
                                // the union of the lists, and a 16-bit word for every block that the rows may see, in whole
                                // pairs, where the windows will be
                                check(p.list >= (p.tile * k < w ? p.tile * k : w), "a tile's list", s, p);
                                check(4 * ((w + 1) / 2) <= windows, "a tile's bits", s, p);
                            }
    if (tiles == 0 || few_waves == 0) {
        std::fprintf(stderr, "FAILED: %lld tiles, %lld of them on fewer than 4 waves\n", tiles, few_waves);
        ++g_failures;
    }
    std::printf("%lld plans, %lld tiles, %lld on fewer than 4 waves, %d failure(s)\n", total, tiles, few_waves, g_failures);
    return g_failures != 0;
}
