// CPU tests of the launch plan of the attention over listed blocks
// (rllm_amd/csrc/sparse_plan.h): whatever the sizes, what the kernel keeps in LDS fits.
//
// usage: test_sparse_plan      (exit status 0 = all passed)
#include "../../rllm_amd/csrc/sparse_plan.h"

#include <cstdio>

using namespace rllm;

static int g_failures = 0;
static void check(bool ok, const char* what, const SparseShape& s, const SparsePlan& p) {
    if (ok) return;
    if (++g_failures <= 10)
        std::fprintf(stderr, "FAILED %s: rows %lld hq %lld hkv %lld d %d bs %d maxb %lld k %lld: tile %d list %d waves %d splits %d\n",
                     what, (long long)s.rows, (long long)s.hq, (long long)s.hkv, s.d, 1 << s.bs_log2, (long long)s.maxb,
                     (long long)s.k, p.tile, p.list, p.waves, p.splits);
}

int main() {
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
