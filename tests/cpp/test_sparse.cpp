// Tests of the wrappers of the C++ host mirror (rllm_amd/host/rllm_host.hpp) for attention
// over selected cache blocks: refusals on the host (cpu) and, on a GPU, one sequence appended
// a token at a time, its bounds, its selection and its attention, against sums in double.
//
// usage: test_sparse cpu | gpu      (exit status 0 = all passed)
#include "../../rllm_amd/host/rllm_host.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

using namespace rllm::kernels;

static int g_failures = 0;
#define CHECK(cond)                                                             \
    do {                                                                        \
        if (!(cond)) {                                                          \
            std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++g_failures;                                                       \
        }                                                                       \
    } while (0)

static float f32(uint16_t b) {
    const uint32_t u = static_cast<uint32_t>(b) << 16;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}
static uint16_t bf16(float f) {   // cut to bf16
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return static_cast<uint16_t>(u >> 16);
}

static void refusals() {
    void* p = reinterpret_cast<void*>(0x1000);   // never dereferenced
    int32_t* i = reinterpret_cast<int32_t*>(0x1000);
    float* f = reinterpret_cast<float*>(0x1000);
    CHECK(key_bounds(p, p, i, i, 2, 8, 100, 16, 4, 10, DType::BF16, 0).is_err());
    CHECK(key_bounds(nullptr, p, i, i, 2, 8, 128, 16, 4, 10, DType::BF16, 0).is_err());
    CHECK(key_bounds(nullptr, nullptr, nullptr, nullptr, 0, 8, 128, 16, 4, 10, DType::BF16, 0).is_ok());
    CHECK(rope_cache_append(p, p, p, p, p, p, p, i, i, nullptr, f, f, 2, 3, 8, 2, 128, 16, 4, 10, 100, DType::BF16, DType::BF16,
                            1.f, 1.f, 0).is_err());
    CHECK(select_blocks(i, p, p, i, i, nullptr, 2, 2, 8, 2, 128, 16, 40, 10, 8, 4, 5, DType::BF16, DType::BF16, 0, p, 1 << 20).is_err());
    CHECK(paged_attention_sparse(p, p, p, p, i, i, nullptr, i, 2, 2, 7, 2, 128, 16, 4, 10, 8, 0.1f, DType::BF16, DType::BF16, 1.f,
                                 1.f, 0).is_err());
}

template <class T> static T* upload(const std::vector<T>& v) {
    void* p = nullptr;
    CHECK(hipMalloc(&p, v.size() * sizeof(T)) == hipSuccess);
    CHECK(hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) == hipSuccess);
    return static_cast<T*>(p);
}
template <class T> static std::vector<T> download(const void* p, size_t n) {
    std::vector<T> v(n);
    CHECK(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost) == hipSuccess);
    return v;
}

static void append_select_attend() {
    const int T = 203, hq = 4, hkv = 2, D = 64, bs = 16, nb = 15, maxb = 13, K = 5;
    std::mt19937 rng(5);
    std::normal_distribution<float> nd;
    std::vector<uint16_t> k(T * hkv * D), v(k.size()), q(hq * D);
    for (auto* x : {&k, &v, &q})
        for (auto& e : *x) e = bf16(nd(rng));
    std::vector<int32_t> bt(maxb);
    for (int j = 0; j < maxb; ++j) bt[j] = (7 * j + 3) % nb;
    // no rotation: cos 1, sin 0
    std::vector<float> cos(T * D / 2, 1.f), sin(T * D / 2, 0.f);
    const std::vector<uint16_t> zero(nb * hkv * D * bs, 0), zero_b(nb * hkv * 2 * D, 0);
    uint16_t *kc = upload(zero), *vc = upload(zero), *kb = upload(zero_b), *kb2 = upload(zero_b);
    uint16_t *dk = upload(k), *dv = upload(v), *dq = upload(q), *out = upload(q);
    int32_t *dbt = upload(bt), *dlen = upload(std::vector<int32_t>{0}), *sel = upload(std::vector<int32_t>(hkv * K, -9));
    float *dc = upload(cos), *dsn = upload(sin);
    for (int t = 0; t < T; ++t) {
        const int32_t len = t + 1;
        CHECK(hipMemcpy(dlen, &len, 4, hipMemcpyHostToDevice) == hipSuccess);
        CHECK(rope_cache_append(nullptr, nullptr, dk + t * hkv * D, dv + t * hkv * D, kc, vc, kb, dbt, dlen, nullptr, dc, dsn, 1, 1,
                                0, hkv, D, bs, maxb, nb, T, DType::BF16, DType::BF16, 1.f, 1.f, 0).is_ok());
    }
    CHECK(key_bounds(kb2, kc, dbt, dlen, 1, hkv, D, bs, maxb, nb, DType::BF16, 0).is_ok());
    CHECK(select_blocks(sel, dq, kb, dbt, dlen, nullptr, 1, 1, hq, hkv, D, bs, maxb, nb, K, 1, 1, DType::BF16, DType::BF16, 0).is_ok());
    const float scale = 0.125f;
    CHECK(paged_attention_sparse(out, dq, kc, vc, dbt, dlen, nullptr, sel, 1, 1, hq, hkv, D, bs, maxb, nb, K, scale, DType::BF16,
                                 DType::BF16, 1.f, 1.f, 0).is_ok());
    CHECK(hipDeviceSynchronize() == hipSuccess);
    const auto b1 = download<uint16_t>(kb, zero_b.size()), b2 = download<uint16_t>(kb2, zero_b.size());
    CHECK(b1 == b2);
    const auto lists = download<int32_t>(sel, hkv * K);
    const auto got = download<uint16_t>(out, hq * D);
    double worst = 0;
    for (int g = 0; g < hkv; ++g) {
        std::vector<std::pair<double, int>> score;   // (-score, block)
        for (int j = 0; j < maxb; ++j) {
            double best = -1e300;
            for (int h = g * 2; h < g * 2 + 2; ++h) {
                double s = 0;
                for (int d = 0; d < D; ++d) {
                    double lo = 1e300, hi = -1e300;
                    for (int t = j * bs; t < std::min(T, (j + 1) * bs); ++t) {
                        lo = std::min<double>(lo, f32(k[(t * hkv + g) * D + d]));
                        hi = std::max<double>(hi, f32(k[(t * hkv + g) * D + d]));
                    }
                    const double x = f32(q[h * D + d]);
                    s += std::max(x * lo, x * hi);
                }
                best = std::max(best, s);
            }
            if (j > 0 && j < maxb - 1) score.push_back({-best, j});
        }
        std::sort(score.begin(), score.end());
        std::vector<int32_t> want = {0, maxb - 1};
        for (int i = 0; i < K - 2; ++i) want.push_back(score[i].second);
        std::sort(want.begin(), want.end());
        CHECK(std::equal(want.begin(), want.end(), lists.begin() + g * K));
        for (int h = g * 2; h < g * 2 + 2; ++h) {
            std::vector<double> o(D, 0.0), mag(D, 0.0);
            double z = 0;
            for (int j : want)
                for (int t = j * bs; t < std::min(T, (j + 1) * bs); ++t) {
                    double s = 0;
                    for (int d = 0; d < D; ++d) s += double(f32(q[h * D + d])) * f32(k[(t * hkv + g) * D + d]);
                    const double p = std::exp(s * scale);
                    z += p;
                    for (int d = 0; d < D; ++d) {
                        const double x = f32(v[(t * hkv + g) * D + d]);
                        o[d] += p * x;
                        mag[d] += p * std::fabs(x);
                    }
                }
            for (int d = 0; d < D; ++d) {
                // half a bf16 step of the output, and 2^-14 of the weighted magnitude for sums, scores and weights
                const double tol = std::fabs(o[d] / z) / 256 + mag[d] / z / 16384;
                worst = std::max(worst, std::fabs(f32(got[h * D + d]) - o[d] / z) / tol);
            }
        }
    }
    CHECK(worst <= 1.0);
    for (void* x : {static_cast<void*>(kc), static_cast<void*>(vc), static_cast<void*>(kb), static_cast<void*>(kb2),
                    static_cast<void*>(dk), static_cast<void*>(dv), static_cast<void*>(dq), static_cast<void*>(out),
                    static_cast<void*>(dbt), static_cast<void*>(dlen), static_cast<void*>(sel), static_cast<void*>(dc),
                    static_cast<void*>(dsn)})
        (void)hipFree(x);
}

int main(int argc, char** argv) {
    refusals();
    if (argc > 1 && std::strcmp(argv[1], "gpu") == 0) append_select_attend();
    std::printf("%d failure(s)\n", g_failures);
    return g_failures != 0;
}
