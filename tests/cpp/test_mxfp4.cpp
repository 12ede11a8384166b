// Tests of the MXFP4 wrappers of the C++ host mirror (rllm_amd/host/rllm_host.hpp):
// refusals on the host (cpu) and, on a GPU, a sequence written row by row, read back,
// attended by decode steps and by one chunk, against sums in double.
//
// usage: test_mxfp4 cpu | gpu      (exit status 0 = all passed)
#include "../../rllm_amd/host/rllm_host.hpp"

#include <hip/hip_runtime.h>

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
static uint16_t bf16(float f) {   // values used here are bf16 already, or cut to it
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return static_cast<uint16_t>(u >> 16);
}

static void refusals() {
    CHECK(mxfp4_page_bytes(128, 16).value() == 16 * 68);
    CHECK(mxfp4_page_bytes(100, 16).is_err() && mxfp4_page_bytes(128, 24).is_err());
    uint16_t* w = reinterpret_cast<uint16_t*>(0x1000);   // never dereferenced
    uint8_t* c = reinterpret_cast<uint8_t*>(0x1000);
    int64_t* s = reinterpret_cast<int64_t*>(0x1000);
    int32_t* i = reinterpret_cast<int32_t*>(0x1000);
    float* f = reinterpret_cast<float*>(0x1000);
    CHECK(cache_write_mxfp4(c, c, w, w, s, 4, 8, 128, 16, 10, DType::FP8E4M3, 0).is_err());
    CHECK(cache_write_mxfp4(c, c, w, w, s, 4, 8, 120, 16, 10, DType::BF16, 0).is_err());
    CHECK(cache_write_mxfp4(nullptr, c, w, w, s, 0, 8, 128, 16, 10, DType::BF16, 0).is_ok());
    CHECK(cache_read_mxfp4(w, w, c, c, nullptr, 4, 8, 128, 16, 10, DType::BF16, 0).is_err());
    CHECK(rope_cache_write_mxfp4(w, w, w, w, c, c, s, i, f, f, 4, 8, 2, 96, 16, 10, 100, DType::BF16, 0).is_err());
    const auto d = paged_attention_decode_mxfp4(w, w, c, c, i, i, 2, 30, 8, 128, 16, 4, 10, 0.1f, DType::BF16, 0);
    CHECK(d.is_err());
    CHECK(paged_attention_prefill_mxfp4(w, w, c, c, i, i, i, 2, 9, 32, 8, 128, 16, 4, 0, 0.1f, DType::BF16, 0).is_err());
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

static void write_read_attend() {
    const int T = 45, hq = 4, hkv = 2, D = 64, bs = 16, nb = 5;
    std::mt19937 rng(3);
    std::normal_distribution<float> nd;
    std::vector<uint16_t> k(T * hkv * D), v(k.size()), q(T * hq * D);
    for (auto* x : {&k, &v, &q})
        for (auto& e : *x) e = bf16(nd(rng));
    const std::vector<int32_t> bt = {3, 0, 4};
    std::vector<int64_t> slots(T);
    for (int t = 0; t < T; ++t) slots[t] = bt[t / bs] * bs + t % bs;
    const size_t bytes = nb * hkv * mxfp4_page_bytes(D, bs).value();
    uint8_t *kc = gpu_alloc(bytes).value(), *vc = gpu_alloc(bytes).value();
    CHECK(cache_zero_sync(kc, bytes).is_ok() && cache_zero_sync(vc, bytes).is_ok());
    uint16_t *dk = upload(k), *dv = upload(v), *dq = upload(q);
    int64_t* ds = upload(slots);
    int32_t *dbt = upload(bt), *dlen = upload(std::vector<int32_t>{T}), *dqsl = upload(std::vector<int32_t>{0, T});
    uint16_t *ok = upload(k), *ov = upload(v), *out = upload(q);
    CHECK(cache_write_mxfp4(kc, vc, dk, dv, ds, T, hkv, D, bs, nb, DType::BF16, 0).is_ok());
    CHECK(cache_read_mxfp4(ok, ov, kc, vc, ds, T, hkv, D, bs, nb, DType::BF16, 0).is_ok());
    const float scale = 0.125f;
    CHECK(paged_attention_prefill_mxfp4(out, dq, kc, vc, dbt, dlen, dqsl, 1, T, hq, hkv, D, bs, 3, nb, scale,
                                        DType::BF16, 0).is_ok());
    CHECK(hipDeviceSynchronize() == hipSuccess);
    const auto kb = download<uint16_t>(ok, k.size()), vb = download<uint16_t>(ov, v.size());
    const auto chunk = download<uint16_t>(out, q.size());
    // the last token again, as a decode step
    CHECK(paged_attention_decode_mxfp4(out, dq + (T - 1) * hq * D, kc, vc, dbt, dlen, 1, hq, hkv, D, bs, 3, nb, scale,
                                       DType::BF16, 0).is_ok());
    CHECK(hipDeviceSynchronize() == hipSuccess);
    const auto step = download<uint16_t>(out, hq * D);
    double worst = 0;
    for (size_t i = 0; i < k.size(); ++i) {
        // a value is at most a quarter of its block's largest off: 8 saturates at 6
        const size_t b = i / 32 * 32;
        float top = 0;
        for (size_t j = b; j < b + 32; ++j) top = std::fmax(top, std::fabs(f32(k[j])));
        CHECK(std::fabs(f32(kb[i]) - f32(k[i])) <= 0.25f * top);
    }
    for (int t = 0; t < T; ++t)
        for (int h = 0; h < hq; ++h) {
            const int g = h / (hq / hkv);
            std::vector<double> p(t + 1);
            double z = 0;
            for (int u = 0; u <= t; ++u) {
                double s = 0;
                for (int d = 0; d < D; ++d) s += double(f32(q[(t * hq + h) * D + d])) * f32(kb[(u * hkv + g) * D + d]);
                z += p[u] = std::exp(s * scale);
            }
            for (int d = 0; d < D; ++d) {
                double o = 0, mag = 0;
                for (int u = 0; u <= t; ++u) {
                    const double x = p[u] / z * f32(vb[(u * hkv + g) * D + d]);
                    o += x;
                    mag += std::fabs(x);
                }
                // half a bf16 step of the output, and of every weight, and the scores' 2^-12
                const double tol = std::fabs(o) / 256 + mag * (1.0 / 256 + 1.0 / 256);
                const double e = std::fabs(f32(chunk[(t * hq + h) * D + d]) - o);
                worst = std::fmax(worst, e / (tol + 1e-30));
                if (t == T - 1) worst = std::fmax(worst, std::fabs(f32(step[h * D + d]) - o) / (tol + 1e-30));
            }
        }
    CHECK(worst <= 1.0);
    for (void* p : {static_cast<void*>(dk), static_cast<void*>(dv), static_cast<void*>(dq), static_cast<void*>(ds),
                    static_cast<void*>(dbt), static_cast<void*>(dlen), static_cast<void*>(dqsl), static_cast<void*>(ok),
                    static_cast<void*>(ov), static_cast<void*>(out)})
        (void)hipFree(p);
    CHECK(gpu_free(kc).is_ok() && gpu_free(vc).is_ok());
}

int main(int argc, char** argv) {
    refusals();
    if (argc > 1 && std::strcmp(argv[1], "gpu") == 0) write_read_attend();
    std::printf("%d failure(s)\n", g_failures);
    return g_failures != 0;
}
