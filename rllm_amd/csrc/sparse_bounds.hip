// Key bounds of cache blocks, and the append that keeps them, for gfx950.
//
// bounds[b, h, 0 / 1, d] = min / max over the rows of block b that hold keys of
// K[row, h, d].  Stored elements are compared as integers in the order of their
// values (ordered2), so a bound is one of the stored keys, in the cache's type.
#include "sparse_blocks.h"
#include "sparse_plan.h"

#include <type_traits>

namespace rllm {
namespace {

// ---------------------------------------------------------------------------
// bounds of whole sequences
// ---------------------------------------------------------------------------

struct BoundsArgs {
    void* kb;
    const void* kc;
    const int32_t *bt, *seq_lens, *first;
    int32_t num_seqs, hkv, d, bs_log2, maxb;
    int64_t num_blocks;
};

// A wave per (sequence, block, kv head): 16-byte loads along the tokens of a
// head_dim row, the lanes of a row reduced with each other.  Bound by HBM (the keys
// are read once): 16 sequences of 1000-8000 tokens in 32-token blocks, 8 kv heads, head_dim
// 128, 38 us, 3.9 TB/s.
template <bool FP8>
__global__ __launch_bounds__(256) void key_bounds_kernel(BoundsArgs a) {
    constexpr int TPL = FP8 ? 16 : 8;                   // tokens of a 16-byte load
    const int lane = threadIdx.x & 63;
    const int bs = 1 << a.bs_log2;
    const int lpr_log2 = a.bs_log2 - (FP8 ? 4 : 3);     // lanes of a row
    const int lpr = 1 << lpr_log2;
    const int64_t items = static_cast<int64_t>(a.num_seqs) * a.maxb;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int s = static_cast<int>(it / a.maxb), j = static_cast<int>(it - static_cast<int64_t>(s) * a.maxb);
        const int held = min(a.seq_lens[s] - (j << a.bs_log2), bs);
        if (held <= 0 || (a.first && a.first[s] >= ((j + 1) << a.bs_log2))) continue;
        const int32_t b = a.bt[it];
        if (b < 0 || b >= a.num_blocks) continue;
        for (int h = threadIdx.x >> 6; h < a.hkv; h += 4) {
            const int64_t row0 = (static_cast<int64_t>(b) * a.hkv + h) * a.d;
            const uint8_t* src = static_cast<const uint8_t*>(a.kc) + (row0 << a.bs_log2) * (FP8 ? 1 : 2);
            const int part = lane & (lpr - 1), n = held - part * TPL;   // keys among this lane's tokens
            const int rows = 64 >> lpr_log2;                   // of a load
            for (int d4 = lane >> lpr_log2; d4 < a.d; d4 += 4 * rows) {
                uint4 w4[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int d = min(d4 + x * rows, a.d - 1);
                    w4[x] = *reinterpret_cast<const uint4*>(src + static_cast<int64_t>((d << lpr_log2) + part) * 16);
                }
#pragma unroll
                for (int x4 = 0; x4 < 4; ++x4) {
                    const int d = d4 + x4 * rows;
                    const uint4 w = w4[x4];
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
                    i16x2 lo = {0x7fff, 0x7fff}, hi = {-0x8000, -0x8000};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
#pragma unroll
                        for (int p = 0; p < (FP8 ? 2 : 1); ++p) {
                            // FP8: tokens 4i, 4i + 2, then 4i + 1, 4i + 3
                            const i16x2 x = ordered2(FP8 ? (p ? u[i] & 0xff00ff00u : (u[i] << 8) & 0xff00ff00u) : u[i]);
                            const int t0 = FP8 ? 4 * i + p : 2 * i, t1 = FP8 ? t0 + 2 : t0 + 1;
                            const i16x2 l = {t0 < n ? x[0] : short(0x7fff), t1 < n ? x[1] : short(0x7fff)};
                            const i16x2 g = {t0 < n ? x[0] : short(-0x8000), t1 < n ? x[1] : short(-0x8000)};
                            lo = __builtin_elementwise_min(lo, l);
                            hi = __builtin_elementwise_max(hi, g);
                        }
                    }
                    int l = min(lo[0], lo[1]), g = max(hi[0], hi[1]);
                    for (int x = 1; x < lpr; x <<= 1) {
                        l = min(l, __shfl_xor(l, x));
                        g = max(g, __shfl_xor(g, x));
                    }
                    if (part == 0 && d < a.d) {
                        const uint16_t lb = ordered1(static_cast<int16_t>(l)), gb = ordered1(static_cast<int16_t>(g));
                        if constexpr (FP8) {
                            uint8_t* o = static_cast<uint8_t*>(a.kb) + row0 * 2 + d;
                            o[0] = static_cast<uint8_t>(lb >> 8);
                            o[a.d] = static_cast<uint8_t>(gb >> 8);
                        } else {
                            uint16_t* o = static_cast<uint16_t*>(a.kb) + row0 * 2 + d;
                            o[0] = lb;
                            o[a.d] = gb;
                        }
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// rotation, append and bounds
// ---------------------------------------------------------------------------

struct AppendArgs {
    uint16_t* q_out;
    const uint16_t *q, *k, *v;
    void *kc, *vc, *kb;
    const int32_t *bt, *seq_lens, *qsl;
    const float *cos, *sin;
    int32_t num_seqs, rows, hq, hkv, d, bs, maxb, max_position, group, roles;
    int64_t num_blocks;
    float k_scale, v_scale;
    int32_t rne;
};

template <int KIND>
__device__ __forceinline__ float in16(uint16_t b) {
    return KIND == KIND_BF16 ? to_f32<bf16_t>(b) : to_f32<f16_t>(b);
}
template <int KIND>
__device__ __forceinline__ uint16_t out16(float x) {
    return KIND == KIND_BF16 ? f32_to_bf16_bits(x) : f32_to_f16_bits(x);
}
// 8 f32 values as the cache stores them: one rounding.  To the nearest by the hardware's
// conversion, saturated before it; NaN is 0x7F, as from the encoders of common.h (4096
// tokens of 32/8 heads, head_dim 128, into E4M3: 38 us with those).
template <int KIND>
__device__ __forceinline__ uint32_t fp8_pair(float x, float y) {
    constexpr float TOP = KIND == KIND_FP8_E4M3 ? 448.f : 57344.f;
    const float a = __builtin_amdgcn_fmed3f(x, -TOP, TOP), b = __builtin_amdgcn_fmed3f(y, -TOP, TOP);
    uint32_t w;
    if constexpr (KIND == KIND_FP8_E4M3) w = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false));
    else w = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false));
    if (x != x) w = (w & 0xff00u) | 0x7fu;
    if (y != y) w = (w & 0xffu) | 0x7f00u;
    return w & 0xffffu;
}
template <int IN, int CK, class E>
__device__ __forceinline__ void stored8(const float (&x)[8], float scale, int32_t rne, E (&e)[8]) {
    if constexpr (sparse_is_fp8<CK>()) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i] / scale;
        if (rne) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const uint32_t w = fp8_pair<CK>(y[i], y[i + 1]);
                e[i] = static_cast<uint8_t>(w);
                e[i + 1] = static_cast<uint8_t>(w >> 8);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = CK == KIND_FP8_E4M3 ? fp8_e4m3_encode(y[i]) : fp8_e5m2_encode(y[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = out16<IN>(x[i]);
    }
}
// elements j .. j + 7 and their partners half a head on, rotated in f32 (each product and the sum rounded, as without contraction)
template <int IN>
__device__ __forceinline__ void rotate8_f32(const uint16_t* x, int half, const float* c, const float* s, float (&y1)[8], float (&y2)[8]) {
#pragma clang fp contract(off)
    const uint4 w1 = *reinterpret_cast<const uint4*>(x), w2 = *reinterpret_cast<const uint4*>(x + half);
    const uint32_t u1[4] = {w1.x, w1.y, w1.z, w1.w}, u2[4] = {w2.x, w2.y, w2.z, w2.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = in16<IN>(static_cast<uint16_t>(u1[i >> 1] >> ((i & 1) * 16)));
        const float b = in16<IN>(static_cast<uint16_t>(u2[i >> 1] >> ((i & 1) * 16)));
        y1[i] = a * c[i] - b * s[i];
        y2[i] = b * c[i] + a * s[i];
    }
}
template <class E>
__device__ __forceinline__ void put8(E* dst, const E (&e)[8]) {   // dst aligned to 8 elements
    if constexpr (sizeof(E) == 2)
        *reinterpret_cast<uint4*>(dst) = make_uint4(e[0] | uint32_t(e[1]) << 16, e[2] | uint32_t(e[3]) << 16,
                                                    e[4] | uint32_t(e[5]) << 16, e[6] | uint32_t(e[7]) << 16);
    else
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(e[0] | uint32_t(e[1]) << 8 | uint32_t(e[2]) << 16 | uint32_t(e[3]) << 24,
                       e[4] | uint32_t(e[5]) << 8 | uint32_t(e[6]) << 16 | uint32_t(e[7]) << 24);
}

constexpr int APPEND_GROUP = 16;                      // most tokens of a workgroup's own
constexpr int APPEND_STAGED = 2 * APPEND_GROUP - 1;   // and the rest of the last one's 16-row group

// Workgroup b: tokens [g * group, ...) of the flat list, g = b / roles.  Role r <
// Hkv writes kv head r: the runs of tokens of one block (a run starts at a
// sequence's first token of the call or at a block's first row) that start among
// them, to their end, so one workgroup has all the new keys of a block and its
// bounds need no atomics.  The last run goes on past the group, 16 cache rows at a
// time, whole rows stored at once.  The other roles rotate the queries, a token each.
// Bound by HBM: 8 prompts of 300-2000 tokens, 32/8 heads, head_dim 128, 55 us, 4.3 TB/s.
template <int IN, int CK>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    using E = typename std::conditional<sparse_is_fp8<CK>(), uint8_t, uint16_t>::type;
    const int role = static_cast<int>(blockIdx.x % a.roles);
    const int t0 = static_cast<int>(blockIdx.x / a.roles) * a.group;
    const int half = a.d >> 1;

    if (role >= a.hkv) {
        const int t = t0 + role - a.hkv;
        if (t >= a.rows) return;
        const SparseRow row = sparse_row(t, a.qsl, a.seq_lens, a.num_seqs);
        if (row.seq < 0) return;
        const int64_t pos = min(max(row.pos, 0), a.max_position - 1);
        const int items = a.d >> 4;                   // of 8 pairs, a head
        for (int it = threadIdx.x; it < a.hq * items; it += 256) {
            const int h = it / items, j = (it - h * items) * 8;
            const int64_t at = (static_cast<int64_t>(t) * a.hq + h) * a.d + j;
            float y1[8], y2[8];
            rotate8_f32<IN>(a.q + at, half, a.cos + pos * half + j, a.sin + pos * half + j, y1, y2);
            uint16_t e1[8], e2[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e1[i] = out16<IN>(y1[i]);
                e2[i] = out16<IN>(y2[i]);
            }
            put8(a.q_out + at, e1);
            put8(a.q_out + at + half, e2);
        }
        return;
    }

    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int32_t s_pos[APPEND_GROUP], s_off[APPEND_GROUP], s_blk[APPEND_GROUP], s_len[APPEND_GROUP];
    __shared__ uint32_t s_lead;
    const int h = role, D = a.d;
    const int stride = D + 16 / static_cast<int>(sizeof(E));
    E* const kl = reinterpret_cast<E*>(lds);                   // [staged token][stride]
    E* const vl = kl + APPEND_STAGED * stride;
    E* const old = vl + APPEND_STAGED * stride;                // [own token][2][D]: bounds that go on
    if (threadIdx.x < 64) {
        bool lead = false;
        const int i = threadIdx.x;
        if (i < a.group && t0 + i < a.rows) {
            const SparseRow row = sparse_row(t0 + i, a.qsl, a.seq_lens, a.num_seqs);
            const int blk = row.pos >= 0 ? row.pos / a.bs : 0, off = row.pos >= 0 ? row.pos - blk * a.bs : 0;
            lead = row.seq >= 0 && row.pos >= 0 && (row.i == 0 || off == 0);
            int32_t b = -1;
            if (lead && blk < a.maxb) b = a.bt[static_cast<int64_t>(row.seq) * a.maxb + blk];
            s_pos[i] = row.pos;
            s_off[i] = off;
            s_blk[i] = b >= 0 && b < a.num_blocks ? b : -1;
            s_len[i] = min(a.bs - off, min(row.n - row.i, a.rows - t0 - i));
        }
        const uint64_t leads = __builtin_amdgcn_ballot_w64(lead);
        if (i == 0) s_lead = static_cast<uint32_t>(leads);
    }
    __syncthreads();
    const uint32_t leads = s_lead;
    if (!leads) return;
    const int first = __builtin_ctz(leads), last = 31 - __builtin_clz(leads);
    const int last_off = s_off[last], last_len = s_len[last], last_pos = s_pos[last];

    // rotated keys and values of flat tokens t0 + [lo, lo + n) into rows lo - base ..;
    // those of the last run have positions that follow its first one's
    auto stage = [&](int lo, int n, int base) __attribute__((always_inline)) {
        const int vit = D >> 3, kit = D >> 4;
        for (int it = threadIdx.x; it < n * vit; it += 256) {
            const int i = it / vit, c = it - i * vit, tok = lo + i;
            const int64_t row = (static_cast<int64_t>(t0 + tok) * a.hkv + h) * D;
            E* const vd = vl + (tok - base) * stride + c * 8;
            if constexpr (!sparse_is_fp8<CK>()) {
                *reinterpret_cast<uint4*>(vd) = *reinterpret_cast<const uint4*>(a.v + row + c * 8);
            } else {
                const uint4 w = *reinterpret_cast<const uint4*>(a.v + row + c * 8);
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
                float y[8];
                E e[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) y[x] = in16<IN>(static_cast<uint16_t>(u[x >> 1] >> ((x & 1) * 16)));
                stored8<IN, CK>(y, a.v_scale, a.rne, e);
                put8(vd, e);
            }
            if (c < kit) {
                const int p = tok >= last ? last_pos + (tok - last) : s_pos[tok];
                const int64_t pos = min(max(p, 0), a.max_position - 1);
                float y1[8], y2[8];
                rotate8_f32<IN>(a.k + row + c * 8, half, a.cos + pos * half + c * 8, a.sin + pos * half + c * 8, y1, y2);
                E e1[8], e2[8];
                stored8<IN, CK>(y1, a.k_scale, a.rne, e1);
                stored8<IN, CK>(y2, a.k_scale, a.rne, e2);
                E* const kd = kl + (tok - base) * stride + c * 8;
                put8(kd, e1);
                put8(kd + half, e2);
            }
        }
    };
    const int b0 = min(16 - (last_off & 15), last_len);       // of the last run, to the end of a 16-row group
    stage(first, last + b0 - first, first);
    for (int it = threadIdx.x; it < a.group * 2 * D; it += 256) {   // bounds that the runs' first rows do not start
        const int tok = it / (2 * D), x = it - tok * 2 * D;
        if ((leads >> tok & 1) && s_off[tok] > 0 && s_blk[tok] >= 0)
            old[it] = static_cast<const E*>(a.kb)[(static_cast<int64_t>(s_blk[tok]) * a.hkv + h) * 2 * D + x];
    }
    __syncthreads();

    // a thread per (K or V, head_dim row), two where head_dim passes 128
    constexpr int SH = sparse_is_fp8<CK>() ? 8 : 0;
    auto ordered = [](E x) __attribute__((always_inline)) { return static_cast<int>(ordered1(static_cast<int16_t>(x << SH))); };
    auto unordered = [](int x) __attribute__((always_inline)) {
        return static_cast<E>(static_cast<uint16_t>(ordered1(static_cast<int16_t>(x))) >> SH);
    };
    int lo[2], hi[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int r = threadIdx.x + 256 * k;
        if (r >= 2 * D) break;
        const bool is_v = r >= D;
        const int d = is_v ? r - D : r;
        const E* const col = (is_v ? vl : kl) + d;
        E* const cache = static_cast<E*>(is_v ? a.vc : a.kc);
        for (uint32_t m = leads; m; m &= m - 1) {
            const int tok = __builtin_ctz(m), blk = s_blk[tok], off = s_off[tok];
            lo[k] = 0x7fff;
            hi[k] = -0x8000;
            if (blk >= 0 && off > 0 && !is_v) {
                lo[k] = ordered(old[2 * tok * D + d]);
                hi[k] = ordered(old[(2 * tok + 1) * D + d]);
            }
            if (tok == last || blk < 0) continue;
            const int n = s_len[tok];                          // a run before the last: within the group
            E* const dst = cache + ((static_cast<int64_t>(blk) * a.hkv + h) * D + d) * a.bs + off;
            for (int i = 0; i < n; ++i) {
                const E x = col[(tok + i - first) * stride];
                dst[i] = x;
                lo[k] = min(lo[k], ordered(x));
                hi[k] = max(hi[k], ordered(x));
            }
            if (is_v) continue;
            E* const o = static_cast<E*>(a.kb) + (static_cast<int64_t>(blk) * a.hkv + h) * 2 * D + d;
            o[0] = unordered(lo[k]);
            o[D] = unordered(hi[k]);
        }
    }

    // the last run, up to 16 rows of a 16-row group at a time
    const int blk = s_blk[last];
    if (blk < 0) return;
    for (int done = 0; done < last_len;) {
        const int off = last_off + done, n = min(16 - (off & 15), last_len - done);
        if (done > 0) {
            __syncthreads();
            stage(last + done, n, last + done);
            __syncthreads();
        }
        const int base = done > 0 ? 0 : last - first;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int r = threadIdx.x + 256 * k;
            if (r >= 2 * D) break;
            const bool is_v = r >= D;
            const int d = is_v ? r - D : r;
            const E* const col = (is_v ? vl : kl) + d + base * stride;
            E* const dst = static_cast<E*>(is_v ? a.vc : a.kc) + ((static_cast<int64_t>(blk) * a.hkv + h) * D + d) * a.bs + off;
            if (n == 16) {
                E e0[8], e1[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    e0[i] = col[i * stride];
                    e1[i] = col[(8 + i) * stride];
                }
                put8(dst, e0);
                put8(dst + 8, e1);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    lo[k] = min(lo[k], min(ordered(e0[i]), ordered(e1[i])));
                    hi[k] = max(hi[k], max(ordered(e0[i]), ordered(e1[i])));
                }
            } else {
                for (int i = 0; i < n; ++i) {
                    const E x = col[i * stride];
                    dst[i] = x;
                    lo[k] = min(lo[k], ordered(x));
                    hi[k] = max(hi[k], ordered(x));
                }
            }
        }
        done += n;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int r = threadIdx.x + 256 * k;
        if (r >= D) break;
        E* const o = static_cast<E*>(a.kb) + (static_cast<int64_t>(blk) * a.hkv + h) * 2 * D + r;
        o[0] = unordered(lo[k]);
        o[D] = unordered(hi[k]);
    }
}

template <int IN, int CK>
int32_t launch_append(const AppendArgs& a, hipStream_t st) {
    constexpr int ES = sparse_is_fp8<CK>() ? 1 : 2;
    const int64_t groups = (static_cast<int64_t>(a.rows) + a.group - 1) / a.group;
    const size_t lds = static_cast<size_t>(2 * APPEND_STAGED * (a.d * ES + 16) + APPEND_GROUP * 2 * a.d * ES);
    hipLaunchKernelGGL((append_kernel<IN, CK>), dim3(static_cast<unsigned>(groups * a.roles)), dim3(256), lds, st, a);
    return launch_status();
}

}  // namespace
}  // namespace rllm

using namespace rllm;

extern "C" {

int32_t rllm_key_bounds(void* k_bounds, const void* key_cache, const int32_t* block_tables, const int32_t* seq_lens,
                        const int32_t* first_positions, int64_t num_seqs, int64_t num_kv_heads, int64_t head_dim,
                        int64_t block_size, int64_t max_num_blocks_per_seq, int64_t num_blocks, int32_t kv_dtype,
                        uintptr_t stream) {
    if (num_seqs <= 0 || max_num_blocks_per_seq <= 0) return 0;
    RLLM_CHECK_ARG(sparse_shape(num_kv_heads, head_dim, block_size));
    RLLM_CHECK_ARG(kv_dtype >= RLLM_DTYPE_F16 && kv_dtype <= RLLM_DTYPE_FP8_E5M2);
    RLLM_CHECK_ARG(num_seqs <= SPARSE_MAX_ROWS && sparse_table(max_num_blocks_per_seq, block_size) && num_blocks >= 0);
    RLLM_CHECK_ARG(k_bounds && key_cache && block_tables && seq_lens);
    RLLM_CHECK_ARG(aligned_to(k_bounds, 16) && aligned_to(key_cache, 16));
    BoundsArgs a = {k_bounds, key_cache, block_tables, seq_lens, first_positions, static_cast<int32_t>(num_seqs),
                    static_cast<int32_t>(num_kv_heads), static_cast<int32_t>(head_dim),
                    __builtin_ctz(static_cast<unsigned>(block_size)), static_cast<int32_t>(max_num_blocks_per_seq), num_blocks};
    const int64_t items = num_seqs * max_num_blocks_per_seq;
    const dim3 grid(static_cast<unsigned>(items < 16384 ? items : 16384));
    if (kv_dtype == RLLM_DTYPE_FP8_E4M3 || kv_dtype == RLLM_DTYPE_FP8_E5M2)
        hipLaunchKernelGGL(key_bounds_kernel<true>, grid, dim3(256), 0, as_stream(stream), a);
    else
        hipLaunchKernelGGL(key_bounds_kernel<false>, grid, dim3(256), 0, as_stream(stream), a);
    return launch_status();
}

int32_t rllm_rope_cache_append(void* q_out, const void* q, const void* k, const void* v, void* key_cache,
                               void* value_cache, void* k_bounds, const int32_t* block_tables, const int32_t* seq_lens,
                               const int32_t* query_start_loc, const float* cos_cache, const float* sin_cache,
                               int64_t num_seqs, int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                               int64_t head_dim, int64_t block_size, int64_t max_num_blocks_per_seq, int64_t num_blocks,
                               int64_t max_position, int32_t dtype, int32_t kv_dtype, float k_scale, float v_scale,
                               int32_t fp8_rounding, uintptr_t stream) {
    if (num_seqs <= 0 || num_tokens <= 0) return 0;
    RLLM_CHECK_ARG(sparse_shape(num_kv_heads, head_dim, block_size) && sparse_types(dtype, kv_dtype));
    RLLM_CHECK_ARG(num_q_heads >= 0 && num_q_heads <= 1024);
    RLLM_CHECK_ARG(num_seqs <= SPARSE_MAX_ROWS && num_tokens <= SPARSE_MAX_ROWS && num_blocks >= 0);
    RLLM_CHECK_ARG(sparse_table(max_num_blocks_per_seq, block_size));
    RLLM_CHECK_ARG(max_position > 0 && max_position <= INT32_MAX);
    RLLM_CHECK_ARG(query_start_loc || num_tokens == num_seqs);
    RLLM_CHECK_ARG(k && v && key_cache && value_cache && k_bounds && seq_lens && cos_cache && sin_cache);
    RLLM_CHECK_ARG(block_tables || max_num_blocks_per_seq == 0);
    RLLM_CHECK_ARG(num_q_heads == 0 || (q && q_out));
    for (const void* p : {static_cast<const void*>(q_out), q, k, v, static_cast<const void*>(key_cache),
                          static_cast<const void*>(value_cache), static_cast<const void*>(k_bounds),
                          static_cast<const void*>(cos_cache), static_cast<const void*>(sin_cache)})
        RLLM_CHECK_ARG(aligned_to(p, 16));
    const bool fp8 = kv_dtype == RLLM_DTYPE_FP8_E4M3 || kv_dtype == RLLM_DTYPE_FP8_E5M2;
    if (fp8) {
        RLLM_CHECK_ARG(std::isfinite(k_scale) && std::isfinite(v_scale) && k_scale > 0.f && v_scale > 0.f);
        RLLM_CHECK_ARG(fp8_rounding == RLLM_FP8_ROUND_TOWARD_ZERO || fp8_rounding == RLLM_FP8_ROUND_NEAREST_EVEN);
    }
    // few tokens: fewer a workgroup, whose runs go one after the other (32/8 heads, head_dim 128, in
    // a graph, 4 and 16 a workgroup: 64 sequences' one token 8.0 and 15.5 us, 512 14.4 and 20.5, 1024
    // 23.5 and 28.8; one sequence's 512 7.8 and 8.6, 640 9.1 both, 1024 11.6 and 10.0; 8 x 512 31 and
    // 24, into E4M3 39 and 31; 9250 of 8 59 and 45)
    const int32_t group = num_tokens <= 512 ? 4 : APPEND_GROUP;
    AppendArgs a = {static_cast<uint16_t*>(q_out), static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                    static_cast<const uint16_t*>(v), key_cache, value_cache, k_bounds, block_tables, seq_lens,
                    query_start_loc, cos_cache, sin_cache, static_cast<int32_t>(num_seqs), static_cast<int32_t>(num_tokens),
                    static_cast<int32_t>(num_q_heads), static_cast<int32_t>(num_kv_heads), static_cast<int32_t>(head_dim),
                    static_cast<int32_t>(block_size), static_cast<int32_t>(max_num_blocks_per_seq),
                    static_cast<int32_t>(max_position), group,
                    static_cast<int32_t>(num_kv_heads) + (num_q_heads > 0 ? group : 0), num_blocks, k_scale, v_scale,
                    fp8_rounding == RLLM_FP8_ROUND_NEAREST_EVEN};
    RLLM_CHECK_ARG((num_tokens + group - 1) / group * a.roles <= MAX_WORKGROUPS);
    const hipStream_t st = as_stream(stream);
    if (dtype == RLLM_DTYPE_BF16) {
        if (kv_dtype == RLLM_DTYPE_FP8_E4M3) return launch_append<KIND_BF16, KIND_FP8_E4M3>(a, st);
        if (kv_dtype == RLLM_DTYPE_FP8_E5M2) return launch_append<KIND_BF16, KIND_FP8_E5M2>(a, st);
        return launch_append<KIND_BF16, KIND_BF16>(a, st);
    }
    if (kv_dtype == RLLM_DTYPE_FP8_E4M3) return launch_append<KIND_F16, KIND_FP8_E4M3>(a, st);
    if (kv_dtype == RLLM_DTYPE_FP8_E5M2) return launch_append<KIND_F16, KIND_FP8_E5M2>(a, st);
    return launch_append<KIND_F16, KIND_F16>(a, st);
}

}  // extern "C"
