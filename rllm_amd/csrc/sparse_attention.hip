// Attention over listed cache blocks, for gfx950: decode rows and chunks of prompts.
//
//   o = softmax(scale q . K^T) V over the keys of the listed blocks that the row sees,
// in one pass with a running maximum and sum.
//
// Bound by HBM (decode) or by what the L2s bring (chunks, whose rows list much the
// same blocks): K and V of the listed blocks are read once per row and 16 query heads.
//
// Work: a workgroup of 4 waves takes one (row, kv head, 16 heads); the list's keys
// stand one after the other and are cut into windows of 128, wave w taking windows
// w, w + 4, ...; the four merge through LDS.  No operand passes through LDS:
//   S^T = K Q^T   v_mfma_16x16x32, rows = tokens, columns = heads.  Lane (r = l % 16,
//                 q = l / 16) loads the 8 tokens of octet 4 (r % 4) + r / 4 of the
//                 window in head_dim rows 32k + 8q .. + 7, along the tokens as the cache has
//                 them, and transposes the 8 x 8 tile with v_perm; product t of the
//                 eight takes token t of every lane's octet.
//   O^T = V^T P^T rows = head_dim, k = tokens.  With that order lane (r, q) holds
//                 the scores of head r for octets 4i + q: the operand of k-step i
//                 as it stands; V's is one 16-byte load of row r, octet 4i + q.
// An octet lies within one block (of 16 rows or more), so only the list tells this
// from attention over whole tables.  Weights enter as two 16-bit terms (generic_mfma.h).
#include "sparse_blocks.h"
#include "generic_mfma.h"

namespace rllm {
namespace {

constexpr int SA_WIN = 128;     // tokens of a wave's window
constexpr int SA_WAVES = 4;

struct SparseArgs {
    uint16_t* out;
    const uint16_t* q;
    const uint8_t *kc, *vc;
    const int32_t *bt, *seq_lens, *qsl, *sel;
    int32_t num_seqs, rows, hq, hkv, bs_log2, maxb, k, head_groups;
    int64_t num_blocks;
    float s_scale, v_scale;     // s_scale: scale * k_scale * log2(e)
};

__device__ __forceinline__ float over_quads_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_quads_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

template <int KVKIND, int D>
constexpr int sa_waves_per_simd() {
    return D > 128 && !gen_is_fp8<KVKIND>() ? 1 : 2;
}

template <int QKIND, int KVKIND, int NK>
__global__ __launch_bounds__(256, (sa_waves_per_simd<KVKIND, 32 * NK>())) void sparse_attention_kernel(SparseArgs a) {
    using M = GenMfma<QKIND>;
    using raw_t = GenRaw<KVKIND>;
    constexpr int D = 32 * NK, ND = D / 16;
    constexpr int VC = sa_waves_per_simd<KVKIND, D>() == 1 || ND < 8 || ND % 4 ? ND : ND == 8 ? (gen_is_fp8<KVKIND>() ? 8 : 4) : ND / 2;
    constexpr int VSTEPS = 4 * (ND / VC);
    constexpr int ES = gen_is_fp8<KVKIND>() ? 1 : 2;
    constexpr int OST = D + 4;                                  // LDS row of one head's partial
    constexpr int MERGE = (SA_WAVES * 16 * OST + 2 * SA_WAVES * 16) * 4, LIST = RLLM_SELECT_MAX_BLOCKS * 8;
    __shared__ __align__(16) uint8_t lds[MERGE > LIST ? MERGE : LIST];
    __shared__ int s_used;
    int2* const s_list = reinterpret_cast<int2*>(lds);          // (block or -1, keys seen in it)
    float* const s_o = reinterpret_cast<float*>(lds);           // after the list: [wave][head][OST]
    float* const s_m = s_o + SA_WAVES * 16 * OST;               // [wave][head]
    float* const s_l = s_m + SA_WAVES * 16;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q4 = lane >> 4;
    const int G = a.hq / a.hkv;
    const int hg = blockIdx.x % a.head_groups;
    const int unit = blockIdx.x / a.head_groups, h = unit % a.hkv, t = unit / a.hkv;
    const SparseRow row = sparse_row(t, a.qsl, a.seq_lens, a.num_seqs);
    if (row.seq < 0) return;
    const int ng = min(16, G - 16 * hg);
    const int64_t row0 = static_cast<int64_t>(t) * a.hq + h * G + 16 * hg;

    // the list, with what the row sees of each block
    if (threadIdx.x == 0) s_used = 0;
    __syncthreads();
    {
        const int32_t* const sel = a.sel + (static_cast<int64_t>(t) * a.hkv + h) * a.k;
        const int32_t* const bt = a.bt + static_cast<int64_t>(row.seq) * a.maxb;
        int used = 0;
        for (int i = threadIdx.x; i < a.k; i += 256) {
            const int j = sel[i], before = i ? sel[i - 1] : -1;
            int b = -1, seen = 0;
            if (j > before && j >= 0 && j < a.maxb && j <= row.pos >> a.bs_log2) {
                b = bt[j];
                if (b < 0 || b >= a.num_blocks) b = -1;
                seen = min(row.pos + 1 - (j << a.bs_log2), 1 << a.bs_log2);
            }
            s_list[i] = make_int2(b, seen);
            if (b >= 0) used = i + 1;
        }
        if (used) atomicMax(&s_used, used);
    }

    // queries, negated where the scale is negative (exact), so that the running max is
    // over c * s with c >= 0
    const float c = __builtin_fabsf(a.s_scale);
    uint4 qreg[NK];
    {
        const uint32_t flip = a.s_scale < 0.f ? 0x80008000u : 0u;
        const uint16_t* qrow = a.q + (row0 + r) * D;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (r < ng) x = *reinterpret_cast<const uint4*>(qrow + 32 * k + 8 * q4);
            qreg[k] = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
        }
    }
    __syncthreads();
    const int end = s_used << a.bs_log2;                        // tokens of the list (at most 4096 * 128)
    const uint8_t* const zero = reinterpret_cast<const uint8_t*>(g_gen_zero);
    const int row_b = ES << a.bs_log2;                          // bytes of a head_dim row of a block
    const int64_t slab_b = static_cast<int64_t>(D) * row_b;
    // offset of an octet's head_dim row 0 in the caches, -1 where there is nothing to read; keep: the keys seen in it
    auto octet = [&](int tok, int& keep) __attribute__((always_inline)) -> int64_t {
        keep = 0;
        if (tok >= end) return -1;
        const int2 e = s_list[tok >> a.bs_log2];
        const int off = tok & ((1 << a.bs_log2) - 1);
        if (e.x < 0 || off >= e.y) return -1;
        keep = e.y - off;
        return (static_cast<int64_t>(e.x) * a.hkv + h) * slab_b + off * ES;
    };

    gm_f32x4 o[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[dt] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    // The loads run ahead of the arithmetic: K one k-step, V one group of tiles, and as
    // a window's V products run, the next window's first K rows.
    raw_t kr[2][8];
    auto load_k = [&](int64_t ko, int k, raw_t* dst) __attribute__((always_inline)) {
        const uint8_t* p = ko >= 0 ? a.kc + ko + static_cast<int64_t>(32 * k + 8 * q4) * row_b : zero;
        const int st = ko >= 0 ? row_b : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = *reinterpret_cast<const raw_t*>(p + static_cast<int64_t>(i) * st);
    };
    const int k_oct = 8 * (4 * (r & 3) + (r >> 2));
    int w0 = SA_WIN * wave, skip;
    int64_t ko = octet(w0 + k_oct, skip), vo[4];
    int keep[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vo[i] = octet(w0 + 8 * (4 * i + q4), keep[i]);
    load_k(ko, 0, kr[0]);
    for (; w0 < end; w0 += SA_WIN * SA_WAVES) {
        // ---- S^T = K Q^T ----
        gm_f32x4 acc[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            if (k + 1 < NK) load_k(ko, k + 1, kr[(k + 1) & 1]);
            uint4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = gen_to16<QKIND, KVKIND>(kr[k & 1][i]);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                auto word = [&](const uint4& v) __attribute__((always_inline)) -> uint32_t {
                    return u < 2 ? v.x : u < 4 ? v.y : u < 6 ? v.z : v.w;
                };
                const uint32_t pick = (u & 1) ? 0x07060302u : 0x05040100u;
                const uint4 kt = make_uint4(__builtin_amdgcn_perm(word(x[1]), word(x[0]), pick),
                                            __builtin_amdgcn_perm(word(x[3]), word(x[2]), pick),
                                            __builtin_amdgcn_perm(word(x[5]), word(x[4]), pick),
                                            __builtin_amdgcn_perm(word(x[7]), word(x[6]), pick));
                acc[u] = M::mma16(kt, qreg[k], acc[u]);
            }
        }

        // V of the first step goes out before the softmax
        raw_t vr[2][VC];
        auto load_v = [&](int st, raw_t* dst) __attribute__((always_inline)) {
            const int i = st / (ND / VC), c0 = st % (ND / VC) * VC;
            const uint8_t* p = vo[i] >= 0 ? a.vc + vo[i] + static_cast<int64_t>(16 * c0 + r) * row_b : zero;
            const int step = vo[i] >= 0 ? 16 * row_b : 0;
#pragma unroll
            for (int dt = 0; dt < VC; ++dt) dst[dt] = *reinterpret_cast<const raw_t*>(p + static_cast<int64_t>(dt) * step);
        };
        load_v(0, vr[0]);

        // ---- weights: lane (head r, q4) holds tokens w0 + 8 (4i + q4) + u ----
        float p[4][8];
        const bool whole = __builtin_amdgcn_ballot_w64(min(min(keep[0], keep[1]), min(keep[2], keep[3])) < 8) == 0;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                p[i][u] = acc[u][i];
                if (!whole && u >= keep[i]) p[i][u] = -INFINITY;
                mx = fmaxf(mx, p[i][u]);
            }
        // the max, lowered by the weights' lift; c = 0 times an infinity must not poison it
        const float m_new = fmaxf(m_run, over_quads_max(mx == -INFINITY ? mx : mx * c - gen_decode_lift<QKIND>()));
        const float ms = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2f(m_run - ms);
        // past 2^20 the roundings of the product and of the lowered max show: the same
        // product on both sides then, and no weight above 2^lift (f16 ends at 2^16)
        const bool large = __builtin_amdgcn_ballot_w64(!(__builtin_fabsf(ms) <= 0x1p20f)) != 0;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float e = fmaf(p[i][u], c, -ms);
                if (large) {
#pragma clang fp contract(off)
                    const float x = p[i][u] * c;
                    e = x - ms > gen_decode_lift<QKIND>() ? gen_decode_lift<QKIND>() : x - ms;   // NaN goes on
                }
                e = __builtin_amdgcn_exp2f(e);
                p[i][u] = whole || u < keep[i] ? e : 0.f;
                sum += p[i][u];
            }
        l_run = l_run * alpha + sum;
        m_run = m_new;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[dt] *= alpha;

        // ---- O^T += V^T P^T ----
        const int w1 = w0 + SA_WIN * SA_WAVES;
        ko = octet(w1 + k_oct, skip);
        int64_t nvo[4];
        int nkeep[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) nvo[i] = octet(w1 + 8 * (4 * i + q4), nkeep[i]);
        uint4 ph, pl;
#pragma unroll
        for (int st = 0; st < VSTEPS; ++st) {
            const int i = st / (ND / VC), c0 = st % (ND / VC) * VC;
            if (st + 1 < VSTEPS) load_v(st + 1, vr[(st + 1) & 1]);
            else load_k(ko, 0, kr[0]);
            if (c0 == 0) gen_split8<QKIND>(p[i], ph, pl);
#pragma unroll
            for (int dt = 0; dt < VC; ++dt) {
                uint4 v = gen_to16<QKIND, KVKIND>(vr[st & 1][dt]);
                if (!whole) v = gen_keep(v, keep[i]);           // stale values follow the last key
                o[c0 + dt] = M::mma16(v, ph, o[c0 + dt]);
                o[c0 + dt] = M::mma16(v, pl, o[c0 + dt]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            vo[i] = nvo[i];
            keep[i] = nkeep[i];
        }
    }

    // ---- merge the four waves ----
    l_run = over_quads_sum(l_run);
    __syncthreads();                                            // the list is done with
    if (q4 == 0) {
        s_m[wave * 16 + r] = m_run;
        s_l[wave * 16 + r] = l_run;
    }
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
        *reinterpret_cast<gm_f32x4*>(s_o + (wave * 16 + r) * OST + 16 * dt + 4 * q4) = o[dt];
    __syncthreads();
    constexpr int quads = D >> 2;
    for (int it = threadIdx.x; it < ng * quads; it += 256) {
        const int hd = it / quads, d0 = (it - hd * quads) * 4;
        float mm[SA_WAVES], mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < SA_WAVES; ++w) {
            mm[w] = s_m[w * 16 + hd];
            mx = fmaxf(mx, mm[w]);
        }
        gm_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < SA_WAVES; ++w) {
            const float lw = s_l[w * 16 + hd];
            if (lw == 0.f) continue;                            // a wave without keys (NaN goes on)
            const float f = exp2f(mm[w] - mx);
            L = fmaf(f, lw, L);
            sum += f * *reinterpret_cast<const gm_f32x4*>(s_o + (w * 16 + hd) * OST + d0);
        }
        const gm_f32x4 v = sum * gen_inv(a.v_scale, L);
        *reinterpret_cast<uint2*>(a.out + (row0 + hd) * D + d0) = make_uint2(M::pack2(v[0], v[1]), M::pack2(v[2], v[3]));
    }
}

template <int QKIND, int KVKIND>
int32_t launch_sparse(const SparseArgs& a, int64_t d, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.rows) * a.hkv * a.head_groups));
    switch (d / 32) {
#define RLLM_SPARSE(N) \
    case N: hipLaunchKernelGGL((sparse_attention_kernel<QKIND, KVKIND, N>), grid, dim3(64 * SA_WAVES), 0, st, a); break;
        RLLM_SPARSE(1) RLLM_SPARSE(2) RLLM_SPARSE(3) RLLM_SPARSE(4) RLLM_SPARSE(5) RLLM_SPARSE(6) RLLM_SPARSE(7) RLLM_SPARSE(8)
#undef RLLM_SPARSE
    }
    return launch_status();
}

}  // namespace
}  // namespace rllm

using namespace rllm;

extern "C" {

int32_t rllm_paged_attention_sparse(void* output, const void* query, const void* key_cache, const void* value_cache,
                                    const int32_t* block_tables, const int32_t* seq_lens, const int32_t* query_start_loc,
                                    const int32_t* selected, int64_t num_seqs, int64_t num_rows, int64_t num_q_heads,
                                    int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                    int64_t max_num_blocks_per_seq, int64_t num_blocks, int64_t num_selected, float scale,
                                    int32_t q_dtype, int32_t kv_dtype, float k_scale, float v_scale, uintptr_t stream) {
    if (num_seqs <= 0 || num_rows <= 0) return 0;
    RLLM_CHECK_ARG(sparse_shape(num_kv_heads, head_dim, block_size) && sparse_heads(num_q_heads, num_kv_heads));
    RLLM_CHECK_ARG(sparse_types(q_dtype, kv_dtype));
    RLLM_CHECK_ARG(num_seqs <= SPARSE_MAX_ROWS && num_rows <= SPARSE_MAX_ROWS && num_blocks >= 0);
    RLLM_CHECK_ARG(sparse_table(max_num_blocks_per_seq, block_size));
    RLLM_CHECK_ARG(query_start_loc || num_rows == num_seqs);
    RLLM_CHECK_ARG(num_selected >= 1 && num_selected <= RLLM_SELECT_MAX_BLOCKS);
    RLLM_CHECK_ARG(output && query && key_cache && value_cache && seq_lens && selected);
    RLLM_CHECK_ARG(block_tables || max_num_blocks_per_seq == 0);
    for (const void* p : {static_cast<const void*>(output), query, key_cache, value_cache}) RLLM_CHECK_ARG(aligned_to(p, 16));
    const bool fp8 = kv_dtype == RLLM_DTYPE_FP8_E4M3 || kv_dtype == RLLM_DTYPE_FP8_E5M2;
    if (!fp8) k_scale = v_scale = 1.f;
    const float s_scale = scale * k_scale * 1.44269504088896340736f;
    RLLM_CHECK_ARG(std::isfinite(scale) && std::isfinite(k_scale) && std::isfinite(v_scale) && std::isfinite(s_scale));
    const int64_t head_groups = (num_q_heads / num_kv_heads + 15) / 16;
    RLLM_CHECK_ARG(num_rows * num_kv_heads * head_groups <= INT32_MAX);
    SparseArgs a = {static_cast<uint16_t*>(output), static_cast<const uint16_t*>(query),
                    static_cast<const uint8_t*>(key_cache), static_cast<const uint8_t*>(value_cache), block_tables, seq_lens,
                    query_start_loc, selected, static_cast<int32_t>(num_seqs), static_cast<int32_t>(num_rows),
                    static_cast<int32_t>(num_q_heads), static_cast<int32_t>(num_kv_heads),
                    __builtin_ctz(static_cast<unsigned>(block_size)), static_cast<int32_t>(max_num_blocks_per_seq),
                    static_cast<int32_t>(num_selected), static_cast<int32_t>(head_groups), num_blocks, s_scale, v_scale};
    const hipStream_t st = as_stream(stream);
    if (q_dtype == RLLM_DTYPE_BF16) {
        if (kv_dtype == RLLM_DTYPE_FP8_E4M3) return launch_sparse<KIND_BF16, KIND_FP8_E4M3>(a, head_dim, st);
        if (kv_dtype == RLLM_DTYPE_FP8_E5M2) return launch_sparse<KIND_BF16, KIND_FP8_E5M2>(a, head_dim, st);
        return launch_sparse<KIND_BF16, KIND_BF16>(a, head_dim, st);
    }
    if (kv_dtype == RLLM_DTYPE_FP8_E4M3) return launch_sparse<KIND_F16, KIND_FP8_E4M3>(a, head_dim, st);
    if (kv_dtype == RLLM_DTYPE_FP8_E5M2) return launch_sparse<KIND_F16, KIND_FP8_E5M2>(a, head_dim, st);
    return launch_sparse<KIND_F16, KIND_F16>(a, head_dim, st);
}

}  // extern "C"
