// Chunked-prefill attention over the MXFP4 KV cache, for gfx950: query token i of
// a sequence's n new ones sits at position seq_len - n + i and attends keys
// 0 .. that position (the new tokens' rows are in the cache already).
//
// Bound by the matrix cores: 4 D operations a (query head, key) pair against 17/16 D
// bytes a key of a kv head, read once per 256 query rows.
//
// Work.  The rows of a (sequence, kv head) are its (token, query head of the
// group) pairs, token by token; a workgroup takes 32 rows a wave.  Keys go by in
// tiles of 64 tokens, staged in LDS by all waves: K's code rows as they are
// ([32-element block][token][16 bytes], one scale byte each), V converted exactly to
// bf16 ([token][D]).  A wave's products: S^T = K Q^T on the block-scaled 32x32x64
// product (A = K from LDS, B = the query terms in registers), so lane l holds the
// scores of row l % 32; the softmax stays in the lane and its partner l ^ 32; the
// weights, rounded to bf16, are the B operand of O^T = V^T P^T as they stand, with V
// read back from LDS transposed.  f16 queries take two terms a weight (16 bits
// against the output's 11); bf16 ones one, like the 16-bit caches' kernel: an error
// of at most half a bf16 step a weight, the size of the output's own rounding.
#include "mxfp4_attention.h"
#include "workspace.h"
#include "../../include/rllm_kernels.h"

namespace rllm {
namespace {

constexpr int MXP_TILE = 64;    // keys
constexpr int MXP_SUBS = MXP_TILE / MX4_TOKENS;

// 8 waves, two a SIMD, up to head_dim 128; past it a wave needs the registers of two
template <int NB> constexpr int mxp_waves() { return NB <= 4 ? 8 : 4; }

struct MxPrefillArgs {
    uint16_t* out;
    const uint16_t* q;
    const uint8_t *kc, *vc;
    const int32_t *bt, *seq_lens, *qsl;
    int32_t num_seqs, num_tokens, hq, hkv;
    int32_t bs, subs;       // tokens, 16-token parts of a block
    uint64_t subs_mul;      // ceil(2^32 / subs)
    int32_t maxb;
    int64_t nb;
    float c;                // scale * log2(e)
    int32_t splits, base_wgs;
    float* part_o;          // [num_tokens * hq][splits][D], relative to the part's max
    float* part_ml;         // [num_tokens * hq][splits][2]
};

// bf16 elements of a V row in LDS: four consecutive rows of a transposing read
// (64 bytes each) on different banks
template <int NB> constexpr int mxp_row() { return 32 * NB + (NB % 2 ? 0 : 32); }

template <int NB>
struct MxTile {   // one buffer
    uint4 k[NB][MXP_TILE];
    uint16_t v[MXP_TILE][mxp_row<NB>()];
    uint8_t ke[NB][MXP_TILE];
    uint8_t bad[NB][MXP_TILE];   // V blocks that are NaN
    int32_t bad_tile;            // the last tile here that had one
};

template <int QKIND, int NB>
__global__ __launch_bounds__(64 * mxp_waves<NB>(), 8 / (NB <= 4 ? 4 : 8)) void mx4_prefill_kernel(
    MxPrefillArgs a, const int32_t* __restrict__ bt) {
    constexpr int D = 32 * NB, WAVES = mxp_waves<NB>(), THREADS = 64 * WAVES, ROWS = 32 * WAVES;
    constexpr int NKS = (NB + 1) / 2;             // 64-wide steps of head_dim
    constexpr int NT = mx4_terms<QKIND>();
    constexpr int PT = QKIND == KIND_BF16 ? 1 : 2;   // terms of a weight
    constexpr int CHUNKS = 2 * MXP_TILE * NB;     // 16-byte chunks of a tile, K's then V's
    constexpr int NCH = (CHUNKS + THREADS - 1) / THREADS;
    constexpr int ROW = mxp_row<NB>();
    __shared__ __align__(16) MxTile<NB> tiles[2];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int l32 = lane & 31, hl = lane >> 5;
    const int G = a.hq / a.hkv;

    // ---- which (kv head, sequence, query tile): a sequence's last tile first ----
    const int base = a.splits > 1 ? blockIdx.x % a.base_wgs : blockIdx.x;
    const int split = a.splits > 1 ? blockIdx.x / a.base_wgs : 0;
    const int h = base % a.hkv;
    int j = base / a.hkv;
    int s = -1, q0 = 0, n = 0, tile = 0;
    for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
        int q0_l = 0, n_l = 0;
        if (s0 + lane < a.num_seqs) {
            q0_l = min(max(a.qsl[s0 + lane], 0), a.num_tokens);
            n_l = min(max(a.qsl[s0 + lane + 1], q0_l), a.num_tokens) - q0_l;
        }
        const int nt_l = static_cast<int>((static_cast<int64_t>(n_l) * G + ROWS - 1) / ROWS);
        const int incl = mx4_scan(nt_l);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(incl - nt_l <= j && j < incl);
        if (hit) {
            const int k = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            s = s0 + k;
            q0 = __builtin_amdgcn_readlane(q0_l, k);
            n = __builtin_amdgcn_readlane(n_l, k);
            tile = __builtin_amdgcn_readlane(incl, k) - 1 - j;
            break;
        }
        j -= __builtin_amdgcn_readlane(incl, 63);
    }
    if (s < 0) return;   // whole workgroup
    s = __builtin_amdgcn_readfirstlane(s);
    const int ctx = min(max(a.seq_lens[s], 0), a.maxb * a.bs);
    const int cached = max(a.seq_lens[s], 0) - n;  // position of the first new token
    const int rows = n * G;
    const int last_tok = (min((tile + 1) * ROWS, rows) - 1) / G;
    const int kv_end = min(max(cached + last_tok + 1, 0), ctx);
    const int ntiles = (kv_end + MXP_TILE - 1) / MXP_TILE;
    const int per = (ntiles + a.splits - 1) / a.splits;
    const int t_lo = min(ntiles, split * per), t_hi = min(ntiles, t_lo + per);

    // ---- this lane's row ----
    const int row = tile * ROWS + 32 * wave + l32;
    const bool live = row < rows;
    const int tok = (live ? row : rows - 1) / G;
    const int pos = cached + tok;                  // below 0: attends nothing
    const int64_t orow = (static_cast<int64_t>(q0) + tok) * a.hq + h * G + ((live ? row : rows - 1) - tok * G);
    const bool wave_live = tile * ROWS + 32 * wave < rows;   // uniform
    // the smallest position among the wave's rows: its first row's
    const int min_pos = __builtin_amdgcn_readfirstlane(pos);

    // ---- staging ----
    const int64_t page_bytes = mx4_page_bytes(D, a.bs);
    const int code_bytes = a.bs * (D / 2);
    const int32_t* bt_row = bt + static_cast<int64_t>(s) * a.maxb;
    struct Ids { int id[MXP_SUBS]; int row[MXP_SUBS]; };
    auto load_ids = [&](int t, Ids& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MXP_SUBS; ++i) {
            const int u = t * MXP_SUBS + i;
            const int blk = static_cast<int>((static_cast<uint32_t>(u) * a.subs_mul) >> 32);
            const bool in = u * MX4_TOKENS < kv_end;
            const int id = in ? bt_row[min(blk, a.maxb - 1)] : -1;
            x.id[i] = id >= 0 && id < a.nb ? id : -1;
            x.row[i] = in ? (u - blk * a.subs) * MX4_TOKENS : 0;
        }
    };
    auto presence = [&](const Ids& x) __attribute__((always_inline)) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < MXP_SUBS; ++i) m |= x.id[i] >= 0 ? 1u << i : 0u;
        return m;
    };
    struct Raw { uint4 w[NCH]; uint32_t e[NCH]; };
    auto fetch = [&](int t, const Ids& x, Raw& r) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int idx = c * THREADS + tid;
            const bool is_v = idx >= MXP_TILE * NB;
            const int at = is_v ? idx - MXP_TILE * NB : idx;
            const int sub = min(at / (MX4_TOKENS * NB), MXP_SUBS - 1), off = at - sub * (MX4_TOKENS * NB);
            int id = x.id[0], r0 = x.row[0];
#pragma unroll
            for (int i = 1; i < MXP_SUBS; ++i) {
                id = sub == i ? x.id[i] : id;
                r0 = sub == i ? x.row[i] : r0;
            }
            r.w[c] = make_uint4(0, 0, 0, 0);
            r.e[c] = 127;
            // rows past the keys any query here sees may hold anything: zeros
            const int key = t * MXP_TILE + sub * MX4_TOKENS + off / NB;
            if ((CHUNKS % THREADS == 0 || idx < CHUNKS) && id >= 0 && key < kv_end) {
                const uint8_t* page = (is_v ? a.vc : a.kc) + (static_cast<int64_t>(id) * a.hkv + h) * page_bytes;
                r.w[c] = *reinterpret_cast<const uint4*>(page + r0 * (D / 2) + 16 * off);
                r.e[c] = page[code_bytes + r0 * NB + off];
            }
        }
    };
    auto store = [&](int t, const Raw& r, MxTile<NB>& buf) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int idx = c * THREADS + tid;
            if (CHUNKS % THREADS != 0 && idx >= CHUNKS) continue;
            const bool is_v = idx >= MXP_TILE * NB;
            const int at = is_v ? idx - MXP_TILE * NB : idx;
            const int key = at / NB, b = at % NB;
            if (!is_v) {
                buf.k[b][key] = r.w[c];
                buf.ke[b][key] = static_cast<uint8_t>(r.e[c]);
            } else {
                // A NaN block enters as zeros and marks its token: a weight of 0
                // for a key that a row does not see would not keep it out.
                const bool bad = r.e[c] > MX4_TOP_SCALE;
                const uint4 w = r.w[c];
                const float f = bad ? 0.f : mx4_factor(r.e[c]);
                // 16-byte chunk i of block b lies at i ^ (b % 4): the 16 lanes of a
                // store (4 keys x 4 blocks, rows 64 bytes apart in the banks) then
                // cover all banks
                uint4* dst = reinterpret_cast<uint4*>(&buf.v[key][32 * b]);
                const int sw = b & 3;
                dst[0 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.x, f), mx4_dec_bf16<1>(w.x, f), mx4_dec_bf16<2>(w.x, f), mx4_dec_bf16<3>(w.x, f));
                dst[1 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.y, f), mx4_dec_bf16<1>(w.y, f), mx4_dec_bf16<2>(w.y, f), mx4_dec_bf16<3>(w.y, f));
                dst[2 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.z, f), mx4_dec_bf16<1>(w.z, f), mx4_dec_bf16<2>(w.z, f), mx4_dec_bf16<3>(w.z, f));
                dst[3 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.w, f), mx4_dec_bf16<1>(w.w, f), mx4_dec_bf16<2>(w.w, f), mx4_dec_bf16<3>(w.w, f));
                buf.bad[b][key] = bad;
                if (bad) buf.bad_tile = t;
            }
        }
    };
    if (tid == 0) tiles[0].bad_tile = tiles[1].bad_tile = -1;

    Ids ids;
    Raw raw;
    uint32_t present = 0, next_present = 0;
    if (t_lo < t_hi) {
        load_ids(t_lo, ids);
        fetch(t_lo, ids, raw);
        present = presence(ids);
    }

    // ---- the query row as E4M3 terms: lane group hl holds elements 16 hl.. and
    // 32 + 16 hl.. of each 64-wide step ----
    mx_i32x8 qt[NT][NKS];
    int qs[NT];
    {
        const uint16_t* src = a.q + orow * D;
        uint4 w[NKS][4];
        uint32_t amax = 0;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d0 = 64 * ks + 32 * (i >> 1) + 16 * hl + 8 * (i & 1);
                w[ks][i] = make_uint4(0, 0, 0, 0);
                if (NB % 2 == 0 || 64 * ks + 32 * (i >> 1) < D) w[ks][i] = *reinterpret_cast<const uint4*>(src + d0);
                amax = max(amax, mx4_amax8(w[ks][i]));
            }
        const int byte0 = mx4_query_byte<QKIND>(mx4_umax_32(amax));
        const float factor = mx4_query_factor(byte0);
#pragma unroll
        for (int t = 0; t < NT; ++t) qs[t] = mx4_term_byte(byte0, t);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t x[NT], y[NT];
                mx4_split4<QKIND>(w[ks][i].x, w[ks][i].y, factor, x);
                mx4_split4<QKIND>(w[ks][i].z, w[ks][i].w, factor, y);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    qt[t][ks][2 * i] = static_cast<int>(x[t]);
                    qt[t][ks][2 * i + 1] = static_cast<int>(y[t]);
                }
            }
    }

    mx_f32x16 o[NB];   // O^T: elements 32 dt + 8 (i / 4) + 4 hl + i % 4 of row l32
#pragma unroll
    for (int dt = 0; dt < NB; ++dt) o[dt] = mx_f32x16{};
    float m = -INFINITY, l = 0.f;   // l: this lane's keys only
    uint32_t nan_blocks = 0;        // output blocks made NaN by a value the row sees

    __syncthreads();   // bad_tile is set
    if (t_lo < t_hi) store(t_lo, raw, tiles[0]);
    if (t_lo + 1 < t_hi) {
        load_ids(t_lo + 1, ids);
        fetch(t_lo + 1, ids, raw);
        next_present = presence(ids);
    }
    __syncthreads();

    // transposing V read: row 4 hl + (lane % 16) / 4, 16 elements from 16 ((lane / 16) & 1) of a block
    const int v_row = 4 * hl + ((lane & 15) >> 2);
    const int v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), v_in = 4 * (lane & 1);

    for (int t = t_lo; t < t_hi; ++t) {
        MxTile<NB>& buf = tiles[(t - t_lo) & 1];
        if (wave_live) {
            // ---- scores ----
            mx_f32x16 st[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                st[half] = mx_f32x16{};
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) {
                    const int b = 2 * ks + hl;
                    const bool have = NB % 2 == 0 || b < NB;
                    const uint4 kk = buf.k[have ? b : 0][32 * half + l32];
                    const int e = have ? buf.ke[b][32 * half + l32] : 127;
#pragma unroll
                    for (int i = 0; i < NT; ++i) st[half] = mx4_mma32(kk, qt[i][ks], st[half], e, qs[i]);
                }
            }
            const int t0 = t * MXP_TILE;
            const bool full = present == (1u << MXP_SUBS) - 1 && t0 + MXP_TILE <= kv_end && t0 + MXP_TILE - 1 <= min_pos;
            float sc[2][16];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[half][i] = st[half][i] * a.c;
            if (!full) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = 32 * half + 8 * (i >> 2) + 4 * hl + (i & 3);
                        const bool ok = ((present >> (key >> 4)) & 1u) && t0 + key <= pos && t0 + key < kv_end;
                        sc[half][i] = ok ? sc[half][i] : -INFINITY;
                    }
            }
            if (buf.bad_tile == t) {
                for (int key = 0; key < MXP_TILE; ++key)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        nan_blocks |= t0 + key <= pos ? static_cast<uint32_t>(buf.bad[b][key]) << b : 0u;
            }
            // ---- weights against a max that moves only when passed by 2^8 ----
            float top = sc[0][0];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[half][i]);
            if (__builtin_amdgcn_ballot_w64(top > m + 8.f || m == -INFINITY)) {
                const float m_new = fmaxf(m, mx4_max_32(top));
                const float alpha = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < NB; ++dt) o[dt] *= alpha;
                m = m_new;
            }
            const float mb = m == -INFINITY ? 0.f : m;
            uint32_t p[PT][2][8];
            float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p0 = __builtin_amdgcn_exp2f(sc[half][2 * i] - mb);
                    const float p1 = __builtin_amdgcn_exp2f(sc[half][2 * i + 1] - mb);
                    sum0 += p0;
                    sum1 += p1;
                    p[0][half][i] = mx4_pack_bf16(p0, p1);
                    if constexpr (PT == 2)
                        p[1][half][i] = mx4_pack_bf16(p0 - bf16_lo(p[0][half][i]), p1 - bf16_hi(p[0][half][i]));
                }
            l += sum0 + sum1;
            // ---- O^T += V^T P^T, 16 keys a step ----
#pragma unroll
            for (int k16 = 0; k16 < MXP_TILE / 16; ++k16) {
                uint4 pb[PT];
#pragma unroll
                for (int i = 0; i < PT; ++i) {
                    const uint32_t* w = &p[i][k16 >> 1][4 * (k16 & 1)];
                    pb[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
#pragma unroll
                for (int dt = 0; dt < NB; ++dt) {
                    const uint16_t* src = &buf.v[16 * k16 + v_row][32 * dt + 8 * (v_chunk ^ (dt & 3)) + v_in];
                    const uint2 v0 = mx4_read_tr16(src), v1 = mx4_read_tr16(src + 8 * ROW);
                    const uint4 vv = make_uint4(v0.x, v0.y, v1.x, v1.y);
#pragma unroll
                    for (int i = 0; i < PT; ++i) o[dt] = mx4_mma32_bf16(vv, pb[i], o[dt]);
                }
            }
        }
        MxTile<NB>& next = tiles[(t - t_lo + 1) & 1];
        if (t + 1 < t_hi) store(t + 1, raw, next);
        present = next_present;
        if (t + 2 < t_hi) {
            load_ids(t + 2, ids);
            fetch(t + 2, ids, raw);
            next_present = presence(ids);
        }
        __syncthreads();
    }
    if (!wave_live) return;   // no barrier follows

    l = mx4_sum_32(l);
    if (!live) return;
    const float nan = __builtin_nanf("");
    if (a.splits > 1) {
        const int64_t slot = orow * a.splits + split;
        float* dst = a.part_o + slot * D + 4 * hl;
#pragma unroll
        for (int dt = 0; dt < NB; ++dt)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                mx_f32x4 y = {o[dt][4 * jj], o[dt][4 * jj + 1], o[dt][4 * jj + 2], o[dt][4 * jj + 3]};
                if ((nan_blocks >> dt) & 1u) y = mx_f32x4{nan, nan, nan, nan};
                *reinterpret_cast<mx_f32x4*>(dst + 32 * dt + 8 * jj) = y;
            }
        if (hl == 0) *reinterpret_cast<mx_f32x2*>(a.part_ml + 2 * slot) = mx_f32x2{m, l};
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* dst = a.out + orow * D + 4 * hl;
#pragma unroll
    for (int dt = 0; dt < NB; ++dt) {
        const float f = (nan_blocks >> dt) & 1u ? nan : inv;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
            *reinterpret_cast<uint2*>(dst + 32 * dt + 8 * jj) =
                make_uint2(mx4_pack16<QKIND>(o[dt][4 * jj] * f, o[dt][4 * jj + 1] * f),
                           mx4_pack16<QKIND>(o[dt][4 * jj + 2] * f, o[dt][4 * jj + 3] * f));
    }
}

// Adds the parts of every row in their order: a wave a row.
template <int QKIND>
__global__ __launch_bounds__(256) void mx4_prefill_merge_kernel(MxPrefillArgs a, int64_t rows, int d) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (r >= rows) return;
    const int64_t tok = r / a.hq;
    if (tok < a.qsl[0] || tok >= a.qsl[a.num_seqs]) return;   // no sequence's token: its output stays
    float mp = -INFINITY, lp = 0.f;
    if (lane < a.splits) {
        const mx_f32x2 x = *reinterpret_cast<const mx_f32x2*>(a.part_ml + 2 * (r * a.splits + lane));
        mp = x[0];
        lp = x[1];
    }
    const float top = wave_max(mp);
    const float f = lp == 0.f ? 0.f : __builtin_amdgcn_exp2f(mp - top);
    const float L = wave_sum(lp == 0.f ? 0.f : f * lp);
    const int d0 = 4 * lane;
    if (d0 >= d) return;
    mx_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const float* po = a.part_o + r * a.splits * d + d0;
    for (int i = 0; i < a.splits; ++i) {
        const float fi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), i));
        if (fi != 0.f) acc += fi * *reinterpret_cast<const mx_f32x4*>(po + static_cast<int64_t>(i) * d);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    *reinterpret_cast<uint2*>(a.out + r * d + d0) =
        make_uint2(mx4_pack16<QKIND>(acc[0] * inv, acc[1] * inv), mx4_pack16<QKIND>(acc[2] * inv, acc[3] * inv));
}

// ---- host ----

template <int QKIND>
int32_t mxp_launch(const MxPrefillArgs& a, int64_t d, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(a.base_wgs) * static_cast<unsigned>(a.splits));
    switch (d / 32) {
#define MXP_CASE(NB)                                                                                              \
    case NB:                                                                                                      \
        hipLaunchKernelGGL((mx4_prefill_kernel<QKIND, NB>), grid, dim3(64 * mxp_waves<NB>()), 0, st, a, a.bt);      \
        break;
        MXP_CASE(1) MXP_CASE(2) MXP_CASE(3) MXP_CASE(4) MXP_CASE(5) MXP_CASE(6) MXP_CASE(7) MXP_CASE(8)
#undef MXP_CASE
        default: return static_cast<int32_t>(hipErrorInvalidValue);
    }
    return launch_status();
}

}  // namespace
}  // namespace rllm

using namespace rllm;

extern "C" int32_t rllm_paged_attention_prefill_mxfp4(
    void* output, const void* query, const uint8_t* key_cache, const uint8_t* value_cache, const int32_t* block_tables,
    const int32_t* seq_lens, const int32_t* query_start_loc, int64_t num_seqs, int64_t num_tokens, int64_t num_q_heads,
    int64_t num_kv_heads, int64_t head_dim, int64_t block_size, int64_t max_num_blocks_per_seq, int64_t num_blocks,
    float scale, int32_t q_dtype, uintptr_t stream) {
    if (num_seqs <= 0 || num_tokens <= 0) return 0;
    RLLM_CHECK_ARG(output && query && key_cache && value_cache && block_tables && seq_lens && query_start_loc);
    RLLM_CHECK_ARG(mx4_shape_ok(num_kv_heads, head_dim, block_size, num_blocks) && num_blocks > 0);
    RLLM_CHECK_ARG(mx4_attention_ok(num_seqs, num_q_heads, num_kv_heads, block_size, max_num_blocks_per_seq));
    RLLM_CHECK_ARG(num_tokens <= (int64_t(1) << 26) && num_tokens * (num_q_heads / num_kv_heads) <= (int64_t(1) << 30));
    RLLM_CHECK_ARG(q_dtype == RLLM_DTYPE_F16 || q_dtype == RLLM_DTYPE_BF16);
    RLLM_CHECK_ARG(std::isfinite(scale));
    RLLM_CHECK_ARG(mx4_aligned16(key_cache) && mx4_aligned16(value_cache) && mx4_aligned16(query));
    RLLM_CHECK_ARG((reinterpret_cast<uintptr_t>(output) & 7) == 0);
    const int64_t group = num_q_heads / num_kv_heads, rows_wg = head_dim <= 128 ? 256 : 128;
    // a sequence's tiles are at most rows / rows_wg + 1; workgroups past the last find none
    const int64_t wgs = (num_tokens * group / rows_wg + num_seqs) * num_kv_heads;
    RLLM_CHECK_ARG(wgs <= INT32_MAX);
    MxPrefillArgs a{};
    a.out = static_cast<uint16_t*>(output);
    a.q = static_cast<const uint16_t*>(query);
    a.kc = key_cache;
    a.vc = value_cache;
    a.bt = block_tables;
    a.seq_lens = seq_lens;
    a.qsl = query_start_loc;
    a.num_seqs = static_cast<int32_t>(num_seqs);
    a.num_tokens = static_cast<int32_t>(num_tokens);
    a.hq = static_cast<int32_t>(num_q_heads);
    a.hkv = static_cast<int32_t>(num_kv_heads);
    a.bs = static_cast<int32_t>(block_size);
    a.subs = static_cast<int32_t>(block_size / MX4_TOKENS);
    a.subs_mul = ((uint64_t(1) << 32) + a.subs - 1) / a.subs;   // exact quotients below 2^23
    a.maxb = static_cast<int32_t>(max_num_blocks_per_seq);
    a.nb = num_blocks;
    a.c = scale * MX4_LOG2E;
    a.base_wgs = static_cast<int32_t>(wgs);
    a.splits = 1;
    // few query tiles over long contexts: several workgroups a tile, each on a part of the keys
    int dev = 0, cus = 0;
    RLLM_TRY(hipGetDevice(&dev));
    RLLM_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    const int64_t tiles = (max_num_blocks_per_seq * block_size + MXP_TILE - 1) / MXP_TILE;
    int64_t splits = cus / wgs;
    if (splits > tiles / 4) splits = tiles / 4;
    if (splits > 64) splits = 64;
    hipStream_t st = as_stream(stream);
    WorkspaceHold hold;
    if (splits > 1) {
        const int64_t rows = num_tokens * num_q_heads;
        void* ws = nullptr;
        RLLM_TRY(static_cast<hipError_t>(g_workspaces.get(stream, WS_MX4_PREFILL, rows * splits * (head_dim + 2) * 4, false, &ws, &hold)));
        if (ws) {   // else captured before any eager call of this size: unsplit
            a.splits = static_cast<int32_t>(splits);
            a.part_o = static_cast<float*>(ws);
            a.part_ml = a.part_o + rows * splits * head_dim;
        }
    }
    int32_t rc = q_dtype == RLLM_DTYPE_BF16 ? mxp_launch<KIND_BF16>(a, head_dim, st) : mxp_launch<KIND_F16>(a, head_dim, st);
    if (rc || a.splits == 1) return rc;
    const int64_t rows = num_tokens * num_q_heads;
    auto merge = q_dtype == RLLM_DTYPE_BF16 ? mx4_prefill_merge_kernel<KIND_BF16> : mx4_prefill_merge_kernel<KIND_F16>;
    hipLaunchKernelGGL(merge, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, st, a, rows, static_cast<int>(head_dim));
    return launch_status();
}
