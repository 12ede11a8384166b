// Decode attention (one query token a sequence) over the MXFP4 KV cache, for
// gfx950: o = softmax(scale q K^T) V per (sequence, query head).
//
// Bound by HBM: a context token of one kv head is 2 * D * 17 / 32 bytes (136 at D
// 128) against 4 D G operations for its G query heads.
//
// Work.  A row is a (sequence, kv head, group of up to 16 of its query heads); its
// context is cut into items of 32 tokens (an empty context is one, so every output
// is written).  The rows' items form one list, of which every workgroup takes an
// equal share; the host sees only the tables' width, so the shares come from the
// lengths on the device.  The four waves of a workgroup take a row's items in
// turn and join at the row's end in LDS.  A row cut between workgroups leaves
// partials (sum of p v relative to the piece's max, max, sum of p); the workgroup
// that completes the row's arrival counter adds the pieces in their order, so
// repeated calls give the same bits whichever comes last.  Partials are written
// and read as relaxed agent-scope atomics, which pass by the XCDs' own L2, and each
// wave waits for its stores before the count (the order of the stream decode
// kernel's merge).
//
// A 32-token item of a wave: K's codes from memory straight into the block-scaled
// product (two 16-token products a 128-wide step); the weights stay in registers,
// the product's result layout being the next product's operand with tokens
// {4g..4g+3, 16+4g..} of lane group g; V is converted exactly to bf16 in registers
// and turned through LDS, [32 tokens][D] private to the wave, read back
// transposed.  Weights enter as two bf16 terms, p = hi + lo (16 bits against the
// output's 8 or 11), whatever the query's type: the matrix cores have the time.
// Items are loaded one ahead of use.
#include "mxfp4_attention.h"
#include "workspace.h"
#include "../../include/rllm_kernels.h"

namespace rllm {
namespace {

constexpr int MXD_WAVES = 4;
constexpr int MXD_THREADS = 64 * MXD_WAVES;
constexpr int MXD_ITEM = 32;          // tokens
constexpr int MXD_HEADS = 16;         // query heads a row
constexpr int MXD_MAX_PIECES = 64;    // of a row

// workgroups a CU: two waves a SIMD, one where a wave needs more than half its registers
__host__ __device__ constexpr int mxd_per_cu(int64_t d) { return d <= 128 ? 2 : 1; }

struct MxDecodeArgs {
    uint16_t* out;
    const uint16_t* q;
    const uint8_t *kc, *vc;
    const int32_t *bt, *seq_lens;
    int32_t num_seqs, hq, hkv, groups;   // groups of query heads a kv head
    int32_t bs, subs;                    // tokens, 16-token parts of a block
    uint64_t subs_mul;                   // ceil(2^32 / subs)
    int32_t maxb;
    int64_t nb;
    float c;                             // scale * log2(e)
    uint32_t* counters;                  // [workgroups]
    float* part_o;                       // [2 * workgroups][16][D]
    float* part_ml;                      // [2 * workgroups][16][2]
};

// bf16 elements of a V row in LDS (a multiple of 64 bytes apart in the banks, see
// the transposing read)
template <int NB> constexpr int mxd_row() { return 32 * NB + (NB % 2 ? 0 : 32); }

template <int NB>
constexpr int mxd_lds_words() {   // 4-byte words: the waves' V tiles, or their outputs at a row's end
    return MXD_WAVES * MXD_ITEM * mxd_row<NB>() / 2 > MXD_WAVES * MXD_HEADS * 32 * NB
               ? MXD_WAVES * MXD_ITEM * mxd_row<NB>() / 2
               : MXD_WAVES * MXD_HEADS * 32 * NB;
}

// One item's operands as loaded.
template <int NB>
struct MxItem {
    static constexpr int NK = (NB + 3) / 4;     // 128-wide steps of head_dim
    static constexpr int NV = (NB + 1) / 2;     // 16-byte V chunks a lane
    uint4 k[2][NK], v[NV];
    uint32_t ke[2][NK], ve[NV];
};

// A row at hand: row r of sequence s, its first item in the list of all, its items
// (all of them, and lo .. hi - 1 of this workgroup) and keys.
struct MxRow {
    int s, r, first, items, lo, hi, ctx;
};

template <int QKIND, int NB>
__global__ __launch_bounds__(MXD_THREADS, mxd_per_cu(32 * NB)) void mx4_decode_kernel(MxDecodeArgs a) {
    constexpr int D = 32 * NB;
    constexpr int NK = MxItem<NB>::NK, NV = MxItem<NB>::NV;
    constexpr int NT = mx4_terms<QKIND>();
    constexpr int ROW = mxd_row<NB>();
    __shared__ __align__(16) uint32_t lds[mxd_lds_words<NB>()];
    __shared__ float ml_lds[MXD_WAVES][MXD_HEADS][2];
    __shared__ float w_lds[MXD_MAX_PIECES][MXD_HEADS];
    __shared__ int last_lds;

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int l16 = lane & 15, grp = lane >> 4;
    uint16_t* const v_lds = reinterpret_cast<uint16_t*>(lds) + wave * MXD_ITEM * ROW;
    const int rows_seq = a.hkv * a.groups;      // rows of a sequence
    const int page_bytes = static_cast<int>(mx4_page_bytes(D, a.bs));
    const int code_bytes = a.bs * (D / 2);      // of a page
    const int width = a.maxb * a.bs;            // tokens a table can hold

    auto items_of = [&](int len) __attribute__((always_inline)) {
        return max((min(len, width) + MXD_ITEM - 1) / MXD_ITEM, 1);
    };

    MxRow row{};
    int end, share;   // the end of this workgroup's items in the list, and the items of a workgroup
    if (!a.counters) {
        // no scratch: a workgroup a row
        row.s = blockIdx.x / rows_seq;
        row.r = blockIdx.x % rows_seq;
        row.items = items_of(a.seq_lens[row.s]);
        end = share = row.items;
    } else {
        // ---- the share: every wave works it out from the lengths.  The lengths of
        // up to 64 sequences are read once ----
        int len0 = lane < a.num_seqs ? items_of(a.seq_lens[lane]) : 0;
        int total = 0, longest = 1;
        for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
            const int n = s0 == 0 ? len0 : s0 + lane < a.num_seqs ? items_of(a.seq_lens[s0 + lane]) : 0;
            total += __builtin_amdgcn_readlane(mx4_scan(n), 63);
            longest = max(longest, mx4_wave_max(n));
        }
        total *= rows_seq;
        // n items span at most ceil(n / share) + 1 pieces
        const int least = max(MXD_WAVES, (longest + MXD_MAX_PIECES - 3) / (MXD_MAX_PIECES - 2));
        share = __builtin_amdgcn_readfirstlane(max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), least));
        const int64_t pos64 = static_cast<int64_t>(share) * blockIdx.x;
        if (pos64 >= total) return;   // whole workgroup
        const int pos = static_cast<int>(pos64);
        end = static_cast<int>(min<int64_t>(pos64 + share, total));
        int before = 0;   // items of one row of each earlier sequence
        for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
            const int n = s0 == 0 ? len0 : s0 + lane < a.num_seqs ? items_of(a.seq_lens[s0 + lane]) : 0;
            const int incl = mx4_scan(n);
            const int first = (before + incl - n) * rows_seq;
            const uint64_t hit = __builtin_amdgcn_ballot_w64(n > 0 && first <= pos && pos - first < n * rows_seq);
            if (hit) {
                const int j = __ffsll(static_cast<unsigned long long>(hit)) - 1;
                row.s = s0 + j;
                row.items = __builtin_amdgcn_readlane(n, j);
                const int f = __builtin_amdgcn_readlane(first, j);
                row.r = static_cast<int>(static_cast<uint32_t>(pos - f) / static_cast<uint32_t>(row.items));
                row.first = f + row.r * row.items;
                break;
            }
            before += __builtin_amdgcn_readlane(incl, 63);
        }
        row.s = __builtin_amdgcn_readfirstlane(row.s);
        row.r = __builtin_amdgcn_readfirstlane(row.r);
        row.first = __builtin_amdgcn_readfirstlane(row.first);
        row.items = __builtin_amdgcn_readfirstlane(row.items);
        row.lo = pos - row.first;
    }
    row.hi = min(end - row.first, row.items);
    row.ctx = min(max(a.seq_lens[row.s], 0), width);

    // the row after this one, empty (lo == hi) past the share
    auto next_row = [&](const MxRow& x) __attribute__((always_inline)) -> MxRow {
        MxRow y = x;
        y.first = x.first + x.items;
        y.lo = 0;
        y.hi = 0;
        if (y.first >= end) return y;
        if (++y.r == rows_seq) {
            y.r = 0;
            ++y.s;   // within the batch: the list goes on
            const int len = a.seq_lens[y.s];
            y.items = items_of(len);
            y.ctx = min(max(len, 0), width);
        }
        y.hi = min(end - y.first, y.items);
        return y;
    };

    // ---- this wave's items of a row are lo + wave + 4 k.  Lane j holds what 16-token
    // part j % 2 of item k0 + j / 2 needs of the table: its page (-1: none, a key
    // past the context among it) and row in the page ----
    struct Ids { int id, row; };
    auto load_ids = [&](const MxRow& x, int k0) __attribute__((always_inline)) -> Ids {
        const int i = x.lo + wave + MXD_WAVES * (k0 + (lane >> 1));
        const int u = 2 * i + (lane & 1);
        const int blk = static_cast<int>((static_cast<uint32_t>(u) * a.subs_mul) >> 32);
        Ids y{-1, 0};
        if (i < x.hi && u * MX4_TOKENS < x.ctx) {
            const int id = a.bt[static_cast<int64_t>(x.s) * a.maxb + min(blk, a.maxb - 1)];
            y.id = id < a.nb ? id : -1;
            y.row = (u - blk * a.subs) * MX4_TOKENS;
        }
        return y;
    };
    struct Part { const uint8_t *k, *v; int codes, scales; bool ok; };   // pages and byte offsets, uniform
    auto part_of = [&](const Ids& ids, int at, int h) __attribute__((always_inline)) -> Part {
        const int id = __builtin_amdgcn_readlane(ids.id, at), r0 = __builtin_amdgcn_readlane(ids.row, at);
        Part p;
        p.ok = id >= 0;
        const int64_t page = (static_cast<int64_t>(max(id, 0)) * a.hkv + h) * page_bytes;
        p.k = a.kc + page;
        p.v = a.vc + page;
        p.codes = r0 * (D / 2);
        p.scales = code_bytes + r0 * NB;
        return p;
    };
    // loads of an item's keys and values; `at` its lane in ids.  Every address lies in a page of the cache
    const uint32_t k_off = l16 * (D / 2) + 16 * grp, ke_off = l16 * NB + grp;
    auto load_k = [&](const Ids& ids, int at, int h, MxItem<NB>& x) __attribute__((always_inline)) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const Part p = part_of(ids, at + sub, h);
            const uint8_t *codes = p.k + p.codes, *scales = p.k + p.scales;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                x.k[sub][kk] = make_uint4(0, 0, 0, 0);
                x.ke[sub][kk] = 127;
                if (4 * (kk + 1) <= NB || 4 * kk + grp < NB) {
                    x.k[sub][kk] = *reinterpret_cast<const uint4*>(codes + (k_off + 64 * kk));
                    x.ke[sub][kk] = scales[ke_off + 4 * kk];
                }
            }
        }
    };
    auto load_v = [&](const Ids& ids, int at, int h, MxItem<NB>& x) __attribute__((always_inline)) -> uint32_t {
        const Part p0 = part_of(ids, at, h), p1 = part_of(ids, at + 1, h);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            constexpr int SUB = MX4_TOKENS * NB;   // chunks of a 16-token part
            if constexpr (NB % 4 == 0) {           // a load lies in one part
                const Part& p = 64 * j >= SUB ? p1 : p0;
                const uint32_t at_c = (64 * j) % SUB + lane;
                x.v[j] = *reinterpret_cast<const uint4*>(p.v + p.codes + 16 * at_c);
                x.ve[j] = (p.v + p.scales)[at_c];
            } else {
                const int idx = 64 * j + lane;
                const bool second = idx >= SUB;
                const int at_c = second ? idx - SUB : idx;
                const uint8_t* page = second ? p1.v : p0.v;
                x.v[j] = make_uint4(0, 0, 0, 0);
                x.ve[j] = 127;
                if (NB % 2 == 0 || idx < 2 * SUB) {
                    x.v[j] = *reinterpret_cast<const uint4*>(page + (second ? p1.codes : p0.codes) + 16 * at_c);
                    x.ve[j] = page[(second ? p1.scales : p0.scales) + at_c];
                }
            }
        }
        return (p0.ok ? 1u : 0u) | (p1.ok ? 2u : 0u);
    };

    // transposing V read: lane's row 4 grp + l16 / 4 (and 16 more); 16-byte chunk i of
    // block b of row t lies at i ^ (b % 4) ^ (2 (t / 4 % 2)).  With rows a multiple of 64
    // bytes apart, the stores of 16 lanes (4 rows x 4 blocks) and the reads of 32 (8
    // rows x 32 bytes) are then spread over all banks.
    const int vr_row = 4 * grp + (l16 >> 2), vr_sw = 2 * (grp & 1);
    const uint16_t* const vr = v_lds + vr_row * ROW + 4 * (l16 & 1);
    const int vr_half = (l16 & 3) >> 1;

    Ids ids = load_ids(row, 0);
    MxItem<NB> set[2];
    uint32_t present[2] = {0, 0};
    // the first two items of a row
    auto start = [&](const MxRow& x, const Ids& y) __attribute__((always_inline)) {
        const int h = x.r / a.groups;
#pragma unroll
        for (int b = 0; b < 2; ++b)
            if (x.lo + wave + MXD_WAVES * b < x.hi) {
                load_k(y, 2 * b, h, set[b]);
                present[b] = load_v(y, 2 * b, h, set[b]);
            }
    };
    start(row, ids);

    while (row.lo < row.hi) {
        const int h = row.r / a.groups, hg = row.r % a.groups;
        const int g_all = a.hq / a.hkv;
        const int heads = min(g_all - hg * MXD_HEADS, MXD_HEADS);           // of this row
        const int64_t q_row = static_cast<int64_t>(row.s) * a.hq + h * g_all + hg * MXD_HEADS;
        const MxRow nxt = next_row(row);
        const Ids nxt_ids = load_ids(nxt, 0);

        // ---- the query rows as E4M3 terms: lane group g holds elements 16 g.. and
        // 64 + 16 g.. of each 128-wide step (the 8-bit operand's order) ----
        mx_i32x8 qt[NT][NK];
        int qs[NT];
        {
            const uint16_t* src = a.q + (q_row + min(l16, heads - 1)) * D;
            uint32_t raw[NK][16];
            float amax = 0.f;
            bool finite = true;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int d0 = 128 * kk + 64 * hf + 16 * grp;
                    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                    if (NB % 4 == 0 || d0 < D) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const uint32_t*>(src + d0 + 2 * j);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        raw[kk][8 * hf + j] = w[j];
                        const float lo = QKIND == KIND_BF16 ? bf16_lo(w[j]) : f16_lo(w[j]);
                        const float hi = QKIND == KIND_BF16 ? bf16_hi(w[j]) : f16_hi(w[j]);
                        finite = finite && __builtin_fabsf(lo) < INFINITY && __builtin_fabsf(hi) < INFINITY;
                        amax = fmaxf(amax, fmaxf(__builtin_fabsf(lo), __builtin_fabsf(hi)));
                    }
                }
            amax = mx4_max_16(finite ? amax : INFINITY);
            const int byte0 = mx4_query_byte(amax);
            const int shift = byte0 == 255 ? 0 : 127 - byte0;
#pragma unroll
            for (int t = 0; t < NT; ++t) qs[t] = mx4_term_byte(byte0, t);
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t w = raw[kk][2 * j + e];
                        x[2 * e] = ldexpf(QKIND == KIND_BF16 ? bf16_lo(w) : f16_lo(w), shift);
                        x[2 * e + 1] = ldexpf(QKIND == KIND_BF16 ? bf16_hi(w) : f16_hi(w), shift);
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) qt[t][kk][j] = static_cast<int>(mx4_term4(x));
                }
        }

        mx_f32x4 o[2 * NB];   // O^T: rows 16 j + 4 grp + 0..3 of column l16
#pragma unroll
        for (int j = 0; j < 2 * NB; ++j) o[j] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;   // l: this lane's tokens only
        const int count = (row.hi - row.lo - wave + MXD_WAVES - 1) / MXD_WAVES;   // this wave's items

        // item k from set x; the set's loads of item k + 2 go out as its registers come free
        auto item = [&](int k, MxItem<NB>& x, uint32_t& here) __attribute__((always_inline)) {
            const bool more = k + 2 < count;
            const int at = 2 * ((k + 2) & 31);
            // ---- scores, in units of log2 ----
            float sc[8];
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                mx_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        acc = mx4_mma16(x.k[sub][kk], qt[t][kk], acc, static_cast<int>(x.ke[sub][kk]), qs[t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[4 * sub + e] = acc[e] * a.c;
            }
            if (more) {
                if (at == 0) ids = load_ids(row, k + 2);   // every 32 items
                load_k(ids, at, h, x);
            }
            const int t0 = (row.lo + wave + MXD_WAVES * k) * MXD_ITEM;
            const bool full = here == 3u && t0 + MXD_ITEM <= row.ctx;
            if (!full) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool ok = ((here >> (e >> 2)) & 1u) && t0 + 16 * (e >> 2) + 4 * grp + (e & 3) < row.ctx;
                    sc[e] = ok ? sc[e] : -INFINITY;
                }
            }
            // ---- weights against a running max that moves only when a score
            // passes it by 2^8: no weight passes 2^8, and the outputs are rarely
            // rescaled ----
            const float top = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
            if (__builtin_amdgcn_ballot_w64(top > m + 8.f || m == -INFINITY)) {
                const float m_new = fmaxf(m, mx4_max_16(top));
                const float alpha = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
                l *= alpha;
#pragma unroll
                for (int j = 0; j < 2 * NB; ++j) o[j] *= alpha;
                m = m_new;
            }
            const float base = m == -INFINITY ? 0.f : m;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p0 = __builtin_amdgcn_exp2f(sc[2 * e] - base), p1 = __builtin_amdgcn_exp2f(sc[2 * e + 1] - base);
                l += p0 + p1;
                hi[e] = mx4_pack_bf16(p0, p1);
                lo[e] = mx4_pack_bf16(p0 - bf16_lo(hi[e]), p1 - bf16_hi(hi[e]));
            }
            // ---- V: exact bf16 rows in LDS ----
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int idx = 64 * j + lane;
                const int tok = idx / NB, b = idx % NB;
                uint4 w = x.v[j];
                uint32_t e = x.ve[j];
                if (!full) {   // rows that no query sees may hold anything: zeros
                    const bool ok = ((here >> (tok >> 4)) & 1u) && t0 + tok < row.ctx;
                    w = ok ? w : make_uint4(0, 0, 0, 0);
                    e = ok ? e : 127u;
                }
                const float f = e > MX4_TOP_SCALE ? INFINITY : mx4_factor(e);   // NaN
                if (NB % 2 == 0 || idx < 2 * MX4_TOKENS * NB) {
                    uint4* dst = reinterpret_cast<uint4*>(v_lds + tok * ROW + 32 * b);
                    const int sw = (b & 3) ^ (2 * ((tok >> 2) & 1));
                    dst[0 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.x, f), mx4_dec_bf16<1>(w.x, f), mx4_dec_bf16<2>(w.x, f), mx4_dec_bf16<3>(w.x, f));
                    dst[1 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.y, f), mx4_dec_bf16<1>(w.y, f), mx4_dec_bf16<2>(w.y, f), mx4_dec_bf16<3>(w.y, f));
                    dst[2 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.z, f), mx4_dec_bf16<1>(w.z, f), mx4_dec_bf16<2>(w.z, f), mx4_dec_bf16<3>(w.z, f));
                    dst[3 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.w, f), mx4_dec_bf16<1>(w.w, f), mx4_dec_bf16<2>(w.w, f), mx4_dec_bf16<3>(w.w, f));
                }
            }
            if (more) here = load_v(ids, at, h, x);
            // a wave's LDS accesses stay in order; the fence keeps the compiler's too
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const uint4 ph = make_uint4(hi[0], hi[1], hi[2], hi[3]), pl = make_uint4(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
            for (int j = 0; j < 2 * NB; ++j) {   // 16 elements: half j % 2 of block j / 2
                const uint16_t* src = vr + 32 * (j >> 1) + 8 * ((2 * (j & 1) + vr_half) ^ ((j >> 1) & 3) ^ vr_sw);
                const uint2 v0 = mx4_read_tr16(src), v1 = mx4_read_tr16(src + 16 * ROW);
                const uint4 vv = make_uint4(v0.x, v0.y, v1.x, v1.y);
                o[j] = mx4_mma_bf16(vv, ph, o[j]);
                o[j] = mx4_mma_bf16(vv, pl, o[j]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        };
        for (int k = 0; k < count; k += 2) {
            item(k, set[0], present[0]);
            if (k + 1 < count) item(k + 1, set[1], present[1]);
        }
        // the next row's first loads travel while the waves join
        ids = nxt_ids;
        start(nxt, ids);

        // ---- the waves join ----
        l = mx4_sum_16(l);
        if (grp == 0) {
            ml_lds[wave][l16][0] = m;
            ml_lds[wave][l16][1] = l;
        }
        __syncthreads();   // every wave has also left its V tile
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < MXD_WAVES; ++w) mm = fmaxf(mm, ml_lds[w][l16][0]);
#pragma unroll
        for (int w = 0; w < MXD_WAVES; ++w) {
            const float mw = ml_lds[w][l16][0], lw = ml_lds[w][l16][1];
            ll += lw == 0.f ? 0.f : lw * __builtin_amdgcn_exp2f(mw - mm);
        }
        {
            const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - mm);
            float* dst = reinterpret_cast<float*>(lds) + (wave * MXD_HEADS + l16) * D + 4 * grp;
            if (l16 < heads) {
#pragma unroll
                for (int j = 0; j < 2 * NB; ++j) {
                    const mx_f32x4 y = f == 0.f ? mx_f32x4{0.f, 0.f, 0.f, 0.f} : o[j] * f;
                    *reinterpret_cast<mx_f32x4*>(dst + 16 * j) = y;
                }
            }
        }
        // sums of the row's heads beside the outputs
        if (wave == 0 && grp == 0) {
            w_lds[0][l16] = mm;
            w_lds[1][l16] = ll;
        }
        __syncthreads();
        const float* o_lds = reinterpret_cast<const float*>(lds);
        const int first_wg = static_cast<int>(static_cast<uint32_t>(row.first) / static_cast<uint32_t>(share));
        const int pieces = static_cast<int>(static_cast<uint32_t>(row.first + row.items - 1) / static_cast<uint32_t>(share)) - first_wg + 1;
        const bool whole = pieces == 1;
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (row.lo == 0 ? 1 : 0);
        for (int e = 2 * tid; e < heads * D; e += 2 * MXD_THREADS) {
            const int hd = e / D;
            float y0 = 0.f, y1 = 0.f;
#pragma unroll
            for (int w = 0; w < MXD_WAVES; ++w) {
                const mx_f32x2 y = *reinterpret_cast<const mx_f32x2*>(o_lds + w * MXD_HEADS * D + e);
                y0 += y[0];
                y1 += y[1];
            }
            if (whole) {
                const float L = w_lds[1][hd];
                const float inv = L == 0.f ? 0.f : 1.f / L;
                *reinterpret_cast<uint32_t*>(a.out + q_row * D + e) = mx4_pack16<QKIND>(y0 * inv, y1 * inv);
            } else {
                __hip_atomic_store(reinterpret_cast<uint64_t*>(a.part_o + slot * (MXD_HEADS * D) + e),
                                   static_cast<uint64_t>(__float_as_uint(y1)) << 32 | __float_as_uint(y0),
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        if (!whole) {
            if (tid < 2 * MXD_HEADS)
                __hip_atomic_store(a.part_ml + slot * (2 * MXD_HEADS) + tid, w_lds[tid & 1][tid >> 1], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's stores have arrived
            __syncthreads();
            if (tid == 0) {
                const uint32_t n = __hip_atomic_fetch_add(a.counters + first_wg, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last_lds = n + 1 == static_cast<uint32_t>(pieces);
            }
            __syncthreads();
            if (last_lds) {
                if (tid == 0) __hip_atomic_store(a.counters + first_wg, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                // piece p's slot: the row starts in its first workgroup's last
                // piece (slot 2 wg + 1) and goes on in the others' first
                auto slot_of = [&](int p) __attribute__((always_inline)) { return 2 * static_cast<int64_t>(first_wg + p) + (p == 0 ? 1 : 0); };
                // a wave a head, a lane a piece: the pieces' factors and the row's sum
                for (int hd = wave; hd < heads; hd += MXD_WAVES) {
                    float mp = -INFINITY, lp = 0.f;
                    if (lane < pieces) {
                        const float* src = a.part_ml + slot_of(lane) * (2 * MXD_HEADS) + 2 * hd;
                        mp = __hip_atomic_load(src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        lp = __hip_atomic_load(src + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                    const float top = wave_max(mp);
                    const float f = lp == 0.f ? 0.f : __builtin_amdgcn_exp2f(mp - top);
                    const float L = wave_sum(lp == 0.f ? 0.f : f * lp);
                    if (lane < pieces) w_lds[lane][hd] = f;
                    if (lane == 0) ml_lds[0][hd][0] = L == 0.f ? 0.f : 1.f / L;
                }
                __syncthreads();
                for (int e = 2 * tid; e < heads * D; e += 2 * MXD_THREADS) {
                    const int hd = e / D;
                    float y0 = 0.f, y1 = 0.f;
                    for (int p0 = 0; p0 < pieces; p0 += 8) {
                        uint64_t w[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            w[k] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(
                                                         a.part_o + slot_of(min(p0 + k, pieces - 1)) * (MXD_HEADS * D) + e),
                                                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float f = p0 + k < pieces ? w_lds[p0 + k][hd] : 0.f;
                            if (f != 0.f) {   // a piece that saw nothing adds nothing, NaN goes on
                                y0 += f * __uint_as_float(static_cast<uint32_t>(w[k]));
                                y1 += f * __uint_as_float(static_cast<uint32_t>(w[k] >> 32));
                            }
                        }
                    }
                    const float inv = ml_lds[0][hd][0];
                    *reinterpret_cast<uint32_t*>(a.out + q_row * D + e) = mx4_pack16<QKIND>(y0 * inv, y1 * inv);
                }
            }
        }
        __syncthreads();   // LDS is free for the next row
        row = nxt;
    }
}

// ---- host ----

// Bytes of the arrival counters, and of all scratch, for `wgs` workgroups.
int64_t mxd_counter_bytes(int64_t wgs) { return (wgs * 4 + 255) & ~int64_t(255); }
int64_t mxd_scratch_bytes(int64_t wgs, int64_t d) {
    return mxd_counter_bytes(wgs) + 2 * wgs * MXD_HEADS * (d + 2) * 4;
}

// Workgroups: what the device holds, fewer where the tables hold less than one item a wave.
int32_t mxd_workgroups(int64_t num_seqs, int64_t hq, int64_t hkv, int64_t d, int64_t bs, int64_t maxb, int64_t* wgs) {
    int dev = 0, cus = 0;
    RLLM_TRY(hipGetDevice(&dev));
    RLLM_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    const int64_t groups = (hq / hkv + MXD_HEADS - 1) / MXD_HEADS, rows = num_seqs * hkv * groups;
    const int64_t items = (maxb * bs + MXD_ITEM - 1) / MXD_ITEM;
    const int64_t most = rows * ((items + MXD_WAVES - 1) / MXD_WAVES > 0 ? (items + MXD_WAVES - 1) / MXD_WAVES : 1);
    const int64_t held = static_cast<int64_t>(cus) * mxd_per_cu(d);
    *wgs = most < held ? most : held;
    return 0;
}

int32_t mxd_check(int64_t num_seqs, int64_t hq, int64_t hkv, int64_t d, int64_t bs, int64_t maxb, int64_t nb) {
    RLLM_CHECK_ARG(mx4_shape_ok(hkv, d, bs, nb));
    RLLM_CHECK_ARG(mx4_attention_ok(num_seqs, hq, hkv, bs, maxb));
    // the items of all rows are counted in 32 bits
    const int64_t rows = num_seqs * hkv * ((hq / hkv + MXD_HEADS - 1) / MXD_HEADS);
    RLLM_CHECK_ARG(rows * ((maxb * bs + MXD_ITEM - 1) / MXD_ITEM + 1) <= INT32_MAX);
    return 0;
}

template <int QKIND>
int32_t mxd_launch(const MxDecodeArgs& a, int64_t d, int64_t wgs, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(wgs)), block(MXD_THREADS);
    switch (d / 32) {
#define MXD_CASE(NB) case NB: hipLaunchKernelGGL((mx4_decode_kernel<QKIND, NB>), grid, block, 0, st, a); break;
        MXD_CASE(1) MXD_CASE(2) MXD_CASE(3) MXD_CASE(4) MXD_CASE(5) MXD_CASE(6) MXD_CASE(7) MXD_CASE(8)
#undef MXD_CASE
        default: return static_cast<int32_t>(hipErrorInvalidValue);
    }
    return launch_status();
}

}  // namespace
}  // namespace rllm

using namespace rllm;

extern "C" {

int64_t rllm_paged_attention_decode_mxfp4_workspace_size(int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads,
                                                         int64_t head_dim, int64_t block_size,
                                                         int64_t max_num_blocks_per_seq) {
    if (num_seqs <= 0) return 0;
    if (mxd_check(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, 0)) return -1;
    int64_t wgs = 0;
    if (mxd_workgroups(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, &wgs)) return -1;
    return mxd_scratch_bytes(wgs, head_dim);
}

int32_t rllm_paged_attention_decode_mxfp4(void* output, const void* query, const uint8_t* key_cache,
                                          const uint8_t* value_cache, const int32_t* block_tables,
                                          const int32_t* seq_lens, int64_t num_seqs, int64_t num_q_heads,
                                          int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                          int64_t max_num_blocks_per_seq, int64_t num_blocks, float scale,
                                          int32_t q_dtype, void* workspace, int64_t workspace_bytes,
                                          uintptr_t stream) {
    if (num_seqs <= 0) return 0;
    RLLM_CHECK_ARG(output && query && key_cache && value_cache && block_tables && seq_lens);
    const int32_t bad = mxd_check(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, num_blocks);
    if (bad) return bad;
    RLLM_CHECK_ARG(num_blocks > 0);
    RLLM_CHECK_ARG(q_dtype == RLLM_DTYPE_F16 || q_dtype == RLLM_DTYPE_BF16);
    RLLM_CHECK_ARG(std::isfinite(scale));
    RLLM_CHECK_ARG(mx4_aligned16(key_cache) && mx4_aligned16(value_cache));
    RLLM_CHECK_ARG(((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(output)) & 3) == 0);
    int64_t wgs = 0;
    const int32_t rc = mxd_workgroups(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, &wgs);
    if (rc) return rc;
    const int64_t need = mxd_scratch_bytes(wgs, head_dim);
    void* ws = workspace;
    if (ws) {
        RLLM_CHECK_ARG(mx4_aligned16(ws) && workspace_bytes >= need);
    } else {
        RLLM_TRY(static_cast<hipError_t>(g_workspaces.get(stream, WS_MX4_DECODE, need, true, &ws)));
        if (!ws) {   // captured before any eager call of this size: a workgroup a row
            wgs = num_seqs * num_kv_heads * ((num_q_heads / num_kv_heads + MXD_HEADS - 1) / MXD_HEADS);
            RLLM_CHECK_ARG(wgs <= INT32_MAX);
        }
    }
    MxDecodeArgs a{};
    a.out = static_cast<uint16_t*>(output);
    a.q = static_cast<const uint16_t*>(query);
    a.kc = key_cache;
    a.vc = value_cache;
    a.bt = block_tables;
    a.seq_lens = seq_lens;
    a.num_seqs = static_cast<int32_t>(num_seqs);
    a.hq = static_cast<int32_t>(num_q_heads);
    a.hkv = static_cast<int32_t>(num_kv_heads);
    a.groups = static_cast<int32_t>((num_q_heads / num_kv_heads + MXD_HEADS - 1) / MXD_HEADS);
    a.bs = static_cast<int32_t>(block_size);
    a.subs = static_cast<int32_t>(block_size / MX4_TOKENS);
    a.subs_mul = ((uint64_t(1) << 32) + a.subs - 1) / a.subs;   // exact quotients below 2^23
    a.maxb = static_cast<int32_t>(max_num_blocks_per_seq);
    a.nb = num_blocks;
    a.c = scale * MX4_LOG2E;
    if (ws) {
        a.counters = static_cast<uint32_t*>(ws);
        a.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + mxd_counter_bytes(wgs));
        a.part_ml = a.part_o + 2 * wgs * MXD_HEADS * head_dim;
    }
    return q_dtype == RLLM_DTYPE_BF16 ? mxd_launch<KIND_BF16>(a, head_dim, wgs, as_stream(stream))
                                      : mxd_launch<KIND_F16>(a, head_dim, wgs, as_stream(stream));
}

}  // extern "C"
