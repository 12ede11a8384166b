// Decode attention over the MXFP4 KV cache, for gfx950: o = softmax(scale q K^T) V per
// (sequence, query head), for one query token a sequence, and for chunks of few (see
// mxfp4_prefill.hip, which sends them here): a sequence's query token i of n attends keys
// 0 .. seq_len - n + i.
//
// Bound by HBM: a context token of one kv head is 2 * D * 17 / 32 bytes (136 at D
// 128) against 4 D operations for each of its columns, a column being a (query token,
// query head of the group) pair.
//
// Work.  A row is up to 16 columns of a (sequence, kv head), the width of the product;
// its context is cut into items of 32 tokens (an empty context is one, so every output
// is written).  The host sees only the tables' width, so how rows go to workgroups
// comes from the lengths on the device: where the rows are alike each gets workgroups
// of its own; else the rows' items form one list, cut into equal shares.  The waves
// of a workgroup take a row's items in turn and join at the row's end in LDS.  A row cut
// between workgroups leaves partials (sum of p v relative to the piece's m, m, sum of
// p); the workgroup that completes the row's arrival counter adds the pieces in their
// order, so repeated calls give the same bits whichever comes last.  Partials are written
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
// Items are loaded one ahead of use, over a row's end too.
//
// Measured (32/8 heads, head_dim 128, bf16): 64 contexts of 128-4096 tokens, 146 MB,
// 39.1 us (3.7 TB/s); 24 of 4000-32000 (24/8 heads, f16), 506 MB, 102 us (4.95 TB/s,
// a large copy's rate); one of 700 tokens 8 us, nearly all latency: a launch, lengths, table
// entries, a part's loads, the join.
#pragma once
#include "mxfp4_attention.h"
#include "workspace.h"
#include "../../include/rllm_kernels.h"

namespace rllm {
namespace {

constexpr int MXD_ITEM = 32;          // tokens
constexpr int MXD_HEADS = 16;         // query heads a row
constexpr int MXD_MAX_PIECES = 64;    // of a row
// What a row's start and join cost beside its items, in items: a workgroup whose share
// starts more rows gets fewer.  64 contexts of 128-4096 tokens (32/8 heads, head_dim
// 128): 53.6 us without, 44 with 4, 39.5 with 8, 41 with 12.
constexpr int MXD_VIRT = 8;
// A row's pieces are joined by one workgroup, so pieces that its joining would outlast
// are not cut: a piece holds at least sqrt(items * elements / threads * this) items.
// One sequence's 4 new tokens on 8000 (32/8 heads, head_dim 128), whose 16 columns make a
// join four times a token's: 31.8 us without, 21.9 with half of this, 20.3, 21.6 with twice.
constexpr float MXD_JOIN = 0.1875f;
constexpr int MXD_JOIN_LOADS = 8;   // pieces of a join in flight: 8.6 us against 9.1 of 16, 1 context of 1024

// workgroups a CU
__host__ __device__ constexpr int mxd_per_cu(int64_t d, int waves) { return 4 * mxd_per_simd(d) / waves; }

struct MxDecodeArgs {
    uint16_t* out;
    const uint16_t* q;
    const uint8_t *kc, *vc;
    const int32_t *bt, *seq_lens;
    const int32_t* qsl;                  // chunks: their query tokens; else null
    int32_t num_seqs, num_tokens, hq, hkv;
    int32_t most_cols;                   // chunks: sequences of more columns are not for this kernel
    int32_t bs, subs;                    // tokens, 16-token parts of a block
    uint64_t subs_mul;                   // ceil(2^32 / subs)
    int32_t maxb;
    int32_t nb;
    float c;                             // scale * log2(e)
    uint32_t* counters;                  // [workgroups]
    float* part_o;                       // [2 * workgroups][16][D]
    float* part_ml;                      // [2 * workgroups][16][2]
};

// bf16 elements of a V row in LDS (a multiple of 64 bytes apart in the banks, see
// the transposing read)
template <int NB> constexpr int mxd_row() { return 32 * NB + (NB % 2 ? 0 : 32); }

// One item's operands as loaded.
template <int NB>
struct MxItem {
    static constexpr int NK = (NB + 3) / 4;     // 128-wide steps of head_dim
    static constexpr int NV = (NB + 1) / 2;     // 16-byte V chunks a lane
    uint4 k[2][NK], v[NV];
    uint32_t ke[2][NK], ve[NV];
};

// A row at hand: row r of sequence s, its first item in the list of all, its items
// (all of them, and lo .. hi - 1 of this workgroup) and keys; the sequence's n query
// tokens from q0 on, the first of them at position cached.
struct MxRow {
    int s, r, first, items, lo, hi, ctx, n, q0, cached;
};

// The columns of a row: up to 16 (query token, query head) pairs of a kv head, token
// by token, from column `col` of the sequence's.
struct MxCols {
    int h, col, count, q0;
};

// A piece of a row cut between workgroups: the row's columns, its first workgroup and its pieces.
struct Piece {
    MxCols cols;
    int first_wg, count;
};

// two floats past the XCD's own L2, as one access
__device__ __forceinline__ void store2(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void load2(const float* p, float& x, float& y) {
    const uint64_t w = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = __uint_as_float(static_cast<uint32_t>(w));
    y = __uint_as_float(static_cast<uint32_t>(w >> 32));
}

template <int QKIND, int NB, int WAVES, bool CHUNK>
__global__ __launch_bounds__(64 * WAVES, mxd_per_simd(32 * NB)) void mx4_decode_kernel(MxDecodeArgs a) {
    constexpr int THREADS = 64 * WAVES;
    constexpr int D = 32 * NB;
    constexpr int NK = MxItem<NB>::NK, NV = MxItem<NB>::NV;
    constexpr int NT = mx4_terms<QKIND>();
    constexpr int ROW = mxd_row<NB>();
    __shared__ __align__(16) uint32_t lds[WAVES * MXD_ITEM * ROW / 2];   // a V tile a wave
    __shared__ float ml_lds[WAVES][MXD_HEADS][2];
    __shared__ float w_lds[MXD_MAX_PIECES][MXD_HEADS];
    __shared__ int last_lds[2];
    __shared__ uint32_t nan_lds[WAVES][MXD_HEADS];   // chunks: value blocks that are NaN in a column

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int l16 = lane & 15, grp = lane >> 4;
    uint16_t* const v_lds = reinterpret_cast<uint16_t*>(lds) + wave * MXD_ITEM * ROW;
    const int G = a.hq / a.hkv;
    const int page_bytes = static_cast<int>(mx4_page_bytes(D, a.bs));
    const int code_bytes = a.bs * (D / 2);      // of a page
    const int width = a.maxb * a.bs;            // tokens a table can hold

    auto items_of = [&](int len) __attribute__((always_inline)) {
        return max((min(len, width) + MXD_ITEM - 1) / MXD_ITEM, 1);
    };

    // groups of 16 columns a kv head of a sequence of n query tokens has
    auto groups_of = [&](int n) __attribute__((always_inline)) { return (n * G + MXD_HEADS - 1) / MXD_HEADS; };
    // a sequence's query tokens, and the first of them
    auto tokens_of = [&](int s, int& q0) __attribute__((always_inline)) {
        if constexpr (!CHUNK) {
            q0 = s;
            return 1;
        } else {
            q0 = a.qsl[s];
            const int n = a.qsl[s + 1] - q0;
            return n * G <= a.most_cols ? n : 0;
        }
    };
    auto open_row = [&](MxRow& x, int len) __attribute__((always_inline)) {
        x.items = items_of(len);
        x.ctx = min(max(len, 0), width);
        x.cached = max(len, 0) - x.n;
    };

    MxRow row{};
    int virt = 0;     // items a row's start counts for in the list; -1: rows are cut apart
    int end, share;   // the end of this workgroup's items in the list, and the items of a workgroup
    {
        // ---- the share: every wave works it out from the lengths.  Those of up to 64
        // sequences are read once ----
        const int len0 = a.seq_lens[min(lane, a.num_seqs - 1)];
        auto len_at = [&](int s0) __attribute__((always_inline)) {
            return s0 == 0 ? len0 : a.seq_lens[min(s0 + lane, a.num_seqs - 1)];
        };
        auto rows_at = [&](int s0) __attribute__((always_inline)) {   // of sequence s0 + lane
            int q0;
            return s0 + lane < a.num_seqs ? a.hkv * groups_of(tokens_of(min(s0 + lane, a.num_seqs - 1), q0)) : 0;
        };
        int total = 0, longest = 1, all_rows = 0;
        for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
            if constexpr (CHUNK) {   // starts that fall or leave the batch: nothing below would hold
                const int s = min(s0 + lane, a.num_seqs - 1), q0 = a.qsl[s], q1 = a.qsl[s + 1];
                if (__builtin_amdgcn_ballot_w64(q0 < 0 || q1 < q0 || q1 > a.num_tokens)) return;   // whole workgroup
            }
            const int rows = rows_at(s0), n = rows ? items_of(len_at(s0)) : 0;
            total += __builtin_amdgcn_readlane(mx4_scan(rows * n), 63);
            all_rows += CHUNK ? __builtin_amdgcn_readlane(mx4_scan(rows), 63) : 0;
            longest = max(longest, mx4_wave_max(n));
        }
        if constexpr (!CHUNK) all_rows = a.num_seqs * a.hkv * groups_of(1);
        if (all_rows == 0) return;   // no query tokens for this kernel
        // Where each row can have `own` workgroups of its own and the longest row's part is
        // no more than an equal share of the list, starts and joins counted, every row is cut
        // at multiples of that part (or larger ones, see MXD_JOIN) and no workgroup touches two
        // rows.  Else the list is
        // cut into equal shares, a row's start in it as `virt` items.
        const int grid = gridDim.x;
        const int even = (total + MXD_VIRT * all_rows + grid - 1) / grid;
        const int own = static_cast<int>(static_cast<uint32_t>(grid) / static_cast<uint32_t>(all_rows));
        int part = own ? max((longest + own - 1) / own, max(WAVES, (longest + MXD_MAX_PIECES - 1) / MXD_MAX_PIECES)) : 0;
        const bool apart = !a.counters || (own && part <= max(even, WAVES));
        const int joins = min(CHUNK ? MXD_HEADS : G, MXD_HEADS) * D;   // elements of a row
        const int worth = static_cast<int>(__builtin_sqrtf(static_cast<float>(longest) * joins * (MXD_JOIN / THREADS)));
        part = max(part, worth);
        if (!a.counters) part = longest;   // no scratch: a workgroup a row
        int stride = 0;   // of rows cut apart
        if (apart) {
            share = __builtin_amdgcn_readfirstlane(part);
            stride = __builtin_amdgcn_readfirstlane((longest + part - 1) / part) * share;
            total = all_rows * stride;
        } else {
            virt = __builtin_amdgcn_readfirstlane(min(MXD_VIRT, even / 2));
            total += virt * all_rows;
            // n items span at most ceil(n / share) + 1 pieces
            const int least = max(max(WAVES, worth), (longest + virt + MXD_MAX_PIECES - 3) / (MXD_MAX_PIECES - 2));
            share = __builtin_amdgcn_readfirstlane(max((total + grid - 1) / grid, least));
        }
        const int64_t pos64 = static_cast<int64_t>(share) * blockIdx.x;
        if (pos64 >= total) return;   // whole workgroup
        const int pos = static_cast<int>(pos64);
        end = static_cast<int>(min<int64_t>(pos64 + share, total));
        int before = 0;   // of the list in earlier sequences
        for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
            const int raw = len_at(s0), rows = rows_at(s0);
            const int len = apart ? stride : items_of(raw) + virt;   // of a row in the list
            const int incl = mx4_scan(rows * len), first = before + incl - rows * len;
            const uint64_t hit = __builtin_amdgcn_ballot_w64(first <= pos && pos - first < rows * len);
            if (hit) {
                const int j = __ffsll(static_cast<unsigned long long>(hit)) - 1;
                row.s = s0 + j;
                const int f = __builtin_amdgcn_readlane(first, j), row_len = __builtin_amdgcn_readlane(len, j);
                row.r = static_cast<int>(static_cast<uint32_t>(pos - f) / static_cast<uint32_t>(row_len));
                row.first = f + row.r * row_len + virt;
                row.n = tokens_of(row.s, row.q0);
                open_row(row, __builtin_amdgcn_readlane(raw, j));
                break;
            }
            before += __builtin_amdgcn_readlane(incl, 63);
        }
        row.s = __builtin_amdgcn_readfirstlane(row.s);
        row.r = __builtin_amdgcn_readfirstlane(row.r);
        row.first = __builtin_amdgcn_readfirstlane(row.first);
        row.items = __builtin_amdgcn_readfirstlane(row.items);
        row.ctx = __builtin_amdgcn_readfirstlane(row.ctx);
        row.n = __builtin_amdgcn_readfirstlane(row.n);
        row.q0 = __builtin_amdgcn_readfirstlane(row.q0);
        row.cached = __builtin_amdgcn_readfirstlane(row.cached);
        row.lo = max(pos - row.first, 0);
        if (apart) virt = -1;   // no other row in this share
    }
    row.hi = min(end - row.first, row.items);

    // the row after this one, empty (lo == hi) past the share
    auto next_row = [&](const MxRow& x) __attribute__((always_inline)) -> MxRow {
        MxRow y = x;
        y.lo = 0;
        y.hi = 0;
        if (virt < 0) return y;   // rows cut apart: their strides' sum may be just below 2^31
        y.first = x.first + x.items + virt;
        if (y.first >= end) return y;
        if (++y.r == a.hkv * groups_of(x.n)) {
            y.r = 0;
            do ++y.s;   // within the batch: the list goes on
            while ((y.n = tokens_of(y.s, y.q0)) == 0);
            open_row(y, a.seq_lens[y.s]);
        }
        y.hi = min(end - y.first, y.items);
        return y;
    };
    auto cols_of = [&](const MxRow& x) __attribute__((always_inline)) -> MxCols {
        const int groups = groups_of(x.n), g = x.r % groups;
        return MxCols{x.r / groups, g * MXD_HEADS, min(x.n * G - g * MXD_HEADS, MXD_HEADS), x.q0};
    };
    // a column's query row
    auto q_row_of = [&](const MxCols& x, int c) __attribute__((always_inline)) -> int64_t {
        if constexpr (!CHUNK) return static_cast<int64_t>(x.q0) * a.hq + x.h * G + x.col + c;
        const int at = x.col + c, tok = static_cast<int>(static_cast<uint32_t>(at) / static_cast<uint32_t>(G));
        return (static_cast<int64_t>(x.q0) + tok) * a.hq + x.h * G + (at - tok * G);
    };

    // ---- this wave's items of a row are lo + wave + WAVES k.  Lane j holds the table entry
    // of 16-token part j % 2 of item k0 + j / 2, and the part's row in the page (-1: past
    // the context).  Nothing looks at the entry here: its load, a row ahead, would have
    // to be waited for ----
    struct Ids { int id, row; };
    auto load_ids = [&](const MxRow& x, int k0) __attribute__((always_inline)) -> Ids {
        const int i = x.lo + wave + WAVES * (k0 + (lane >> 1));
        const int u = 2 * i + (lane & 1);
        const int blk = static_cast<int>((static_cast<uint32_t>(u) * a.subs_mul) >> 32);
        Ids y{-1, i < x.hi && u * MX4_TOKENS < x.ctx ? (u - blk * a.subs) * MX4_TOKENS : -1};
        if (a.maxb > 0) y.id = a.bt[static_cast<int64_t>(x.s) * a.maxb + min(blk, a.maxb - 1)];
        return y;
    };
    // The same resolved for kv head h: lane j's byte offset of the part's first code
    // row in a cache, the distance from there to its first scale row, and which of the
    // parts exist (the others point to page 0, and get no weight)
    struct Parts { uint32_t lo, hi; int scales; uint64_t ok; };
    auto resolve = [&](const Ids& x, int h) __attribute__((always_inline)) -> Parts {
        const bool ok = x.row >= 0 && static_cast<uint32_t>(x.id) < static_cast<uint32_t>(a.nb);
        const int r0 = ok ? x.row : 0;
        const int64_t at = (static_cast<int64_t>(ok ? x.id : 0) * a.hkv + h) * page_bytes + r0 * (D / 2);
        return Parts{static_cast<uint32_t>(at), static_cast<uint32_t>(at >> 32), code_bytes + r0 * (NB - D / 2),
                     __builtin_amdgcn_ballot_w64(ok)};
    };
    struct Part { int64_t at; int scales; };   // uniform
    auto part_of = [&](const Parts& x, int j) __attribute__((always_inline)) -> Part {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x.lo), j);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(x.hi), j);
        return Part{static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo), __builtin_amdgcn_readlane(x.scales, j)};
    };
    // loads of an item's keys and values from its parts.  Every address lies in a page of the cache
    const uint32_t k_off = l16 * (D / 2) + 16 * grp, ke_off = l16 * NB + grp;
    auto load_k = [&](const Part& p0, const Part& p1, MxItem<NB>& x) __attribute__((always_inline)) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const Part& p = sub ? p1 : p0;
            const uint8_t *codes = a.kc + p.at, *scales = codes + p.scales;
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
    auto load_v = [&](const Part& p0, const Part& p1, MxItem<NB>& x) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            constexpr int SUB = MX4_TOKENS * NB;   // chunks of a 16-token part
            if constexpr (NB % 4 == 0) {           // a load lies in one part
                const Part& p = 64 * j >= SUB ? p1 : p0;
                const uint8_t* codes = a.vc + p.at;
                const uint32_t at_c = (64 * j) % SUB + lane;
                x.v[j] = *reinterpret_cast<const uint4*>(codes + 16 * at_c);
                x.ve[j] = (codes + p.scales)[at_c];
            } else {
                const int idx = 64 * j + lane;
                const bool second = idx >= SUB;
                const int at_c = second ? idx - SUB : idx;
                const uint8_t* codes = a.vc + (second ? p1.at : p0.at);
                x.v[j] = make_uint4(0, 0, 0, 0);
                x.ve[j] = 127;
                if (NB % 2 == 0 || idx < 2 * SUB) {
                    x.v[j] = *reinterpret_cast<const uint4*>(codes + 16 * at_c);
                    x.ve[j] = codes[(second ? p1.scales : p0.scales) + at_c];
                }
            }
        }
    };

    // transposing V read: lane's row 4 grp + l16 / 4 (and 16 more); 16-byte chunk i of
    // block b of row t lies at i ^ (b % 4) ^ (2 (t / 4 % 2)).  With rows a multiple of 64
    // bytes apart, the stores of 16 lanes (4 rows x 4 blocks) and the reads of 32 (8
    // rows x 32 bytes) are then spread over all banks.
    const int vr_row = 4 * grp + (l16 >> 2), vr_sw = 2 * (grp & 1);
    const uint16_t* const vr = v_lds + vr_row * ROW + 4 * (l16 & 1);
    const int vr_half = (l16 & 3) >> 1;

    // a row's first workgroup and pieces: one that lies in this share needs no division
    auto piece_of = [&](const MxRow& x) __attribute__((always_inline)) -> Piece {
        Piece y{cols_of(x), static_cast<int>(blockIdx.x), 1};
        if (x.lo > 0) y.first_wg = static_cast<int>(static_cast<uint32_t>(x.first) / static_cast<uint32_t>(share));
        if (x.lo > 0 || x.hi < x.items)
            y.count = static_cast<int>(static_cast<uint32_t>(x.first + x.items - 1) / static_cast<uint32_t>(share)) - y.first_wg + 1;
        return y;
    };
    Piece head{}, tail{};   // pieces of rows cut at the share's start and end

    // the query rows, 4-byte aligned: lane group g holds elements 16 g.. and 64 + 16 g..
    // of each 128-wide step (the order of the 8-bit operand)
    uint4 q_raw[NK][4];
    auto load_q = [&](const MxRow& x) __attribute__((always_inline)) {
        const MxCols cols = cols_of(x);
        const uint16_t* src = a.q + q_row_of(cols, min(l16, cols.count - 1)) * D;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d0 = 128 * kk + 64 * (i >> 1) + 16 * grp + 8 * (i & 1);
                q_raw[kk][i] = make_uint4(0, 0, 0, 0);
                if (NB % 4 == 0 || d0 < D) {
                    const mx_u32x4 w = *reinterpret_cast<const mx_u32x4*>(src + d0);
                    q_raw[kk][i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
    };

    MxItem<NB> set[2];
    uint32_t present[2] = {0, 0};   // an item's parts that exist
    Parts parts;                    // of the items whose loads go out next
    // the first two items of a row
    auto start = [&](const MxRow& x) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
            if (x.lo + wave + WAVES * b < x.hi) {
                const Part p0 = part_of(parts, 2 * b), p1 = part_of(parts, 2 * b + 1);
                load_k(p0, p1, set[b]);
                load_v(p0, p1, set[b]);
                present[b] = static_cast<uint32_t>(parts.ok >> (2 * b)) & 3u;
            }
    };
    parts = resolve(load_ids(row, 0), cols_of(row).h);
    load_q(row);
    start(row);

    while (row.lo < row.hi) {
        const MxCols cols = cols_of(row);
        const int h = cols.h, heads = cols.count;
        const MxRow nxt = next_row(row);
        const int nxt_h = cols_of(nxt).h;
        // keys this lane's column sees (a chunk's tokens: up to their own positions), and
        // those that every column of the row does
        int seen = row.ctx, seen_all = row.ctx;
        if constexpr (CHUNK) {
            const int tok = static_cast<int>(static_cast<uint32_t>(cols.col + min(l16, heads - 1)) / static_cast<uint32_t>(G));
            seen = min(seen, row.cached + tok + 1);
            seen_all = min(seen_all, row.cached + static_cast<int>(static_cast<uint32_t>(cols.col) / static_cast<uint32_t>(G)) + 1);
        }
        uint32_t nan_blocks = 0;   // chunks: value blocks that are NaN in this lane's column
        const Ids nxt_ids = load_ids(nxt, 0);

        // ---- the query rows as E4M3 terms ----
        mx_i32x8 qt[NT][NK];
        int qs[NT];
        {
            uint32_t amax = 0;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) amax = max(amax, mx4_amax8(q_raw[kk][i]));
            const int byte0 = mx4_query_byte<QKIND>(mx4_umax_16(amax));
            const float factor = mx4_query_factor(byte0);
#pragma unroll
            for (int t = 0; t < NT; ++t) qs[t] = mx4_term_byte(byte0, t);
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t x[NT], y[NT];
                    mx4_split4<QKIND>(q_raw[kk][i].x, q_raw[kk][i].y, factor, x);
                    mx4_split4<QKIND>(q_raw[kk][i].z, q_raw[kk][i].w, factor, y);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        qt[t][kk][2 * i] = static_cast<int>(x[t]);
                        qt[t][kk][2 * i + 1] = static_cast<int>(y[t]);
                    }
                }
        }

        mx_f32x4 o[2 * NB];   // O^T: rows 16 j + 4 grp + 0..3 of column l16
#pragma unroll
        for (int j = 0; j < 2 * NB; ++j) o[j] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;   // l: this lane's tokens only
        const int count = (row.hi - row.lo - wave + WAVES - 1) / WAVES;   // this wave's items

        // item k from set x.  As the set's registers come free, the loads of item k + 2
        // go out, or, at a row's end, of the next row's first two items
        const int nxt_count = count < 2 ? 0 : (nxt.hi - nxt.lo - wave + WAVES - 1) / WAVES;
        auto item = [&](int k, MxItem<NB>& x, uint32_t& here) __attribute__((always_inline)) {
            const bool last2 = k + 2 >= count;
            const int ahead = last2 ? k + 2 - count : k + 2;
            const bool more = !last2 || ahead < nxt_count;
            const int at = 2 * (ahead & 31);
            Part p0{}, p1{};
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
            if (last2 && ahead == 0) parts = resolve(nxt_ids, nxt_h);
            if (more) {
                if (!last2 && at == 0) parts = resolve(load_ids(row, ahead), h);   // every 32 items
                p0 = part_of(parts, at);
                p1 = part_of(parts, at + 1);
                load_k(p0, p1, x);
            }
            const int t0 = (row.lo + wave + WAVES * k) * MXD_ITEM;
            const bool full = here == 3u && t0 + MXD_ITEM <= seen_all;
            if (!full) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool ok = ((here >> (e >> 2)) & 1u) && t0 + 16 * (e >> 2) + 4 * grp + (e & 3) < seen;
                    sc[e] = ok ? sc[e] : -INFINITY;
                }
            }
            // ---- weights against m, 2^8 times the running max when it last moved, which
            // it does only when a score passes m: the outputs are rarely rescaled, and no
            // weight passes 1, so that sums of large values overflow no sooner than the
            // softmax's own ----
            const float top = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
            if (__builtin_amdgcn_ballot_w64(top > m || m == -INFINITY)) {
                const float m_new = fmaxf(m, mx4_max_16(top) + MX4_AHEAD);
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
                float f = e > MX4_TOP_SCALE ? INFINITY : mx4_factor(e);   // NaN
                if constexpr (CHUNK) {
                    // A NaN block enters with a finite factor and marks the columns that see its
                    // token: a weight of 0 would not keep NaN out of the others.
                    uint64_t bad = __builtin_amdgcn_ballot_w64(e > MX4_TOP_SCALE);
                    f = e > MX4_TOP_SCALE ? 1.f : f;
                    for (; bad; bad &= bad - 1) {
                        const int at_lane = 64 * j + __ffsll(static_cast<unsigned long long>(bad)) - 1;
                        nan_blocks |= t0 + at_lane / NB < seen ? 1u << (at_lane % NB) : 0u;
                    }
                }
                if (NB % 2 == 0 || idx < 2 * MX4_TOKENS * NB) {
                    uint4* dst = reinterpret_cast<uint4*>(v_lds + tok * ROW + 32 * b);
                    const int sw = (b & 3) ^ (2 * ((tok >> 2) & 1));
                    dst[0 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.x, f), mx4_dec_bf16<1>(w.x, f), mx4_dec_bf16<2>(w.x, f), mx4_dec_bf16<3>(w.x, f));
                    dst[1 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.y, f), mx4_dec_bf16<1>(w.y, f), mx4_dec_bf16<2>(w.y, f), mx4_dec_bf16<3>(w.y, f));
                    dst[2 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.z, f), mx4_dec_bf16<1>(w.z, f), mx4_dec_bf16<2>(w.z, f), mx4_dec_bf16<3>(w.z, f));
                    dst[3 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.w, f), mx4_dec_bf16<1>(w.w, f), mx4_dec_bf16<2>(w.w, f), mx4_dec_bf16<3>(w.w, f));
                }
            }
            if (more) {
                load_v(p0, p1, x);
                here = static_cast<uint32_t>(parts.ok >> at) & 3u;
            }
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
        if (nxt.lo < nxt.hi) load_q(nxt);
        if (count < 2) {
            parts = resolve(nxt_ids, nxt_h);
            start(nxt);
        } else if (count & 1) {
            const MxItem<NB> x = set[0];
            set[0] = set[1];
            set[1] = x;
            const uint32_t p = present[0];
            present[0] = present[1];
            present[1] = p;
        }

        // ---- the waves join: outputs and sums in LDS (each in its own V tile) ----
        l = mx4_sum_16(l);
        if (l16 < heads) {
            if (grp == 0) {
                ml_lds[wave][l16][0] = m;
                ml_lds[wave][l16][1] = l;
                if constexpr (CHUNK) nan_lds[wave][l16] = nan_blocks;
            }
            float* dst = reinterpret_cast<float*>(v_lds) + l16 * D + 4 * grp;
#pragma unroll
            for (int j = 0; j < 2 * NB; ++j) *reinterpret_cast<mx_f32x4*>(dst + 16 * j) = o[j];
        }
        __syncthreads();
        const Piece piece = piece_of(row);
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (row.lo == 0 ? 1 : 0);
        for (int e = 2 * tid; e < heads * D; e += 2 * THREADS) {
            const int hd = e / D;
            float mw[WAVES], lw[WAVES], mm = -INFINITY, ll = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                mw[w] = ml_lds[w][hd][0];
                lw[w] = ml_lds[w][hd][1];
                mm = fmaxf(mm, mw[w]);
            }
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const mx_f32x2 y = *reinterpret_cast<const mx_f32x2*>(lds + w * MXD_ITEM * ROW / 2 + e);
                if (lw[w] != 0.f) {   // a wave that saw nothing adds nothing, NaN goes on
                    const float f = __builtin_amdgcn_exp2f(mw[w] - mm);
                    ll += f * lw[w];
                    y0 += f * y[0];
                    y1 += f * y[1];
                }
            }
            if constexpr (CHUNK) {
                uint32_t nans = 0;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) nans |= nan_lds[w][hd];
                if ((nans >> (e % D / MX4_BLOCK)) & 1u) y0 = y1 = __builtin_nanf("");
            }
            if (piece.count == 1) {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                *reinterpret_cast<uint32_t*>(a.out + q_row_of(cols, hd) * D + e % D) = mx4_pack16<QKIND>(y0 * inv, y1 * inv);
            } else {
                store2(a.part_o + slot * (MXD_HEADS * D) + e, y0, y1);
                if (e == hd * D) store2(a.part_ml + slot * (2 * MXD_HEADS) + 2 * hd, mm, ll);
            }
        }
        if (piece.count > 1) {
            if (row.lo == 0) tail = piece;
            else head = piece;
        }
        __syncthreads();   // LDS is free for the next row
        row = nxt;
    }

    // ---- the share's (at most two) pieces of cut rows are counted; whoever completes
    // a row adds its pieces ----
    if (head.count == 0 && tail.count == 0) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's stores have arrived
    __syncthreads();
    if (tid == 0) {
        uint32_t n0 = 0, n1 = 0;
        if (head.count) n0 = __hip_atomic_fetch_add(a.counters + head.first_wg, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (tail.count) n1 = __hip_atomic_fetch_add(a.counters + tail.first_wg, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_lds[0] = head.count && n0 + 1 == static_cast<uint32_t>(head.count);
        last_lds[1] = tail.count && n1 + 1 == static_cast<uint32_t>(tail.count);
    }
    __syncthreads();
    for (int side = 0; side < 2; ++side) {
        if (!last_lds[side]) continue;   // uniform
        const Piece x = side ? tail : head;
        const int heads = x.cols.count;
        if (tid == 0) __hip_atomic_store(a.counters + x.first_wg, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // piece p's slot: the row starts in its first workgroup's last piece
        // (slot 2 wg + 1) and goes on in the others' first
        auto slot_of = [&](int p) __attribute__((always_inline)) { return 2 * static_cast<int64_t>(x.first_wg + p) + (p == 0 ? 1 : 0); };
        // the first pieces' outputs travel with the factors
        const int e0 = 2 * tid;
        float u[MXD_JOIN_LOADS], v[MXD_JOIN_LOADS];
        auto load_some = [&](int p0, int e) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < MXD_JOIN_LOADS; ++k)
                load2(a.part_o + slot_of(min(p0 + k, x.count - 1)) * (MXD_HEADS * D) + e, u[k], v[k]);
        };
        if (e0 < heads * D) load_some(0, e0);
        // a wave a head, a lane a piece: the pieces' factors and the row's sum
        for (int hd = wave; hd < heads; hd += WAVES) {
            float mp = -INFINITY, lp = 0.f;
            if (lane < x.count) load2(a.part_ml + slot_of(lane) * (2 * MXD_HEADS) + 2 * hd, mp, lp);
            const float top = wave_max(mp);
            // a piece that saw a key keeps a factor, however small: NaN values go on
            const float f = lp == 0.f ? 0.f : fmaxf(__builtin_amdgcn_exp2f(mp - top), MX4_LEAST);
            const float L = wave_sum(lp == 0.f ? 0.f : f * lp);
            if (lane < x.count) w_lds[lane][hd] = f;
            if (lane == 0) ml_lds[0][hd][0] = L == 0.f ? 0.f : 1.f / L;
        }
        __syncthreads();
        for (int e = e0; e < heads * D; e += 2 * THREADS) {
            const int hd = e / D;
            float y0 = 0.f, y1 = 0.f;
            for (int p0 = 0; p0 < x.count; p0 += MXD_JOIN_LOADS) {
                if (p0 > 0 || e > e0) load_some(p0, e);
#pragma unroll
                for (int k = 0; k < MXD_JOIN_LOADS; ++k) {
                    const float f = p0 + k < x.count ? w_lds[p0 + k][hd] : 0.f;
                    if (f != 0.f) {
                        y0 += f * u[k];
                        y1 += f * v[k];
                    }
                }
            }
            const float inv = ml_lds[0][hd][0];
            *reinterpret_cast<uint32_t*>(a.out + q_row_of(x.cols, hd) * D + e % D) = mx4_pack16<QKIND>(y0 * inv, y1 * inv);
        }
        __syncthreads();   // before the other row's factors
    }
}

// ---- host ----

// The arrival counters have a place of their own at the scratch's start, the same for
// every call: what one call leaves in its partials never lies under another's counters.
constexpr int64_t MXD_COUNTER_BYTES = 16384, MXD_MAX_WGS = MXD_COUNTER_BYTES / 4;
int64_t mxd_scratch_bytes(int64_t wgs, int64_t d) {
    return MXD_COUNTER_BYTES + 2 * wgs * MXD_HEADS * (d + 2) * 4;
}

// Workgroups: what the device holds, fewer where the tables hold less than one item a wave.
int64_t mxd_at_most(int64_t rows, int64_t d, int64_t bs, int64_t maxb, int cus, int waves) {
    const int64_t items = (maxb * bs + MXD_ITEM - 1) / MXD_ITEM;
    const int64_t most = rows * (items > waves ? (items + waves - 1) / waves : 1);
    int64_t held = static_cast<int64_t>(cus) * mxd_per_cu(d, waves);
    if (held > MXD_MAX_WGS) held = MXD_MAX_WGS;
    return most < held ? most : held;
}

template <int QKIND, int WAVES, bool CHUNK>
int32_t mxd_launch(const MxDecodeArgs& a, int64_t d, int64_t wgs, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(wgs)), block(64 * WAVES);
    switch (d / 32) {
#define MXD_CASE(NB) case NB: hipLaunchKernelGGL((mx4_decode_kernel<QKIND, NB, WAVES, CHUNK>), grid, block, 0, st, a); break;
        MXD_CASE(1) MXD_CASE(2) MXD_CASE(3) MXD_CASE(4) MXD_CASE(5) MXD_CASE(6) MXD_CASE(7) MXD_CASE(8)
#undef MXD_CASE
        default: return static_cast<int32_t>(hipErrorInvalidValue);
    }
    return launch_status();
}

MxDecodeArgs mxd_args(void* out, const void* q, const uint8_t* kc, const uint8_t* vc, const int32_t* bt,
                      const int32_t* seq_lens, int64_t num_seqs, int64_t hq, int64_t hkv, int64_t d, int64_t bs,
                      int64_t maxb, int64_t nb, float scale, void* ws, int64_t wgs) {
    MxDecodeArgs a{};
    a.out = static_cast<uint16_t*>(out);
    a.q = static_cast<const uint16_t*>(q);
    a.kc = kc;
    a.vc = vc;
    a.bt = bt;
    a.seq_lens = seq_lens;
    a.num_seqs = static_cast<int32_t>(num_seqs);
    a.hq = static_cast<int32_t>(hq);
    a.hkv = static_cast<int32_t>(hkv);
    a.bs = static_cast<int32_t>(bs);
    a.subs = static_cast<int32_t>(bs / MX4_TOKENS);
    a.subs_mul = ((uint64_t(1) << 32) + a.subs - 1) / a.subs;   // exact quotients below 2^23
    a.maxb = static_cast<int32_t>(maxb);
    a.nb = static_cast<int32_t>(nb);
    a.c = scale * MX4_LOG2E;
    if (ws) {
        a.counters = static_cast<uint32_t*>(ws);
        a.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + MXD_COUNTER_BYTES);
        a.part_ml = a.part_o + 2 * wgs * MXD_HEADS * d;
    }
    return a;
}

}  // namespace
}  // namespace rllm
