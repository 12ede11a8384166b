// Chunked-prefill attention over the MXFP4 KV cache, for gfx950: query token i of
// a sequence's n new ones sits at position seq_len - n + i and attends keys
// 0 .. that position (the new tokens' rows are in the cache already).
//
// Bound by the matrix cores: 4 D operations a (query head, key) pair against 17/16 D
// bytes a key of a kv head, read once per 256 query rows.
//
// Work.  The rows of a (sequence, kv head) are its (token, query head of the
// group) pairs, token by token; a workgroup takes 32 rows a wave.  Keys go by in
// tiles of 64 tokens, staged in LDS: K's code rows as they are ([32-element
// block][token][16 bytes], one scale byte each), V converted exactly to bf16
// ([token][D]).  A wave's products: S^T = K Q^T on the block-scaled 32x32x64
// product (A = K from LDS, B = the query terms in registers), so lane l holds the
// scores of row l % 32; the softmax stays in the lane and its partner l ^ 32; the
// weights, rounded to bf16, are the B operand of O^T = V^T P^T as they stand, with V
// read back from LDS transposed.  f16 queries take two terms a weight (16 bits
// against the output's 11); bf16 ones one, like the 16-bit caches' kernel: an error
// of at most half a bf16 step a weight, the size of the output's own rounding.
//
// The waves are two groups, one a turn behind the other: while one group's wave on a
// SIMD keeps the matrix core, the other's does its softmax and its copy (group 0 brings
// V, group 1 K).  With all waves in step, staging together, 2 chunks of 1500-2048 tokens on
// 14000 took 1038 us, in turns 909 (800 after the later steps).  That holds up to head_dim
// 128.  Past it a SIMD has registers for one wave, the groups are on different SIMDs, and
// a SIMD's matrix core idles while its wave is in its softmax.
//
// Measured (32/8 heads, head_dim 128, bf16): 8 sequences of 512 new tokens on 2048, 155
// GF, 150 us (1029 TF/s); 2 of 1500-2048 on 14000, 963 GF, 800 us (1204 TF/s), where a
// large bf16 product runs at 1242 on the same card.  Replayed from a graph, us of bf16 /
// f16, whose three 8-bit query terms and two 16-bit weight terms for two and one are 1.75
// times the matrix time: the first 174 / 229, the second 817 / 1186; the first at head_dim 64 131 / 162, with 16/4
// heads at 192 193 / 232, at 224 - / 290, at 256 233 / 398.  f16 spills registers to memory at
// head_dim 64 (36 bytes a lane), 224 (68) and 256 (236), bf16 nowhere.
#include "mxfp4_attention.h"
#include "workspace.h"
#include "../../include/rllm_kernels.h"

namespace rllm {
namespace {

constexpr int MXP_TILE = 64;    // keys
constexpr int MXP_SUBS = MXP_TILE / MX4_TOKENS;
// Rounds of workgroups up to which the query tiles go by falling key counts: with
// more, the last round is a small part.
constexpr int MXP_SORTED_ROUNDS = 4;

// Sequences of few new tokens leave most of a workgroup's 256 rows empty, and stream their
// context at the pace of a single wave's turns: the decode kernel takes them, a column a
// row, 16 columns a pass over the context.
//  - In a batch that may hold both (more than one sequence, no key split, not too many
//    columns a sequence on average: past MXP_SOME_SHORT the short ones are a small part of
//    the time, and the second launch costs 3 us) each sequence goes where its own columns
//    say, up to MXP_SHORT_COLS (twice that past head_dim 128, where this kernel has one wave a
//    SIMD).  32/8 heads, head_dim 128, us of this kernel / of both: 64 sequences of 4 tokens
//    on 2000 107 / 38.7, 32 of 8 55.5 / 37.9, 256 of 4 on 500 144 / 69.4; 63 of 1 and one of 512
//    on 2000 155 / 107; 32 of 4 on 4000 (64/4 heads, head_dim 256) 190 / 138.  What it costs: the
//    first launch where few or none are short, as only the device knows the lengths (64 of 64
//    on 500 69.5 / 72.6, 64 of 16 on 500 45.6 / 48.4, 32 of 16 on 2000 57.0 / 60.4, 8 of 512 on
//    2048 168.6 / 171.4, 64 of 1-400 on 2000 572 / 580); and parts that no longer overlap where
//    neither fills the card (15 of 1 and one of 512 on 8000 219 / 253).
//  - Where tables are at most MXP_ALL_SHORT tokens wide and the rows of 16 columns no more
//    than the workgroups the device holds, the call is all latency and the decode kernel cuts
//    it finer: 120 fresh tokens 14.9 / 9.5 us, on 500 25.4 / 20.6, on 1000 24.2 / 23.1, on 2000
//    26.6 / 28.1.  Slower: 8 of 4 on 1000 16.2 / 18.1, 8 of 6 16.6 / 19.3, 8 of 8 16.8 / 19.6.  The
//    host knows the tables' width alone: 120 fresh tokens under tables of 4096 take 22 us.
constexpr int64_t MXP_SHORT_COLS = 32, MXP_SOME_SHORT = 1024, MXP_ALL_SHORT = 1024;

// 8 waves, two a SIMD (one of each group), up to head_dim 128; past it a wave needs the
// registers of two
template <int NB> constexpr int mxp_waves() { return NB <= 4 ? 8 : 4; }

struct MxPrefillArgs {
    uint16_t* out;
    const uint16_t* q;
    const uint8_t *kc, *vc;
    const int32_t *bt, *seq_lens, *qsl;
    int32_t num_seqs, num_tokens, hq, hkv;
    int32_t bs, subs;       // tokens, 16-token parts of a block
    int32_t maxb;
    int32_t nb;
    float c;                // scale * log2(e)
    int32_t splits, base_wgs;
    int32_t longest_first;  // query tiles by falling key counts
    int32_t short_cols;     // sequences of up to this many rows are not for this kernel
    float* part_o;          // [num_tokens * hq][splits][D], relative to 2^8 times the part's max
    float* part_ml;         // [num_tokens * hq][splits][2]
};

// bf16 elements of a V row in LDS: four consecutive rows of a transposing read
// (64 bytes each) on different banks
template <int NB> constexpr int mxp_row() { return 32 * NB + (NB % 2 ? 0 : 32); }

// Tile `rank` of the batch by falling key counts, in steps of MXP_TILE keys: the
// workgroups of a launch start in order, so the long ones run first and the short
// ones fill the last round.  Lane i brings sequence i's new tokens n (nt query tiles)
// and context ctx.  The step is searched for: a sequence's tiles with more than T steps
// of keys are its last ones, and their number is a shift away.  -1 past the last tile.
template <int ROWS>
__device__ __forceinline__ int mxp_longest(int n, int ctx, int nt, int G, int rank, int& tile) {
    static_assert((ROWS & (ROWS - 1)) == 0, "tiles are counted by shifts");
    constexpr int SH = __builtin_ctz(ROWS);
    ctx = min(max(ctx, 0), 1 << 27);
    auto above = [&](int steps) __attribute__((always_inline)) {
        // tile i's last token is (ROWS (i + 1) - 1) / G, and attends it and ctx - n more;
        // below 0 steps every tile counts, those without a key (ctx < n) too
        if (steps < 0) return nt;
        const int x = min(max(steps * MXP_TILE - (ctx - n), 0), n);
        return nt > 0 && ctx > steps * MXP_TILE ? nt - min(nt - 1, (x * G) >> SH) : 0;
    };
    auto all_above = [&](int steps) __attribute__((always_inline)) {
        return __builtin_amdgcn_readlane(mx4_scan(above(steps)), 63);
    };
    int lo = -1, hi = (mx4_wave_max(ctx) + MXP_TILE - 1) / MXP_TILE;   // all_above(lo) counts every tile, (hi) none
    if (rank >= all_above(lo)) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (all_above(mid) > rank) lo = mid;
        else hi = mid;
    }
    const int longer = above(hi), band = above(lo) - longer;
    const int r = rank - all_above(hi);
    const int before = mx4_scan(band) - band;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(before <= r && r < before + band);
    const int s = __ffsll(static_cast<unsigned long long>(hit)) - 1;
    tile = __builtin_amdgcn_readlane(nt - longer - 1 - (r - before), s);
    return s;
}

// LDS: K codes of two tiles, V rows of two, and beside them K's scales and marks of
// NaN blocks of V (a tile's number where it has one).
template <int NB>
struct MxTiles {
    uint4 k[2][NB][MXP_TILE];
    uint16_t v[2][MXP_TILE][mxp_row<NB>()];
    uint8_t ke[2][NB][MXP_TILE];
    uint8_t bad[2][NB][MXP_TILE];
    int32_t bad_tile[2];
};

template <int QKIND, int NB>
__global__ __launch_bounds__(64 * mxp_waves<NB>(), mxp_waves<NB>() / 4) void mx4_prefill_kernel(
    MxPrefillArgs a, const int32_t* __restrict__ bt) {
    constexpr int D = 32 * NB, WAVES = mxp_waves<NB>(), ROWS = 32 * WAVES;
    constexpr int GROUP = 64 * (WAVES / 2);       // threads of a group
    constexpr int NKS = (NB + 1) / 2;             // 64-wide steps of head_dim
    constexpr int NT = mx4_terms<QKIND>();
    constexpr int PT = QKIND == KIND_BF16 ? 1 : 2;   // terms of a weight
    constexpr int CHUNKS = MXP_TILE * NB;         // 16-byte chunks of a tile's K (V): group 1 (0) copies them
    constexpr int NCH = (CHUNKS + GROUP - 1) / GROUP;
    constexpr int ROW = mxp_row<NB>();
    __shared__ __align__(16) MxTiles<NB> tiles;

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int grp = wave / (WAVES / 2), gtid = tid - grp * GROUP;
    const int l32 = lane & 31, hl = lane >> 5;
    const int G = a.hq / a.hkv;

    // ---- which (kv head, sequence, query tile) ----
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
            n_l = n_l * G <= a.short_cols ? 0 : n_l;
        }
        const int nt_l = (n_l * G + ROWS - 1) / ROWS;
        if (a.longest_first) {   // at most 64 sequences
            const int ctx_l = s0 + lane < a.num_seqs ? a.seq_lens[s0 + lane] : 0;
            s = mxp_longest<ROWS>(n_l, ctx_l, nt_l, G, j, tile);
            if (s >= 0) {
                q0 = __builtin_amdgcn_readlane(q0_l, s);
                n = __builtin_amdgcn_readlane(n_l, s);
            }
            break;
        }
        // sequence by sequence, a sequence's last tile (the most keys) first
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

    // ---- copies: group 0 brings V, group 1 K.  A thread's chunks are 16 bytes of codes
    // and their scale; its table entries are loaded a tile before the chunks ----
    const int64_t page_bytes = mx4_page_bytes(D, a.bs);
    const int code_bytes = a.bs * (D / 2);
    const int32_t* bt_row = bt + static_cast<int64_t>(s) * a.maxb;
    const uint8_t* const cache = (grp == 0 ? a.vc : a.kc) + h * page_bytes;
    const uint64_t block_bytes = static_cast<uint64_t>(a.hkv) * page_bytes;
    // A place in the context: the 16-token part `rem` of table entry `blk`.  Four parts
    // (a tile) further on by additions alone: this runs every tile, and integer
    // products take four issue slots.
    struct Place { int blk, rem; };
    const int adv_blk = MXP_SUBS / a.subs, adv_rem = MXP_SUBS % a.subs;
    auto place_of = [&](int u) __attribute__((always_inline)) { return Place{u / a.subs, u % a.subs}; };
    auto advance = [&](Place& x) __attribute__((always_inline)) {
        x.rem += adv_rem;
        const bool over = x.rem >= a.subs;
        x.rem -= over ? a.subs : 0;
        x.blk += adv_blk + (over ? 1 : 0);
    };
    // this thread's chunks: their places in the tile whose entries are loaded next and,
    // for part lane % 4, what says whether it exists
    Place at[NCH], at_part;
    int id[NCH], id_part, rem[NCH];   // entries as loaded, and the chunks' parts of them
    const int part = lane & (MXP_SUBS - 1);
    auto begin_ids = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            at[c] = place_of(t * MXP_SUBS + min((c * GROUP + gtid) / (MX4_TOKENS * NB), MXP_SUBS - 1));
        at_part = place_of(t * MXP_SUBS + part);
    };
    auto load_ids = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            id[c] = bt_row[min(at[c].blk, a.maxb - 1)];
            rem[c] = at[c].rem;
            advance(at[c]);
        }
        id_part = bt_row[min(at_part.blk, a.maxb - 1)];
        advance(at_part);
    };
    // bit i: part i of tile t exists
    auto presence = [&](int t) __attribute__((always_inline)) {
        const bool ok = static_cast<uint32_t>(id_part) < static_cast<uint32_t>(a.nb) && (t * MXP_SUBS + part) * MX4_TOKENS < kv_end;
        return static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ok)) & ((1u << MXP_SUBS) - 1);
    };
    // a chunk's byte offsets in its part's codes and scales, and its key in the tile
    int c_off[NCH], c_key[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int idx = c * GROUP + gtid;
        c_off[c] = idx % (MX4_TOKENS * NB);
        c_key[c] = CHUNKS % GROUP == 0 || idx < CHUNKS ? idx / NB : 1 << 30;   // past any context
    }
    struct Raw { uint4 w[NCH]; uint32_t e[NCH]; };
    auto fetch = [&](int t, Raw& r) __attribute__((always_inline)) {
        const int room = kv_end - t * MXP_TILE;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            r.w[c] = make_uint4(0, 0, 0, 0);
            r.e[c] = 127;
            // rows past the keys any query here sees may hold anything: zeros
            if (static_cast<uint32_t>(id[c]) < static_cast<uint32_t>(a.nb) && c_key[c] < room) {
                const uint8_t* page = cache + static_cast<uint64_t>(static_cast<uint32_t>(id[c])) * block_bytes;
                r.w[c] = *reinterpret_cast<const uint4*>(page + (rem[c] * (MX4_TOKENS * D / 2) + 16 * c_off[c]));
                r.e[c] = page[code_bytes + rem[c] * (MX4_TOKENS * NB) + c_off[c]];
            }
        }
    };
    auto store = [&](int t, const Raw& r) __attribute__((always_inline)) {
        const int buf = (t - t_lo) & 1;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int idx = c * GROUP + gtid;
            if (CHUNKS % GROUP != 0 && idx >= CHUNKS) continue;
            const int key = idx / NB, b = idx % NB;
            if (grp == 1) {
                tiles.k[buf][b][key] = r.w[c];
                tiles.ke[buf][b][key] = static_cast<uint8_t>(r.e[c]);
            } else {
                // A NaN block enters as zeros and marks its token: a weight of 0
                // for a key that a row does not see would not keep it out.
                const bool bad = r.e[c] > MX4_TOP_SCALE;
                const uint4 w = r.w[c];
                const float f = bad ? 0.f : mx4_factor(r.e[c]);
                // 16-byte chunk i of block b lies at i ^ (b % 4): the 16 lanes of a
                // store (4 keys x 4 blocks, rows 64 bytes apart in the banks) then
                // cover all banks
                uint4* dst = reinterpret_cast<uint4*>(&tiles.v[buf][key][32 * b]);
                const int sw = b & 3;
                dst[0 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.x, f), mx4_dec_bf16<1>(w.x, f), mx4_dec_bf16<2>(w.x, f), mx4_dec_bf16<3>(w.x, f));
                dst[1 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.y, f), mx4_dec_bf16<1>(w.y, f), mx4_dec_bf16<2>(w.y, f), mx4_dec_bf16<3>(w.y, f));
                dst[2 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.z, f), mx4_dec_bf16<1>(w.z, f), mx4_dec_bf16<2>(w.z, f), mx4_dec_bf16<3>(w.z, f));
                dst[3 ^ sw] = make_uint4(mx4_dec_bf16<0>(w.w, f), mx4_dec_bf16<1>(w.w, f), mx4_dec_bf16<2>(w.w, f), mx4_dec_bf16<3>(w.w, f));
                tiles.bad[buf][b][key] = bad;
                if (bad) tiles.bad_tile[buf] = t;
            }
        }
    };

    // presences of the tiles ahead, four bits each
    uint32_t ring = 0;
    auto note = [&](int t) __attribute__((always_inline)) {
        const int sh = 4 * ((t - t_lo) & 7);
        ring = (ring & ~(15u << sh)) | presence(t) << sh;
    };
    // the next tile's copy: stored from its registers, the one after it fetched and the
    // table entries of one more asked for
    Raw raw;
    auto copy = [&](int t) __attribute__((always_inline)) {
        if (t < t_hi) store(t, raw);
        if (t + 1 < t_hi) {
            fetch(t + 1, raw);
            note(t + 1);
            if (t + 2 < t_hi) load_ids();
        }
    };
    if (tid == 0) tiles.bad_tile[0] = tiles.bad_tile[1] = -1;
    if (t_lo < t_hi) {
        begin_ids(t_lo);
        load_ids();
        fetch(t_lo, raw);
        note(t_lo);
        if (t_lo + 1 < t_hi) load_ids();
    }

    // ---- the query row as E4M3 terms: lane group hl holds elements 16 hl.. and
    // 32 + 16 hl.. of each 64-wide step ----
    mx_i32x8 qt[NT][NKS];
    int qs[NT];
    {
        const uint16_t* src = a.q + orow * D;
        const MxScale sign = mx4_scale(a.c);
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
                w[ks][i] = mx4_scaled(w[ks][i], sign);
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

    const float c = mx4_scale(a.c).c;
    mx_f32x16 st[2];               // S^T of the tile's 32-key halves
    uint32_t p[PT][2][8];          // the weights, packed pairs, same order

    // transposing V read: row 4 hl + (lane % 16) / 4, 16 elements from 16 ((lane / 16) & 1) of a block
    const int v_row = 4 * hl + ((lane & 15) >> 2);
    const int v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), v_in = 4 * (lane & 1);

    // ---- products ----
    auto load_v = [&](int t, int k16, uint4 (&v)[NB]) __attribute__((always_inline)) {
        const uint16_t* base = &tiles.v[(t - t_lo) & 1][16 * k16 + v_row][v_in];
#pragma unroll
        for (int dt = 0; dt < NB; ++dt) {
            const uint16_t* src = base + 32 * dt + 8 * (v_chunk ^ (dt & 3));
            const uint2 v0 = mx4_read_tr16(src), v1 = mx4_read_tr16(src + 8 * ROW);
            v[dt] = make_uint4(v0.x, v0.y, v1.x, v1.y);
        }
    };
    struct KOp { uint4 k[2]; int e[2]; };   // both halves of a 64-wide step
    auto load_k = [&](int t, int ks, KOp& x) __attribute__((always_inline)) {
        const int buf = (t - t_lo) & 1, b = 2 * ks + hl;
        const bool have = NB % 2 == 0 || b < NB;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            x.k[half] = tiles.k[buf][have ? b : 0][32 * half + l32];
            x.e[half] = have ? tiles.ke[buf][b][32 * half + l32] : 127;
        }
    };
    // O^T += V^T P^T over tile t, 16 keys a step
    auto values = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int k16 = 0; k16 < MXP_TILE / 16; ++k16) {
            uint4 v[NB];
            load_v(t, k16, v);
#pragma unroll
            for (int i = 0; i < PT; ++i) {
                const uint32_t* w = &p[i][k16 >> 1][4 * (k16 & 1)];
                const uint4 pb = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
                for (int dt = 0; dt < NB; ++dt) o[dt] = mx4_mma32_bf16(v[dt], pb, o[dt]);
            }
        }
    };
    int bad_before = -1;   // bad_tile of the tile before, read where LDS is waited for anyway
    auto products = [&](int t) __attribute__((always_inline)) {
        if (t > t_lo) values(t - 1);
        bad_before = tiles.bad_tile[(t - 1 - t_lo) & 1];
        st[0] = st[1] = mx_f32x16{};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            KOp k;
            load_k(t, ks, k);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    st[half] = mx4_mma32(k.k[half], qt[i][ks], st[half], k.e[half], qs[i]);
        }
        bad_before = __builtin_amdgcn_readfirstlane(bad_before);
    };
    // value blocks of tile t that are NaN in a row that sees them
    auto mark_nan = [&](int t) __attribute__((always_inline)) {
        const int buf = (t - t_lo) & 1;
        if (t < t_lo || tiles.bad_tile[buf] != t) return;
        for (int key = 0; key < MXP_TILE; ++key)
#pragma unroll
            for (int b = 0; b < NB; ++b)
                nan_blocks |= t * MXP_TILE + key <= pos ? static_cast<uint32_t>(tiles.bad[buf][b][key]) << b : 0u;
    };
    // ---- scores of tile t -> weights against 2^8 times the max as it stands, which moves
    // only when a lane's weights sum past 1: the tile's own max is not looked for before, and
    // sums of large values overflow no sooner than the softmax's own ----
    auto mask = [&](int t) __attribute__((always_inline)) {
        const int t0 = t * MXP_TILE;
        const uint32_t present = ring >> (4 * ((t - t_lo) & 7)) & ((1u << MXP_SUBS) - 1);
        const bool full = present == (1u << MXP_SUBS) - 1 && t0 + MXP_TILE <= kv_end && t0 + MXP_TILE - 1 <= min_pos;
        if (!full) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = 32 * half + 8 * (i >> 2) + 4 * hl + (i & 3);
                    const bool ok = ((present >> (key >> 4)) & 1u) && t0 + key <= pos && t0 + key < kv_end;
                    st[half][i] = ok ? st[half][i] : -INFINITY;
                }
        }
    };
    auto rescale = [&]() __attribute__((always_inline)) {
        float top = st[0][0];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, st[half][i]);
        const float m_new = fmaxf(m, mx4_max_32(top));
        const float alpha = m_new == m ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < NB; ++dt) o[dt] *= alpha;
        m = m_new;
    };
    auto weights = [&]() __attribute__((always_inline)) -> float {   // their sum
        const float mc = m == -INFINITY ? 0.f : __builtin_fmaf(m, c, MX4_AHEAD);
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[half][2 * i], c, -mc));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[half][2 * i + 1], c, -mc));
                sum0 += p0;
                sum1 += p1;
                p[0][half][i] = mx4_pack_bf16(p0, p1);
                if constexpr (PT == 2) p[1][half][i] = mx4_pack_bf16(p0 - bf16_lo(p[0][half][i]), p1 - bf16_hi(p[0][half][i]));
            }
        return sum0 + sum1;
    };

    // ---- the turns.  In turn 2t group 0 issues tile t's products (and tile t-1's
    // V products), in turn 2t + 1 its softmax and the copy of V(t); group 1 is one turn
    // behind, with the copy of K(t + 2).  Where a SIMD holds a wave of each (head_dim up to
    // 128), one keeps the matrix core while the other works on the vector units.  K(t) is read in turns 2t
    // and 2t + 1, V(t) in 2t + 2 and 2t + 3; K(t + 2) is written over K(t) in turn 2t + 2, V(t)
    // over V(t - 2) in turn 2t + 1. ----
    if (t_lo < t_hi) {
        if (grp == 1) copy(t_lo);
        __syncthreads();
        if (grp == 1) {   // while group 0 begins
            copy(t_lo + 1);
            __syncthreads();
        }
        // A tile that moves the max or follows one with NaN values leaves the loop and comes
        // back: what it needs, in the loop's body, costs every tile 5%.
        for (int t = t_lo; t < t_hi;) {
            bool rare = false;
            for (; t < t_hi; ++t) {
                if (wave_live) products(t);
                __syncthreads();
                if (wave_live) {
                    mask(t);
                    const float sum = weights();
                    rare = __builtin_amdgcn_ballot_w64(!(sum <= 1.f) || m == -INFINITY) || bad_before == t - 1;
                    if (rare) break;
                    l += sum;
                }
                copy(grp == 0 ? t : t + 2);
                __syncthreads();
            }
            if (!rare) break;
            mark_nan(t - 1);
            rescale();
            l += weights();
            copy(grp == 0 ? t : t + 2);
            __syncthreads();
            ++t;
        }
        if (grp == 0) __syncthreads();   // group 1's last softmax
        if (wave_live) {
            mark_nan(t_hi - 1);
            values(t_hi - 1);
        }
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
        if (hl == 0) *reinterpret_cast<mx_f32x2*>(a.part_ml + 2 * slot) = mx_f32x2{m * c, l};
        return;
    }
    // lanes l and l + 32 hold the two halves of each 8-element run; swapped in pairs of
    // runs, lane l stores the whole of the first and lane l + 32 of the second
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* dst = a.out + orow * D + 8 * hl;
#pragma unroll
    for (int dt = 0; dt < NB; ++dt) {
        const float f = (nan_blocks >> dt) & 1u ? nan : inv;
#pragma unroll
        for (int jj = 0; jj < 4; jj += 2) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t even = mx4_pack16<QKIND>(o[dt][4 * jj + 2 * i] * f, o[dt][4 * jj + 2 * i + 1] * f);
                const uint32_t odd = mx4_pack16<QKIND>(o[dt][4 * jj + 4 + 2 * i] * f, o[dt][4 * jj + 5 + 2 * i] * f);
                mx4_swap_32(even, odd, w[i], w[2 + i]);
            }
            *reinterpret_cast<mx_out8*>(dst + 32 * dt + 8 * jj) = mx_out8{w[0], w[1], w[2], w[3]};
        }
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
    const float f = lp == 0.f ? 0.f : fmaxf(__builtin_amdgcn_exp2f(mp - top), MX4_LEAST);   // NaN values go on
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
    RLLM_CHECK_ARG(std::isfinite(scale * MX4_LOG2E));
    RLLM_CHECK_ARG(mx4_aligned16(key_cache) && mx4_aligned16(value_cache) && mx4_aligned16(query));
    RLLM_CHECK_ARG((reinterpret_cast<uintptr_t>(output) & 7) == 0);
    const int64_t group = num_q_heads / num_kv_heads, rows_wg = head_dim <= 128 ? 256 : 128;
    // ceil(r / rows_wg) <= (r - 1) / rows_wg + 1 for every r >= 0; workgroups past the last tile find none
    const int64_t wgs = ((num_tokens * group - num_seqs) / rows_wg + num_seqs) * num_kv_heads;
    RLLM_CHECK_ARG(wgs * 512 <= MX4_MAX_THREADS);
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
    a.maxb = static_cast<int32_t>(max_num_blocks_per_seq);
    a.nb = static_cast<int32_t>(num_blocks);
    a.c = scale * MX4_LOG2E;
    a.base_wgs = static_cast<int32_t>(wgs);
    a.splits = 1;
    int dev = 0, cus = 0;
    RLLM_TRY(hipGetDevice(&dev));
    RLLM_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    const int64_t width = max_num_blocks_per_seq * block_size;
    const int64_t every = num_tokens * group;   // columns
    auto short_rows = [&](int64_t most) {
        return mx4_short_rows(num_seqs, num_tokens, num_q_heads, num_kv_heads, block_size, max_num_blocks_per_seq, most);
    };
    auto short_chunks = [&](int64_t most) {
        return mx4_short_chunks(output, query, key_cache, value_cache, block_tables, seq_lens, query_start_loc, num_seqs,
                                num_tokens, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq,
                                num_blocks, scale, q_dtype, most, stream);
    };
    if (width <= MXP_ALL_SHORT) {
        const int64_t rows = short_rows(every);
        if (rows > 0 && rows <= static_cast<int64_t>(cus) * mxd_per_simd(head_dim)) return short_chunks(every);
    }
    if (num_seqs > 1 && every <= MXP_SOME_SHORT * num_seqs && 2 * wgs > cus) {
        const int64_t most = head_dim <= 128 ? MXP_SHORT_COLS : 2 * MXP_SHORT_COLS;
        if (short_rows(most) > 0) {
            const int32_t rc = short_chunks(most);
            if (rc) return rc;
            a.short_cols = static_cast<int32_t>(most);
        }
    }
    // few query tiles over long contexts: several workgroups a tile, each on a part of the keys
    const int64_t tiles = (width + MXP_TILE - 1) / MXP_TILE;
    a.longest_first = num_seqs > 1 && num_seqs <= 64 && wgs > cus && wgs <= MXP_SORTED_ROUNDS * cus;
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
