// Selection of the cache blocks that a query attends, for gfx950.
//
//   score(b) = max over the heads of the group of sum_d max(q_d lo_bd, q_d hi_bd)
//
// is an upper bound of q . k over the keys of block b.  With q- = min(q, 0) and q+ =
// max(q, 0) the sum is q- . lo + q+ . hi, a matrix product over 2 head_dim whose
// right side lies in memory as it is needed.
//
// The lists are those of the scores in 64 bits.  The matrix cores give each score in
// f32 (products of 16-bit values are exact there, sums are not) and a bound E of
// its error; with T the K-th largest f32 score, every block above T + 2E is in, every
// one below T - 2E is out, and only those between are scored again in f64.  Equal
// ones go to the lowest block.
#include "sparse_blocks.h"
#include "sparse_plan.h"
#include "generic_mfma.h"
#include "workspace.h"

namespace rllm {
namespace {

struct SelectArgs {
    int32_t* sel;
    const uint16_t* q;
    const void* kb;
    const int32_t *bt, *seq_lens, *qsl;
    uint32_t* keys;     // [rows of the launch, hkv, pitch]: scores in their order, 0 = not to be chosen
    uint8_t* state;     // OUT, MID or IN of each, for lists whose candidates are not held in registers
    float* kmax;        // [rows of the launch, hkv, chunks]: largest |bound| of a chunk, at a sequence's last row of the launch
    int32_t num_seqs, row0, rows, hq, hkv, d, bs_log2, maxb, k, first, last, chunk, chunks;
    int32_t tiles;      // whether rows were scored in tiles
    int32_t group_log2; // heads of a group, as a power of two, where rows go in tiles
    int64_t num_blocks, pitch;
};

// blocks of its sequence that a row sees
__device__ __forceinline__ int visible_blocks(const SelectArgs& a, const SparseRow& r) {
    return r.pos < 0 ? 0 : min((r.pos >> a.bs_log2) + 1, a.maxb);
}

// f32 as integers in the order of its values, never 0; NaN above all
__device__ __forceinline__ uint32_t order32(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);            // -0 is 0
    return x != x ? 0xffffffffu : u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unorder32(uint32_t k) {
    return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t order64(double x) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));   // -0 is 0
    return x != x ? ~uint64_t(0) : u >> 63 ? ~u : u | (uint64_t(1) << 63);
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t umin(uint32_t a, uint32_t b) { return a < b ? a : b; }

// q- and q+ of 8 elements (NaN in one of them)
__device__ __forceinline__ void split_signs(const uint4& x, uint4& neg, uint4& pos) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
    uint32_t n[4], p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t m = (u[j] >> 15 & 0x00010001u) * 0xffffu;
        n[j] = u[j] & m;
        p[j] = u[j] & ~m;
    }
    neg = make_uint4(n[0], n[1], n[2], n[3]);
    pos = make_uint4(p[0], p[1], p[2], p[3]);
}
// A chunk's largest magnitude, which lies highest as 16 bits do.  It may be of a block that a row which reads it does
// not see (rows of a tile share them): NaN is an infinity there, so that the others' size counts as not known.
template <class TAG>
__device__ __forceinline__ float chunk_max(uint32_t bits) {
    const float x = to_f32<TAG>(static_cast<uint16_t>(bits));
    return x == x ? x : INFINITY;
}

// A workgroup per (row, chunk of its blocks), a wave kv heads w, w + 4, ..., 16 blocks at
// a time: v_mfma_16x16x32, rows = heads, columns = blocks, k = channels of lo, then of
// hi.  Each lane loads 8 channels of its column's block, the operand as it stands.
// Bound by HBM: the bounds are read once a row.  The heads of a block lie in a run, so
// the waves of a workgroup read whole runs between them (64 rows of 250-2000 blocks, 8 kv
// heads, head_dim 128: 72 us, 4.0 TB/s; 84 where a workgroup kept to one head).
template <int QKIND, int KVKIND, int NK>
__global__ __launch_bounds__(256) void select_score_kernel(SelectArgs a) {
    using M = GenMfma<QKIND>;
    using raw_t = GenRaw<KVKIND>;
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    constexpr int ES = gen_is_fp8<KVKIND>() ? 1 : 2, D = 32 * NK;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, kq = lane >> 4;
    const int chunk = blockIdx.x % a.chunks, t = a.row0 + blockIdx.x / a.chunks;
    const SparseRow row = sparse_row(t, a.qsl, a.seq_lens, a.num_seqs);
    const int nv = visible_blocks(a, row);
    if (row.seq < 0 || nv <= a.k) return;
    const int c0 = max(chunk * a.chunk, a.first), c1 = min((chunk + 1) * a.chunk, nv - a.last);
    if (c0 >= c1) return;
    const int G = a.hq / a.hkv, hgs = (G + 15) / 16;
    const int32_t* const bt = a.bt + static_cast<int64_t>(row.seq) * a.maxb;
    for (int h = wave; h < a.hkv; h += 4) {
        const int64_t unit = static_cast<int64_t>(t - a.row0) * a.hkv + h;
        uint32_t top = 0;                                   // largest magnitudes, two 16-bit halves
        uint32_t* const keys = a.keys + unit * a.pitch;
        uint4 qn[NK], qp[NK];
        auto load_q = [&](int hg) __attribute__((always_inline)) {
            const bool live = 16 * hg + col < G;
            const uint16_t* src = a.q + (static_cast<int64_t>(t) * a.hq + h * G + 16 * hg + col) * D;
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const uint4 x = live ? *reinterpret_cast<const uint4*>(src + 32 * i + 8 * kq) : make_uint4(0, 0, 0, 0);
                split_signs(x, qn[i], qp[i]);
            }
        };
        load_q(0);
        // the next tile's bounds are on their way while this one's are worked on, and its blocks' ids
        auto block_at = [&](int b0) __attribute__((always_inline)) -> int32_t {
            const int j = b0 + col;
            int32_t b = -1;
            if (j >= c0 && j < c1) {
                b = bt[j];
                if (b >= a.num_blocks) b = -1;
            }
            return b;
        };
        raw_t raw[2 * NK];
        auto load = [&](int32_t b) __attribute__((always_inline)) {
            const uint8_t* src = b >= 0 ? static_cast<const uint8_t*>(a.kb) + (static_cast<int64_t>(b) * a.hkv + h) * (2 * D * ES)
                                        : reinterpret_cast<const uint8_t*>(g_gen_zero);
            const int st = b >= 0 ? ES : 0;
#pragma unroll
            for (int i = 0; i < 2 * NK; ++i) raw[i] = *reinterpret_cast<const raw_t*>(src + (32 * i + 8 * kq) * st);
        };
        const int first_tile = chunk * a.chunk;
        int32_t b = block_at(first_tile), b_next = block_at(first_tile + 16);
        load(b);
        for (int b0 = first_tile; b0 < c1; b0 += 16) {
            const int j = b0 + col;
            uint4 x[2 * NK];
#pragma unroll
            for (int i = 0; i < 2 * NK; ++i) x[i] = gen_to16<QKIND, KVKIND>(raw[i]);
            const bool here = b >= 0;
            b = b_next;
            if (b0 + 16 < c1) {
                load(b);
                b_next = block_at(b0 + 32);
            }
            u16x2 m = __builtin_bit_cast(u16x2, top);
#pragma unroll
            for (int i = 0; i < 2 * NK; ++i) {
                const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u[e] & 0x7fff7fffu));
            }
            top = __builtin_bit_cast(uint32_t, m);
            uint32_t best = 0;
            for (int hg = 0; hg < hgs; ++hg) {
                if (hgs > 1) load_q(hg);
                gm_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NK; ++i) acc = M::mma16(qn[i], x[i], acc);
#pragma unroll
                for (int i = 0; i < NK; ++i) acc = M::mma16(qp[i], x[NK + i], acc);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (16 * hg + 4 * kq + i < G) best = umax(best, order32(acc[i]));
            }
            best = quads_umax(best);
            if (kq == 0 && j >= c0 && j < c1) keys[j] = here ? best : 0;
        }
        const uint32_t t16 = wave_umax(umax(top & 0xffffu, top >> 16));
        if (lane == 0) a.kmax[unit * a.chunks + chunk] = chunk_max<typename M::tag>(t16);
    }
}

// Rows of a chunk: a workgroup has a tile of them, 256 (row, head) pairs (128 past head_dim
// 128) of one sequence and kv head, a quarter a wave, their queries in registers.  The
// bounds of 16 blocks at a time go to LDS in whole runs, the next ones on their way,
// and serve every row of the tile.  704 rows of 1250-1650
// blocks, 32/8 heads, head_dim 128: 58 us; vector instructions are busy for 39% of them
// (1339 a wave, 101 of them products), and half of a wave's cycles go in waiting.
template <int QKIND, int KVKIND, int NK>
__global__ __launch_bounds__(256, 2) void select_score_tile_kernel(SelectArgs a) {
    using M = GenMfma<QKIND>;
    using raw_t = GenRaw<KVKIND>;
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    constexpr int ES = gen_is_fp8<KVKIND>() ? 1 : 2, D = 32 * NK, MT = select_m_tiles(D);
    constexpr int PIECES = 2 * D * ES / 16, ROW = 2 * D * ES + 16;    // 16-byte pieces of a block's bounds; a block in LDS
    constexpr int NP = (16 * PIECES + 255) / 256;                      // of a thread
    __shared__ __align__(16) uint8_t s_bounds[2][16 * ROW];
    __shared__ uint32_t s_max[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, kq = lane >> 4;
    const int h = blockIdx.x % a.hkv, chunk = blockIdx.x / a.hkv % a.chunks;
    const int G = a.hq / a.hkv, gl = a.group_log2, tile = 64 * MT >> gl;
    const SparseTile x = sparse_tile(blockIdx.x / a.hkv / a.chunks, tile, a.qsl, a.num_seqs);
    if (x.seq < 0 || x.row < 0) return;
    const int nt = min(min(tile, x.n - x.i), a.row0 + a.rows - x.row);        // rows of the tile within the launch
    if (nt <= 0 || x.row + nt <= a.row0) return;
    const int pos = a.seq_lens[x.seq] - x.n + x.i;
    const SparseRow last = {x.seq, 0, 0, pos + nt - 1};
    const int nv = visible_blocks(a, last);
    if (nv <= a.k) return;
    const int c0 = max(chunk * a.chunk, a.first), c1 = min((chunk + 1) * a.chunk, nv - a.last);
    if (c0 >= c1) return;
    const int32_t* const bt = a.bt + static_cast<int64_t>(x.seq) * a.maxb;
    const int wave_tok = wave * (16 * MT >> gl);                       // the wave's first row of the tile
    uint4 qn[MT][NK], qp[MT][NK];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r = 16 * m + col, tok = wave_tok + (r >> gl), g = r & ((1 << gl) - 1);
        const bool live = tok < nt && g < G;
        const uint16_t* src = a.q + (static_cast<int64_t>(x.row + tok) * a.hq + h * G + g) * D;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const uint4 y = live ? *reinterpret_cast<const uint4*>(src + 32 * i + 8 * kq) : make_uint4(0, 0, 0, 0);
            split_signs(y, qn[m][i], qp[m][i]);
        }
    }
    // the last rows of the sequence see every block that the others see: their workgroups
    // alone take the bounds' magnitudes
    const bool widest = x.row + nt == min(x.row - x.i + x.n, a.row0 + a.rows);
    u16x2 top = {0, 0};
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 next[NP];
    auto usable = [&](int j) __attribute__((always_inline)) -> int32_t {
        int32_t b = -1;
        if (j >= c0 && j < c1) {
            b = bt[j];
            if (b >= a.num_blocks) b = -1;
        }
        return b;
    };
    auto load = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int i = threadIdx.x + 256 * p, blk = i / PIECES;
            const int32_t b = blk < 16 ? usable(b0 + blk) : -1;
            next[p] = u32x4{0, 0, 0, 0};
            if (b >= 0)
                next[p] = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.kb) +
                                                          (static_cast<int64_t>(b) * a.hkv + h) * (2 * D * ES) + (i - blk * PIECES) * 16);
        }
    };
    auto store = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int i = threadIdx.x + 256 * p, blk = i / PIECES;
            if (16 * PIECES % 256 == 0 || blk < 16) *reinterpret_cast<u32x4*>(s_bounds[buffer] + blk * ROW + (i - blk * PIECES) * 16) = next[p];
        }
    };
    // where the lane's results go: row wave_tok + ((16 m + 4 kq) >> gl) for groups of 4 heads or more
    const int64_t row_pitch = a.hkv * a.pitch;
    uint32_t* const keys0 = a.keys + (static_cast<int64_t>(x.row - a.row0) * a.hkv + h) * a.pitch;
    uint32_t* keys_m[MT];
    uint32_t owns = 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int tok = wave_tok + ((16 * m + 4 * kq) >> gl);
        keys_m[m] = keys0 + tok * row_pitch;
        if (gl >= 2 && tok < nt && x.row + tok >= a.row0 && (kq & ((1 << (gl - 2)) - 1)) == 0) owns |= 1u << m;
    }
    const bool full = 1 << gl == G;
    const int first_tile = chunk * a.chunk;
    load(first_tile);
    store(0);
    int buffer = 0;
    for (int b0 = first_tile; b0 < c1; b0 += 16, buffer ^= 1) {
        __syncthreads();                                               // this tile is there, the other's readers are done
        if (b0 + 16 < c1) load(b0 + 16);
        const int j = b0 + col;
        const bool here = usable(j) >= 0;
        uint4 y[2 * NK];
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i)
            y[i] = gen_to16<QKIND, KVKIND>(*reinterpret_cast<const raw_t*>(s_bounds[buffer] + col * ROW + (32 * i + 8 * kq) * ES));
        if (widest) {
#pragma unroll
            for (int i = 0; i < 2 * NK; ++i) {
                const uint32_t u[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, u[e] & 0x7fff7fffu));
            }
        }
        gm_f32x4 acc[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = M::mma16(qn[m][i], y[i], acc[m]);
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = M::mma16(qp[m][i], y[NK + i], acc[m]);
        const bool in = j >= c0 && j < c1;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            // a NaN among values that are added up shows in the sum
            float v[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = w[i] = acc[m][i];
            if (!full) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (((4 * kq + i) & ((1 << gl) - 1)) >= G) {
                        v[i] = -INFINITY;
                        w[i] = 0.f;
                    }
            }
            if (gl >= 2) {
                const float z = (w[0] + w[1]) + (w[2] + w[3]);
                uint32_t key = order32(z != z ? z : fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
                if (gl >= 3) key = umax(key, __shfl_xor(key, 16));
                if (gl >= 4) key = umax(key, __shfl_xor(key, 32));
                if (in && (owns >> m & 1)) keys_m[m][j] = here ? key : 0;
                continue;
            }
            // rows 4 kq + i of the tile's m-th 16, of one head or two
            auto put = [&](int tok, uint32_t key) __attribute__((always_inline)) {
                if (in && tok < nt && x.row + tok >= a.row0) keys0[tok * row_pitch + j] = here ? key : 0;
            };
            if (gl == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) put(wave_tok + 16 * m + 4 * kq + i, order32(v[i]));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float z = w[i] + w[i + 1];
                    put(wave_tok + 8 * m + 2 * kq + i / 2, order32(z != z ? z : fmaxf(v[i], v[i + 1])));
                }
            }
        }
        if (b0 + 16 < c1) store(buffer ^ 1);
    }
    uint32_t t16 = wave_umax(umax(top[0], top[1]));
    if (lane == 0) s_max[wave] = t16;
    __syncthreads();
    t16 = umax(umax(s_max[0], s_max[1]), umax(s_max[2], s_max[3]));
    if (widest && threadIdx.x == 0)
        a.kmax[(static_cast<int64_t>(x.row + nt - 1 - a.row0) * a.hkv + h) * a.chunks + chunk] =
            chunk_max<typename M::tag>(t16);
}

enum : uint8_t { OUT = 0, MID = 1, IN = 2 };

// sums over the workgroup; every thread calls
struct Team {
    uint32_t* s;          // [2][waves]
    int waves, wave, turn;
    __device__ __forceinline__ int sum(int wave_value) {
        if (waves == 1) return wave_value;
        uint32_t* const b = s + (turn ^= 1) * waves;
        if ((threadIdx.x & 63) == 0) b[wave] = wave_value;
        __syncthreads();
        int n = 0;
        for (int w = 0; w < waves; ++w) n += b[w];
        return n;
    }
    // the sum, and that of the waves before this one
    __device__ __forceinline__ int scan(int wave_value, int& before) {
        before = 0;
        if (waves == 1) return wave_value;
        uint32_t* const b = s + (turn ^= 1) * waves;
        if ((threadIdx.x & 63) == 0) b[wave] = wave_value;
        __syncthreads();
        int n = 0;
        for (int w = 0; w < waves; ++w) {
            if (w == wave) before = n;
            n += b[w];
        }
        return n;
    }
    __device__ __forceinline__ uint32_t max(uint32_t wave_value) {
        if (waves == 1) return wave_value;
        uint32_t* const b = s + (turn ^= 1) * waves;
        if ((threadIdx.x & 63) == 0) b[wave] = wave_value;
        __syncthreads();
        uint32_t n = 0;
        for (int w = 0; w < waves; ++w) n = umax(n, b[w]);
        return n;
    }
};
__device__ __forceinline__ int wave_count(bool p) { return __popcll(__builtin_amdgcn_ballot_w64(p)); }

// The K-th largest key among those in the middle (there are K of them at least), by
// its bits from the top; the bits that all of them share are not searched.
template <int NT>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* keys, const uint8_t* state, int n, int K, Team& team) {
    uint32_t hi = 0, low = 0;
    for (int i = threadIdx.x; i < n; i += NT)
        if (state[i] == MID) {
            hi = umax(hi, keys[i]);
            low = umax(low, ~keys[i]);
        }
    hi = team.max(wave_umax(hi));
    const uint32_t lo = ~team.max(wave_umax(low));
    if (hi == lo) return hi;
    const int b0 = 31 - __builtin_clz(hi ^ lo);
    uint32_t p = b0 == 31 ? 0 : hi >> (b0 + 1) << (b0 + 1);
    for (int b = b0; b >= 0; --b) {
        const uint32_t test = p | 1u << b;
        int c = 0;
        for (int i0 = 0; i0 < n; i0 += NT) {
            const int i = i0 + threadIdx.x;
            c += wave_count(i < n && state[i] == MID && keys[i] >= test);
        }
        if (team.sum(c) >= K) p = test;
    }
    return p;
}

// Settles the middle by its keys: those above the K-th largest are in, those below
// out, equal ones stay if there are more of them than places.  Returns the places left for them.
template <int NT>
__device__ __forceinline__ int settle(const uint32_t* keys, uint8_t* state, int n, int K, Team& team) {
    const uint32_t th = kth_largest<NT>(keys, state, n, K, team);
    int c = 0;
    for (int i0 = 0; i0 < n; i0 += NT) {
        const int i = i0 + threadIdx.x;
        const bool mid = i < n && state[i] == MID;
        const bool in = mid && keys[i] > th;
        if (in) state[i] = IN;
        else if (mid && keys[i] < th) state[i] = OUT;
        c += wave_count(in);
    }
    return K - team.sum(c);
}

// score in 64 bits, the same in every lane of the wave
template <int QKIND, int KVKIND>
__device__ double exact_score(const SelectArgs& a, int t, int h, int64_t block) {
    using tag = typename GenMfma<QKIND>::tag;
    const int lane = threadIdx.x & 63, D = a.d, G = a.hq / a.hkv;
    const int64_t at = (block * a.hkv + h) * 2 * D;
    float lo[4], hi[4];
    auto bound = [&](int64_t i) __attribute__((always_inline)) -> float {
        if constexpr (gen_is_fp8<KVKIND>()) {
            const uint32_t w = static_cast<const uint8_t*>(a.kb)[i];
            const uint32_t x = KVKIND == KIND_FP8_E4M3 ? e4m3x2_to_bf16x2(w, false) : e5m2x2_to_bf16x2(w, false);
            return bf16_lo(x);
        } else {
            return to_f32<tag>(static_cast<const uint16_t*>(a.kb)[i]);
        }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        lo[i] = d < D ? bound(at + d) : 0.f;
        hi[i] = d < D ? bound(at + D + d) : 0.f;
    }
    double best = -INFINITY;
    bool nan = false;
    for (int g = 0; g < G; ++g) {
        const uint16_t* qrow = a.q + (static_cast<int64_t>(t) * a.hq + h * G + g) * D;
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            if (d >= D) continue;
            const double q = to_f32<tag>(qrow[d]);
            const double x = q * lo[i], y = q * hi[i];
            s += x != x || y != y ? __builtin_nan("") : x > y ? x : y;
        }
        for (int x = 1; x < 64; x <<= 1) s += __shfl_xor(s, x);
        nan |= s != s;
        best = s > best ? s : best;
    }
    return nan ? __builtin_nan("") : best;
}

// What the lists of a row and kv head are made from.
struct Pick {
    const SelectArgs& a;
    const int32_t* bt;
    int32_t* sel;
    int unit, h, t, nv;
    int widest;             // the sequence's last row of the launch
    int base, n;            // candidates: blocks base .. base + n - 1
    __device__ __forceinline__ bool usable(int j) const {
        const int32_t b = bt[j];
        return b >= 0 && b < a.num_blocks;
    }
};

// A bound of the f32 scores' error (not finite: none is known); and the f32 scores that are certainly above, or below,
// the K-th largest in 64 bits, th being the K-th largest in f32 (false: not finite).
template <int QKIND, int NT>
__device__ __forceinline__ float select_error(const Pick& p, Team& team) {
    using tag = typename GenMfma<QKIND>::tag;
    const SelectArgs& a = p.a;
    const int lane = threadIdx.x & 63, G = a.hq / a.hkv;
    // E = (D + 32) 2^-23 max_h |q_h|_1 max |bound|: D products that are not 0, each with a sum whose rounding may
    // be a whole last bit, and room for this bound's own roundings
    float qs = 0.f;
    for (int r = team.wave; r < G; r += NT / 64) {
        const uint16_t* qrow = a.q + (static_cast<int64_t>(p.t) * a.hq + p.h * G + r) * a.d;
        float s = 0.f;
        for (int d = 2 * lane; d < a.d; d += 128) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(qrow + d);
            s += __builtin_fabsf(to_f32<tag>(static_cast<uint16_t>(w))) + __builtin_fabsf(to_f32<tag>(static_cast<uint16_t>(w >> 16)));
        }
        qs = fmaxf(qs, wave_sum(s));
    }
    float km = 0.f;
    const float* const kmax = a.kmax + (static_cast<int64_t>(p.widest - a.row0) * a.hkv + p.h) * a.chunks;
    const int ch0 = p.base / a.chunk, ch1 = (p.base + p.n - 1) / a.chunk;
    for (int i = ch0 + lane; i <= ch1; i += 64) km = fmaxf(km, kmax[i]);
    qs = __uint_as_float(team.max(__float_as_uint(qs)));
    km = wave_max(km);
    // either 0: every score is exactly 0.  The product of both may be below f32's range, as the scores may: 2^-100 stands for those
    return qs == 0.f || km == 0.f ? 0.f : (a.d + 32) * 0x1p-23f * (qs * km) + 0x1p-100f;
}
__device__ __forceinline__ bool select_window(float th, float eps, float& over, float& under) {
    const float slack = 2.f * eps + (eps > 0.f ? __builtin_fabsf(th) * 0x1p-22f : 0.f);
    over = th + slack;
    under = th - slack;
    return gen_finite(over) && gen_finite(under);
}

// The list of a row of any number of candidates, whatever their scores: keys and states in memory.
template <int QKIND, int KVKIND, int NT>
__device__ __forceinline__ void pick_slowly(const SelectArgs& a, int unit, int h, int t, int seq, int nv, int widest, uint32_t* s_team) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Team team = {s_team, NT / 64, wave, 0};
    const int32_t* const bt = a.bt + static_cast<int64_t>(seq) * a.maxb;
    int32_t* const sel = a.sel + (static_cast<int64_t>(t) * a.hkv + h) * a.k;
    const bool all = nv <= a.k;
    const int base = a.first, n = all ? 0 : nv - a.last - a.first;
    const Pick p = {a, bt, sel, unit, h, t, nv, widest, base, n};
    auto usable = [&](int j) __attribute__((always_inline)) { return p.usable(j); };
    uint32_t* const keys = a.keys + unit * a.pitch + base;
    uint8_t* const state = a.state + unit * a.pitch + base;
    __syncthreads();
    int K = 0, ties = 0;
    if (!all) {
        int c = 0, f = 0;
        for (int i0 = 0; i0 < a.first + a.last; i0 += NT) {
            const int i = i0 + threadIdx.x;
            f += wave_count(i < a.first + a.last && usable(i < a.first ? i : nv - a.last + (i - a.first)));
        }
        bool odd = false;
        for (int i0 = 0; i0 < n; i0 += NT) {
            const int i = i0 + threadIdx.x;
            uint32_t key = 0;
            if (i < n) {
                key = keys[i];
                state[i] = key ? MID : OUT;
            }
            const float x = unorder32(key);
            odd |= key && !gen_finite(x);
            c += wave_count(key != 0);
        }
        K = a.k - team.sum(f);
        const int eligible = team.sum(c);
        if (eligible <= K) {
            ties = K;          // the whole middle goes in
        } else if (K > 0) {
            const bool any_odd = team.max(__builtin_amdgcn_ballot_w64(odd) != 0) != 0;
            bool again = any_odd;
            if (!any_odd) {
                float over, under;
                const float th = unorder32(kth_largest<NT>(keys, state, n, K, team));
                again = !select_window(th, select_error<QKIND, NT>(p, team), over, under);
                if (!again) {
                    int in = 0, mid = 0;
                    for (int i0 = 0; i0 < n; i0 += NT) {
                        const int i = i0 + threadIdx.x;
                        const bool was = i < n && state[i] == MID;
                        const float x = was ? unorder32(keys[i]) : 0.f;
                        const bool is_in = was && x > over, is_mid = was && x >= under && x <= over;
                        if (was) state[i] = is_in ? IN : is_mid ? MID : OUT;
                        in += wave_count(is_in);
                        mid += wave_count(is_mid);
                    }
                    K -= team.sum(in);
                    again = team.sum(mid) > K;
                }
            }
            ties = K;
            if (again) {
                // the middle once more in 64 bits: upper half, and where that is equal the lower
                for (int half = 0; half < 2; ++half) {
                    __syncthreads();
                    int mid = 0;
                    for (int i0 = 64 * wave; i0 < n; i0 += NT) {
                        uint64_t m = __builtin_amdgcn_ballot_w64(i0 + lane < n && state[i0 + lane] == MID);
                        mid += __popcll(m);
                        for (; m; m &= m - 1) {
                            const int i = i0 + __builtin_ctzll(m);
                            const uint64_t key = order64(exact_score<QKIND, KVKIND>(a, t, h, bt[base + i]));
                            if (lane == 0) keys[i] = static_cast<uint32_t>(half ? key : key >> 32);
                        }
                    }
                    if (team.sum(mid) <= ties) break;
                    __syncthreads();
                    ties = settle<NT>(keys, state, n, ties, team);
                }
            }
        }
        __syncthreads();
    }
    // the list, in the blocks' order; of the middle the first `ties`
    int out = 0, mids = 0;
    const int total = nv;
    for (int j0 = 0; j0 < total && out < a.k; j0 += NT) {
        const int j = j0 + threadIdx.x;
        bool in = false, mid = false;
        if (j < total) {
            if (all || j < a.first || j >= nv - a.last) in = usable(j);
            else {
                in = state[j - base] == IN;
                mid = state[j - base] == MID;
            }
        }
        int before;
        const uint64_t below = (uint64_t(1) << lane) - 1;
        const uint64_t mm = __builtin_amdgcn_ballot_w64(mid);
        const int found = team.scan(__popcll(mm), before);
        in |= mid && mids + before + __popcll(mm & below) < ties;
        mids += found;
        const uint64_t mi = __builtin_amdgcn_ballot_w64(in);
        const int taken = team.scan(__popcll(mi), before);
        const int at = out + before + __popcll(mi & below);
        if (in && at < a.k) sel[at] = j;
        out += taken;
    }
    for (int i = out + threadIdx.x; i < a.k; i += NT) sel[i] = -1;
}

// Scores of up to four candidates at once, 16 lanes each: the lane's own, in all 16.
template <int QKIND, int KVKIND>
__device__ __forceinline__ double exact_score16(const Pick& p, int j) {
    using tag = typename GenMfma<QKIND>::tag;
    using raw_t = GenRaw<KVKIND>;
    constexpr int ES = gen_is_fp8<KVKIND>() ? 1 : 2;
    const SelectArgs& a = p.a;
    const int l = threadIdx.x & 15, D = a.d, G = a.hq / a.hkv;
    const uint8_t* const at = static_cast<const uint8_t*>(a.kb) + (static_cast<int64_t>(p.bt[j]) * a.hkv + p.h) * 2 * D * ES;
    double best = -INFINITY;
    bool nan = false;
    for (int g = 0; g < G; ++g) {
        const uint16_t* qrow = a.q + (static_cast<int64_t>(p.t) * a.hq + p.h * G + g) * D;
        double s = 0.0;
        for (int d0 = 8 * l; d0 < D; d0 += 128) {
            const uint4 q = *reinterpret_cast<const uint4*>(qrow + d0);
            const uint4 lo = gen_to16<QKIND, KVKIND>(*reinterpret_cast<const raw_t*>(at + d0 * ES));
            const uint4 hi = gen_to16<QKIND, KVKIND>(*reinterpret_cast<const raw_t*>(at + (D + d0) * ES));
            const uint32_t qu[4] = {q.x, q.y, q.z, q.w}, lu[4] = {lo.x, lo.y, lo.z, lo.w}, hu[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int w = i >> 1, sh = (i & 1) * 16;
                const double qd = to_f32<tag>(static_cast<uint16_t>(qu[w] >> sh));
                const double x = qd * to_f32<tag>(static_cast<uint16_t>(lu[w] >> sh));
                const double y = qd * to_f32<tag>(static_cast<uint16_t>(hu[w] >> sh));
                s += x > y ? x : y;                          // finite: the window was
            }
        }
        s = row_sum16(s);
        nan |= s != s;
        best = s > best ? s : best;
    }
    return nan ? __builtin_nan("") : best;
}

// f(0) .. f(n - 1) with constant arguments, n <= MOST: one branch leaves the rest out
// (a condition each made a taken branch each: 1250 candidates of one row and 8 heads 16.5 us, 13.0 so)
template <int J, int MOST, class F>
__device__ __forceinline__ void upto(int n, F& f) {
    if constexpr (J < MOST) {
        if (J < n) {
            f(J);
            upto<J + 1, MOST>(n, f);
        }
    }
}

// A workgroup per (row, kv head), each thread KPT candidates in registers: wave w the
// w-th part of them, so that a list comes out in order.  Latency counts here: bits
// that all keys share are not searched, and the search ends where K keys remain (64 of 1250
// blocks: 8 lists 12 us, 512 of 250-2000 18, 5632 of 1250-1650 58).
template <int QKIND, int KVKIND, int NT, int KPT>
__global__ __launch_bounds__(NT) void select_pick_kernel(SelectArgs a) {
    constexpr int NW = NT / 64, REFINE = 64;
    __shared__ uint32_t s_team[2 * NW];
    __shared__ uint64_t s_exact[REFINE];
    __shared__ int s_cand[REFINE];
    __shared__ uint8_t s_take[REFINE];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = blockIdx.x, h = unit % a.hkv, t = a.row0 + unit / a.hkv;
    const SparseRow row = sparse_row(t, a.qsl, a.seq_lens, a.num_seqs);
    if (row.seq < 0) return;
    const int nv = visible_blocks(a, row);
    const int n = nv - a.last - a.first;
    // where its chunks' largest bounds are: with the last row where rows went in tiles
    const int widest = a.tiles ? min(t - row.i + row.n, a.row0 + a.rows) - 1 : t;
    auto quickly = [&]() __attribute__((always_inline)) -> bool {
        Team team = {s_team, NW, wave, 0};
        const Pick p = {a, a.bt + static_cast<int64_t>(row.seq) * a.maxb, a.sel + (static_cast<int64_t>(t) * a.hkv + h) * a.k,
                        unit, h, t, nv, widest, a.first, n};
        const uint64_t below = (uint64_t(1) << lane) - 1;

        const uint32_t* const keys = a.keys + unit * a.pitch + p.base;
        const int kpw = (n + NT - 1) / NT, i0 = wave * kpw * 64 + lane;      // keys of a lane, its first candidate
        uint32_t key[KPT], hi = 0, low = 0;
        int eligible = 0;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < KPT; ++j) key[j] = j < kpw && i0 + 64 * j < n ? keys[i0 + 64 * j] : 0;
        const float eps = select_error<QKIND, NT>(p, team);              // its loads go with the keys'
        auto each = [&](auto f) __attribute__((always_inline)) { upto<0, KPT>(kpw, f); };
        // the forced blocks, by every wave for itself
        int nf = 0, nl = 0;
        for (int x = 0; x < a.first; x += 64) nf += wave_count(x + lane < a.first && p.usable(x + lane));
        for (int x = 0; x < a.last; x += 64) nl += wave_count(x + lane < a.last && p.usable(nv - a.last + x + lane));
        each([&](int j) __attribute__((always_inline)) {
            eligible += wave_count(key[j] != 0);
            hi = umax(hi, key[j]);
            if (key[j]) {
                low = umax(low, ~key[j]);
                odd |= !gen_finite(unorder32(key[j]));
            }
        });
        eligible = team.sum(eligible);
        int K = a.k - nf - nl;
        uint32_t over_key = 0xffffffffu, under_key = 0xffffffffu;            // above: in; from under on: in the middle
        int places = 0;                                                      // for the middle
        bool refine = false, slow = false;
        if (eligible <= K) {
            over_key = 0;
        } else if (K > 0) {
            hi = team.max(wave_umax(hi));
            const uint32_t lo = ~team.max(wave_umax(low));
            slow = team.max(__builtin_amdgcn_ballot_w64(odd) != 0) != 0;
            uint32_t th = hi;
            if (!slow && hi != lo) {
                const int b0 = 31 - __builtin_clz(hi ^ lo);
                uint32_t pre = b0 == 31 ? 0 : hi >> (b0 + 1) << (b0 + 1);
                bool exact = false;
                for (int b = b0; b >= 0 && !exact; --b) {
                    const uint32_t test = pre | 1u << b;
                    int c = 0;
                    each([&](int j) __attribute__((always_inline)) {
                        c += wave_count(key[j] >= test);
                    });
                    c = team.sum(c);
                    if (c >= K) pre = test;
                    exact = c == K;
                }
                th = pre;
                if (exact) {                                                 // the least of the K
                    uint32_t least = 0;
#pragma unroll
                    for (int j = 0; j < KPT; ++j)
                        if (key[j] >= pre) least = umax(least, ~key[j]);
                    th = ~team.max(wave_umax(least));
                }
            }
            float over = 0.f, under = 0.f;
            if (!slow) slow = !select_window(unorder32(th), eps, over, under);
            if (!slow) {
                over_key = order32(over);
                under_key = order32(under);
                int in = 0, mid = 0;
                each([&](int j) __attribute__((always_inline)) {
                    in += wave_count(key[j] > over_key);
                    mid += wave_count(key[j] >= under_key);
                });
                in = team.sum(in);
                mid = team.sum(mid) - in;
                places = K - in;
                refine = mid > places && over_key != under_key;
                slow = refine && mid > REFINE;
                if (refine && !slow) {
                    int mine = 0, before;
                    each([&](int j) __attribute__((always_inline)) {
                        mine += wave_count(key[j] >= under_key && key[j] <= over_key);
                    });
                    team.scan(mine, before);
                    each([&](int j) __attribute__((always_inline)) {
                        const bool is = key[j] >= under_key && key[j] <= over_key;
                        const uint64_t m = __builtin_amdgcn_ballot_w64(is);
                        if (is) s_cand[before + __popcll(m & below)] = i0 + 64 * j;
                        before += __popcll(m);
                    });
                    __syncthreads();
                    for (int e = threadIdx.x >> 4; e < mid; e += NT / 16) {
                        const uint64_t k64 = order64(exact_score16<QKIND, KVKIND>(p, p.base + s_cand[e]));
                        if ((lane & 15) == 0) s_exact[e] = k64;
                    }
                    __syncthreads();
                    if (static_cast<int>(threadIdx.x) < mid) {               // candidates stand in their order: ties to the lower
                        const uint64_t me = s_exact[threadIdx.x];
                        int rank = 0;
                        for (int e = 0; e < mid; ++e) rank += s_exact[e] > me || (s_exact[e] == me && e < static_cast<int>(threadIdx.x));
                        s_take[threadIdx.x] = rank < places;
                    }
                    __syncthreads();
                }
            }
        }
        if (slow) return false;

        // the list: the first blocks, the candidates in order, the last blocks, -1
        int mine = 0, taken = 0, mids, outs;
        if (eligible > K) {
            int m = 0;
            each([&](int j) __attribute__((always_inline)) {
                m += wave_count(key[j] >= under_key && key[j] <= over_key);
            });
            team.scan(m, mids);
        } else {
            mids = 0;
        }
        const int mids0 = mids;
        auto chosen = [&](int j) __attribute__((always_inline)) -> bool {    // and moves `mids` on
            const bool is = key[j] >= under_key && key[j] <= over_key;
            const uint64_t m = __builtin_amdgcn_ballot_w64(is);
            const int at = mids + __popcll(m & below);
            mids += __popcll(m);
            return key[j] > over_key || (is && (refine ? s_take[at] != 0 : at < places));
        };
        each([&](int j) __attribute__((always_inline)) {
            mine += wave_count(chosen(j));
        });
        taken = team.scan(mine, outs);
        mids = mids0;
        outs += nf;
        each([&](int j) __attribute__((always_inline)) {
            const bool in = chosen(j);
            const uint64_t m = __builtin_amdgcn_ballot_w64(in);
            if (in) p.sel[outs + __popcll(m & below)] = p.base + i0 + 64 * j;
            outs += __popcll(m);
        });
        if (wave == 0) {
            int at = 0;
            auto forced = [&](int j0, int count) __attribute__((always_inline)) {
                for (int x = 0; x < count; x += 64) {
                    const bool in = x + lane < count && p.usable(j0 + x + lane);
                    const uint64_t m = __builtin_amdgcn_ballot_w64(in);
                    if (in) p.sel[at + __popcll(m & below)] = j0 + x + lane;
                    at += __popcll(m);
                }
            };
            forced(0, a.first);
            at += taken;
            forced(nv - a.last, a.last);
            for (int i = at + lane; i < a.k; i += 64) p.sel[i] = -1;
        }
        return true;
    };
    if (nv > a.k && n <= NT * KPT && quickly()) return;
    pick_slowly<QKIND, KVKIND, NT>(a, unit, h, t, row.seq, nv, widest, s_team);
}

template <int QKIND, int KVKIND>
int32_t launch_select(const SelectArgs& a, hipStream_t st) {
    const int64_t units = static_cast<int64_t>(a.rows) * a.hkv;
    if (a.chunks > 0) {
        if (a.tiles) {
            const int64_t count = select_tiles(static_cast<int64_t>(a.row0) + a.rows, a.num_seqs, a.d, a.group_log2);
            const dim3 grid(static_cast<unsigned>(count * a.hkv * a.chunks));
            switch (a.d / 32) {
#define RLLM_SCORE(N) \
    case N: hipLaunchKernelGGL((select_score_tile_kernel<QKIND, KVKIND, N>), grid, dim3(256), 0, st, a); break;
                RLLM_SCORE(1) RLLM_SCORE(2) RLLM_SCORE(3) RLLM_SCORE(4) RLLM_SCORE(5) RLLM_SCORE(6) RLLM_SCORE(7) RLLM_SCORE(8)
#undef RLLM_SCORE
            }
        } else {
            const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.rows) * a.chunks));
            switch (a.d / 32) {
#define RLLM_SCORE(N) \
    case N: hipLaunchKernelGGL((select_score_kernel<QKIND, KVKIND, N>), grid, dim3(256), 0, st, a); break;
                RLLM_SCORE(1) RLLM_SCORE(2) RLLM_SCORE(3) RLLM_SCORE(4) RLLM_SCORE(5) RLLM_SCORE(6) RLLM_SCORE(7) RLLM_SCORE(8)
#undef RLLM_SCORE
            }
        }
        const int32_t rc = launch_status();
        if (rc) return rc;
    }
    // a wave a row where rows are many and short enough, else four (8 heads, 1250-1650 blocks, with the scores,
    // in a graph, by one wave and by four: one row 31.5 and 20.6 us, 128 158 and 147, 256, the border, 279 and
    // 277, 384 358 and 359, 512 465 and 472; 704 of two chunks 121 and 127; 256 of 60-250 44.2 and 49.5)
    if (units >= 2048 && a.maxb <= 64 * 32)
        hipLaunchKernelGGL((select_pick_kernel<QKIND, KVKIND, 64, 32>), dim3(static_cast<unsigned>(units)), dim3(64), 0, st, a);
    else if (a.maxb <= 256 * 8)
        hipLaunchKernelGGL((select_pick_kernel<QKIND, KVKIND, 256, 8>), dim3(static_cast<unsigned>(units)), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((select_pick_kernel<QKIND, KVKIND, 256, 32>), dim3(static_cast<unsigned>(units)), dim3(256), 0, st, a);
    return launch_status();
}

}  // namespace
}  // namespace rllm

using namespace rllm;

extern "C" {

int64_t rllm_select_blocks_workspace_size(int64_t num_rows, int64_t num_kv_heads, int64_t max_num_blocks_per_seq) {
    if (num_rows < 0 || num_rows > SPARSE_MAX_ROWS || num_kv_heads < 1 || num_kv_heads > 1024 ||
        !sparse_table(max_num_blocks_per_seq, 16))
        return -1;
    int64_t pitch;
    return select_bytes(num_rows, select_row_bytes(num_kv_heads, max_num_blocks_per_seq, pitch));
}

int32_t rllm_select_blocks(int32_t* selected, const void* query, const void* k_bounds, const int32_t* block_tables,
                           const int32_t* seq_lens, const int32_t* query_start_loc, int64_t num_seqs, int64_t num_rows,
                           int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                           int64_t max_num_blocks_per_seq, int64_t num_blocks, int64_t num_selected, int64_t num_first,
                           int64_t num_last, int32_t q_dtype, int32_t kv_dtype, void* workspace, int64_t workspace_bytes,
                           uintptr_t stream) {
    if (num_seqs <= 0 || num_rows <= 0) return 0;
    RLLM_CHECK_ARG(sparse_shape(num_kv_heads, head_dim, block_size) && sparse_heads(num_q_heads, num_kv_heads));
    RLLM_CHECK_ARG(sparse_types(q_dtype, kv_dtype));
    RLLM_CHECK_ARG(num_seqs <= SPARSE_MAX_ROWS && num_rows <= SPARSE_MAX_ROWS && num_blocks >= 0);
    RLLM_CHECK_ARG(sparse_table(max_num_blocks_per_seq, block_size));
    RLLM_CHECK_ARG(query_start_loc || num_rows == num_seqs);
    RLLM_CHECK_ARG(num_selected >= 1 && num_selected <= RLLM_SELECT_MAX_BLOCKS);
    RLLM_CHECK_ARG(num_first >= 0 && num_last >= 1 && num_first <= num_selected && num_last <= num_selected - num_first);
    RLLM_CHECK_ARG(selected && query && k_bounds && seq_lens && (block_tables || max_num_blocks_per_seq == 0));
    RLLM_CHECK_ARG(aligned_to(query, 16) && aligned_to(k_bounds, 16));
    const SelectPlan p = select_plan(num_rows, num_seqs, num_q_heads, num_kv_heads, head_dim, max_num_blocks_per_seq,
                                     num_selected, query_start_loc != nullptr);
    WorkspaceHold hold;
    void* ws = workspace;
    if (workspace) {
        RLLM_CHECK_ARG(workspace_bytes >= p.need && aligned_to(workspace, 16));
    } else if (p.need > 0) {
        const int32_t rc = g_workspaces.get(stream, WS_SELECT, p.need, false, &ws, &hold);
        if (rc) return rc;
        if (!ws) return static_cast<int32_t>(hipErrorStreamCaptureUnsupported);
    }
    SelectArgs a = {};
    a.sel = selected;
    a.q = static_cast<const uint16_t*>(query);
    a.kb = k_bounds;
    a.bt = block_tables;
    a.seq_lens = seq_lens;
    a.qsl = query_start_loc;
    a.keys = static_cast<uint32_t*>(ws);
    a.num_seqs = static_cast<int32_t>(num_seqs);
    a.hq = static_cast<int32_t>(num_q_heads);
    a.hkv = static_cast<int32_t>(num_kv_heads);
    a.d = static_cast<int32_t>(head_dim);
    a.bs_log2 = __builtin_ctz(static_cast<unsigned>(block_size));
    a.maxb = static_cast<int32_t>(max_num_blocks_per_seq);
    a.k = static_cast<int32_t>(num_selected);
    a.first = static_cast<int32_t>(num_first);
    a.last = static_cast<int32_t>(num_last);
    a.chunk = static_cast<int32_t>(p.chunk);
    a.chunks = static_cast<int32_t>(p.chunks);
    a.num_blocks = num_blocks;
    a.pitch = p.pitch;
    a.tiles = p.tiles;
    a.group_log2 = p.group_log2;
    const hipStream_t st = as_stream(stream);
    for (int64_t r = 0; r < num_rows; r += p.slab) {
        a.row0 = static_cast<int32_t>(r);
        a.rows = static_cast<int32_t>(num_rows - r < p.slab ? num_rows - r : p.slab);
        const int64_t units = p.slab * num_kv_heads;     // the scratch's layout is that of a whole slab
        a.kmax = reinterpret_cast<float*>(a.keys + units * p.pitch);
        a.state = reinterpret_cast<uint8_t*>(a.kmax + units * (p.pitch / SELECT_CHUNK_MIN));
        int32_t rc;
        if (q_dtype == RLLM_DTYPE_BF16)
            rc = kv_dtype == RLLM_DTYPE_FP8_E4M3   ? launch_select<KIND_BF16, KIND_FP8_E4M3>(a, st)
                 : kv_dtype == RLLM_DTYPE_FP8_E5M2 ? launch_select<KIND_BF16, KIND_FP8_E5M2>(a, st)
                                                   : launch_select<KIND_BF16, KIND_BF16>(a, st);
        else
            rc = kv_dtype == RLLM_DTYPE_FP8_E4M3   ? launch_select<KIND_F16, KIND_FP8_E4M3>(a, st)
                 : kv_dtype == RLLM_DTYPE_FP8_E5M2 ? launch_select<KIND_F16, KIND_FP8_E5M2>(a, st)
                                                   : launch_select<KIND_F16, KIND_F16>(a, st);
        if (rc) return rc;
    }
    return 0;
}

}  // extern "C"
