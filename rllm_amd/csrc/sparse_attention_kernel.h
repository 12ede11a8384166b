// Attention over listed cache blocks, for gfx950: decode rows and chunks of prompts.
// The kernel and its launches; a translation unit for each type of cache.
//
//   o = softmax(scale q . K^T) V over the keys of the listed blocks that the row sees,
// in one pass with a running maximum and sum.
//
// Bound by HBM (decode) or by what the L2s bring (chunks, whose rows list much the
// same blocks): K and V of the listed blocks are read once per row and 16 query heads.
//
// Work: a workgroup of 4 or 8 waves takes one (row, kv head, 16 heads), or in a chunk
// a tile of consecutive rows of one sequence that fill the 16 columns with the heads of
// one kv head: the tile attends the union of its rows' lists, and each row's weights of blocks
// that it does not list are 0.  The list's keys stand one after the other and are cut
// into windows of 64, wave w taking windows w, w + waves, ...; the waves merge
// through LDS.  Per window and wave:
//   copies        K and V arrive by 16-byte loads whose lanes read runs of memory (the
//                 next window's on the way while this one is worked on) and go to the
//                 wave's part of LDS as groups of 16 tokens, [group][head_dim][16].
//   S^T = K Q^T   v_mfma_16x16x32, rows = the tokens of a group, columns = heads; the K
//                 operand by transposing LDS reads of 16 head_dim rows in a run.
//   O^T = V^T P^T rows = head_dim, k = the tokens of two groups, four of each a lane:
//                 the scores of a lane are the weights it needs, V's operand two 8-byte
//                 LDS reads.
// Loads that gave every lane the 8 x 8 tile it transposes itself read 16 bytes here
// and there, without LDS: no faster for 64 rows on 128 blocks (head_dim 128, 99 us either way, 5.4
// TB/s), and 311 us for 704 rows of two chunks on 64, where whole runs and tiles take 148.
// Weights enter as two 16-bit terms (generic_mfma.h), in bf16 16 bits of them, in f16 22.
// A third term in bf16 made 167 of 262144 outputs of the 64 rows differ from f32 weights' by a
// last bit instead of 524, with the same error against 64 bits (the output's rounding,
// 2^-9, hides both), and the chunks 150 us instead of 144: left out.
#pragma once

#include "sparse_blocks.h"
#include "sparse_plan.h"
#include "generic_mfma.h"
#include "workspace.h"

namespace rllm {

static_assert(SA_MAX_LIST >= RLLM_SELECT_MAX_BLOCKS, "a row's list fits");

struct SparseArgs {
    uint16_t* out;
    const uint16_t* q;
    const uint8_t *kc, *vc;
    const int32_t *bt, *seq_lens, *qsl, *sel;
    int32_t num_seqs, rows, hq, hkv, bs_log2, maxb, k, head_groups;
    int32_t splits;             // workgroups of a unit, joined by the last to end
    int32_t* count;             // arrivals of a unit, 0 between calls
    float* part;                // [unit][split][16 columns][head_dim + 4]: sum, max, sum of weights, two unused
    int32_t tile, list;         // rows of a workgroup (1, or 16 / heads of a kv head), and the entries its list has room for
    int64_t num_blocks;
    float s_scale, v_scale;     // s_scale: scale * k_scale * log2(e)
};

namespace {

__device__ __forceinline__ float over_quads_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_quads_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

typedef uint32_t sa_u32x4 __attribute__((ext_vector_type(4)));   // (uint4 arrays of these loads end up in scratch)
typedef short sa_i16x4 __attribute__((ext_vector_type(4)));
// Transposing LDS read: in each 16 lanes, lane j addresses 4 consecutive 16-bit values
// M[j][0..3]; lane i receives M[4 k + i / 4][i % 4], k = 0..3.  (Not in the kernel
// templates themselves: the host pass does not know the builtin.)
__device__ __forceinline__ uint2 sa_read_tr16(const uint8_t* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sa_i16x4*)(p)));
}

// One row and head by a wave, key by key: what a tile falls back to where its outputs are
// not finite.
template <int QKIND, int KVKIND>
__device__ __forceinline__ void sparse_one(const SparseArgs& a, int t, int h, int g, int seq, int pos, int D, int bs_log2) {
    using tag = typename GenMfma<QKIND>::tag;
    const int lane = threadIdx.x & 63, hkv = a.hkv;
    const int64_t row = (static_cast<int64_t>(t) * a.hq + h * (a.hq / hkv) + g) * D;
    const int32_t* const sel = a.sel + (static_cast<int64_t>(t) * hkv + h) * a.k;
    const int32_t* const bt = a.bt + static_cast<int64_t>(seq) * a.maxb;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    for (int x = 0; x < 4; ++x) q[x] = lane + 64 * x < D ? to_f32<tag>(a.q[row + lane + 64 * x]) : 0.f;
    auto value = [&](const uint8_t* cache, int64_t i) {
        if constexpr (gen_is_fp8<KVKIND>()) {
            const uint32_t w = cache[i];
            return bf16_lo(KVKIND == KIND_FP8_E4M3 ? e4m3x2_to_bf16x2(w, false) : e5m2x2_to_bf16x2(w, false));
        } else {
            return to_f32<tag>(reinterpret_cast<const uint16_t*>(cache)[i]);
        }
    };
    int before = -1;
    for (int e = 0; e < a.k; ++e) {
        const int j = sel[e], last = before;
        before = j;
        if (j <= last || j < 0) break;
        if (j >= a.maxb || j > pos >> bs_log2) continue;
        const int b = bt[j];
        if (b < 0 || b >= a.num_blocks) continue;
        const int64_t at = (static_cast<int64_t>(b) * hkv + h) * D;
        const int seen = min(pos + 1 - (j << bs_log2), 1 << bs_log2);
        for (int k = 0; k < seen; ++k) {
            float s = 0.f;
            for (int x = 0; x < 4; ++x)
                if (lane + 64 * x < D) s += q[x] * value(a.kc, ((at + lane + 64 * x) << bs_log2) + k);
            s = wave_sum(s) * a.s_scale;
            const float mn = s > m ? s : m, al = m == mn ? 1.f : exp2f(m - mn), p = s == -INFINITY ? 0.f : exp2f(s - mn);
            l = l * al + p;
            for (int x = 0; x < 4; ++x)
                if (lane + 64 * x < D) o[x] = o[x] * al + p * value(a.vc, ((at + lane + 64 * x) << bs_log2) + k);
            m = mn;
        }
    }
    const float f = gen_inv(a.v_scale, l);
    for (int x = 0; x < 4; ++x)
        if (lane + 64 * x < D) a.out[row + lane + 64 * x] = from_f32<tag>(o[x] * f);
}

template <int QKIND, int KVKIND, int NK, int RUN>
__global__ __launch_bounds__(64 * sa_max_waves(32 * NK), (sa_max_waves(32 * NK) / 4)) void sparse_attention_kernel(SparseArgs a) {
    using M = GenMfma<QKIND>;
    constexpr bool FP8 = gen_is_fp8<KVKIND>();
    constexpr int D = 32 * NK, ND = D / 16, ES = FP8 ? 1 : 2;
    constexpr int NL = (FP8 ? 2 : 4) * NK;                      // 16-byte loads of K, or V, of a window
    constexpr int NB = SA_WIN >> RUN;                           // blocks of a window
    constexpr bool EVEN = !FP8 || NK % 2 == 0 || RUN > 4;       // a load instruction lies in one block
    const int bs_log2 = RUN < 6 ? RUN : a.bs_log2;              // of a block; past 64 tokens a window is a part of one
    constexpr int GB = sa_group_bytes(D), STAGE = sa_stage_bytes(D);
    constexpr int OST = D + 4;                                  // row of one head's partial
    static_assert(STAGE >= (16 * OST + 32) * 4, "a wave's partials go where its windows were");
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int s_used, s_end[16];                           // entries of the list, and of each row's
    __shared__ int s_count[8];
    const int waves = blockDim.x >> 6, threads = blockDim.x;
    int32_t* const s_list = reinterpret_cast<int32_t*>(lds + waves * STAGE);    // cache blocks, -1 = nothing to attend
    int32_t* const s_num = s_list + a.list;                                     // their numbers within the sequence
    uint16_t* const s_mask = reinterpret_cast<uint16_t*>(s_num + a.list);       // rows of the tile that list them

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q4 = lane >> 4;
    const int G = a.hq / a.hkv;
    const int hg = blockIdx.x % a.head_groups;
    const int split = blockIdx.x / a.head_groups % a.splits;
    const int unit = blockIdx.x / a.head_groups / a.splits, h = unit % a.hkv;
    // column r: row r >> gl of the tile, head 16 hg + (r & (2^gl - 1)) of the group
    const int gl = a.tile > 1 ? 31 - __builtin_clz(16 / a.tile) : 4;
    const int col_row = r >> gl, col_head = 16 * hg + (r & ((1 << gl) - 1));
    const float c = __builtin_fabsf(a.s_scale);
    const uint8_t* const zero = reinterpret_cast<const uint8_t*>(g_gen_zero);

    // A load's 16-byte chunks, 64 a load, count block by block of the window, row by
    // row, along the tokens: chunks of a row, as a power of two, and a lane's place.
    constexpr int cl = RUN - (FP8 ? 4 : 3);
    const int row_b = ES << bs_log2;                          // bytes of a head_dim row of a block
    const int64_t slab_b = static_cast<int64_t>(D) * row_b;
    const int lane_row = lane >> cl, lane_chunk = lane & ((1 << cl) - 1);
    const uint32_t lane_src = lane_row * row_b + lane_chunk * 16;
    uint8_t* const stage = lds + wave * STAGE;
    // A row's two 16-byte halves change places in rows 8 .. 15 of 16: the V operand's
    // rows r and r + 8 then lie on different banks.
    auto swap16 = [](int d) __attribute__((always_inline)) { return (d & 8) << 1; };
    uint8_t* const lane_dst = stage + lane_row * 32 + (FP8 ? lane_chunk * GB : (lane_chunk >> 1) * GB);
    const int lane_half = FP8 ? 0 : (lane_chunk & 1) * 16;
    constexpr int groups_log2 = RUN - 4;                        // 16-token groups of a block within a window

    // the rows: t .. t + nt - 1 of sequence seq, the first at position pos
    int t, nt, seq, pos;
    if (a.tile > 1) {
        const SparseTile x = sparse_tile(unit / a.hkv, a.tile, a.qsl, a.num_seqs);
        if (x.seq < 0) return;
        seq = x.seq;
        t = x.row;
        nt = min(min(a.tile, x.n - x.i), a.rows - t);
        pos = a.seq_lens[seq] - x.n + x.i;
        if (nt <= 0 || t < 0) return;
    } else {
        t = unit / a.hkv;
        const SparseRow x = sparse_row(t, a.qsl, a.seq_lens, a.num_seqs);
        if (x.seq < 0) return;
        seq = x.seq;
        nt = 1;
        pos = x.pos;
    }
    const int32_t* const bt = a.bt + static_cast<int64_t>(seq) * a.maxb;
    const int32_t* const sel = a.sel + (static_cast<int64_t>(t) * a.hkv + h) * a.k;
    const int64_t sel_row = static_cast<int64_t>(a.hkv) * a.k;
    // a list ends at its first entry that is not above the one before it
    auto ends = [&](int j, int before) __attribute__((always_inline)) { return j <= before || j < 0; };
    auto seen = [&](int j, int p) __attribute__((always_inline)) { return j < a.maxb && j <= p >> bs_log2; };
    auto block_of = [&](int j) __attribute__((always_inline)) -> int {
        const int b = bt[j];
        return b >= 0 && b < a.num_blocks ? b : -1;
    };
    if (threadIdx.x == 0) s_used = 0;
    if (threadIdx.x < 16) s_end[threadIdx.x] = a.k;
    if (nt == 1) {
        __syncthreads();
        int most = 0;
        for (int i0 = 0; i0 < a.k; i0 += threads) {
            const int i = i0 + threadIdx.x;
            const int j = i < a.k ? sel[i] : 0x7fffffff, before = i > 0 && i < a.k ? sel[i - 1] : -1;
            const uint64_t over = __builtin_amdgcn_ballot_w64(ends(j, before));
            if (over && lane == 0) atomicMin(&s_end[0], i + __builtin_ctzll(over));
            if (i < a.k) {
                const int b = !ends(j, before) && seen(j, pos) ? block_of(j) : -1;
                s_list[i] = b;
                s_num[i] = j;
                s_mask[i] = 1;
                if (b >= 0) most = i + 1;
            }
        }
        most = static_cast<int>(wave_umax(static_cast<uint32_t>(most)));
        if (lane == 0 && most) atomicMax(&s_used, most);
    } else {
        // the union: a word of bits for every block of the sequence, where the windows will be
        uint16_t* const s_bits = reinterpret_cast<uint16_t*>(lds);
        const int nv = pos + nt - 1 < 0 ? 0 : min(((pos + nt - 1) >> bs_log2) + 1, a.maxb);
        const int words = (nv + 1) >> 1;
        for (int i = threadIdx.x; i < words; i += threads) reinterpret_cast<uint32_t*>(s_bits)[i] = 0;
        __syncthreads();
        auto entry = [&](int i, int& x, int& e, int& before) __attribute__((always_inline)) -> int {
            x = i / a.k;
            e = i - x * a.k;
            before = e ? sel[x * sel_row + e - 1] : -1;
            return sel[x * sel_row + e];
        };
        int x, e, before;
        for (int i = threadIdx.x; i < nt * a.k; i += threads)
            if (ends(entry(i, x, e, before), before)) atomicMin(&s_end[x], e);
        __syncthreads();
        for (int i = threadIdx.x; i < nt * a.k; i += threads) {
            const int j = entry(i, x, e, before);
            if (e < s_end[x] && seen(j, pos + x)) atomicOr(reinterpret_cast<uint32_t*>(s_bits) + (j >> 1), 1u << (16 * (j & 1) + x));
        }
        __syncthreads();
        // wave w the w-th part of the blocks
        const int part = (nv + 64 * waves - 1) / (64 * waves) * 64;
        const int j0 = wave * part, j1 = min(j0 + part, nv);
        int n = 0;
        for (int j = j0; j < j1; j += 64) n += __popcll(__builtin_amdgcn_ballot_w64(j + lane < j1 && s_bits[j + lane]));
        if (lane == 0) s_count[wave] = n;
        __syncthreads();
        int at = 0;
        for (int w = 0; w < waves; ++w) {
            if (w == wave) n = at;
            at += s_count[w];
        }
        for (int j = j0; j < j1; j += 64) {
            const uint32_t bits = j + lane < j1 ? s_bits[j + lane] : 0;
            const uint64_t m = __builtin_amdgcn_ballot_w64(bits != 0);
            if (bits) {
                const int i = n + __popcll(m & ((uint64_t(1) << lane) - 1));
                s_list[i] = block_of(j + lane);
                s_num[i] = j + lane;
                s_mask[i] = static_cast<uint16_t>(bits);
            }
            n += __popcll(m);
        }
        if (threadIdx.x == 0) s_used = at;
    }

    // queries, negated where the scale is negative (exact), so that the running max is
    // over c * s with c >= 0
    const bool col_live = col_row < nt && col_head < G && (a.tile > 1 || col_head < 16 * hg + 16);
    const int64_t out_row = static_cast<int64_t>(t + col_row) * a.hq + h * G + col_head;
    uint4 qreg[NK];
    {
        const uint32_t flip = a.s_scale < 0.f ? 0x80008000u : 0u;
        const uint16_t* qrow = a.q + out_row * D;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (col_live) {
                const uint2 y = *reinterpret_cast<const uint2*>(qrow + 32 * k + 4 * q4);
                const uint2 z = *reinterpret_cast<const uint2*>(qrow + 32 * k + 16 + 4 * q4);
                x = make_uint4(y.x, y.y, z.x, z.y);
            }
            qreg[k] = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
        }
    }
    __syncthreads();
    const int used = __builtin_amdgcn_readfirstlane(nt == 1 ? min(s_used, s_end[0]) : s_used);
    const int end = used << bs_log2;                        // tokens of the list
    const int first_own = pos < 0 ? 0 : pos >> bs_log2;     // blocks before it every row sees whole
    const int last_seen = pos + nt;                         // keys of the sequence that the last row sees

    sa_u32x4 kbuf[NL], vbuf[NL];
    // entries of the window at token w, one a lane: cache blocks, numbers, masks
    auto entries = [&](int w, int& block, int& num, int& mask) __attribute__((always_inline)) {
        const int e = (w >> bs_log2) + (lane & (NB - 1));
        block = -1;
        num = 0x7fffffff;
        mask = 0;
        if (e < used) {
            block = s_list[e];
            num = s_num[e];
            mask = s_mask[e];
        }
    };
    const uint32_t full = (1u << nt) - 1;
    auto load = [&](const uint8_t* cache, int w, int blocks, sa_u32x4 (&buf)[NL]) __attribute__((always_inline)) {
        if constexpr (EVEN) {
#pragma unroll
            for (int bi = 0; bi < NB; ++bi) {
                const int b = __builtin_amdgcn_readlane(blocks, bi);
                const int within = RUN < 6 ? 0 : (w & ((1 << bs_log2) - 1)) * ES;
                const uint8_t* const base = b >= 0 ? cache + (static_cast<int64_t>(b) * a.hkv + h) * slab_b + within : zero;
                const uint32_t off = b >= 0 ? lane_src : 0u;
                const int rs = b >= 0 ? (64 >> cl) * row_b : 0;          // bytes from a load's rows to the next one's
#pragma unroll
                for (int n = 0; n < NL / NB; ++n)
                    buf[bi * (NL / NB) + n] = *reinterpret_cast<const sa_u32x4*>(base + n * rs + off);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NL; ++n) {
                const int at = (64 * n + lane) >> cl, bi = at / D;
                const int b = __shfl(blocks, bi);
                const uint8_t* p = b >= 0 ? cache + (static_cast<int64_t>(b) * a.hkv + h) * slab_b +
                                                ((at - bi * D) * row_b + lane_chunk * 16)
                                          : zero;
                buf[n] = *reinterpret_cast<const sa_u32x4*>(p);
            }
        }
    };
    auto store = [&](const sa_u32x4 (&buf)[NL]) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            uint8_t* dst;
            int half;
            if constexpr (EVEN) {
                // row1 is a multiple of 8, and of 16 where a lane's row passes 7
                const int bi = n / (NL / NB), row1 = (n - bi * (NL / NB)) * (64 >> cl);
                dst = lane_dst + (bi << groups_log2) * GB + row1 * 32;
                half = lane_half ^ swap16(lane_row) ^ swap16(row1);
            } else {
                const int at = (64 * n + lane) >> cl, bi = at / D, d = at - bi * D;
                dst = stage + ((bi << groups_log2) + lane_chunk) * GB + d * 32;
                half = swap16(d);
            }
            if constexpr (FP8) {
                *reinterpret_cast<uint4*>(dst + half) = gen_to16<QKIND, KVKIND>(make_uint2(buf[n][0], buf[n][1]));
                *reinterpret_cast<uint4*>(dst + (half ^ 16)) = gen_to16<QKIND, KVKIND>(make_uint2(buf[n][2], buf[n][3]));
            } else {
                *reinterpret_cast<sa_u32x4*>(dst + half) = buf[n];
            }
        }
        __builtin_amdgcn_wave_barrier();
    };

    gm_f32x4 o[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[dt] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;
    const int stride = SA_WIN * waves * a.splits;               // from a wave's window to its next
    int w0 = SA_WIN * (split * waves + wave);
    int blocks, nums, masks;
    entries(w0, blocks, nums, masks);
    if (w0 < end) {
        load(a.kc, w0, blocks, kbuf);
        load(a.vc, w0, blocks, vbuf);
    }
    const uint8_t* const k_src = stage + (4 * q4 + (r >> 2)) * 32 + (((r & 3) * 8) ^ swap16(4 * q4));
    const uint8_t* const v_src = stage + r * 32 + ((q4 * 8) ^ swap16(r));
    while (w0 < end) {
        const int w1 = w0 + stride;
        int next, next_nums, next_masks;
        entries(w1, next, next_nums, next_masks);
        // ---- S^T = K Q^T ----
        store(kbuf);
        if (w1 < end) load(a.kc, w1, next, kbuf);
        gm_f32x4 acc[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            acc[g] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const uint2 x = sa_read_tr16(k_src + g * GB + k * 1024), y = sa_read_tr16(k_src + g * GB + k * 1024 + 512);
                acc[g] = M::mma16(make_uint4(x.x, x.y, y.x, y.y), qreg[k], acc[g]);
            }
        }
        __builtin_amdgcn_wave_barrier();
        store(vbuf);

        // Keys of each group that the column sees: 16 of a block that its row lists and that
        // lies before its own, as long as no block of the window is at the rows' own.
        const bool near = __builtin_amdgcn_ballot_w64(nums >= first_own) != 0;
        bool whole = !near;
        int n[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int bi = g >> groups_log2;
            const int b = __builtin_amdgcn_readlane(blocks, bi);
            const uint32_t mask = __builtin_amdgcn_readlane(masks, bi);
            whole = whole && b >= 0 && mask == full;
            n[g] = b >= 0 && (mask >> col_row & 1) ? 16 : 0;
        }
        if (near) {
            const int off = RUN < 6 ? 0 : w0 & ((1 << bs_log2) - 1);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int bi = g >> groups_log2;
                const int g0 = (__builtin_amdgcn_readlane(nums, bi) << bs_log2) + off + 16 * (g & ((1 << groups_log2) - 1));   // the group's first position
                n[g] = min(n[g], max(pos + col_row + 1 - g0, 0));
                // values behind the sequence's last key may be anything
                const int held = min(max(last_seen - g0, 0), 16);
                if (held < 16 && __builtin_amdgcn_readlane(blocks, bi) >= 0) {
                    for (int d = lane; d < D; d += 64) {
                        uint4* const v = reinterpret_cast<uint4*>(stage + g * GB + d * 32);
                        v[swap16(d) >> 4] = gen_keep(v[swap16(d) >> 4], held);
                        v[1 - (swap16(d) >> 4)] = gen_keep(v[1 - (swap16(d) >> 4)], held - 8);
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }

        // ---- weights: lane (head r, q4) holds tokens 4 q4 + i of every group ----
        float p[2][8];
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[g >> 1][4 * (g & 1) + i] = acc[g][i];
        if (!whole) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * q4 + i >= n[g]) p[g >> 1][4 * (g & 1) + i] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fmaxf(p[0][i], p[1][i]));
        // the max, lowered by the weights' lift; c = 0 times an infinity must not poison it
        const float m_new = fmaxf(m_run, over_quads_max(mx == -INFINITY ? mx : mx * c - gen_decode_lift<QKIND>()));
        const float ms = m_new == -INFINITY ? 0.f : m_new;
        if (__builtin_amdgcn_ballot_w64(!(__builtin_fabsf(ms) <= 0x1p20f)) == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[0][i] = __builtin_amdgcn_exp2f(fmaf(p[0][i], c, -ms));
                p[1][i] = __builtin_amdgcn_exp2f(fmaf(p[1][i], c, -ms));
            }
        } else {
            // past 2^20 the roundings of the product and of the lowered max show: the same product
            // on both sides then, and no weight above 2^lift (f16 ends at 2^16)
#pragma clang fp contract(off)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = p[i >> 3][i & 7] * c, e = y - ms;
                p[i >> 3][i & 7] = __builtin_amdgcn_exp2f(e > gen_decode_lift<QKIND>() ? gen_decode_lift<QKIND>() : e);   // NaN goes on
            }
        }
        if (!whole && c == 0.f) {                               // 0 * -inf
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * q4 + i >= n[g]) p[g >> 1][4 * (g & 1) + i] = 0.f;
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += p[0][i] + p[1][i];
        if (__builtin_amdgcn_ballot_w64(m_new != m_run)) {
            const float alpha = exp2f(m_run - ms);
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) o[dt] *= alpha;
        }
        l_run += sum;
        m_run = m_new;

        // ---- O^T += V^T P^T ----
        if (w1 < end) load(a.vc, w1, next, vbuf);
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
            uint4 ph, pl;
            gen_split8<QKIND>(p[pair], ph, pl);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                const uint2 x = *reinterpret_cast<const uint2*>(v_src + (2 * pair) * GB + dt * 512);
                const uint2 y = *reinterpret_cast<const uint2*>(v_src + (2 * pair + 1) * GB + dt * 512);
                const uint4 v = make_uint4(x.x, x.y, y.x, y.y);
                o[dt] = M::mma16(v, ph, o[dt]);
                o[dt] = M::mma16(v, pl, o[dt]);
            }
        }
        __builtin_amdgcn_wave_barrier();
        w0 = w1;
        blocks = next;
        nums = next_nums;
        masks = next_masks;
    }

    // ---- merge the waves: their partials where their windows were ----
    l_run = over_quads_sum(l_run);
    auto s_o = [&](int w) __attribute__((always_inline)) { return reinterpret_cast<float*>(lds + w * STAGE); };   // [column][OST], max, sum
    if (q4 == 0) {
        s_o(wave)[16 * OST + r] = m_run;
        s_o(wave)[16 * OST + 16 + r] = l_run;
    }
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) *reinterpret_cast<gm_f32x4*>(s_o(wave) + r * OST + 16 * dt + 4 * q4) = o[dt];
    __syncthreads();
    constexpr int quads = D >> 2;
    const int64_t part_unit = static_cast<int64_t>(unit) * a.head_groups + hg;
    bool bad = false;
    for (int it = threadIdx.x; it < 16 * quads; it += threads) {
        const int col = it / quads, d0 = (it - col * quads) * 4;
        const int cr = col >> gl, ch = 16 * hg + (col & ((1 << gl) - 1));
        if (cr >= nt || ch >= G) continue;
        float mx = -INFINITY;
        for (int w = 0; w < waves; ++w) mx = fmaxf(mx, s_o(w)[16 * OST + col]);
        gm_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        float L = 0.f;
        for (int w = 0; w < waves; ++w) {
            const float lw = s_o(w)[16 * OST + 16 + col];
            if (lw == 0.f) continue;                            // a wave without keys (NaN goes on)
            const float f = exp2f(s_o(w)[16 * OST + col] - mx);
            L = fmaf(f, lw, L);
            sum += f * *reinterpret_cast<const gm_f32x4*>(s_o(w) + col * OST + d0);
        }
        if (a.splits > 1) {
            float* const x = a.part + ((part_unit * a.splits + split) * 16 + col) * (D + 4);
            *reinterpret_cast<gm_f32x4*>(x + d0) = sum;
            if (d0 == 0) *reinterpret_cast<gm_f32x4*>(x + D) = gm_f32x4{mx, L, 0.f, 0.f};
            continue;
        }
        const gm_f32x4 v = sum * gen_inv(a.v_scale, L);
        bad |= !(gen_finite(v[0]) && gen_finite(v[1]) && gen_finite(v[2]) && gen_finite(v[3]));
        *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(t + cr) * a.hq + h * G + ch) * D + d0) =
            make_uint2(M::pack2(v[0], v[1]), M::pack2(v[2], v[3]));
    }
    if (a.splits > 1) {
        // The last workgroup of the unit joins its parts, in their order.  Each wave's parts
        // have left the CU before the arrival that releases them to the other XCDs.
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (threadIdx.x == 0) {
            const int before = __hip_atomic_fetch_add(a.count + part_unit, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
            s_used = before == a.splits - 1;
            if (s_used) __hip_atomic_store(a.count + part_unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!s_used) return;
        for (int it = threadIdx.x; it < 16 * quads; it += threads) {
            const int col = it / quads, d0 = (it - col * quads) * 4;
            if (16 * hg + col >= G) continue;
            const float* const x = a.part + (part_unit * a.splits * 16 + col) * (D + 4);
            constexpr int step = 16 * (D + 4);
            gm_f32x4 v[SA_MAX_SPLITS];
            gm_f32x2 ml[SA_MAX_SPLITS];
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < SA_MAX_SPLITS; ++i) {
                const int j = min(i, a.splits - 1);
                v[i] = *reinterpret_cast<const gm_f32x4*>(x + j * step + d0);
                ml[i] = *reinterpret_cast<const gm_f32x2*>(x + j * step + D);
                mx = fmaxf(mx, ml[i][0]);
            }
            gm_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
            float L = 0.f;
#pragma unroll
            for (int i = 0; i < SA_MAX_SPLITS; ++i) {
                if (i >= a.splits || ml[i][1] == 0.f) continue;
                const float f = exp2f(ml[i][0] - mx);
                L = fmaf(f, ml[i][1], L);
                sum += f * v[i];
            }
            sum *= gen_inv(a.v_scale, L);
            *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(t) * a.hq + h * G + 16 * hg + col) * D + d0) =
                make_uint2(M::pack2(sum[0], sum[1]), M::pack2(sum[2], sum[3]));
        }
        return;
    }
    // 0 * Inf from a block that another row of the tile lists would show here: rows by themselves
    if (nt > 1 && __syncthreads_or(bad))
        for (int x = 0; x < nt; ++x)
            for (int g = wave; g < G; g += waves) sparse_one<QKIND, KVKIND>(a, t + x, h, g, seq, pos + x, D, bs_log2);
}

template <int QKIND, int KVKIND, int RUN>
int32_t launch_sparse_run(const SparseArgs& a, int64_t d, int waves, hipStream_t st) {
    const int64_t tiles = a.tile > 1 ? (static_cast<int64_t>(a.rows) + a.tile - 1) / a.tile + a.num_seqs : a.rows;
    const int64_t count = tiles * a.hkv * a.head_groups * a.splits;
    RLLM_CHECK_ARG(count <= MAX_WORKGROUPS);                  // (of 512 threads where units are few)
    const dim3 grid(static_cast<unsigned>(count)), block(64 * waves);
    const size_t lds = static_cast<size_t>(waves) * sa_stage_bytes(static_cast<int>(d)) + a.list * SA_ENTRY;
    switch (d / 32) {
#define RLLM_SPARSE(N) \
    case N: hipLaunchKernelGGL((sparse_attention_kernel<QKIND, KVKIND, N, RUN>), grid, block, lds, st, a); break;
        RLLM_SPARSE(1) RLLM_SPARSE(2) RLLM_SPARSE(3) RLLM_SPARSE(4) RLLM_SPARSE(5) RLLM_SPARSE(6) RLLM_SPARSE(7) RLLM_SPARSE(8)
#undef RLLM_SPARSE
    }
    return launch_status();
}

template <int QKIND, int KVKIND>
int32_t launch_sparse(SparseArgs a, int64_t d, hipStream_t st) {
    const SparseShape shape = {a.rows, a.num_seqs, a.hq, a.hkv, a.maxb, a.k, static_cast<int>(d), a.bs_log2, a.qsl != nullptr};
    void* ws = nullptr;
    if (sparse_few(shape)) {
        const int32_t rc = g_workspaces.get(reinterpret_cast<uintptr_t>(st), WS_SPARSE, 1024 + 256 * 16 * (d + 4) * 4, true, &ws);
        if (rc) return rc;
        if (ws) {
            a.count = static_cast<int32_t*>(ws);
            a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + 1024);
        }
    }
    const SparsePlan plan = sparse_plan(shape, ws != nullptr);
    const int waves = plan.waves;
    a.splits = plan.splits;
    a.tile = plan.tile;
    a.list = plan.list;
    if (a.bs_log2 == 4) return launch_sparse_run<QKIND, KVKIND, 4>(a, d, waves, st);
    if (a.bs_log2 == 5) return launch_sparse_run<QKIND, KVKIND, 5>(a, d, waves, st);
    return launch_sparse_run<QKIND, KVKIND, 6>(a, d, waves, st);
}

}  // namespace

// the launches by cache type (arguments checked by the entry point)
int32_t launch_sparse_16(const SparseArgs& a, int32_t q_dtype, int64_t d, hipStream_t st);
int32_t launch_sparse_e4m3(const SparseArgs& a, int32_t q_dtype, int64_t d, hipStream_t st);
int32_t launch_sparse_e5m2(const SparseArgs& a, int32_t q_dtype, int64_t d, hipStream_t st);

}  // namespace rllm
