// Shared pieces of the operators over selected cache blocks (sparse_bounds.hip,
// sparse_select.hip, sparse_attention.hip): shape rules, where a query row stands
// in its sequence, and the order of stored elements.
//
// The bounds of a block are the smallest and the largest key of each channel over
// the block's rows that hold keys, k_bounds [num_blocks, num_kv_heads, 2, head_dim]
// in the cache's own element type (a minimum of stored keys is a stored key, so
// nothing is rounded).
#pragma once

#include "common.h"
#include "../../include/rllm_kernels.h"

#include <cmath>

namespace rllm {

// shapes every operator here takes
static inline bool sparse_shape(int64_t hkv, int64_t d, int64_t bs) {
    return hkv > 0 && hkv <= 1024 && d > 0 && d <= 256 && d % 32 == 0 && (bs == 16 || bs == 32 || bs == 64 || bs == 128);
}
static inline bool sparse_heads(int64_t hq, int64_t hkv) { return hq > 0 && hq <= 1024 && hq % hkv == 0; }
static inline bool sparse_types(int32_t q_dtype, int32_t kv_dtype) {
    return (q_dtype == RLLM_DTYPE_F16 || q_dtype == RLLM_DTYPE_BF16) &&
           (kv_dtype == q_dtype || kv_dtype == RLLM_DTYPE_FP8_E4M3 || kv_dtype == RLLM_DTYPE_FP8_E5M2);
}
static inline bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
constexpr int64_t SPARSE_MAX_ROWS = int64_t(1) << 24;    // rows of a call, and sequences
static inline bool sparse_table(int64_t maxb, int64_t bs) { return maxb >= 0 && maxb <= INT32_MAX / bs; }   // positions are 32-bit

namespace {

template <int KIND> constexpr bool sparse_is_fp8() { return KIND == KIND_FP8_E4M3 || KIND == KIND_FP8_E5M2; }

// A query row (or new token): its sequence, the place among the sequence's rows
// of the call, their number, and the row's position; seq -1 for a row that no
// sequence has.
struct SparseRow {
    int32_t seq, i, n, pos;
};
__device__ __forceinline__ SparseRow sparse_row(int32_t t, const int32_t* qsl, const int32_t* seq_lens, int32_t num_seqs) {
    if (!qsl) return {t, 0, 1, seq_lens[t] - 1};
    int32_t lo = 0, hi = num_seqs;       // the first sequence that ends past t
    while (lo < hi) {
        const int32_t mid = (lo + hi) >> 1;
        if (qsl[mid + 1] <= t) lo = mid + 1;
        else hi = mid;
    }
    if (lo >= num_seqs) return {-1, 0, 0, -1};
    const int32_t q0 = qsl[lo], n = qsl[lo + 1] - q0;
    if (t < q0) return {-1, 0, 0, -1};
    return {lo, t - q0, n, seq_lens[lo] - n + (t - q0)};
}

struct SparseTile {
    int32_t seq, row, i, n;
};
// Tile x of the sequences' rows, each sequence's cut into tiles of its own: its sequence
// (-1: there are fewer), first row, place among the sequence's rows, and their number.
__device__ __forceinline__ SparseTile sparse_tile(int x, int tile, const int32_t* qsl, int num_seqs) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < num_seqs; s0 += 64) {
        const int s = s0 + lane;
        const int q0 = s < num_seqs ? qsl[s] : 0, n = s < num_seqs ? max(qsl[s + 1] - q0, 0) : 0;
        const int tiles = (n + tile - 1) / tile;
        int sum = tiles;
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(sum, d);
            if (lane >= d) sum += y;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(sum > x);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int i = (x - __builtin_amdgcn_readlane(sum - tiles, l)) * tile;
            return {s0 + l, __builtin_amdgcn_readlane(q0, l) + i, i, __builtin_amdgcn_readlane(n, l)};
        }
        x -= __builtin_amdgcn_readlane(sum, 63);
    }
    return {-1, 0, 0, 0};
}

// Stored elements as 16-bit integers that rise with the value (an FP8 byte in the
// upper half): the sign's magnitude is turned round.  Its own inverse.  A positive
// NaN lies above +inf, a negative one below -inf, so one of the two bounds keeps it.
typedef short i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ i16x2 ordered2(uint32_t w) {
    const i16x2 x = __builtin_bit_cast(i16x2, w);
    return x ^ ((x >> 15) & i16x2{0x7fff, 0x7fff});
}
__device__ __forceinline__ int16_t ordered1(int16_t x) { return static_cast<int16_t>(x ^ ((x >> 15) & 0x7fff)); }

// lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ uint32_t quads_umax(uint32_t v) {
    const auto x = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(static_cast<uint32_t>(x[0]), static_cast<uint32_t>(x[1]));
    const auto y = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(static_cast<uint32_t>(y[0]), static_cast<uint32_t>(y[1]));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}
// of all 64 lanes
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    v = max(v, dpp_u<DPP_QUAD_XOR1>(v));
    v = max(v, dpp_u<DPP_QUAD_XOR2>(v));
    v = max(v, dpp_u<DPP_ROW_HALF_MIRROR>(v));
    v = max(v, dpp_u<DPP_ROW_MIRROR>(v));
    return quads_umax(v);
}
// the sum of 16 lanes, in each of them
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
    const uint64_t w = static_cast<uint64_t>(dpp_u<CTRL>(static_cast<uint32_t>(u >> 32))) << 32 | dpp_u<CTRL>(static_cast<uint32_t>(u));
    return __longlong_as_double(static_cast<long long>(w));
}
__device__ __forceinline__ double row_sum16(double v) {
    v += dpp_d<DPP_QUAD_XOR1>(v);
    v += dpp_d<DPP_QUAD_XOR2>(v);
    v += dpp_d<DPP_ROW_HALF_MIRROR>(v);
    return v + dpp_d<DPP_ROW_MIRROR>(v);
}

}  // namespace
}  // namespace rllm
