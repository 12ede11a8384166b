// Pieces of the attention kernels over the MXFP4 KV cache (mxfp4_decode.hip,
// mxfp4_prefill.hip).
//
// Scores.  S = K Q^T runs on the block-scaled matrix product with K as it lies in
// the cache: a lane's 16 bytes are the 32 codes of one scale, its scale byte the
// product's E8M0 scale, so K is never converted.  The other operand is 8 bits a
// value; a query row is split into E4M3 terms that add up to it: x0 = e4m3(x),
// x1 = e4m3(16 (x - x0)), x2 = e4m3(16 (16 (x - x0) - x1)), with a power of two per row
// (largest element in [128, 256)) and 2^-4 more per term in the scale operand.
// Four significant bits a term: two hold a bf16 (8 bits), three an f16 (11),
// exactly for elements down to 2^-13 of the row's largest, below that within 2^-21
// (bf16; f16 2^-25) of it.  Against 64 bits the summed products of such terms are
// off by 4e-6 of the scores' rms (200 random 128-wide tiles; 3e-5 with 30-fold
// outlier channels): the product's own sums carry about 17 bits below its largest
// terms.
//
// Values.  O^T = V^T P^T runs in bf16: code * 2^(e - 127) is exact in bf16 (two
// significant bits, the f32 exponent range), whatever the query's type.
#pragma once

#include "mxfp4.h"

namespace rllm {
namespace {

// x / factor as four E4M3 bytes, and x less what they stand for (wrappers of target
// builtins, not templates)
__device__ __forceinline__ uint32_t mx4_enc_e4m3(const float (&x)[4], float factor) {
    mx_i16x2 w = {0, 0};
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[0], x[1], factor, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[2], x[3], factor, true);
    return __builtin_bit_cast(uint32_t, w);
}
__device__ __forceinline__ void mx4_sub_e4m3(float (&x)[4], uint32_t w, float factor) {
    const mx_f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, factor, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, factor, true);
    x[0] -= a[0];
    x[1] -= a[1];
    x[2] -= b[0];
    x[3] -= b[1];
}

// What the weights' base is taken ahead of the running max, in log2
constexpr float MX4_AHEAD = 8.f;
// the least factor of a part of a row that saw a key (f32's smallest normal)
constexpr float MX4_LEAST = 1.17549435e-38f;

// terms of a query element
template <int QKIND> constexpr int mx4_terms() { return QKIND == KIND_BF16 ? 2 : 3; }

__device__ __forceinline__ mx_f32x4 mx4_mma16(const uint4& k, const mx_i32x8& q, const mx_f32x4& c, int ks, int qs) {
    const mx_i32x8 a = {static_cast<int>(k.x), static_cast<int>(k.y), static_cast<int>(k.z), static_cast<int>(k.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, c, 4, 0, 0, ks, 0, qs);
}
__device__ __forceinline__ mx_f32x16 mx4_mma32(const uint4& k, const mx_i32x8& q, const mx_f32x16& c, int ks, int qs) {
    const mx_i32x8 a = {static_cast<int>(k.x), static_cast<int>(k.y), static_cast<int>(k.z), static_cast<int>(k.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, q, c, 4, 0, 0, ks, 0, qs);
}
__device__ __forceinline__ mx_f32x4 mx4_mma_bf16(const uint4& a, const uint4& b, const mx_f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_bf16x8, a), __builtin_bit_cast(mx_bf16x8, b), c,
                                                   0, 0, 0);
}
__device__ __forceinline__ mx_f32x16 mx4_mma32_bf16(const uint4& a, const uint4& b, const mx_f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(mx_bf16x8, a), __builtin_bit_cast(mx_bf16x8, b), c,
                                                   0, 0, 0);
}

// Transposing LDS read: in each group of 16 lanes, lane j addresses 4
// consecutive 16-bit values M[j][0..3]; lane i receives M[4k + i/4][i%4] for k = 0..3.
__device__ __forceinline__ uint2 mx4_read_tr16(const uint16_t* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) mx_i16x4*)(p)));
}

__device__ __forceinline__ uint32_t mx4_pack_bf16(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(mx_f32x2{lo, hi}, mx_bf16x2));
}
template <int QKIND> __device__ __forceinline__ uint32_t mx4_pack16(float lo, float hi) {
    if constexpr (QKIND == KIND_BF16) return mx4_pack_bf16(lo, hi);
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(mx_f32x2{lo, hi}, mx_f16x2));
}

// Four query elements (two packed pairs) as E4M3 terms, byte t of w[t]: term t is in
// units of factor * 2^-4t.  Every step is exact but the conversions to E4M3 (nearest,
// ties to even; in range, see mx4_query_byte).
template <int QKIND>
__device__ __forceinline__ void mx4_split4(uint32_t p0, uint32_t p1, float factor, uint32_t (&w)[mx4_terms<QKIND>()]) {
    constexpr int NT = mx4_terms<QKIND>();
    float x[4];
    x[0] = QKIND == KIND_BF16 ? bf16_lo(p0) : f16_lo(p0);
    x[1] = QKIND == KIND_BF16 ? bf16_hi(p0) : f16_hi(p0);
    x[2] = QKIND == KIND_BF16 ? bf16_lo(p1) : f16_lo(p1);
    x[3] = QKIND == KIND_BF16 ? bf16_hi(p1) : f16_hi(p1);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        w[t] = mx4_enc_e4m3(x, factor);
        if (t + 1 < NT) {
            mx4_sub_e4m3(x, w[t], factor);
            factor *= 0.0625f;
        }
    }
}

__device__ __forceinline__ uint32_t mx4_umax_32(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
}
__device__ __forceinline__ uint32_t mx4_umax_16(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return mx4_umax_32(max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1])));
}

// max / sum over the lanes that share l % 16 (XOR 16, 32), or l % 32 (XOR 32 alone)
__device__ __forceinline__ float mx4_max_32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float mx4_sum_32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// x: a of lanes < 32, then b of lanes < 32; y: a of lanes >= 32, then b of lanes >= 32
__device__ __forceinline__ void mx4_swap_32(uint32_t a, uint32_t b, uint32_t& x, uint32_t& y) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    x = r[0];
    y = r[1];
}
__device__ __forceinline__ float mx4_max_16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return mx4_max_32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float mx4_sum_16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return mx4_sum_32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// inclusive prefix sum over the wave
__device__ __forceinline__ int mx4_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);   // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);   // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);   // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast:15 into rows 1, 3
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast:31 into rows 2, 3
}

// largest value (>= 0) of the wave
__device__ __forceinline__ int mx4_wave_max(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}

// The softmax's exponents are score * c, c = scale * log2(e) > 0: a negative scale
// turns the query's sign, and of scale 0 the query is 0 and c 1.
struct MxScale {
    uint32_t keep, flip;   // of a packed pair of query elements
    float c;
};
__device__ __forceinline__ MxScale mx4_scale(float c) {
    return MxScale{c == 0.f ? 0u : 0xffffffffu, c < 0.f ? 0x80008000u : 0u, c == 0.f ? 1.f : __builtin_fabsf(c)};
}
__device__ __forceinline__ uint4 mx4_scaled(const uint4& w, const MxScale& x) {
    return make_uint4((w.x & x.keep) ^ x.flip, (w.y & x.keep) ^ x.flip, (w.z & x.keep) ^ x.flip, (w.w & x.keep) ^ x.flip);
}

// The power of two of a query row (its largest element in [128, 256)) as the
// scale byte of its first term, from the row's largest pattern; the terms' bytes are
// this less 4 each and stay above 0.  255 (NaN) for a row with an infinity or a NaN.
template <int QKIND>
__device__ __forceinline__ int mx4_query_byte(uint32_t amax) {
    const float x = QKIND == KIND_BF16 ? __uint_as_float(amax << 16) : f16_bits_to_f32(static_cast<uint16_t>(amax));
    const int e = static_cast<int>(__float_as_uint(x) >> 23);   // 127 + floor(log2)
    return amax < (QKIND == KIND_BF16 ? 0x7f80u : 0x7c00u) ? max(e - 7, 9) : 255;
}
// the terms' unit; of a NaN row any will do, its scales make it NaN
__device__ __forceinline__ float mx4_query_factor(int byte0) {
    return __uint_as_float(static_cast<uint32_t>(byte0 == 255 ? 127 : byte0) << 23);
}

// the block scales of a term: 255 stays NaN
__device__ __forceinline__ int mx4_term_byte(int byte0, int term) { return byte0 == 255 ? 255 : byte0 - 4 * term; }

// waves a SIMD of the decode kernel: two, one where a wave needs more than half its registers
__host__ __device__ constexpr int mxd_per_simd(int64_t d) { return d <= 128 ? 2 : 1; }
}  // namespace

// Chunks of few new tokens on the decode kernel, a (token, query head) pair a column: sequences of
// at most most_cols columns a kv head; the others' outputs stay.  Its rows, at most (a workgroup's
// least work), or -1 where the batch passes its counters, which the launch refuses.
int64_t mx4_short_rows(int64_t num_seqs, int64_t num_tokens, int64_t hq, int64_t hkv, int64_t bs, int64_t maxb,
                       int64_t most_cols);
int32_t mx4_short_chunks(void* out, const void* q, const uint8_t* kc, const uint8_t* vc, const int32_t* bt,
                         const int32_t* seq_lens, const int32_t* qsl, int64_t num_seqs, int64_t num_tokens, int64_t hq,
                         int64_t hkv, int64_t d, int64_t bs, int64_t maxb, int64_t nb, float scale, int32_t q_dtype,
                         int64_t most_cols, uintptr_t stream);

}  // namespace rllm
