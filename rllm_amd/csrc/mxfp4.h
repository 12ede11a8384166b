// The microscaled 4-bit (MXFP4) KV cache: layout, element conversion and the
// pieces its kernels share.
//
// One layer's K (and V) is uint8 [num_blocks, num_kv_heads, page] with
// page = block_size * head_dim * 17 / 32 bytes: block_size rows of head_dim / 2
// code bytes, then block_size rows of head_dim / 32 scale bytes.  Byte i of a
// code row holds elements 2i (low four bits) and 2i + 1; a code is E2M1 (sign,
// two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), a scale byte
// e the factor 2^(e - 127) of 32 elements (E8M0; 255 = NaN).  Rows are whole
// per token, unlike the 16-bit and FP8 caches' [head_dim][block_size]: a lane's
// 16-byte load is then the 32 elements of one scale, which is the operand of the
// gfx950 block-scaled matrix product as it stands, and a token's write touches
// no byte of another's.  block_size is a multiple of 16, so every row and page
// starts on 16 bytes and 16 tokens never straddle a page.
#pragma once

#include "common.h"

#include <cmath>

namespace rllm {

constexpr int MX4_BLOCK = 32;       // elements of one scale
constexpr int MX4_TOKENS = 16;      // block_size is a multiple of this
constexpr int64_t MX4_MAX_DIM = 256;
// the largest scale byte a write makes (bf16 values up to 2^128): 6 * 2^125 is finite in f32
constexpr uint32_t MX4_TOP_SCALE = 252;
constexpr float MX4_LOG2E = 1.4426950408889634f;

__host__ __device__ inline int64_t mx4_page_bytes(int64_t d, int64_t bs) { return bs * (d / 32) * 17; }

// the shapes of all five operators
inline bool mx4_shape_ok(int64_t hkv, int64_t d, int64_t bs, int64_t nb) {
    return hkv > 0 && hkv <= 1024 && d >= MX4_BLOCK && d % MX4_BLOCK == 0 && d <= MX4_MAX_DIM && bs >= MX4_TOKENS &&
           bs % MX4_TOKENS == 0 && bs <= 4096 && nb >= 0 && nb <= (int64_t(1) << 31) - 1;
}

constexpr int64_t MX4_MAX_THREADS = (int64_t(1) << 32) - 1;   // of a launch

// the tables and heads of the two attention operators
inline bool mx4_attention_ok(int64_t num_seqs, int64_t hq, int64_t hkv, int64_t bs, int64_t maxb) {
    return hq > 0 && hq <= 1024 && hq % hkv == 0 && num_seqs <= (int64_t(1) << 20) && maxb >= 0 &&
           maxb <= (int64_t(1) << 24) && maxb * bs <= (int64_t(1) << 27);
}

inline bool mx4_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t mx_u32x4a __attribute__((ext_vector_type(4)));
typedef uint32_t mx_out8 __attribute__((ext_vector_type(4), aligned(8)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef short mx_i16x4 __attribute__((ext_vector_type(4)));
typedef short mx_i16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short mx_u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 mx_f16x2 __attribute__((ext_vector_type(2)));

// Non-template wrappers of the target builtins (a template that names one is
// dropped by the host pass).  The fp4 conversions round to nearest, ties to the
// even code, saturate at 6 and keep the sign of zero: an in-bounds sweep of every
// 16-bit pattern at four scales, and of f32 values around every border, matched
// that rule exactly.

// two values / scale -> codes in byte SEL of `old`, the first in the low four bits
template <int SEL> __device__ uint32_t mx4_enc_bf16(uint32_t old, uint32_t pair, float scale);
template <int SEL> __device__ uint32_t mx4_enc_f16(uint32_t old, uint32_t pair, float scale);
template <int SEL> __device__ uint32_t mx4_enc_f32(uint32_t old, float a, float b, float scale);
// byte SEL's two codes * scale -> two packed bf16 / f16
template <int SEL> __device__ uint32_t mx4_dec_bf16(uint32_t w, float scale);
template <int SEL> __device__ uint32_t mx4_dec_f16(uint32_t w, float scale);
#define MX4_CONVERSIONS(SEL)                                                                                           \
    template <> __device__ __forceinline__ uint32_t mx4_enc_bf16<SEL>(uint32_t old, uint32_t pair, float scale) {      \
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(mx_bf16x2, pair), scale, SEL);        \
    }                                                                                                                  \
    template <> __device__ __forceinline__ uint32_t mx4_enc_f16<SEL>(uint32_t old, uint32_t pair, float scale) {       \
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(mx_f16x2, pair), scale, SEL);          \
    }                                                                                                                  \
    template <> __device__ __forceinline__ uint32_t mx4_enc_f32<SEL>(uint32_t old, float a, float b, float scale) {    \
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, scale, SEL);                                        \
    }                                                                                                                  \
    template <> __device__ __forceinline__ uint32_t mx4_dec_bf16<SEL>(uint32_t w, float scale) {                       \
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));                 \
    }                                                                                                                  \
    template <> __device__ __forceinline__ uint32_t mx4_dec_f16<SEL>(uint32_t w, float scale) {                        \
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));                  \
    }
MX4_CONVERSIONS(0)
MX4_CONVERSIONS(1)
MX4_CONVERSIONS(2)
MX4_CONVERSIONS(3)
#undef MX4_CONVERSIONS

// A scale byte as the conversions' factor: 2^(e - 127); 255 gives Inf, which
// they turn into NaN for every code.  2^-127 is subnormal.
__device__ __forceinline__ float mx4_factor(uint32_t e) {
    return __uint_as_float(max(e << 23, 0x00400000u));
}

// The scale byte of a block from its largest magnitude: OCP's rule
// floor(log2 amax) - 2, kept within 1 .. 254 (amax below 2^-124, zero among it, takes 1),
// and 255 where the block holds an infinity or a NaN.
__device__ __forceinline__ uint32_t mx4_scale_byte(float amax, bool finite) {
    const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 2;
    return finite ? static_cast<uint32_t>(max(e, 1)) : 255u;
}

// the largest u32 of the lane's group of four
__device__ __forceinline__ uint32_t mx4_quad_max(uint32_t v) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), DPP_QUAD_XOR1, 0xF, 0xF, false)));
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), DPP_QUAD_XOR2, 0xF, 0xF, false)));
}

// largest magnitude of 8 16-bit floats, as their 15-bit pattern (patterns rise
// with the magnitude, infinities and NaNs above every finite value)
__device__ __forceinline__ uint32_t mx4_amax8(const uint4& w) {
    const mx_u16x2 a = __builtin_bit_cast(mx_u16x2, w.x & 0x7fff7fffu), b = __builtin_bit_cast(mx_u16x2, w.y & 0x7fff7fffu);
    const mx_u16x2 c = __builtin_bit_cast(mx_u16x2, w.z & 0x7fff7fffu), d = __builtin_bit_cast(mx_u16x2, w.w & 0x7fff7fffu);
    const mx_u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(a, b), __builtin_elementwise_max(c, d));
    return max(static_cast<uint32_t>(m[0]), static_cast<uint32_t>(m[1]));
}

}  // namespace rllm
