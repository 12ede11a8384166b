// Writes into and reads from the MXFP4 KV cache (layout in mxfp4.h), for gfx950.
//
//   write   x [num_tokens, Hkv, D] 16-bit -> rows slot_mapping[t] of the cache:
//           per 32 elements e = clamp(floor(log2 max|x|) - 2, -126, 127), code =
//           x / 2^e rounded to E2M1 (nearest, ties to even, at most 6)
//   rope    the same after a rotation of k by halves (y1 = x1 c - x2 s,
//           y2 = x2 c + x1 s); q rotated beside it
//   read    code * 2^e of rows slot_mapping[t] -> 16 bits
//
// All three move data once and compute little: HBM-bound where large, launch
// latency where small.  Eight elements a lane, so that 16-bit rows go by 16-byte
// accesses a lane, whole lines a wave; four neighbouring lanes hold the 32
// elements of one scale and find its magnitude by two lane swaps.
//
// Measured (8 kv heads, D 128): 8 prompts of 300-2000 tokens, f16, 37 MB each way, written
// 9.6 us and read back 9.1 (4 TB/s); 4096 tokens rotated and written, 32 q heads, 88 MB 17.2 us
// (5.1 TB/s); 16 contexts of 1000-8000 read back, 329 MB 57.8 us (5.7 TB/s, past a copy's
// rate: four fifths of it are stores past the L2); a step of 64 tokens 3.1 us, a launch.
#include "mxfp4.h"
#include "../../include/rllm_kernels.h"

namespace rllm {
namespace {

constexpr int MXC_THREADS = 256;

struct MxSlot {
    int64_t page;   // byte offset of the (block, kv head) page, -1: skipped
    int64_t off;    // token row in the page
};

// slots are below 2^32 in any cache under 17 GB a head: the 64-bit division is
// the rare path
__device__ __forceinline__ MxSlot mx_slot(int64_t slot, int bs, int64_t nb, int hkv, int h, int64_t page_bytes) {
    MxSlot r;
    r.page = -1;
    r.off = 0;
    if (slot < 0) return r;
    int64_t blk;
    if ((slot >> 32) == 0) blk = static_cast<uint32_t>(slot) / static_cast<uint32_t>(bs);
    else blk = slot / bs;
    if (blk >= nb) return r;
    r.off = slot - blk * bs;
    r.page = (blk * hkv + h) * page_bytes;
    return r;
}

// 8 elements of this lane's quarter of a 32-element block -> 4 code bytes, and
// the block's scale byte (equal in the four lanes)
template <int KIND>
__device__ __forceinline__ uint32_t quantise8(const uint4& w, uint32_t& e) {
    const uint32_t top = mx4_quad_max(mx4_amax8(w));
    const bool finite = top < (KIND == KIND_BF16 ? 0x7f80u : 0x7c00u);
    e = mx4_scale_byte(KIND == KIND_BF16 ? __uint_as_float(top << 16) : f16_bits_to_f32(static_cast<uint16_t>(top)),
                       finite);
    if (!finite) return 0u;
    const float s = __uint_as_float(e << 23);
    uint32_t c = 0;
    if constexpr (KIND == KIND_BF16) {
        c = mx4_enc_bf16<0>(c, w.x, s);
        c = mx4_enc_bf16<1>(c, w.y, s);
        c = mx4_enc_bf16<2>(c, w.z, s);
        c = mx4_enc_bf16<3>(c, w.w, s);
    } else {
        c = mx4_enc_f16<0>(c, w.x, s);
        c = mx4_enc_f16<1>(c, w.y, s);
        c = mx4_enc_f16<2>(c, w.z, s);
        c = mx4_enc_f16<3>(c, w.w, s);
    }
    return c;
}

__device__ __forceinline__ uint32_t quantise8_f32(const float (&x)[8], uint32_t& e) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = mx4_quad_max(top);
    const bool finite = top < 0x7f800000u;
    e = mx4_scale_byte(__uint_as_float(top), finite);
    if (!finite) return 0u;
    const float s = __uint_as_float(e << 23);
    uint32_t c = 0;
    c = mx4_enc_f32<0>(c, x[0], x[1], s);
    c = mx4_enc_f32<1>(c, x[2], x[3], s);
    c = mx4_enc_f32<2>(c, x[4], x[5], s);
    return mx4_enc_f32<3>(c, x[6], x[7], s);
}

// 4 code bytes and the scale byte of chunk c (8 elements) of a token row
__device__ __forceinline__ void store8(uint8_t* cache, const MxSlot& at, int d, int bs, int c, uint32_t codes,
                                       uint32_t e) {
    if (at.page < 0) return;
    uint8_t* page = cache + at.page;
    *reinterpret_cast<uint32_t*>(page + at.off * (d / 2) + 4 * c) = codes;
    if ((c & 3) == 0) page[static_cast<int64_t>(bs) * (d / 2) + at.off * (d / 32) + (c >> 2)] = static_cast<uint8_t>(e);
}

// ---------------------------------------------------------------------------
// write: one lane per 8 elements of a token's K and of its V
// ---------------------------------------------------------------------------
template <int KIND>
__global__ __launch_bounds__(MXC_THREADS) void mx4_write_kernel(uint8_t* kc, uint8_t* vc, const uint4* __restrict__ nk,
                                                                const uint4* __restrict__ nv,
                                                                const int64_t* __restrict__ slots, int64_t chunks,
                                                                int hkv, int d, int bs, int64_t nb) {
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * MXC_THREADS;
    const int64_t i = i0 + threadIdx.x;
    // a token's chunks are a multiple of four: the lanes of one scale leave together
    if (i >= chunks) return;
    const int per_head = d / 8, per_tok = hkv * per_head;
    const int64_t t0 = i0 / per_tok;   // uniform
    const int r = static_cast<int>(i0 - t0 * per_tok) + static_cast<int>(threadIdx.x);
    const int64_t t = t0 + r / per_tok;
    const int hc = r % per_tok, h = hc / per_head, c = hc % per_head;
    const uint4 k = nk[i], v = nv[i];
    const MxSlot at = mx_slot(slots[t], bs, nb, hkv, h, mx4_page_bytes(d, bs));
    uint32_t ek, ev;
    const uint32_t ck = quantise8<KIND>(k, ek), cv = quantise8<KIND>(v, ev);
    store8(kc, at, d, bs, c, ck, ek);
    store8(vc, at, d, bs, c, cv, ev);
}

// ---------------------------------------------------------------------------
// rope: one lane per 8 elements of a head's first half and their partners in the
// second, of q, k or v
// ---------------------------------------------------------------------------
template <int KIND>
__device__ __forceinline__ void to_f32x8(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = KIND == KIND_BF16 ? bf16_lo(u[i]) : f16_lo(u[i]);
        x[2 * i + 1] = KIND == KIND_BF16 ? bf16_hi(u[i]) : f16_hi(u[i]);
    }
}

template <int KIND>
__device__ __forceinline__ uint4 from_f32x8(const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const mx_f32x2 p = {x[2 * i], x[2 * i + 1]};
        u[i] = KIND == KIND_BF16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(p, mx_bf16x2))
                                 : __builtin_bit_cast(uint32_t, __builtin_convertvector(p, mx_f16x2));
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// Both products and their sum are each rounded to f32, with no contraction: the
// rotated key decides codes at their borders, so its bits are part of the
// operator's definition.  q is rounded to 16 bits once.
__device__ __forceinline__ void rotate8(float (&x1)[8], float (&x2)[8], const float (&cs)[8], const float (&sn)[8]) {
#pragma clang fp contract(off)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = x1[i], b = x2[i];
        const float ac = a * cs[i], bs = b * sn[i], bc = b * cs[i], as = a * sn[i];
        x1[i] = ac - bs;
        x2[i] = bc + as;
    }
}

struct MxRopeArgs {
    uint16_t* q_out;
    const uint16_t *q, *k, *v;
    uint8_t *kc, *vc;
    const int64_t* slots;
    const int32_t* pos;
    const float *cs, *sn;
    int64_t items;
    int32_t hq, hkv, d, bs;
    int64_t nb;
    int32_t maxp;
};

template <int KIND>
__global__ __launch_bounds__(MXC_THREADS) void mx4_rope_kernel(MxRopeArgs a) {
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * MXC_THREADS;
    if (i0 + threadIdx.x >= a.items) return;
    const int per_head = a.d / 16, per_tok = (a.hq + 2 * a.hkv) * per_head;
    const int64_t t0 = i0 / per_tok;   // uniform
    const int r = static_cast<int>(i0 - t0 * per_tok) + static_cast<int>(threadIdx.x);
    const int64_t t = t0 + r / per_tok;
    const int hc = r % per_tok, h = hc / per_head, c = hc % per_head;
    const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
    const int hk = is_v ? h - a.hq - a.hkv : h - a.hq;   // kv head of a k or v item
    const int half = a.d / 2;
    const uint16_t* src = is_q ? a.q + (t * a.hq + h) * a.d : (is_v ? a.v : a.k) + (t * a.hkv + hk) * a.d;
    const uint4 w1 = *reinterpret_cast<const uint4*>(src + 8 * c);
    const uint4 w2 = *reinterpret_cast<const uint4*>(src + half + 8 * c);
    MxSlot at;
    if (!is_q) at = mx_slot(a.slots[t], a.bs, a.nb, a.hkv, hk, mx4_page_bytes(a.d, a.bs));
    if (is_v) {
        uint32_t e1, e2;
        const uint32_t c1 = quantise8<KIND>(w1, e1), c2 = quantise8<KIND>(w2, e2);
        store8(a.vc, at, a.d, a.bs, c, c1, e1);
        store8(a.vc, at, a.d, a.bs, half / 8 + c, c2, e2);
        return;
    }
    const int p = min(max(a.pos[t], 0), a.maxp - 1);
    const float4* cr = reinterpret_cast<const float4*>(a.cs + static_cast<int64_t>(p) * half + 8 * c);
    const float4* sr = reinterpret_cast<const float4*>(a.sn + static_cast<int64_t>(p) * half + 8 * c);
    const float4 c0 = cr[0], c1 = cr[1], s0 = sr[0], s1 = sr[1];
    const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
    float x1[8], x2[8];
    to_f32x8<KIND>(w1, x1);
    to_f32x8<KIND>(w2, x2);
    rotate8(x1, x2, cs, sn);
    if (is_q) {
        uint16_t* dst = a.q_out + (t * a.hq + h) * a.d;
        *reinterpret_cast<uint4*>(dst + 8 * c) = from_f32x8<KIND>(x1);
        *reinterpret_cast<uint4*>(dst + half + 8 * c) = from_f32x8<KIND>(x2);
        return;
    }
    uint32_t e1, e2;
    const uint32_t k1 = quantise8_f32(x1, e1), k2 = quantise8_f32(x2, e2);
    store8(a.kc, at, a.d, a.bs, c, k1, e1);
    store8(a.kc, at, a.d, a.bs, half / 8 + c, k2, e2);
}

// ---------------------------------------------------------------------------
// read: one lane per 8 elements of a row of K and of V
// ---------------------------------------------------------------------------
template <int KIND>
__device__ __forceinline__ uint4 values8(uint32_t codes, uint32_t e) {
    const float s = mx4_factor(e);
    if constexpr (KIND == KIND_BF16)
        return make_uint4(mx4_dec_bf16<0>(codes, s), mx4_dec_bf16<1>(codes, s), mx4_dec_bf16<2>(codes, s),
                          mx4_dec_bf16<3>(codes, s));
    else
        return make_uint4(mx4_dec_f16<0>(codes, s), mx4_dec_f16<1>(codes, s), mx4_dec_f16<2>(codes, s),
                          mx4_dec_f16<3>(codes, s));
}

template <int KIND>
__global__ __launch_bounds__(MXC_THREADS) void mx4_read_kernel(uint4* __restrict__ ok, uint4* __restrict__ ov,
                                                               const uint8_t* __restrict__ kc,
                                                               const uint8_t* __restrict__ vc,
                                                               const int64_t* __restrict__ slots, int64_t chunks,
                                                               int hkv, int d, int bs, int64_t nb) {
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * MXC_THREADS;
    const int64_t i = i0 + threadIdx.x;
    if (i >= chunks) return;
    const int per_head = d / 8, per_tok = hkv * per_head;
    const int64_t t0 = i0 / per_tok;   // uniform
    const int r = static_cast<int>(i0 - t0 * per_tok) + static_cast<int>(threadIdx.x);
    const int64_t t = t0 + r / per_tok;
    const int hc = r % per_tok, h = hc / per_head, c = hc % per_head;
    const MxSlot at = mx_slot(slots[t], bs, nb, hkv, h, mx4_page_bytes(d, bs));
    uint4 k = make_uint4(0, 0, 0, 0), v = k;   // a skipped row reads as zeros
    if (at.page >= 0) {
        const int64_t co = at.page + at.off * (d / 2) + 4 * c;
        const int64_t so = at.page + static_cast<int64_t>(bs) * (d / 2) + at.off * (d / 32) + (c >> 2);
        const uint32_t ck = *reinterpret_cast<const uint32_t*>(kc + co), cv = *reinterpret_cast<const uint32_t*>(vc + co);
        const uint32_t ek = kc[so], ev = vc[so];
        k = values8<KIND>(ck, ek);
        v = values8<KIND>(cv, ev);
    }
    // The rows go past the L2: written through it they take turns with the reads (128k
    // rows of 8 x 128, 330 MB in all: 76 -> 58.5 us; 4000 rows 6.0 -> 4.9; 777 rows of 8 x 64
    // 2.7 -> 2.9).
    __builtin_nontemporal_store(mx_u32x4a{k.x, k.y, k.z, k.w}, reinterpret_cast<mx_u32x4a*>(ok + i));
    __builtin_nontemporal_store(mx_u32x4a{v.x, v.y, v.z, v.w}, reinterpret_cast<mx_u32x4a*>(ov + i));
}

// arguments the write and the read share; *grid = the workgroups
int32_t check_rows(const void* kc, const void* vc, const void* k, const void* v, const int64_t* slots, int64_t n,
                   int64_t hkv, int64_t d, int64_t bs, int64_t nb, int32_t dtype, int64_t* chunks, unsigned* grid) {
    RLLM_CHECK_ARG(kc && vc && k && v && slots);
    RLLM_CHECK_ARG(mx4_shape_ok(hkv, d, bs, nb));
    RLLM_CHECK_ARG(dtype == RLLM_DTYPE_F16 || dtype == RLLM_DTYPE_BF16);
    RLLM_CHECK_ARG(mx4_aligned16(kc) && mx4_aligned16(vc) && mx4_aligned16(k) && mx4_aligned16(v));
    RLLM_CHECK_ARG(n <= (int64_t(1) << 31) - 1);
    *chunks = n * hkv * (d / 8);
    const int64_t wgs = (*chunks + MXC_THREADS - 1) / MXC_THREADS;
    RLLM_CHECK_ARG(wgs * MXC_THREADS <= MX4_MAX_THREADS);
    *grid = static_cast<unsigned>(wgs);
    return 0;
}

}  // namespace
}  // namespace rllm

using namespace rllm;

extern "C" {

int64_t rllm_mxfp4_page_bytes(int64_t head_dim, int64_t block_size) {
    if (!mx4_shape_ok(1, head_dim, block_size, 0)) return -1;
    return mx4_page_bytes(head_dim, block_size);
}

int32_t rllm_cache_write_mxfp4(uint8_t* key_cache, uint8_t* value_cache, const uint16_t* new_key,
                               const uint16_t* new_value, const int64_t* slot_mapping, int64_t num_tokens,
                               int64_t num_kv_heads, int64_t head_dim, int64_t block_size, int64_t num_blocks,
                               int32_t input_dtype, uintptr_t stream) {
    if (num_tokens <= 0) return 0;
    int64_t chunks;
    unsigned grid;
    const int32_t rc = check_rows(key_cache, value_cache, new_key, new_value, slot_mapping, num_tokens, num_kv_heads,
                                  head_dim, block_size, num_blocks, input_dtype, &chunks, &grid);
    if (rc) return rc;
    auto kern = input_dtype == RLLM_DTYPE_BF16 ? mx4_write_kernel<KIND_BF16> : mx4_write_kernel<KIND_F16>;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(MXC_THREADS), 0, as_stream(stream), key_cache, value_cache,
                       reinterpret_cast<const uint4*>(new_key), reinterpret_cast<const uint4*>(new_value), slot_mapping,
                       chunks, static_cast<int>(num_kv_heads), static_cast<int>(head_dim),
                       static_cast<int>(block_size), num_blocks);
    return launch_status();
}

int32_t rllm_cache_read_mxfp4(uint16_t* out_key, uint16_t* out_value, const uint8_t* key_cache,
                              const uint8_t* value_cache, const int64_t* slot_mapping, int64_t num_tokens,
                              int64_t num_kv_heads, int64_t head_dim, int64_t block_size, int64_t num_blocks,
                              int32_t output_dtype, uintptr_t stream) {
    if (num_tokens <= 0) return 0;
    int64_t chunks;
    unsigned grid;
    const int32_t rc = check_rows(key_cache, value_cache, out_key, out_value, slot_mapping, num_tokens, num_kv_heads,
                                  head_dim, block_size, num_blocks, output_dtype, &chunks, &grid);
    if (rc) return rc;
    auto kern = output_dtype == RLLM_DTYPE_BF16 ? mx4_read_kernel<KIND_BF16> : mx4_read_kernel<KIND_F16>;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(MXC_THREADS), 0, as_stream(stream), reinterpret_cast<uint4*>(out_key),
                       reinterpret_cast<uint4*>(out_value), key_cache, value_cache, slot_mapping, chunks,
                       static_cast<int>(num_kv_heads), static_cast<int>(head_dim), static_cast<int>(block_size),
                       num_blocks);
    return launch_status();
}

int32_t rllm_rope_cache_write_mxfp4(void* q_out, const void* q, const void* k, const void* v, uint8_t* key_cache,
                                    uint8_t* value_cache, const int64_t* slot_mapping, const int32_t* positions,
                                    const float* cos_cache, const float* sin_cache, int64_t num_tokens,
                                    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                    int64_t num_blocks, int64_t max_position, int32_t dtype, uintptr_t stream) {
    if (num_tokens <= 0) return 0;
    RLLM_CHECK_ARG(num_tokens <= (int64_t(1) << 31) - 1);
    RLLM_CHECK_ARG(dtype == RLLM_DTYPE_F16 || dtype == RLLM_DTYPE_BF16);
    RLLM_CHECK_ARG(mx4_shape_ok(num_kv_heads, head_dim, block_size, num_blocks));
    RLLM_CHECK_ARG(head_dim % 64 == 0);   // a scale's 32 elements lie in one half
    RLLM_CHECK_ARG(num_q_heads >= 0 && num_q_heads <= 1024);
    RLLM_CHECK_ARG(max_position >= 1 && max_position <= (int64_t(1) << 31) - 1);
    RLLM_CHECK_ARG(k && v && key_cache && value_cache && slot_mapping && positions && cos_cache && sin_cache);
    RLLM_CHECK_ARG(num_q_heads == 0 || (q && q_out));
    RLLM_CHECK_ARG(mx4_aligned16(k) && mx4_aligned16(v) && mx4_aligned16(cos_cache) && mx4_aligned16(sin_cache));
    RLLM_CHECK_ARG(mx4_aligned16(key_cache) && mx4_aligned16(value_cache));
    RLLM_CHECK_ARG(num_q_heads == 0 || (mx4_aligned16(q) && mx4_aligned16(q_out)));
    MxRopeArgs a{};
    a.q_out = static_cast<uint16_t*>(q_out);
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.kc = key_cache;
    a.vc = value_cache;
    a.slots = slot_mapping;
    a.pos = positions;
    a.cs = cos_cache;
    a.sn = sin_cache;
    a.items = num_tokens * (num_q_heads + 2 * num_kv_heads) * (head_dim / 16);
    a.hq = static_cast<int32_t>(num_q_heads);
    a.hkv = static_cast<int32_t>(num_kv_heads);
    a.d = static_cast<int32_t>(head_dim);
    a.bs = static_cast<int32_t>(block_size);
    a.nb = num_blocks;
    a.maxp = static_cast<int32_t>(max_position);
    const int64_t wgs = (a.items + MXC_THREADS - 1) / MXC_THREADS;
    RLLM_CHECK_ARG(wgs * MXC_THREADS <= MX4_MAX_THREADS);
    auto kern = dtype == RLLM_DTYPE_BF16 ? mx4_rope_kernel<KIND_BF16> : mx4_rope_kernel<KIND_F16>;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(wgs)), dim3(MXC_THREADS), 0, as_stream(stream), a);
    return launch_status();
}

}  // extern "C"
