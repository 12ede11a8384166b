// C++ host side of the MI355X paged-attention library: the operator interface
// of the reference's `rllm-kernels` crate, restated over the C ABI of
// include/rllm_kernels.h with the same names, argument meaning and error
// behaviour.
//
//   reference (Rust)                                  here
//   crates/rllm-core/src/dtype.rs:3-26  DType         rllm::kernels::DType
//   crates/rllm-core/src/ids.rs:23      BlockId       rllm::kernels::BlockId
//   crates/rllm-kernels/src/cuda.rs:39-52
//                CudaKernelError, check()             CudaKernelError, Result<T>, check()
//   crates/rllm-kernels/src/attention.rs:15-48        AttentionParams
//   crates/rllm-kernels/src/attention.rs:56-259       AttentionMetadata
//   crates/rllm-kernels/src/attention.rs:425-779      paged_attention_{decode,prefill}_{f16,fp8}[_sync]
//   crates/rllm-kernels/src/cache_ops.rs:106-347      cache_write_*, cache_block_copy*, cache_zero*,
//                                                     gpu_alloc, gpu_free
//   crates/rllm-kernels/src/cache_ops.rs:350-490      GpuKVCache
//   crates/rllm-worker/src/model_runner.rs:806-826    compute_slot_mappings
//   crates/rllm-model/src/rope.rs:5-55                RotaryEmbedding (host cos / sin tables)
//   rope.rs:57-82 + cache_ops.rs:106-347              rope_cache_write (fused, additive)
//   crates/rllm-cache/src/offload.rs:7-84             CpuKvOffloadStore (+ swap_out / swap_in records)
//   block_pool.rs:286-302 + cache_ops.cu:252-292      cache_copy_blocks (copy-on-write data, additive)
//
// Differences: Rust's `Result<T, CudaKernelError>` is Result<T> here (no
// exceptions); `GpuKVCache::new` is a factory returning Result<GpuKVCache>;
// `Option<usize>` is std::optional<size_t>; compute_slot_mappings returns all
// -1 for block_size 0 (the Rust code would divide by zero).  The library is
// always present, so the NotAvailable variant only appears for an unsupported
// element type.
#pragma once

#include "../../include/rllm_kernels.h"

#include <algorithm>
#include <array>
#include <cmath>
#include <cstddef>
#include <cstdlib>
#include <cstdint>
#include <map>
#include <optional>
#include <string>
#include <utility>
#include <vector>

namespace rllm {
namespace kernels {

// ---------------------------------------------------------------------------
// element types (dtype.rs:3-26)
// ---------------------------------------------------------------------------
enum class DType { F32, F16, BF16, FP8E4M3, FP8E5M2, INT8, INT4 };

inline size_t bytes_per_scalar(DType d) {
    switch (d) {
    case DType::F32: return 4;
    case DType::F16:
    case DType::BF16: return 2;
    default: return 1;   // FP8E4M3, FP8E5M2, INT8, INT4 (packed two per byte in practice)
    }
}

// the C ABI's RLLM_DTYPE_* code of a cache / activation type, -1 if it has none
inline int32_t abi_dtype(DType d) {
    switch (d) {
    case DType::F16: return RLLM_DTYPE_F16;
    case DType::BF16: return RLLM_DTYPE_BF16;
    case DType::FP8E4M3: return RLLM_DTYPE_FP8_E4M3;
    case DType::FP8E5M2: return RLLM_DTYPE_FP8_E5M2;
    default: return -1;
    }
}

struct BlockId {
    uint32_t value;
};

// crates/rllm-core/src/ids.rs RequestId (an opaque id; ordered for map keys)
struct RequestId {
    uint64_t value;
};

// ---------------------------------------------------------------------------
// errors (cuda.rs:39-52)
// ---------------------------------------------------------------------------
struct CudaKernelError {
    enum class Kind { KernelError, NotAvailable };
    Kind kind = Kind::KernelError;
    int32_t code = 0;   // the non-zero return code of the C entry point

    std::string message() const {
        return kind == Kind::NotAvailable ? std::string("GPU kernels are not available for this call")
                                          : "GPU kernel returned error code " + std::to_string(code);
    }
};

template <class T>
class Result {
public:
    static Result ok(T v) { return Result(std::move(v)); }
    static Result err(CudaKernelError e) { return Result(e); }
    bool is_ok() const { return ok_; }
    bool is_err() const { return !ok_; }
    const T& value() const { return value_; }
    T& value() { return value_; }
    const CudaKernelError& error() const { return error_; }

private:
    explicit Result(T v) : ok_(true), value_(std::move(v)) {}
    explicit Result(CudaKernelError e) : ok_(false), value_(), error_(e) {}
    bool ok_;
    T value_;
    CudaKernelError error_{};
};

template <>
class Result<void> {
public:
    static Result ok() { return Result(true, {}); }
    static Result err(CudaKernelError e) { return Result(false, e); }
    bool is_ok() const { return ok_; }
    bool is_err() const { return !ok_; }
    const CudaKernelError& error() const { return error_; }

private:
    Result(bool ok, CudaKernelError e) : ok_(ok), error_(e) {}
    bool ok_;
    CudaKernelError error_;
};

// check(): 0 -> Ok, anything else -> KernelError { code }
inline Result<void> check(int32_t rc) {
    if (rc == 0) return Result<void>::ok();
    return Result<void>::err(CudaKernelError{CudaKernelError::Kind::KernelError, rc});
}

// ---------------------------------------------------------------------------
// AttentionParams (attention.rs:15-48)
// ---------------------------------------------------------------------------
struct AttentionParams {
    size_t num_q_heads = 0;
    size_t num_kv_heads = 0;
    size_t head_dim = 0;
    size_t block_size = 0;
    float scale = 0.f;

    static AttentionParams create(size_t num_q_heads, size_t num_kv_heads, size_t head_dim,
                                  size_t block_size) {
        AttentionParams p;
        p.num_q_heads = num_q_heads;
        p.num_kv_heads = num_kv_heads;
        p.head_dim = head_dim;
        p.block_size = block_size;
        p.scale = 1.0f / std::sqrt(static_cast<float>(head_dim));
        return p;
    }
    size_t gqa_ratio() const { return num_q_heads / num_kv_heads; }
    size_t kv_head_for_q_head(size_t q_head) const { return q_head * num_kv_heads / num_q_heads; }
    size_t num_blocks_for_seq_len(size_t seq_len) const { return (seq_len + block_size - 1) / block_size; }
};

// ---------------------------------------------------------------------------
// AttentionMetadata (attention.rs:56-259)
// ---------------------------------------------------------------------------
struct AttentionMetadata {
    std::vector<uint32_t> seq_lens;
    std::vector<uint32_t> query_start_loc{0};
    std::vector<std::vector<int32_t>> block_tables;
    std::vector<int64_t> slot_mapping;
    size_t num_prefill_tokens = 0;
    size_t num_decode_tokens = 0;
    size_t max_num_blocks_per_seq = 0;
    size_t common_prefix_blocks = 0;
    std::optional<size_t> sliding_window;

    static AttentionMetadata create() { return AttentionMetadata{}; }

    // one query token per sequence: query_start_loc = 0, 1, ..., num_seqs
    static AttentionMetadata for_decode(std::vector<uint32_t> seq_lens,
                                        std::vector<std::vector<int32_t>> block_tables,
                                        size_t max_num_blocks_per_seq) {
        AttentionMetadata m;
        const size_t n = seq_lens.size();
        m.query_start_loc.resize(n + 1);
        for (size_t i = 0; i <= n; ++i) m.query_start_loc[i] = static_cast<uint32_t>(i);
        m.seq_lens = std::move(seq_lens);
        m.block_tables = std::move(block_tables);
        m.num_decode_tokens = n;
        m.max_num_blocks_per_seq = max_num_blocks_per_seq;
        return m;
    }

    static AttentionMetadata for_decode_with_options(std::vector<uint32_t> seq_lens,
                                                     std::vector<std::vector<int32_t>> block_tables,
                                                     size_t max_num_blocks_per_seq,
                                                     size_t common_prefix_blocks,
                                                     std::optional<size_t> sliding_window) {
        AttentionMetadata m = for_decode(std::move(seq_lens), std::move(block_tables), max_num_blocks_per_seq);
        m.common_prefix_blocks = common_prefix_blocks;
        m.sliding_window = sliding_window;
        return m;
    }

    static AttentionMetadata for_prefill(std::vector<uint32_t> seq_lens,
                                         const std::vector<uint32_t>& prompt_tokens_per_seq,
                                         std::vector<std::vector<int32_t>> block_tables,
                                         size_t max_num_blocks_per_seq) {
        AttentionMetadata m;
        m.query_start_loc.clear();
        m.query_start_loc.reserve(seq_lens.size() + 1);
        m.query_start_loc.push_back(0);
        uint32_t cumulative = 0;
        for (uint32_t c : prompt_tokens_per_seq) {
            cumulative += c;
            m.query_start_loc.push_back(cumulative);
        }
        m.seq_lens = std::move(seq_lens);
        m.block_tables = std::move(block_tables);
        m.num_prefill_tokens = cumulative;
        m.max_num_blocks_per_seq = max_num_blocks_per_seq;
        return m;
    }

    // [num_seqs * max_num_blocks_per_seq] row-major, -1 padded, rows cut at the width
    std::vector<int32_t> flatten_block_tables() const {
        std::vector<int32_t> flat(seq_lens.size() * max_num_blocks_per_seq, -1);
        for (size_t s = 0; s < block_tables.size() && s < seq_lens.size(); ++s) {
            const size_t len = std::min(block_tables[s].size(), max_num_blocks_per_seq);
            std::copy(block_tables[s].begin(), block_tables[s].begin() + static_cast<std::ptrdiff_t>(len),
                      flat.begin() + static_cast<std::ptrdiff_t>(s * max_num_blocks_per_seq));
        }
        return flat;
    }

    size_t num_seqs() const { return seq_lens.size(); }
    size_t num_tokens() const { return num_prefill_tokens + num_decode_tokens; }

    // leading block ids shared by every table (0 for fewer than two tables)
    void detect_common_prefix_blocks() {
        if (block_tables.size() < 2) {
            common_prefix_blocks = 0;
            return;
        }
        const auto& first = block_tables[0];
        size_t common = first.size();
        for (size_t t = 1; t < block_tables.size(); ++t) {
            const auto& bt = block_tables[t];
            size_t count = 0;
            while (count < first.size() && count < bt.size() && first[count] == bt[count]) ++count;
            common = std::min(common, count);
        }
        common_prefix_blocks = common;
    }

    // per sequence (start, end) of the attended KV range under the window
    std::vector<std::pair<uint32_t, uint32_t>> sliding_window_ranges() const {
        std::vector<std::pair<uint32_t, uint32_t>> r;
        r.reserve(seq_lens.size());
        for (uint32_t len : seq_lens) {
            if (!sliding_window) {
                r.emplace_back(0u, len);
            } else {
                const uint32_t win = static_cast<uint32_t>(*sliding_window);
                r.emplace_back(len <= win ? 0u : len - win, len);
            }
        }
        return r;
    }

    size_t num_window_tokens() const {
        size_t t = 0;
        for (uint32_t len : seq_lens) t += sliding_window ? std::min<size_t>(len, *sliding_window) : len;
        return t;
    }
};

// ---------------------------------------------------------------------------
// paged attention (attention.rs:425-779)
// ---------------------------------------------------------------------------
inline Result<void> paged_attention_decode_f16(uint16_t* output, const uint16_t* query,
                                               const uint16_t* key_cache, const uint16_t* value_cache,
                                               const int32_t* block_tables, const int32_t* seq_lens,
                                               int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads,
                                               int64_t head_dim, int64_t block_size,
                                               int64_t max_num_blocks_per_seq, float scale, uintptr_t stream) {
    return check(rllm_paged_attention_decode_f16(output, query, key_cache, value_cache, block_tables, seq_lens,
                                                 num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                                                 max_num_blocks_per_seq, scale, stream));
}

inline Result<void> paged_attention_decode_f16_sync(uint16_t* output, const uint16_t* query,
                                                    const uint16_t* key_cache, const uint16_t* value_cache,
                                                    const int32_t* block_tables, const int32_t* seq_lens,
                                                    int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads,
                                                    int64_t head_dim, int64_t block_size,
                                                    int64_t max_num_blocks_per_seq, float scale) {
    return check(rllm_paged_attention_decode_f16_sync(output, query, key_cache, value_cache, block_tables,
                                                      seq_lens, num_seqs, num_q_heads, num_kv_heads, head_dim,
                                                      block_size, max_num_blocks_per_seq, scale));
}

inline Result<void> paged_attention_decode_fp8(uint16_t* output, const uint16_t* query, const uint8_t* key_cache,
                                               const uint8_t* value_cache, const int32_t* block_tables,
                                               const int32_t* seq_lens, int64_t num_seqs, int64_t num_q_heads,
                                               int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                               int64_t max_num_blocks_per_seq, float scale, bool is_e5m2,
                                               uintptr_t stream) {
    return check(rllm_paged_attention_decode_fp8(output, query, key_cache, value_cache, block_tables, seq_lens,
                                                 num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                                                 max_num_blocks_per_seq, scale, is_e5m2 ? 1 : 0, stream));
}

inline Result<void> paged_attention_decode_fp8_sync(uint16_t* output, const uint16_t* query,
                                                    const uint8_t* key_cache, const uint8_t* value_cache,
                                                    const int32_t* block_tables, const int32_t* seq_lens,
                                                    int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads,
                                                    int64_t head_dim, int64_t block_size,
                                                    int64_t max_num_blocks_per_seq, float scale, bool is_e5m2) {
    return check(rllm_paged_attention_decode_fp8_sync(output, query, key_cache, value_cache, block_tables,
                                                      seq_lens, num_seqs, num_q_heads, num_kv_heads, head_dim,
                                                      block_size, max_num_blocks_per_seq, scale, is_e5m2 ? 1 : 0));
}

inline Result<void> paged_attention_prefill_f16(uint16_t* output, const uint16_t* query,
                                                const uint16_t* key_cache, const uint16_t* value_cache,
                                                const int32_t* block_tables, const int32_t* seq_lens,
                                                const int32_t* query_start_loc, int64_t num_seqs,
                                                int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                                                int64_t head_dim, int64_t block_size,
                                                int64_t max_num_blocks_per_seq, float scale, uintptr_t stream) {
    return check(rllm_paged_attention_prefill_f16(output, query, key_cache, value_cache, block_tables, seq_lens,
                                                  query_start_loc, num_seqs, num_tokens, num_q_heads,
                                                  num_kv_heads, head_dim, block_size, max_num_blocks_per_seq,
                                                  scale, stream));
}

inline Result<void> paged_attention_prefill_f16_sync(uint16_t* output, const uint16_t* query,
                                                     const uint16_t* key_cache, const uint16_t* value_cache,
                                                     const int32_t* block_tables, const int32_t* seq_lens,
                                                     const int32_t* query_start_loc, int64_t num_seqs,
                                                     int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                                                     int64_t head_dim, int64_t block_size,
                                                     int64_t max_num_blocks_per_seq, float scale) {
    return check(rllm_paged_attention_prefill_f16_sync(output, query, key_cache, value_cache, block_tables,
                                                       seq_lens, query_start_loc, num_seqs, num_tokens,
                                                       num_q_heads, num_kv_heads, head_dim, block_size,
                                                       max_num_blocks_per_seq, scale));
}

inline Result<void> paged_attention_prefill_fp8(uint16_t* output, const uint16_t* query, const uint8_t* key_cache,
                                                const uint8_t* value_cache, const int32_t* block_tables,
                                                const int32_t* seq_lens, const int32_t* query_start_loc,
                                                int64_t num_seqs, int64_t num_tokens, int64_t num_q_heads,
                                                int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                                int64_t max_num_blocks_per_seq, float scale, bool is_e5m2,
                                                uintptr_t stream) {
    return check(rllm_paged_attention_prefill_fp8(output, query, key_cache, value_cache, block_tables, seq_lens,
                                                  query_start_loc, num_seqs, num_tokens, num_q_heads,
                                                  num_kv_heads, head_dim, block_size, max_num_blocks_per_seq,
                                                  scale, is_e5m2 ? 1 : 0, stream));
}

inline Result<void> paged_attention_prefill_fp8_sync(uint16_t* output, const uint16_t* query,
                                                     const uint8_t* key_cache, const uint8_t* value_cache,
                                                     const int32_t* block_tables, const int32_t* seq_lens,
                                                     const int32_t* query_start_loc, int64_t num_seqs,
                                                     int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                                                     int64_t head_dim, int64_t block_size,
                                                     int64_t max_num_blocks_per_seq, float scale, bool is_e5m2) {
    return check(rllm_paged_attention_prefill_fp8_sync(output, query, key_cache, value_cache, block_tables,
                                                       seq_lens, query_start_loc, num_seqs, num_tokens,
                                                       num_q_heads, num_kv_heads, head_dim, block_size,
                                                       max_num_blocks_per_seq, scale, is_e5m2 ? 1 : 0));
}

// ---------------------------------------------------------------------------
// cache operations (cache_ops.rs:106-347)
// ---------------------------------------------------------------------------
inline Result<void> cache_write_f16(uint16_t* key_cache, uint16_t* value_cache, const uint16_t* new_key,
                                    const uint16_t* new_value, const int64_t* slot_mapping, int64_t num_tokens,
                                    int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                    int64_t num_blocks, uintptr_t stream) {
    return check(rllm_cache_write_f16(key_cache, value_cache, new_key, new_value, slot_mapping, num_tokens,
                                      num_kv_heads, head_dim, block_size, num_blocks, stream));
}

inline Result<void> cache_write_f16_sync(uint16_t* key_cache, uint16_t* value_cache, const uint16_t* new_key,
                                         const uint16_t* new_value, const int64_t* slot_mapping,
                                         int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
                                         int64_t block_size, int64_t num_blocks) {
    return check(rllm_cache_write_f16_sync(key_cache, value_cache, new_key, new_value, slot_mapping, num_tokens,
                                           num_kv_heads, head_dim, block_size, num_blocks));
}

inline Result<void> cache_write_fp8(uint8_t* key_cache, uint8_t* value_cache, const uint16_t* new_key,
                                    const uint16_t* new_value, const int64_t* slot_mapping, int64_t num_tokens,
                                    int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                    int64_t num_blocks, bool is_e5m2, uintptr_t stream) {
    return check(rllm_cache_write_fp8(key_cache, value_cache, new_key, new_value, slot_mapping, num_tokens,
                                      num_kv_heads, head_dim, block_size, num_blocks, is_e5m2 ? 1 : 0, stream));
}

inline Result<void> cache_write_fp8_sync(uint8_t* key_cache, uint8_t* value_cache, const uint16_t* new_key,
                                         const uint16_t* new_value, const int64_t* slot_mapping,
                                         int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
                                         int64_t block_size, int64_t num_blocks, bool is_e5m2) {
    return check(rllm_cache_write_fp8_sync(key_cache, value_cache, new_key, new_value, slot_mapping, num_tokens,
                                           num_kv_heads, head_dim, block_size, num_blocks, is_e5m2 ? 1 : 0));
}

inline Result<void> cache_block_copy(const uint8_t* src, uint8_t* dst, int64_t block_nbytes, int64_t num_blocks,
                                     uintptr_t stream) {
    return check(rllm_cache_block_copy(src, dst, block_nbytes, num_blocks, stream));
}

inline Result<void> cache_block_copy_sync(const uint8_t* src, uint8_t* dst, int64_t block_nbytes,
                                          int64_t num_blocks) {
    return check(rllm_cache_block_copy_sync(src, dst, block_nbytes, num_blocks));
}

inline Result<void> cache_zero(uint8_t* ptr, int64_t nbytes, uintptr_t stream) {
    return check(rllm_cache_zero(ptr, nbytes, stream));
}

inline Result<void> cache_zero_sync(uint8_t* ptr, int64_t nbytes) { return check(rllm_cache_zero_sync(ptr, nbytes)); }

inline Result<uint8_t*> gpu_alloc(size_t nbytes) {
    void* p = nullptr;
    const Result<void> r = check(rllm_gpu_alloc(&p, static_cast<int64_t>(nbytes)));
    if (r.is_err()) return Result<uint8_t*>::err(r.error());
    return Result<uint8_t*>::ok(static_cast<uint8_t*>(p));
}

inline Result<void> gpu_free(uint8_t* ptr) { return check(rllm_gpu_free(ptr)); }

// ---------------------------------------------------------------------------
// RotaryEmbedding (rope.rs:5-55): the f32 cos / sin tables
// [max_seq_len][dim / 2] built on the host (f64 angles, rope.rs:13-33).  The
// caller uploads cos_cache() / sin_cache() once per model; rope_cache_write
// then rotates q and k (rope.rs:57-82) and writes the rotated key and the value
// into the paged cache in one launch.
// ---------------------------------------------------------------------------
class RotaryEmbedding {
public:
    static Result<RotaryEmbedding> create(size_t dim, size_t max_seq_len, float theta) {
        RotaryEmbedding r;
        r.dim_ = dim;
        r.max_seq_len_ = max_seq_len;
        r.cos_.resize(max_seq_len * (dim / 2));
        r.sin_.resize(r.cos_.size());
        const Result<void> c = check(rllm_rope_tables(r.cos_.data(), r.sin_.data(), static_cast<int64_t>(max_seq_len),
                                                      static_cast<int64_t>(dim), theta));
        if (c.is_err()) return Result<RotaryEmbedding>::err(c.error());
        return Result<RotaryEmbedding>::ok(std::move(r));
    }
    const std::vector<float>& cos_cache() const { return cos_; }
    const std::vector<float>& sin_cache() const { return sin_; }
    size_t dim() const { return dim_; }
    size_t max_seq_len() const { return max_seq_len_; }

private:
    std::vector<float> cos_, sin_;
    size_t dim_ = 0, max_seq_len_ = 0;
};

// q_out may equal q; dtype is F16 or BF16, kv_dtype dtype or an FP8 type
inline Result<void> rope_cache_write(void* q_out, const void* q, const void* k, const void* v, void* key_cache,
                                     void* value_cache, const int64_t* slot_mapping, const int32_t* positions,
                                     const float* cos_cache, const float* sin_cache, int64_t num_tokens,
                                     int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                     int64_t num_blocks, int64_t max_position, DType dtype, DType kv_dtype,
                                     float k_scale, float v_scale, uintptr_t stream,
                                     int32_t fp8_rounding = RLLM_FP8_ROUND_TOWARD_ZERO) {
    return check(rllm_rope_cache_write_ex(q_out, q, k, v, key_cache, value_cache, slot_mapping, positions,
                                          cos_cache, sin_cache, num_tokens, num_q_heads, num_kv_heads, head_dim,
                                          block_size, num_blocks, max_position, abi_dtype(dtype),
                                          abi_dtype(kv_dtype), k_scale, v_scale, fp8_rounding, stream));
}

// ---------------------------------------------------------------------------
// MXFP4 KV cache (additive entry points): pages of 4-bit codes with a scale per 32
// elements, uint8 [num_blocks, num_kv_heads, mxfp4_page_bytes(head_dim, block_size)]
// ---------------------------------------------------------------------------
inline Result<size_t> mxfp4_page_bytes(size_t head_dim, size_t block_size) {
    const int64_t n = rllm_mxfp4_page_bytes(static_cast<int64_t>(head_dim), static_cast<int64_t>(block_size));
    if (n < 0) return Result<size_t>::err(CudaKernelError{CudaKernelError::Kind::KernelError, 1});   // hipErrorInvalidValue
    return Result<size_t>::ok(static_cast<size_t>(n));
}

inline Result<void> cache_write_mxfp4(uint8_t* key_cache, uint8_t* value_cache, const uint16_t* new_key,
                                      const uint16_t* new_value, const int64_t* slot_mapping, int64_t num_tokens,
                                      int64_t num_kv_heads, int64_t head_dim, int64_t block_size, int64_t num_blocks,
                                      DType input_dtype, uintptr_t stream) {
    return check(rllm_cache_write_mxfp4(key_cache, value_cache, new_key, new_value, slot_mapping, num_tokens,
                                        num_kv_heads, head_dim, block_size, num_blocks, abi_dtype(input_dtype), stream));
}

inline Result<void> cache_read_mxfp4(uint16_t* out_key, uint16_t* out_value, const uint8_t* key_cache,
                                     const uint8_t* value_cache, const int64_t* slot_mapping, int64_t num_tokens,
                                     int64_t num_kv_heads, int64_t head_dim, int64_t block_size, int64_t num_blocks,
                                     DType output_dtype, uintptr_t stream) {
    return check(rllm_cache_read_mxfp4(out_key, out_value, key_cache, value_cache, slot_mapping, num_tokens,
                                       num_kv_heads, head_dim, block_size, num_blocks, abi_dtype(output_dtype), stream));
}

// q_out may equal q; dtype is F16 or BF16
inline Result<void> rope_cache_write_mxfp4(void* q_out, const void* q, const void* k, const void* v,
                                           uint8_t* key_cache, uint8_t* value_cache, const int64_t* slot_mapping,
                                           const int32_t* positions, const float* cos_cache, const float* sin_cache,
                                           int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                                           int64_t head_dim, int64_t block_size, int64_t num_blocks,
                                           int64_t max_position, DType dtype, uintptr_t stream) {
    return check(rllm_rope_cache_write_mxfp4(q_out, q, k, v, key_cache, value_cache, slot_mapping, positions, cos_cache,
                                             sin_cache, num_tokens, num_q_heads, num_kv_heads, head_dim, block_size,
                                             num_blocks, max_position, abi_dtype(dtype), stream));
}

// workspace null: library-owned scratch
inline Result<void> paged_attention_decode_mxfp4(void* output, const void* query, const uint8_t* key_cache,
                                                 const uint8_t* value_cache, const int32_t* block_tables,
                                                 const int32_t* seq_lens, int64_t num_seqs, int64_t num_q_heads,
                                                 int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                                 int64_t max_num_blocks_per_seq, int64_t num_blocks, float scale,
                                                 DType q_dtype, uintptr_t stream, void* workspace = nullptr,
                                                 int64_t workspace_bytes = 0) {
    return check(rllm_paged_attention_decode_mxfp4(output, query, key_cache, value_cache, block_tables, seq_lens,
                                                   num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                                                   max_num_blocks_per_seq, num_blocks, scale, abi_dtype(q_dtype),
                                                   workspace, workspace_bytes, stream));
}

inline Result<void> paged_attention_prefill_mxfp4(void* output, const void* query, const uint8_t* key_cache,
                                                  const uint8_t* value_cache, const int32_t* block_tables,
                                                  const int32_t* seq_lens, const int32_t* query_start_loc,
                                                  int64_t num_seqs, int64_t num_tokens, int64_t num_q_heads,
                                                  int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                                  int64_t max_num_blocks_per_seq, int64_t num_blocks, float scale,
                                                  DType q_dtype, uintptr_t stream) {
    return check(rllm_paged_attention_prefill_mxfp4(output, query, key_cache, value_cache, block_tables, seq_lens,
                                                    query_start_loc, num_seqs, num_tokens, num_q_heads, num_kv_heads,
                                                    head_dim, block_size, max_num_blocks_per_seq, num_blocks, scale,
                                                    abi_dtype(q_dtype), stream));
}

// ---------------------------------------------------------------------------
// block lists: copy-on-write copies and swap records (additive entry points)
// ---------------------------------------------------------------------------
inline Result<void> cache_copy_blocks(const uint64_t* key_caches, const uint64_t* value_caches, int64_t num_layers,
                                      const int64_t* block_pairs, int64_t num_pairs, int64_t num_blocks,
                                      int64_t block_nbytes, uintptr_t stream) {
    return check(rllm_cache_copy_blocks(key_caches, value_caches, num_layers, block_pairs, num_pairs, num_blocks,
                                        block_nbytes, stream));
}

inline Result<void> cache_swap_out(const uint64_t* key_caches, const uint64_t* value_caches, int64_t num_layers,
                                   const int64_t* block_ids, int64_t num_ids, int64_t num_blocks, int64_t block_nbytes,
                                   const int64_t* record_slots, int64_t num_records, uint8_t* host_records,
                                   uintptr_t stream) {
    return check(rllm_cache_swap_out(key_caches, value_caches, num_layers, block_ids, num_ids, num_blocks,
                                     block_nbytes, record_slots, num_records, host_records, stream));
}

inline Result<void> cache_swap_in(const uint64_t* key_caches, const uint64_t* value_caches, int64_t num_layers,
                                  const int64_t* block_ids, int64_t num_ids, int64_t num_blocks, int64_t block_nbytes,
                                  const int64_t* record_slots, int64_t num_records, const uint8_t* host_records,
                                  uintptr_t stream) {
    return check(rllm_cache_swap_in(key_caches, value_caches, num_layers, block_ids, num_ids, num_blocks,
                                    block_nbytes, record_slots, num_records, host_records, stream));
}

// ---------------------------------------------------------------------------
// CpuKvOffloadStore (offload.rs:7-84): pinned host records keyed by
// (request, block).  put / get / remove / usage keep the reference's
// semantics (put of a wrong-sized block and put into a full store fail with
// its messages; a second put of a key reuses its slot).  reserve() / slot_of()
// expose record slots so a GPU swap (cache_swap_out / _in with record_slots)
// can move the bytes of many blocks straight into / out of storage().
// ---------------------------------------------------------------------------
struct CpuKvOffloadUsage {
    size_t capacity_blocks, used_blocks, free_blocks;
    bool operator==(const CpuKvOffloadUsage& o) const {
        return capacity_blocks == o.capacity_blocks && used_blocks == o.used_blocks && free_blocks == o.free_blocks;
    }
};

class CpuKvOffloadStore {
public:
    static Result<CpuKvOffloadStore> create(size_t capacity_blocks, size_t block_size_bytes) {
        CpuKvOffloadStore s;
        s.block_size_bytes_ = block_size_bytes;
        s.capacity_blocks_ = capacity_blocks;
        for (size_t i = capacity_blocks; i-- > 0;) s.free_slots_.push_back(i);   // pops 0 first
        // pinned (hipHostMalloc) so GPU swaps can use it; without a GPU runtime a
        // zeroed heap buffer, as PinnedBuffer::alloc (rllm-tensor/src/pinned.rs:
        // 22-31, 98-103), which the swap entry points refuse
        const size_t bytes = std::max<size_t>(capacity_blocks * block_size_bytes, 1);
        void* p = nullptr;
        if (rllm_gpu_alloc_host(&p, static_cast<int64_t>(bytes)) == 0 && p) {
            std::fill(static_cast<uint8_t*>(p), static_cast<uint8_t*>(p) + bytes, uint8_t{0});
            s.pinned_ = true;
        } else {
            p = std::calloc(bytes, 1);
            if (!p) return Result<CpuKvOffloadStore>::err(CudaKernelError{CudaKernelError::Kind::KernelError, 2});
        }
        s.storage_ = static_cast<uint8_t*>(p);
        return Result<CpuKvOffloadStore>::ok(std::move(s));
    }

    CpuKvOffloadStore() = default;
    CpuKvOffloadStore(const CpuKvOffloadStore&) = delete;
    CpuKvOffloadStore& operator=(const CpuKvOffloadStore&) = delete;
    CpuKvOffloadStore(CpuKvOffloadStore&& o) noexcept { *this = std::move(o); }
    CpuKvOffloadStore& operator=(CpuKvOffloadStore&& o) noexcept {
        if (this != &o) {
            release();
            block_size_bytes_ = o.block_size_bytes_;
            capacity_blocks_ = o.capacity_blocks_;
            free_slots_ = std::move(o.free_slots_);
            slots_ = std::move(o.slots_);
            storage_ = o.storage_;
            pinned_ = o.pinned_;
            o.storage_ = nullptr;
        }
        return *this;
    }
    ~CpuKvOffloadStore() { release(); }

    // nullopt on success, else the reference's error message
    std::optional<std::string> put(RequestId request, BlockId block, const uint8_t* bytes, size_t len) {
        if (len != block_size_bytes_)
            return "offloaded block has " + std::to_string(len) + " bytes, expected " +
                   std::to_string(block_size_bytes_);
        const std::optional<size_t> slot = reserve(request, block);
        if (!slot) return std::string("CPU KV offload store is full");
        std::copy(bytes, bytes + len, storage_ + *slot * block_size_bytes_);
        return std::nullopt;
    }

    std::optional<std::vector<uint8_t>> get(RequestId request, BlockId block) const {
        const std::optional<size_t> slot = slot_of(request, block);
        if (!slot) return std::nullopt;
        const uint8_t* p = storage_ + *slot * block_size_bytes_;
        return std::vector<uint8_t>(p, p + block_size_bytes_);
    }

    bool remove(RequestId request, BlockId block) {
        auto it = slots_.find(key(request, block));
        if (it == slots_.end()) return false;
        free_slots_.push_back(it->second);
        slots_.erase(it);
        return true;
    }

    CpuKvOffloadUsage usage() const { return {capacity_blocks_, slots_.size(), free_slots_.size()}; }

    // the record slot of (request, block), taking a free one for a new key;
    // nullopt when the store is full
    std::optional<size_t> reserve(RequestId request, BlockId block) {
        if (auto s = slot_of(request, block)) return s;
        if (free_slots_.empty()) return std::nullopt;
        const size_t slot = free_slots_.back();
        free_slots_.pop_back();
        slots_.emplace(key(request, block), slot);
        return slot;
    }
    std::optional<size_t> slot_of(RequestId request, BlockId block) const {
        auto it = slots_.find(key(request, block));
        if (it == slots_.end()) return std::nullopt;
        return it->second;
    }
    uint8_t* storage() { return storage_; }
    bool pinned() const { return pinned_; }
    size_t block_size_bytes() const { return block_size_bytes_; }
    size_t capacity_blocks() const { return capacity_blocks_; }

private:
    static std::pair<uint64_t, uint32_t> key(RequestId r, BlockId b) { return {r.value, b.value}; }
    void release() {
        if (storage_ && pinned_)
            rllm_gpu_free_host(storage_);
        else if (storage_)
            std::free(storage_);
        storage_ = nullptr;
    }

    bool pinned_ = false;
    size_t block_size_bytes_ = 0, capacity_blocks_ = 0;
    std::vector<size_t> free_slots_;
    std::map<std::pair<uint64_t, uint32_t>, size_t> slots_;
    uint8_t* storage_ = nullptr;
};

// ---------------------------------------------------------------------------
// GpuKVCache (cache_ops.rs:350-490): per-layer K and V device tensors
// [num_blocks, num_kv_heads, head_dim, block_size], zero-filled at creation,
// freed on destruction.
// ---------------------------------------------------------------------------
class GpuKVCache {
public:
    static Result<GpuKVCache> create(size_t num_blocks, size_t num_layers, size_t num_kv_heads, size_t head_dim,
                                     size_t block_size, DType dtype) {
        GpuKVCache c;
        c.num_blocks_ = num_blocks;
        c.num_kv_heads_ = num_kv_heads;
        c.head_dim_ = head_dim;
        c.block_size_ = block_size;
        c.element_size_ = bytes_per_scalar(dtype);
        c.dtype_ = dtype;
        const size_t per = num_blocks * num_kv_heads * head_dim * block_size * c.element_size_;
        for (size_t l = 0; l < num_layers; ++l) {
            Result<uint8_t*> k = gpu_alloc(per);
            if (k.is_err()) return Result<GpuKVCache>::err(k.error());
            Result<uint8_t*> v = gpu_alloc(per);
            if (v.is_err()) {
                gpu_free(k.value());
                return Result<GpuKVCache>::err(v.error());
            }
            c.layer_ptrs_.emplace_back(k.value(), v.value());
            c.layer_sizes_.emplace_back(per, per);
            for (uint8_t* p : {k.value(), v.value()}) {
                const Result<void> z = cache_zero(p, static_cast<int64_t>(per), 0);
                if (z.is_err()) return Result<GpuKVCache>::err(z.error());
            }
        }
        return Result<GpuKVCache>::ok(std::move(c));
    }

    GpuKVCache() = default;
    GpuKVCache(const GpuKVCache&) = delete;
    GpuKVCache& operator=(const GpuKVCache&) = delete;
    GpuKVCache(GpuKVCache&& o) noexcept { *this = std::move(o); }
    GpuKVCache& operator=(GpuKVCache&& o) noexcept {
        if (this != &o) {
            release();
            layer_ptrs_ = std::move(o.layer_ptrs_);
            layer_sizes_ = std::move(o.layer_sizes_);
            o.layer_ptrs_.clear();
            o.layer_sizes_.clear();
            num_blocks_ = o.num_blocks_;
            num_kv_heads_ = o.num_kv_heads_;
            head_dim_ = o.head_dim_;
            block_size_ = o.block_size_;
            element_size_ = o.element_size_;
            dtype_ = o.dtype_;
        }
        return *this;
    }
    ~GpuKVCache() { release(); }

    const uint8_t* key_ptr(size_t layer) const { return layer_ptrs_[layer].first; }
    const uint8_t* value_ptr(size_t layer) const { return layer_ptrs_[layer].second; }
    std::array<size_t, 4> key_shape() const { return {num_blocks_, num_kv_heads_, head_dim_, block_size_}; }
    std::array<size_t, 4> value_shape() const { return key_shape(); }
    DType dtype() const { return dtype_; }
    size_t num_layers() const { return layer_ptrs_.size(); }
    size_t total_bytes() const {
        size_t t = 0;
        for (const auto& kv : layer_sizes_) t += kv.first + kv.second;
        return t;
    }
    size_t num_blocks() const { return num_blocks_; }
    size_t block_size() const { return block_size_; }
    size_t element_size() const { return element_size_; }

    // slot = block * block_size + offset
    std::vector<int64_t> compute_slots(const std::vector<std::pair<BlockId, size_t>>& positions) const {
        std::vector<int64_t> s;
        s.reserve(positions.size());
        for (const auto& p : positions)
            s.push_back(static_cast<int64_t>(p.first.value) * static_cast<int64_t>(block_size_) +
                        static_cast<int64_t>(p.second));
        return s;
    }

private:
    void release() {
        for (auto& kv : layer_ptrs_) {
            gpu_free(kv.first);
            gpu_free(kv.second);
        }
        layer_ptrs_.clear();
        layer_sizes_.clear();
    }

    std::vector<std::pair<uint8_t*, uint8_t*>> layer_ptrs_;
    std::vector<std::pair<size_t, size_t>> layer_sizes_;
    size_t num_blocks_ = 0, num_kv_heads_ = 0, head_dim_ = 0, block_size_ = 0, element_size_ = 0;
    DType dtype_ = DType::F16;
};

// ---------------------------------------------------------------------------
// model_runner.rs:806-826: slot(pos) = block_table[pos / bs] * bs + pos % bs,
// or -1 past the table (or on overflow)
// ---------------------------------------------------------------------------
inline std::vector<int64_t> compute_slot_mappings(const std::vector<uint32_t>& positions,
                                                  const std::vector<uint32_t>& block_table, size_t block_size) {
    std::vector<int64_t> out(positions.size(), -1);
    if (block_size == 0 || block_size > 0xFFFFFFFFull) return out;
    const uint32_t bs = static_cast<uint32_t>(block_size);
    for (size_t i = 0; i < positions.size(); ++i) {
        const uint32_t bi = positions[i] / bs, off = positions[i] % bs;
        int64_t slot;
        if (bi < block_table.size() &&
            !__builtin_mul_overflow(static_cast<int64_t>(block_table[bi]), static_cast<int64_t>(bs), &slot) &&
            !__builtin_add_overflow(slot, static_cast<int64_t>(off), &slot))
            out[i] = slot;
    }
    return out;
}

}  // namespace kernels
}  // namespace rllm
