// Attention over listed cache blocks: the entry point, and the launches over 16-bit
// caches (the kernel is in sparse_attention_kernel.h).
#include "sparse_attention_kernel.h"

namespace rllm {

int32_t launch_sparse_16(const SparseArgs& a, int32_t q_dtype, int64_t d, hipStream_t st) {
    return q_dtype == RLLM_DTYPE_BF16 ? launch_sparse<KIND_BF16, KIND_BF16>(a, d, st) : launch_sparse<KIND_F16, KIND_F16>(a, d, st);
}

}  // namespace rllm

using namespace rllm;

extern "C" {

int32_t rllm_paged_attention_sparse(void* output, const void* query, const void* key_cache, const void* value_cache,
                                    const int32_t* block_tables, const int32_t* seq_lens, const int32_t* query_start_loc,
                                    const int32_t* selected, int64_t num_seqs, int64_t num_rows, int64_t num_q_heads,
                                    int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                    int64_t max_num_blocks_per_seq, int64_t num_blocks, int64_t num_selected, float scale,
                                    int32_t q_dtype, int32_t kv_dtype, float k_scale, float v_scale, uintptr_t stream) {
    if (num_seqs <= 0 || num_rows <= 0) return 0;
    RLLM_CHECK_ARG(sparse_shape(num_kv_heads, head_dim, block_size) && sparse_heads(num_q_heads, num_kv_heads));
    RLLM_CHECK_ARG(sparse_types(q_dtype, kv_dtype));
    RLLM_CHECK_ARG(num_seqs <= SPARSE_MAX_ROWS && num_rows <= SPARSE_MAX_ROWS && num_blocks >= 0);
    RLLM_CHECK_ARG(sparse_table(max_num_blocks_per_seq, block_size));
    RLLM_CHECK_ARG(query_start_loc || num_rows == num_seqs);
    RLLM_CHECK_ARG(num_selected >= 1 && num_selected <= RLLM_SELECT_MAX_BLOCKS);
    RLLM_CHECK_ARG(output && query && key_cache && value_cache && seq_lens && selected);
    RLLM_CHECK_ARG(output != query);                   // a row may be computed again
    RLLM_CHECK_ARG(block_tables || max_num_blocks_per_seq == 0);
    for (const void* p : {static_cast<const void*>(output), query, key_cache, value_cache}) RLLM_CHECK_ARG(aligned_to(p, 16));
    const bool fp8 = kv_dtype == RLLM_DTYPE_FP8_E4M3 || kv_dtype == RLLM_DTYPE_FP8_E5M2;
    if (!fp8) k_scale = v_scale = 1.f;
    const float s_scale = scale * k_scale * 1.44269504088896340736f;
    RLLM_CHECK_ARG(std::isfinite(scale) && std::isfinite(k_scale) && std::isfinite(v_scale) && std::isfinite(s_scale));
    const int64_t head_groups = (num_q_heads / num_kv_heads + 15) / 16;
    RLLM_CHECK_ARG(num_rows * num_kv_heads * head_groups <= INT32_MAX);   // (and what is launched: MAX_WORKGROUPS)
    SparseArgs a = {};
    a.out = static_cast<uint16_t*>(output);
    a.q = static_cast<const uint16_t*>(query);
    a.kc = static_cast<const uint8_t*>(key_cache);
    a.vc = static_cast<const uint8_t*>(value_cache);
    a.bt = block_tables;
    a.seq_lens = seq_lens;
    a.qsl = query_start_loc;
    a.sel = selected;
    a.num_seqs = static_cast<int32_t>(num_seqs);
    a.rows = static_cast<int32_t>(num_rows);
    a.hq = static_cast<int32_t>(num_q_heads);
    a.hkv = static_cast<int32_t>(num_kv_heads);
    a.bs_log2 = __builtin_ctz(static_cast<unsigned>(block_size));
    a.maxb = static_cast<int32_t>(max_num_blocks_per_seq);
    a.k = static_cast<int32_t>(num_selected);
    a.head_groups = static_cast<int32_t>(head_groups);
    a.num_blocks = num_blocks;
    a.s_scale = s_scale;
    a.v_scale = v_scale;
    const hipStream_t st = as_stream(stream);
    if (kv_dtype == RLLM_DTYPE_FP8_E4M3) return launch_sparse_e4m3(a, q_dtype, head_dim, st);
    if (kv_dtype == RLLM_DTYPE_FP8_E5M2) return launch_sparse_e5m2(a, q_dtype, head_dim, st);
    return launch_sparse_16(a, q_dtype, head_dim, st);
}

}  // extern "C"
