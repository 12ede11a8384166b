// Entry points of decode attention over the MXFP4 KV cache (the kernel:
// mxfp4_decode_kernel.h).
#include "mxfp4_decode_kernel.h"

namespace rllm {
namespace {

// Waves a workgroup: four share a row's items, two where rows are many and short, so
// that a workgroup joins less often for the same waves on the chip.  With a
// row or more for every pair of waves, us of four / two: 256 contexts (32/8 heads,
// head_dim 128) of 64 tokens 20.0 / 13.8, 256 28.0 / 23.1, 512 39.3 / 34.2, 2048 132 / 133, of
// 32-512 38 / 35; 128 of 4096 126 / 130.  With fewer rows two cut them more often: 64 of
// 512 12.5 / 17.0.  The host knows the tables' width alone: under tables of 4096 tokens those
// 256 contexts of 64 run four waves, 21.8 us, of 256 30.7.
constexpr int64_t MXD_SHORT = 2048;   // tokens

// *wgs, *waves: of this call; *most: workgroups of any call of these heads with no more
// sequences and no wider tables, for which scratch is sized.  Where rows are many, narrow
// tables take more (of two waves) than wide ones.
int32_t mxd_workgroups(int64_t num_seqs, int64_t hq, int64_t hkv, int64_t d, int64_t bs, int64_t maxb, int64_t* wgs,
                       int* waves, int64_t* most) {
    int dev = 0, cus = 0;
    RLLM_TRY(hipGetDevice(&dev));
    RLLM_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    const int64_t groups = (hq / hkv + MXD_HEADS - 1) / MXD_HEADS, rows = num_seqs * hkv * groups;
    const bool many = rows >= static_cast<int64_t>(cus) * mxd_per_cu(d, 2);
    *waves = many && maxb * bs <= MXD_SHORT ? 2 : 4;
    *wgs = mxd_at_most(rows, d, bs, maxb, cus, *waves);
    *most = mxd_at_most(rows, d, bs, maxb, cus, many ? 2 : 4);
    return 0;
}

int32_t mxd_check(int64_t num_seqs, int64_t hq, int64_t hkv, int64_t d, int64_t bs, int64_t maxb, int64_t nb) {
    RLLM_CHECK_ARG(mx4_shape_ok(hkv, d, bs, nb));
    RLLM_CHECK_ARG(mx4_attention_ok(num_seqs, hq, hkv, bs, maxb));
    // the items of all rows are counted in 32 bits
    const int64_t rows = num_seqs * hkv * ((hq / hkv + MXD_HEADS - 1) / MXD_HEADS);
    RLLM_CHECK_ARG(rows * ((maxb * bs + MXD_ITEM - 1) / MXD_ITEM + 1 + MXD_VIRT) <= INT32_MAX);
    return 0;
}

}  // namespace
}  // namespace rllm

using namespace rllm;

extern "C" {

int64_t rllm_paged_attention_decode_mxfp4_workspace_size(int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads,
                                                         int64_t head_dim, int64_t block_size,
                                                         int64_t max_num_blocks_per_seq) {
    if (num_seqs <= 0) return 0;
    if (mxd_check(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, 0)) return -1;
    int64_t wgs = 0, most = 0;
    int waves = 0;
    if (mxd_workgroups(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, &wgs, &waves, &most))
        return -1;
    return mxd_scratch_bytes(most, head_dim);
}

int32_t rllm_paged_attention_decode_mxfp4(void* output, const void* query, const uint8_t* key_cache,
                                          const uint8_t* value_cache, const int32_t* block_tables,
                                          const int32_t* seq_lens, int64_t num_seqs, int64_t num_q_heads,
                                          int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                          int64_t max_num_blocks_per_seq, int64_t num_blocks, float scale,
                                          int32_t q_dtype, void* workspace, int64_t workspace_bytes,
                                          uintptr_t stream) {
    if (num_seqs <= 0) return 0;
    RLLM_CHECK_ARG(output && query && key_cache && value_cache && block_tables && seq_lens);
    const int32_t bad = mxd_check(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, num_blocks);
    if (bad) return bad;
    RLLM_CHECK_ARG(num_blocks > 0);
    RLLM_CHECK_ARG(q_dtype == RLLM_DTYPE_F16 || q_dtype == RLLM_DTYPE_BF16);
    RLLM_CHECK_ARG(std::isfinite(scale * MX4_LOG2E));
    RLLM_CHECK_ARG(mx4_aligned16(key_cache) && mx4_aligned16(value_cache));
    RLLM_CHECK_ARG(((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(output)) & 3) == 0);
    int64_t wgs = 0, most = 0;
    int waves = 0;
    const int32_t rc = mxd_workgroups(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, &wgs, &waves, &most);
    if (rc) return rc;
    void* ws = workspace;
    if (ws) {
        RLLM_CHECK_ARG(mx4_aligned16(ws) && workspace_bytes >= mxd_scratch_bytes(wgs, head_dim));
    } else {
        RLLM_TRY(static_cast<hipError_t>(g_workspaces.get(stream, WS_MX4_DECODE, mxd_scratch_bytes(most, head_dim), true, &ws)));
        if (!ws) {   // captured before any eager call of this size: a workgroup a row
            wgs = num_seqs * num_kv_heads * ((num_q_heads / num_kv_heads + MXD_HEADS - 1) / MXD_HEADS);
            RLLM_CHECK_ARG(wgs * 64 * waves <= MX4_MAX_THREADS);
        }
    }
    const MxDecodeArgs a = mxd_args(output, query, key_cache, value_cache, block_tables, seq_lens, num_seqs, num_q_heads,
                                    num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, num_blocks, scale, ws, wgs);
    hipStream_t st = as_stream(stream);
    if (waves == 2)
        return q_dtype == RLLM_DTYPE_BF16 ? mxd_launch<KIND_BF16, 2, false>(a, head_dim, wgs, st)
                                          : mxd_launch<KIND_F16, 2, false>(a, head_dim, wgs, st);
    return q_dtype == RLLM_DTYPE_BF16 ? mxd_launch<KIND_BF16, 4, false>(a, head_dim, wgs, st)
                                      : mxd_launch<KIND_F16, 4, false>(a, head_dim, wgs, st);
}

}  // extern "C"
