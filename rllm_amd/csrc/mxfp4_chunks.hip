// Chunks of few new tokens on the decode kernel, for mxfp4_prefill.hip.
#include "mxfp4_decode_kernel.h"

namespace rllm {

int64_t mx4_short_rows(int64_t num_seqs, int64_t num_tokens, int64_t hq, int64_t hkv, int64_t bs, int64_t maxb,
                       int64_t most_cols) {
    // ceil(c / 16) <= (c - 1) / 16 + 1 for the c > 0 columns of a sequence
    const int64_t used = num_seqs < num_tokens ? num_seqs : num_tokens;
    int64_t rows = ((num_tokens * (hq / hkv) - used) / MXD_HEADS + used) * hkv;
    const int64_t most = used * hkv * ((most_cols + MXD_HEADS - 1) / MXD_HEADS);
    if (rows > most) rows = most;
    // the items of all rows are counted in 32 bits; without scratch a row is a workgroup
    return rows * 256 <= MX4_MAX_THREADS && rows * ((maxb * bs + MXD_ITEM - 1) / MXD_ITEM + 1 + MXD_VIRT) <= INT32_MAX ? rows : -1;
}

int32_t mx4_short_chunks(void* out, const void* q, const uint8_t* kc, const uint8_t* vc, const int32_t* bt,
                         const int32_t* seq_lens, const int32_t* qsl, int64_t num_seqs, int64_t num_tokens, int64_t hq,
                         int64_t hkv, int64_t d, int64_t bs, int64_t maxb, int64_t nb, float scale, int32_t q_dtype,
                         int64_t most_cols, uintptr_t stream) {
    int dev = 0, cus = 0;
    RLLM_TRY(hipGetDevice(&dev));
    RLLM_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    const int64_t rows = mx4_short_rows(num_seqs, num_tokens, hq, hkv, bs, maxb, most_cols);
    RLLM_CHECK_ARG(rows > 0);
    const int64_t wgs_at_most = mxd_at_most(rows, d, bs, maxb, cus, 4);
    void* ws = nullptr;
    RLLM_TRY(static_cast<hipError_t>(g_workspaces.get(stream, WS_MX4_DECODE, mxd_scratch_bytes(wgs_at_most, d), true, &ws)));
    const int64_t wgs = ws ? wgs_at_most : rows;   // captured before any eager call of this size: a workgroup a row
    MxDecodeArgs a = mxd_args(out, q, kc, vc, bt, seq_lens, num_seqs, hq, hkv, d, bs, maxb, nb, scale, ws, wgs);
    a.qsl = qsl;
    a.num_tokens = static_cast<int32_t>(num_tokens);
    a.most_cols = static_cast<int32_t>(most_cols);
    return q_dtype == RLLM_DTYPE_BF16 ? mxd_launch<KIND_BF16, 4, true>(a, d, wgs, as_stream(stream))
                                      : mxd_launch<KIND_F16, 4, true>(a, d, wgs, as_stream(stream));
}

}  // namespace rllm
