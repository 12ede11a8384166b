// Attention over listed blocks of FP8 E4M3 caches (the kernel is in sparse_attention_kernel.h).
#include "sparse_attention_kernel.h"

namespace rllm {

int32_t launch_sparse_e4m3(const SparseArgs& a, int32_t q_dtype, int64_t d, hipStream_t st) {
    return q_dtype == RLLM_DTYPE_BF16 ? launch_sparse<KIND_BF16, KIND_FP8_E4M3>(a, d, st) : launch_sparse<KIND_F16, KIND_FP8_E4M3>(a, d, st);
}

}  // namespace rllm
