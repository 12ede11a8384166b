// Attention over listed blocks of FP8 E5M2 caches (the kernel is in sparse_attention_kernel.h).
#include "sparse_attention_kernel.h"

namespace rllm {

int32_t launch_sparse_e5m2(const SparseArgs& a, int32_t q_dtype, int64_t d, hipStream_t st) {
    return q_dtype == RLLM_DTYPE_BF16 ? launch_sparse<KIND_BF16, KIND_FP8_E5M2>(a, d, st) : launch_sparse<KIND_F16, KIND_FP8_E5M2>(a, d, st);
}

}  // namespace rllm
