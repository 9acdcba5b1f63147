// adapter_gemm_bf16.cu — the adapter's tensor-core products for bfloat16 results.
#include "adapter_gemm.cuh"

namespace xvec {
namespace adapter {

xvec_gpu_status gemm_bf16(const GemmCall& c, cudaStream_t s) { return gemm_by_mode<bf16>(c, s); }

}  // namespace adapter
}  // namespace xvec
