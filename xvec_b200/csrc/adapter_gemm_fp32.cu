// adapter_gemm_fp32.cu — the adapter's tensor-core products for float results.
#include "adapter_gemm.cuh"

namespace xvec {
namespace adapter {

xvec_gpu_status gemm_fp32(const GemmCall& c, cudaStream_t s) { return gemm_by_mode<float>(c, s); }

}  // namespace adapter
}  // namespace xvec
