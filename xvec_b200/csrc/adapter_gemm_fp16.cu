// adapter_gemm_fp16.cu — the adapter's tensor-core products for __half results.
#include "adapter_gemm.cuh"

namespace xvec {
namespace adapter {

xvec_gpu_status gemm_fp16(const GemmCall& c, cudaStream_t s) { return gemm_by_mode<__half>(c, s); }

}  // namespace adapter
}  // namespace xvec
