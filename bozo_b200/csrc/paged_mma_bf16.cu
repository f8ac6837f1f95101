// paged_mma_bf16.cu — the tensor-core decode kernel over bf16 pages.
#include "paged_mma.cuh"

namespace bozo {

cudaError_t launch_paged_mma_bf16(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  return launch_paged_mma<BOZO_DT_BF16>(p, pl, st);
}

}  // namespace bozo
