// paged_mma_f16.cu — the tensor-core decode kernel over fp16 pages.
#include "paged_mma.cuh"

namespace bozo {

cudaError_t launch_paged_mma_f16(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  return launch_paged_mma<BOZO_DT_F16>(p, pl, st);
}

}  // namespace bozo
