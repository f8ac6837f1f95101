// paged_mma_f4.cu — the tensor-core decode kernel over 4-bit pages.
#include "paged_mma.cuh"

namespace bozo {

cudaError_t launch_paged_mma_f4(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  return launch_paged_mma<BOZO_DT_F4E2M1>(p, pl, st);
}

}  // namespace bozo
