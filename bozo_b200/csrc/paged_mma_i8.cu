// paged_mma_i8.cu — the tensor-core decode kernel over int8 pages.
#include "paged_mma.cuh"

namespace bozo {

cudaError_t launch_paged_mma_i8(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  return launch_paged_mma<BOZO_DT_I8>(p, pl, st);
}

}  // namespace bozo
