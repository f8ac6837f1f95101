// paged_mma_f8.cu — the tensor-core decode kernel over e4m3 pages.
#include "paged_mma.cuh"

namespace bozo {

cudaError_t launch_paged_mma_f8(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  return launch_paged_mma<BOZO_DT_F8E4M3>(p, pl, st);
}

}  // namespace bozo
