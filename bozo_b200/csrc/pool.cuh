// pool.cuh — parameter blocks and launchers of the page tables' kernels
// (paged_pool.cu).
#pragma once

#include "paged.cuh"

namespace bozo {

constexpr int kMaxTableRows = 8192;  // sequences of a table: their sums are held in shared memory

struct ReserveP {
  int* table;
  long long ts;
  int B, M, page, P;
  const int* lengths;
  const int* tokens;
  int* refs;
  int* cu;
  int* missing;
  long long rows;
  int* seq;
  int* pos;
  int* slot;
  int* err;
  unsigned cap;  // M·page
  FastDiv div_cap, div_page;
};
cudaError_t launch_paged_reserve(const ReserveP& p, cudaStream_t st, int* launches);

struct ForkP {
  int* table;
  long long ts;
  int B, M, page, P, share;
  const int* lengths;
  const int* parents;
  int* refs;
  int* copies;
  int* missing;
  int* err;
  FastDiv div_page;
};
cudaError_t launch_paged_fork(const ForkP& p, cudaStream_t st);

constexpr int kCopyPools = 128;  // pools of one launch
struct CopyP {
  char* pool[kCopyPools];
  long long bytes[kCopyPools];
  int P;
  const int* copies;
};
cudaError_t launch_paged_copy(const CopyP& p, int pools, long long n, cudaStream_t st);

}  // namespace bozo
