// paged_pool.cu — page tables on the device: pages and places for new tokens
// (bozo_paged_reserve), rows of the table reordered (bozo_paged_fork) and pages copied
// (bozo_paged_copy).
//
// refs[p] counts the table rows that hold page p; 0: it is free.  Both table kernels
// are one cluster.  Every block works out for itself what each sequence wants (the
// prefix sums of a few thousand integers, in shared memory); the pool's counts are
// shared out, a part of them a block, whose numbers of free pages go round through the
// cluster's shared memory.  The i-th free page then finds its place by a search in the
// prefix sums, so nothing depends on an order of atomics.
#include <cooperative_groups.h>

#include "pool.cuh"

namespace bozo {
namespace {

namespace cg = cooperative_groups;
constexpr int kThreads = 1024;

// Inclusive scan of v over the block; `total`: the sum.  `tmp`: 32 words.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* tmp,
                                                         unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) tmp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    unsigned long long w = tmp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    tmp[lane] = w;
  }
  __syncthreads();
  total = tmp[31];
  if (warp) v += tmp[warp - 1];
  __syncthreads();
  return v;
}

// The last i in [0, n) with sums[i] ≤ x (sums[0] ≤ x, non-decreasing).
__device__ __forceinline__ int find(const int* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ bool free_page(const int* refs, int p) { return __ldcg(refs + p) == 0; }

// The part of the pool that this block of the cluster looks after.
struct Part {
  int lo, hi;
  __device__ Part(int pages, unsigned rank, unsigned blocks) {
    const int each = (int)(((long long)pages + blocks - 1) / blocks);
    lo = min(pages, each * (int)rank);
    hi = min(pages, lo + each);
  }
};

// Free pages before this block's part and in all; `count`: one word of shared memory.
__device__ __forceinline__ void count_free(const int* refs, Part part, int* count, unsigned long long* tmp, int& before,
                                           int& all) {
  cg::cluster_group cl = cg::this_cluster();
  int n = 0;
  for (int p = part.lo + threadIdx.x; p < part.hi; p += kThreads) n += free_page(refs, p);
  unsigned long long total;
  block_scan(n, tmp, total);
  if (threadIdx.x == 0) *count = (int)total;
  cl.sync();
  before = all = 0;
  for (unsigned r = 0; r < cl.num_blocks(); ++r) {
    const int c = *cl.map_shared_rank(count, r);
    if (r < cl.block_rank()) before += c;
    all += c;
  }
}

// f(rank, page) for this block's free pages of rank < want, in ascending order.
template <typename F>
__device__ __forceinline__ void give(const int* refs, Part part, int before, int want, unsigned long long* tmp, F f) {
  for (int base = part.lo; base < part.hi && before < want; base += kThreads) {
    const int p = base + threadIdx.x;
    const bool is = p < part.hi && free_page(refs, p);
    unsigned long long total;
    const int rank = before + (int)block_scan(is, tmp, total) - 1;
    if (is && rank < want) f(rank, p);
    before += (int)total;
  }
}

__global__ void __launch_bounds__(kThreads) paged_reserve(ReserveP p) {
  extern __shared__ int sm[];
  int* off = sm;               // wanted pages before each sequence [B + 1]
  int* cu = off + p.B + 1;     // new tokens before it [B + 1]
  int* col = cu + p.B + 1;     // its first new column [B]
  __shared__ unsigned long long tmp[32];
  __shared__ int count;
  cg::cluster_group cl = cg::this_cluster();
  const unsigned rank = cl.block_rank();
  const long long cap = (long long)p.M * p.page;
  unsigned long long carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int want = 0, n = 0, have = 0;
    if (b < p.B) {
      const int t = p.lengths[b];
      if (t >= 0) {
        n = p.tokens ? max(0, p.tokens[b]) : 1;
        if (n > 0x7fffffff / p.B) {  // the sums are held in 31 bits
          atomicCAS(p.err, 0, kErrPaged | 1);
          n = 0;
        }
        have = (int)min((long long)p.M, ((long long)t + p.page - 1) / p.page);
        const int need = n ? (int)min((long long)p.M, ((long long)t + n + p.page - 1) / p.page) : have;
        while (have < need && (unsigned)__ldcg(p.table + b * p.ts + have) < (unsigned)p.P) ++have;
        want = need - have;
      }
    }
    unsigned long long total;
    const unsigned long long v = (unsigned long long)(unsigned)want << 32 | (unsigned)n;
    const unsigned long long before = carry + block_scan(v, tmp, total) - v;
    if (b < p.B) {
      off[b] = (int)(before >> 32);
      cu[b] = (int)(unsigned)before;
      col[b] = have;
    }
    carry += total;
  }
  const int want = (int)(carry >> 32), rows = (int)(unsigned)carry;
  if (threadIdx.x == 0) {
    off[p.B] = want;
    cu[p.B] = rows;
  }
  __syncthreads();
  if (rank == 0)
    for (int b = threadIdx.x; b <= p.B; b += kThreads) p.cu[b] = cu[b];
  int before = 0, all = 0;
  if (want) {
    const Part part(p.P, rank, cl.num_blocks());
    count_free(p.refs, part, &count, tmp, before, all);  // every block has read the table by now
    if (want <= all)
      give(p.refs, part, before, want, tmp, [&](int i, int page) {
        const int b = find(off, p.B, i);
        p.table[b * p.ts + col[b] + i - off[b]] = page;
        p.refs[page] = 1;
      });
    cl.sync();  // the table is whole, and no block's count is read any more
  }
  if (rank == 0 && threadIdx.x == 0) *p.missing = max(0, want - all);
  for (long long i = (long long)rank * kThreads + threadIdx.x; i < p.rows; i += (long long)cl.num_blocks() * kThreads) {
    int b = -1, at = -1, slot = -1;
    if (i < rows) {
      b = find(cu, p.B, (int)i);
      const long long t = (long long)p.lengths[b] + (i - cu[b]), end = (long long)p.lengths[b] + (cu[b + 1] - cu[b]);
      at = (int)t;
      if (t >= end - cap) {
        const int s = (int)(t % cap), j = s / p.page, page = __ldcg(p.table + b * p.ts + j);
        if ((unsigned)page < (unsigned)p.P) slot = page * p.page + (s - j * p.page);
      }
    }
    p.seq[i] = b;
    p.pos[i] = at;
    p.slot[i] = slot;
  }
}

// A row's full and used columns.
struct Used {
  int full, held;
  __device__ Used(const ForkP& p, int t) {
    full = p.share && t > 0 ? (int)min((long long)p.M, (long long)t / p.page) : 0;
    held = t > 0 ? (int)min((long long)p.M, ((long long)t + p.page - 1) / p.page) : 0;
  }
};
__device__ __forceinline__ int parent_of(const ForkP& p, int r) {
  const int x = p.parents[r];
  return (unsigned)x < (unsigned)p.B ? x : -1;
}

__global__ void __launch_bounds__(kThreads) paged_fork(ForkP p, int tile) {
  extern __shared__ int sm[];
  int* children = sm;             // of each row [B]
  int* eldest = children + p.B;   // the first of them [B]
  int* off = eldest + p.B;        // pages wanted before each new row [B + 1]
  int* old = off + p.B + 1;       // `tile` columns of the table [B][tile]
  __shared__ unsigned long long tmp[32];
  __shared__ int count;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), blocks = (int)cl.num_blocks();
  for (int r = threadIdx.x; r < p.B; r += kThreads) {
    children[r] = 0;
    eldest[r] = p.B;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < p.B; r += kThreads) {
    const int x = parent_of(p, r);
    if (x >= 0) {
      atomicAdd(children + x, 1);
      atomicMin(eldest + x, r);
    } else if (p.parents[r] >= 0) {
      atomicCAS(p.err, 0, kErrPaged | 1);
    }
    if (p.share && p.lengths[r] > (long long)p.M * p.page) atomicCAS(p.err, 0, kErrPaged | 1);
  }
  __syncthreads();
  unsigned long long carry = 0;
  for (int r0 = 0; r0 < p.B; r0 += kThreads) {
    const int r = r0 + threadIdx.x;
    unsigned need = 0;
    if (r < p.B) {
      const int x = parent_of(p, r);
      if (x >= 0 && eldest[x] != r) {
        const Used u(p, p.lengths[x]);
        need = u.held - u.full;
      }
    }
    unsigned long long total;
    const unsigned long long before = carry + block_scan(need, tmp, total) - need;
    if (r < p.B) off[r] = (int)before;
    carry += total;
  }
  const int want = (int)carry;
  if (threadIdx.x == 0) off[p.B] = want;
  const long long n_copies = (long long)p.B * (p.share ? 1 : p.M);
  for (long long i = (long long)rank * kThreads + threadIdx.x; i < n_copies; i += (long long)blocks * kThreads)
    reinterpret_cast<int2*>(p.copies)[i] = make_int2(-1, -1);
  // whole columns at a time: their old entries are read before any is written
  for (int c0 = rank * tile; c0 < p.M; c0 += blocks * tile) {
    __syncthreads();
    const int w = min(tile, p.M - c0);
    for (int i = threadIdx.x; i < p.B * w; i += kThreads) {
      const int r = i / w, j = i - r * w;
      old[r * tile + j] = __ldcg(p.table + r * p.ts + c0 + j);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.B * w; i += kThreads) {
      const int r = i / w, j = i - r * w, c = c0 + j, x = parent_of(p, r);
      int page = -1;
      if (x >= 0 && (eldest[x] == r || c < Used(p, p.lengths[x]).full)) page = old[x * tile + j];
      p.table[r * p.ts + c] = page;
      // what the old row gives up, or its further children take
      const int was = old[r * tile + j], n = children[r];
      if ((unsigned)was < (unsigned)p.P) {
        const int d = (c < Used(p, p.lengths[r]).full ? n : min(n, 1)) - 1;
        if (d) atomicAdd(p.refs + was, d);
      }
    }
  }
  cl.sync();
  int before = 0, all = 0;
  if (want) {
    const Part part(p.P, rank, blocks);
    count_free(p.refs, part, &count, tmp, before, all);
    give(p.refs, part, before, want, tmp, [&](int i, int page) {
      const int r = find(off, p.B, i), x = p.parents[r], k = i - off[r];
      const int c = Used(p, p.lengths[x]).full + k;
      const int from = __ldcg(p.table + eldest[x] * p.ts + c);
      p.table[r * p.ts + c] = page;
      p.refs[page] = 1;
      if ((unsigned)from < (unsigned)p.P)
        reinterpret_cast<int2*>(p.copies)[p.share ? r : (long long)r * p.M + c] = make_int2(from, page);
    });
    cl.sync();  // no block's count is read any more
  }
  if (rank == 0 && threadIdx.x == 0) *p.missing = max(0, want - all);
}

constexpr int kCopyThreads = 256;
template <typename T>
__device__ __forceinline__ void copy_page(const char* from, char* to, long long bytes) {
  const T* a = reinterpret_cast<const T*>(from);
  T* b = reinterpret_cast<T*>(to);
  for (long long i = threadIdx.x; i < bytes / (long long)sizeof(T); i += kCopyThreads) b[i] = a[i];
}
__global__ void __launch_bounds__(kCopyThreads) paged_copy(const __grid_constant__ CopyP p) {
  const int2 c = __ldg(reinterpret_cast<const int2*>(p.copies) + blockIdx.x);
  if ((unsigned)c.x >= (unsigned)p.P || (unsigned)c.y >= (unsigned)p.P || c.x == c.y) return;
  char* pool = p.pool[blockIdx.y];
  const long long bytes = p.bytes[blockIdx.y];
  const char* from = pool + (long long)c.x * bytes;
  char* to = pool + (long long)c.y * bytes;
  if (!((reinterpret_cast<uintptr_t>(pool) | bytes) & 15)) copy_page<uint4>(from, to, bytes);
  else copy_page<char>(from, to, bytes);
}

template <typename K, typename P, typename... A>
cudaError_t launch_cluster(K kern, int blocks, size_t smem, cudaStream_t st, const P& p, A... a) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, a...);
}

}  // namespace

cudaError_t launch_paged_reserve(const ReserveP& p, cudaStream_t st) {
  return launch_cluster(paged_reserve, 8, (size_t)(3 * p.B + 2) * sizeof(int), st, p);
}

cudaError_t launch_paged_fork(const ForkP& p, cudaStream_t st) {
  // a sector's worth of columns, fewer where the rows are many
  const int tile = p.B <= 2048 ? 8 : 2;
  return launch_cluster(paged_fork, 8, ((size_t)3 * p.B + 1 + (size_t)p.B * tile) * sizeof(int), st, p, tile);
}

cudaError_t launch_paged_copy(const CopyP& p, int pools, long long n, cudaStream_t st) {
  paged_copy<<<dim3((unsigned)n, (unsigned)pools), kCopyThreads, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace bozo
