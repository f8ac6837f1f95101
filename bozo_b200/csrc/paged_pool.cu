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
// One block does without the cluster's barrier; eight count the pages faster.  In a graph, µs,
// one | eight, 4 and 64 sequences that all need a page: 1024 pages 4.4, 5.0 | 6.3, 6.9; 8192
// 5.4, 7.4 | 6.4, 7.4; 16000 5.8, 9.8 | 6.7, 7.9; 64000 12.1, 29.3 | 7.6, 9.0.
constexpr int kReservePool = 8192;
// A fork has the table to move as well, every second row a copy: 32 × 64 entries over 2400
// pages 6.9 | 7.8, over 16000 7.7 | 8.2, over 64000 13.4 | 8.4; 64 × 64 over 16000 8.6 | 8.2
// (5.5 | 4.1 where nothing forks), 128 × 64 11.6 | 9.2.
constexpr int kForkPool = 16384, kForkTable = 2048;
// Rows whose places the cluster's first kernel writes itself; a second kernel has all SMs but
// has to start: 1024 rows 4.1 | 6.1, 2048 5.2 | 6.5, 4096 7.4 | 7.1, 16384 21.2 | 10.4.
constexpr int kPlacesHere = 4096;

// Sums over the block's threads, one barrier each: every warp adds the warps' totals up
// for itself, and two buffers take turns, so that none is written while it is read.
struct Scan {
  unsigned long long tmp[2][32];
  // v's inclusive sum; `total`: of all threads.  `turn`: the same count in every thread.
  __device__ __forceinline__ unsigned long long run(unsigned long long v, unsigned long long& total, int& turn) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long* t = tmp[turn++ & 1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) t[warp] = v;
    __syncthreads();
    unsigned long long w = t[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const unsigned long long before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return warp ? v + before : v;
  }
};

// The last i in [0, n) with sums[i] ≤ x (sums[0] ≤ x, non-decreasing).
__device__ __forceinline__ int find(const int* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// The pool is shared out in order: a run of consecutive pages a warp, in words of 32 that
// all its lanes read together.
struct Run {
  unsigned from, to, words;  // pages past 2^31 − 32 would pass an int's range in a loop's last step
  __device__ Run(int pages, unsigned rank, unsigned blocks) {
    const long long warps = (long long)blocks * (kThreads / 32), warp = (long long)rank * (kThreads / 32) + (threadIdx.x >> 5);
    words = (unsigned)((pages + warps * 32 - 1) / (warps * 32));
    from = (unsigned)min((long long)pages, warp * words * 32);
    to = (unsigned)min((long long)pages, from + (long long)words * 32);
  }
  __device__ unsigned word(const int* refs, unsigned p) const {
    const unsigned lane = threadIdx.x & 31;
    return __ballot_sync(0xffffffffu, p + lane < to && refs[p + lane] == 0);
  }
  // the warp's free pages; `mask`: which of word `lane` are
  __device__ int count(const int* refs, unsigned& mask) const {
    int n = 0, i = 0;
    mask = 0;
#pragma unroll 8
    for (unsigned p = from; p < to; p += 32, ++i) {
      const unsigned b = word(refs, p);
      n += __popc(b);
      if (i == (int)(threadIdx.x & 31)) mask = b;
    }
    return n;
  }
  // f(rank, page) for its free pages of rank < want, the first of which has rank `before`
  template <typename F>
  __device__ void give(const int* refs, unsigned mask, int n, int before, int want, F f) const {
    const int lane = threadIdx.x & 31;
    if (n == 0) return;
    int i = 0;
    for (unsigned p = from; p < to && before < want; p += 32, ++i) {
      const unsigned b = i < 32 ? __shfl_sync(0xffffffffu, mask, i) : word(refs, p);
      const int rank = before + __popc(b & ((1u << lane) - 1u));
      if (b >> lane & 1 && rank < want) f(rank, (int)(p + lane));
      before += __popc(b);
    }
  }
};

// From each warp's free pages, those before its own and in all; `count`: one word of
// shared memory.  With more than one block the cluster is synchronised in between.
__device__ __forceinline__ void scan_free(int mine, int* count, Scan& scan, int& turn, int& before, int& all) {
  cg::cluster_group cl = cg::this_cluster();
  unsigned long long total;
  before = (int)scan.run((threadIdx.x & 31) == 0 ? mine : 0, total, turn) - mine;
  all = (int)total;
  if (cl.num_blocks() > 1) {
    if (threadIdx.x == 0) *count = all;
    cl.sync();
    all = 0;
    for (unsigned r = 0; r < cl.num_blocks(); ++r) {
      const int c = *cl.map_shared_rank(count, r);
      if (r < cl.block_rank()) before += c;
      all += c;
    }
  }
}
__device__ __forceinline__ void sync_all() {
  cg::cluster_group cl = cg::this_cluster();
  if (cl.num_blocks() > 1) cl.sync();
  else __syncthreads();
}

// Where row i of the packed new tokens goes: sequence b, which has the rows [first, next).
__device__ __forceinline__ void place(const ReserveP& p, int i, int b, int len, int first, int next, int& at, int& slot) {
  const long long t = len, pos = t + (i - first), end = min(t + (next - first), 1LL << 31);
  at = pos < end ? (int)pos : -1;  // positions end at 2^31 − 1
  slot = -1;
  if (pos < end - (long long)p.cap || pos >= end) return;
  const unsigned s = (unsigned)pos - fast_div((unsigned)pos, p.div_cap) * p.cap, j = fast_div(s, p.div_page);
  const int page = __ldcg(p.table + b * p.ts + j);
  if ((unsigned)page < (unsigned)p.P) slot = page * p.page + (int)(s - j * p.page);
}

// Columns that t < 2^32 tokens fill.
__device__ __forceinline__ int pages_of(const ReserveP& p, unsigned t) {
  const unsigned whole = fast_div(t, p.div_page);
  return (int)min((unsigned)p.M, whole + (whole * (unsigned)p.page < t));
}

__global__ void __launch_bounds__(kThreads) paged_reserve(ReserveP p, bool places) {
  extern __shared__ int sm[];
  int* off = sm;               // wanted pages before each sequence [B + 1]
  int* cu = off + p.B + 1;     // new tokens before it [B + 1]
  int* col = cu + p.B + 1;     // its first new column [B]
  int* len = col + p.B;        // the tokens it holds [B]
  __shared__ Scan scan;
  int turn = 0;
  __shared__ int count;
  cg::cluster_group cl = cg::this_cluster();
  const unsigned rank = cl.block_rank();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the places' kernel, which waits for this one
  const Run run(p.P, rank, cl.num_blocks());
  unsigned mask;
  const int mine = run.count(p.refs, mask);
  unsigned long long carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int want = 0, n = 0, have = 0;
    if (b < p.B) {
      const int t = p.lengths[b];
      n = p.tokens ? max(0, p.tokens[b]) : 1;
      len[b] = t;
      if (t < 0) n = 0;
      if (n > 0x7fffffff / p.B) {  // the sums are held in 31 bits
        atomicCAS(p.err, 0, kErrPaged | 1);
        n = 0;
      }
      if (n && (unsigned)t + (unsigned)n > 0x80000000u) atomicCAS(p.err, 0, kErrPaged | 1);
      if (n) {
        have = pages_of(p, t);
        const int need = pages_of(p, (unsigned)t + (unsigned)n);
        while (have < need && (unsigned)__ldcg(p.table + b * p.ts + have) < (unsigned)p.P) ++have;
        want = need - have;
      }
    }
    unsigned long long total;
    const unsigned long long v = (unsigned long long)(unsigned)want << 32 | (unsigned)n;
    const unsigned long long before = carry + scan.run(v, total, turn) - v;
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
    scan_free(mine, &count, scan, turn, before, all);  // every block has read the table by now
    if (want <= all)
      run.give(p.refs, mask, mine, before, want, [&](int i, int page) {
        const int b = find(off, p.B, i);
        p.table[b * p.ts + col[b] + i - off[b]] = page;
        p.refs[page] = 1;
      });
    sync_all();  // the table is whole, and no block's count is read any more
  }
  if (rank == 0 && threadIdx.x == 0) *p.missing = max(0, want - all);
  if (!places) return;
  for (long long i = (long long)rank * kThreads + threadIdx.x; i < p.rows; i += (long long)cl.num_blocks() * kThreads) {
    int b = -1, at = -1, slot = -1;
    if (i < rows) {
      b = find(cu, p.B, (int)i);
      place(p, (int)i, b, len[b], cu[b], cu[b + 1], at, slot);
    }
    p.seq[i] = b;
    p.pos[i] = at;
    p.slot[i] = slot;
  }
}

// The places of many rows, four a thread.
constexpr int kPlaceThreads = 256;
__global__ void __launch_bounds__(kPlaceThreads) paged_places(ReserveP p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long i0 = ((long long)blockIdx.x * kPlaceThreads + threadIdx.x) * 4;
  if (i0 >= p.rows) return;
  const int rows = __ldcg(p.cu + p.B);
  int lo = 0, hi = p.B;  // the last b with cu[b] ≤ i0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid] <= i0) lo = mid; else hi = mid;
  }
  int b = lo, first = p.cu[b], next = p.cu[b + 1];
  int seq[4], at[4], slot[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const long long i = i0 + k;
    seq[k] = at[k] = slot[k] = -1;
    if (i >= rows) continue;
    while (i >= next) {
      ++b;
      first = next;
      next = p.cu[b + 1];
    }
    seq[k] = b;
    place(p, (int)i, b, p.lengths[b], first, next, at[k], slot[k]);
  }
  if (i0 + 4 <= p.rows && !((reinterpret_cast<uintptr_t>(p.seq) | reinterpret_cast<uintptr_t>(p.pos) | reinterpret_cast<uintptr_t>(p.slot)) & 15)) {
    reinterpret_cast<int4*>(p.seq + i0)[0] = make_int4(seq[0], seq[1], seq[2], seq[3]);
    reinterpret_cast<int4*>(p.pos + i0)[0] = make_int4(at[0], at[1], at[2], at[3]);
    reinterpret_cast<int4*>(p.slot + i0)[0] = make_int4(slot[0], slot[1], slot[2], slot[3]);
    return;
  }
  for (int k = 0; k < 4 && i0 + k < p.rows; ++k) {
    p.seq[i0 + k] = seq[k];
    p.pos[i0 + k] = at[k];
    p.slot[i0 + k] = slot[k];
  }
}

__global__ void __launch_bounds__(kThreads) paged_fork(ForkP p, int tile, FastDiv div_tile) {
  extern __shared__ int sm[];
  int* parent = sm;               // of each new row, −1 for none [B]
  int* children = parent + p.B;   // of each old row [B]
  int* eldest = children + p.B;   // the first of them [B]
  int* full = eldest + p.B;       // its columns that its children share [B],
  int* held = full + p.B;         // and those in use [B]
  int* off = held + p.B;          // pages wanted before each new row [B + 1]
  int* old = off + p.B + 1;       // `tile` columns of the table [B][tile]
  __shared__ Scan scan;
  int turn = 0;
  __shared__ int count;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), blocks = (int)cl.num_blocks();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the copies' kernel, which waits for this one
  // the old entries of columns c0 …: thread i has every kThreads-th of a tile's B · tile
  auto load = [&](unsigned c0) {
#pragma unroll 4
    for (int i = threadIdx.x; i < p.B * tile; i += kThreads) {
      const int r = (int)fast_div((unsigned)i, div_tile);
      const unsigned c = c0 + (unsigned)(i - r * tile);
      old[i] = c < (unsigned)p.M ? __ldcg(p.table + r * p.ts + c) : -1;
    }
  };
  const int x0 = (int)threadIdx.x < p.B ? p.parents[threadIdx.x] : 0, t0 = (int)threadIdx.x < p.B ? p.lengths[threadIdx.x] : 0;
  load(rank * tile);
  for (int r = threadIdx.x; r < p.B; r += kThreads) {
    const int x = r < kThreads ? x0 : p.parents[r], t = r < kThreads ? t0 : p.lengths[r];
    parent[r] = (unsigned)x < (unsigned)p.B ? x : -1;
    children[r] = 0;
    eldest[r] = p.B;
    const int whole = t > 0 ? (int)fast_div((unsigned)t, p.div_page) : 0;
    full[r] = p.share ? min(p.M, whole) : 0;
    held[r] = min(p.M, whole + (t > whole * p.page));
    if (x >= p.B || (p.share && t > (long long)p.M * p.page)) atomicCAS(p.err, 0, kErrPaged | 1);
  }
  __syncthreads();
  for (int r = threadIdx.x; r < p.B; r += kThreads) {
    const int x = parent[r];
    if (x < 0) continue;
    atomicAdd(children + x, 1);
    atomicMin(eldest + x, r);
  }
  const long long n_copies = (long long)p.B * (p.share ? 1 : p.M);
  for (long long i = (long long)rank * kThreads + threadIdx.x; i < n_copies; i += (long long)blocks * kThreads)
    reinterpret_cast<int2*>(p.copies)[i] = make_int2(-1, -1);
  __syncthreads();
  unsigned long long carry = 0;
  for (int r0 = 0; r0 < p.B; r0 += kThreads) {
    const int r = r0 + threadIdx.x;
    unsigned need = 0;
    if (r < p.B) {
      const int x = parent[r];
      if (x >= 0 && eldest[x] != r) need = held[x] - full[x];
    }
    unsigned long long total;
    const unsigned long long before = carry + scan.run(need, total, turn) - need;
    if (r < p.B) off[r] = (int)before;
    carry += total;
  }
  const int want = (int)carry;
  if (threadIdx.x == 0) off[p.B] = want;
  // whole columns at a time: their old entries are read before any is written
  for (unsigned c0 = (unsigned)(rank * tile); c0 < (unsigned)p.M; c0 += (unsigned)(blocks * tile)) {
    if (c0 != (unsigned)(rank * tile)) {
      __syncthreads();
      load(c0);
      __syncthreads();
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < p.B * tile; i += kThreads) {
      const int r = (int)fast_div((unsigned)i, div_tile), j = i - r * tile, x = parent[r];
      if (c0 + (unsigned)j >= (unsigned)p.M) continue;
      const int c = (int)(c0 + (unsigned)j);
      p.table[r * p.ts + c] = x >= 0 && (eldest[x] == r || c < full[x]) ? old[x * tile + j] : -1;
      // what the old row gives up, or its further children take
      const int was = old[i], n = children[r], d = (c < full[r] ? n : min(n, 1)) - 1;
      if (d && (unsigned)was < (unsigned)p.P) atomicAdd(p.refs + was, d);
    }
  }
  sync_all();
  int before = 0, all = 0;
  if (want) {
    const Run run(p.P, rank, blocks);
    unsigned mask;
    const int mine = run.count(p.refs, mask);
    scan_free(mine, &count, scan, turn, before, all);
    run.give(p.refs, mask, mine, before, want, [&](int i, int page) {
      const int r = find(off, p.B, i), x = parent[r], c = full[x] + i - off[r];
      const int from = blocks == 1 ? old[x * tile + c] : __ldcg(p.table + eldest[x] * p.ts + c);
      p.table[r * p.ts + c] = page;
      p.refs[page] = 1;
      if ((unsigned)from < (unsigned)p.P)
        reinterpret_cast<int2*>(p.copies)[p.share ? r : (long long)r * p.M + c] = make_int2(from, page);
    });
    if (blocks > 1) cl.sync();  // no block's count is read any more
  }
  if (rank == 0 && threadIdx.x == 0) *p.missing = max(0, want - all);
}

constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = kCopyThreads * 16 * 4;  // of a page, by one block
__global__ void __launch_bounds__(kCopyThreads) paged_copy(const __grid_constant__ CopyP p) {
  const long long bytes = p.bytes[blockIdx.y], lo = (long long)blockIdx.z * kCopyBytes;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (lo >= bytes) return;
  const int2 c = __ldcg(reinterpret_cast<const int2*>(p.copies) + blockIdx.x);
  if ((unsigned)c.x >= (unsigned)p.P || (unsigned)c.y >= (unsigned)p.P || c.x == c.y) return;
  const char* from = p.pool[blockIdx.y] + (long long)c.x * bytes;
  char* to = p.pool[blockIdx.y] + (long long)c.y * bytes;
  const long long hi = blockIdx.z + 1 == gridDim.z ? bytes : min(bytes, lo + kCopyBytes);
  if ((reinterpret_cast<uintptr_t>(p.pool[blockIdx.y]) | bytes) & 15) {
    for (long long i = lo + threadIdx.x; i < hi; i += kCopyThreads) to[i] = from[i];
    return;
  }
  for (long long i0 = lo + threadIdx.x * 16; i0 < hi; i0 += kCopyBytes) {
    uint4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j * kCopyThreads * 16 < hi) x[j] = *reinterpret_cast<const uint4*>(from + i0 + j * kCopyThreads * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j * kCopyThreads * 16 < hi) *reinterpret_cast<uint4*>(to + i0 + j * kCopyThreads * 16) = x[j];
  }
}

template <auto kern, typename P, typename... A>
cudaError_t launch_cluster(int blocks, size_t smem, cudaStream_t st, const P& p, A... a) {
  if (smem > 48 * 1024) {
    const cudaError_t e = allow_shared<kern>();
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

// A kernel that may be launched before the one ahead of it is done, which it waits for.
template <typename P>
cudaError_t launch_after(void (*kern)(P), dim3 grid, int threads, cudaStream_t st, const P& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

cudaError_t launch_paged_reserve(const ReserveP& p, cudaStream_t st, int* launches) {
  const int blocks = p.P <= kReservePool ? 1 : 8;
  const bool here = p.rows <= kPlacesHere;
  cudaError_t e = launch_cluster<paged_reserve>(blocks, (size_t)(4 * p.B + 2) * sizeof(int), st, p, here);
  *launches = here ? 1 : 2;
  if (e != cudaSuccess || here) return e;
  return launch_after(paged_places, dim3((unsigned)((p.rows + 4 * kPlaceThreads - 1) / (4 * kPlaceThreads))),
                      kPlaceThreads, st, p);
}

cudaError_t launch_paged_fork(const ForkP& p, cudaStream_t st) {
  // small tables: one block, whole; else a sector's worth of columns, fewer where the rows are many
  const bool small = p.P <= kForkPool && (long long)p.B * p.M <= kForkTable;
  const int tile = small ? p.M : p.B <= 2048 ? 8 : p.B <= 4096 ? 2 : 1;
  return launch_cluster<paged_fork>(small ? 1 : 8, ((size_t)6 * p.B + 1 + (size_t)p.B * tile) * sizeof(int), st, p, tile,
                        make_fastdiv((unsigned)tile));
}

cudaError_t launch_paged_copy(const CopyP& p, int pools, long long n, cudaStream_t st) {
  long long most = 0;
  for (int i = 0; i < pools; ++i) most = p.bytes[i] > most ? p.bytes[i] : most;
  const long long parts = (most + kCopyBytes - 1) / kCopyBytes;
  return launch_after(paged_copy, dim3((unsigned)n, (unsigned)pools, (unsigned)(parts < 65535 ? parts : 65535)),
                      kCopyThreads, st, p);
}

}  // namespace bozo
