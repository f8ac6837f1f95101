// beam.cu — the best continuations of a beam search's hypotheses (bozo_beam_select).
//
// A continuation is worth score + logit − log Σ exp(logits); within one row the logits
// alone order them.  One cluster a prompt, each block a row, a part of one, or (more
// than kCluster hypotheses) a few rows, and one pass over the logits:
//   * a tile of a row in registers: its largest value and Σ exp(x − largest);
//   * its K best: the K-th largest of 64 groups' maxima is a bound that at least K
//     elements reach, and for unequal logits few more, so that only those are compared
//     with one another (many equal ones: the best are taken out one after the other);
//   * every block's K best keys and sum go to the first block's shared memory, which
//     finds the prompt's best among them in 64 bits.
// Bound by the logits' bytes where rows are many, by the chain of these steps where
// they are few.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "beam.cuh"

namespace bozo {
namespace {

namespace cg = cooperative_groups;
using Key = unsigned long long;
constexpr int kThreads = 512, kWarps = kThreads / 32, kGroups = 64, kCluster = 8;
constexpr int kList = 512;  // elements that reach the bound, at most, before equal ones get a way of their own

// Larger keys come first: the logit, then the lower token.
__device__ __forceinline__ Key key_of(float x, unsigned token) {
  const unsigned u = __float_as_uint(x + 0.f);  // −0 is 0
  const unsigned o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (Key)o << 32 | (unsigned)~token;
}
__device__ __forceinline__ unsigned token_of(Key k) { return ~(unsigned)k; }
__device__ __forceinline__ float logit_of(Key k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }
// What a sum relative to m is worth relative to `to` ≥ m; a sum of nothing nothing (a NaN stays one).
__device__ __forceinline__ float rescale(float m, float to) { return m == -INFINITY ? 0.f : pow2((m - to) * kLog2e); }

// 16 bytes of logits.
template <int DT> struct Vec {
  static constexpr int N = DT == BOZO_DT_F32 ? 4 : 8;
  static constexpr unsigned none = DT == BOZO_DT_F32 ? 0xff800000u : DT == BOZO_DT_BF16 ? 0xff80ff80u : 0xfc00fc00u;
  unsigned w[4];
  __device__ __forceinline__ float at(int i) const {
    if constexpr (DT == BOZO_DT_F32) return __uint_as_float(w[i]);
    else if constexpr (DT == BOZO_DT_BF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
  }
  __device__ __forceinline__ float most() const {
    if constexpr (DT == BOZO_DT_F32) {
      return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3)));
    } else if constexpr (DT == BOZO_DT_BF16) {
      __nv_bfloat162 h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
      const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      __half2 h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __half2*>(&w[i]);
      const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
};

// A row's logits in pieces of 16 bytes from its first token on, so that equal rows are
// summed alike wherever they lie.  Where a row is not aligned a piece is put together from
// two that are (the second is the neighbour's first, out of the L1).
template <int DT> struct Row {
  const char* at;
  int off, V, pieces;  // bytes from a multiple of 16
  static constexpr int N = Vec<DT>::N, size = 16 / N;
  __device__ __forceinline__ Row(const BeamP& p, int row) {
    at = static_cast<const char*>(p.logits) + (long long)row * p.stride * size;
    off = (int)(reinterpret_cast<uintptr_t>(at) & 15);
    V = p.V;
    pieces = (V + N - 1) / N;
  }
  __device__ __forceinline__ Vec<DT> load(int q, int end) const {
    Vec<DT> v;
    const int f = q * N;
    if (off == 0 ? q < end && f + N <= V : q < end && q > 0 && f + 2 * N <= V) {
      const uint4* from = reinterpret_cast<const uint4*>(at - off) + q;
      const uint4 x = __ldg(from);
      v.w[0] = x.x; v.w[1] = x.y; v.w[2] = x.z; v.w[3] = x.w;
      if (off) {
        const uint4 y = __ldg(from + 1);
        unsigned u[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        if (off & 8) {
#pragma unroll
          for (int i = 0; i < 6; ++i) u[i] = u[i + 2];
        }
        if (off & 4) {
#pragma unroll
          for (int i = 0; i < 5; ++i) u[i] = u[i + 1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v.w[i] = __funnelshift_r(u[i], u[i + 1], 8 * (off & 3));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v.w[i] = Vec<DT>::none;
      if (q < end) {  // the ends of a row
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (f + i >= V) continue;
          if constexpr (DT == BOZO_DT_F32) {
            v.w[i] = __ldg(reinterpret_cast<const unsigned*>(at) + f + i);
          } else {
            const unsigned x = __ldg(reinterpret_cast<const unsigned short*>(at) + f + i);
            v.w[i / 2] = i & 1 ? (v.w[i / 2] & 0xffffu) | x << 16 : (v.w[i / 2] & 0xffff0000u) | x;
          }
        }
      }
    }
    return v;
  }
};

struct Best {  // one list in the first block's shared memory: K keys, then
  float m, s;  // its part's largest logit and Σ exp(logit − largest)
};

// Items in order: value, then the lower hypothesis, then the key.
struct Item {
  double value;
  Key key;
  int beam;
};
__device__ __forceinline__ bool ahead(const Item& a, const Item& b) {
  if (a.value != b.value) return a.value > b.value;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}

struct Scratch {
  float top[kGroups], wm[kWarps], ws[kWarps];
  Key list[kList + 32], cur[32], wbest[kWarps];
  float bound;
  int n;
};

// The K best of pieces [q0, q1) of a row, sorted, into sc.cur, and its largest logit and sum.
template <int DT, int NV>
__device__ __forceinline__ void scan(const Row<DT>& row, int q0, int q1, int K, Scratch& sc, float& M, float& S) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int N = Vec<DT>::N;
  float m = -INFINITY, s = 0.f;  // this thread's, over all tiles
  for (int base = q0; base < q1; base += NV * kThreads) {
    Vec<DT> v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = row.load(base + j * kThreads + tid, q1);
    float t = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) t = fmaxf(t, v[j].most());
    const float to = fmaxf(m, t), ref = finite_or_0(to);
    s *= rescale(m, to);
    m = to;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float e[N];
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = pow2((v[j].at(i) - ref) * kLog2e);
#pragma unroll
      for (int o = N / 2; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; ++i) e[i] += e[i + o];
      s += e[0];
    }
    float g = t;
#pragma unroll
    for (int o = 1; o < kThreads / kGroups; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % (kThreads / kGroups) == 0) sc.top[tid / (kThreads / kGroups)] = g;
    const bool more = base != q0;  // the best of the tiles before are in cur
    if (tid == 0) sc.n = more ? K : 0;
    if (more && tid < K) sc.list[tid] = sc.cur[tid];
    __syncthreads();
    // the K-th largest group: each warp ranks its share of them
    const float a = sc.top[lane], b = sc.top[lane + 32];
#pragma unroll
    for (int i = 0; i < kGroups / kWarps; ++i) {
      const int me = warp * (kGroups / kWarps) + i;
      const float x = __shfl_sync(0xffffffffu, me < 32 ? a : b, me & 31);
      const int r = __popc(__ballot_sync(0xffffffffu, a > x || (a == x && lane < me))) +
                    __popc(__ballot_sync(0xffffffffu, b > x || (b == x && lane + 32 < me)));
      if (r == K - 1 && lane == 0) sc.bound = x;
    }
    __syncthreads();
    const float bound = sc.bound;
    // tokens before this tile's were lower: an equal key of theirs comes first by itself
    if (t >= bound) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int q = base + j * kThreads + tid, f = q * N;
        if (v[j].most() < bound || q >= q1) continue;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float x = v[j].at(i);
          if (x >= bound && f + i < row.V) {
            const int at = atomicAdd(&sc.n, 1);
            if (at < kList + 32) sc.list[at] = key_of(x, f + i);
          }
        }
      }
    }
    __syncthreads();
    const int n = sc.n;
    if (n <= kList + 32) {
      // each warp ranks its share of what reached the bound
      for (int i = warp; i < n; i += kWarps) {
        const Key x = sc.list[i];
        int r = 0;
        for (int j = lane; j - lane < n; j += 32) r += __popc(__ballot_sync(0xffffffffu, j < n && sc.list[j] > x));
        if (lane == 0 && r < K) sc.cur[r] = x;
      }
      if (n < K && tid >= n && tid < K) sc.cur[tid] = 0;  // a row with fewer tokens so far
      __syncthreads();
    } else {
      // many equal logits: the largest key below the last, K times
      Key last = ~0ull, mine = more && tid < K ? sc.cur[tid] : 0;
      __syncthreads();
      for (int k = 0; k < K; ++k) {
        Key best = mine < last ? mine : 0;
#pragma unroll 1
        for (int q = base + tid; q < min(q1, base + NV * kThreads); q += kThreads) {
          const Vec<DT> u = row.load(q, q1);
          const int f = q * N;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const Key x = key_of(u.at(i), f + i);
            if (f + i < row.V && x < last && x > best) best = x;
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) sc.wbest[warp] = best;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) best = max(best, sc.wbest[w]);
        if (tid == 0) sc.cur[k] = best;
        last = best;
        __syncthreads();
      }
    }
  }
  float wm = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
  s = warp_sum(s * rescale(m, wm));
  if (lane == 0) {
    sc.wm[warp] = wm;
    sc.ws[warp] = s;
  }
  __syncthreads();
  M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sc.wm[w]);
  S = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) S += sc.ws[w] * rescale(sc.wm[w], M);
}

// Parts of a row and blocks of a cluster: parts · K blocks, or (K > kCluster) blocks that
// take every so many-th row.
template <int DT, int NV>
__global__ void __launch_bounds__(kThreads) beam_select(BeamP p, int parts) {
  __shared__ Scratch sc;
  // of the first block: every list, and what is left of them
  __shared__ Key keys[32 * 32];
  __shared__ Best sums[32];
  __shared__ Item kept[32 * 32];
  __shared__ Item heads[32], limit;
  __shared__ double lse[32];
  __shared__ int kind[32], n;  // 0: scanned, 1: ended, 2: nothing but −infinity
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), blocks = (int)cl.num_blocks();
  const int prompt = blockIdx.x / blocks, K = p.K, L = K * parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (blocks > 1) cl.sync();  // the first block is there
  for (int list = rank; list < L; list += blocks) {
    const int r = prompt * K + list / parts;
    if (!isfinite(p.scores[r]) || (p.done && p.done[r])) continue;
    const Row<DT> row(p, r);
    const int each = (row.pieces + parts - 1) / parts, q0 = min(row.pieces, each * (list % parts));
    float M, S;
    if (tid < K) sc.cur[tid] = 0;  // a part without a piece
    __syncthreads();
    scan<DT, NV>(row, q0, min(row.pieces, q0 + each), K, sc, M, S);
    Key* to = cl.map_shared_rank(keys, 0) + list * K;
    if (tid < K) to[tid] = sc.cur[tid];
    if (tid == 0) *(cl.map_shared_rank(sums, 0) + list) = Best{M, S};
    __syncthreads();
  }
  if (blocks > 1) cl.sync();
  if (rank != 0) return;
  __syncthreads();

  if (tid == 0) n = 0;
  if (tid < K) {
    const float score = p.scores[prompt * K + tid];
    int k = !isfinite(score) ? 2 : p.done && p.done[prompt * K + tid] ? 1 : 0;
    if (k == 0) {
      float m = -INFINITY, s = 0.f;
      for (int i = 0; i < parts; ++i) m = fmaxf(m, sums[tid * parts + i].m);
      for (int i = 0; i < parts; ++i)
        s += sums[tid * parts + i].s * rescale(sums[tid * parts + i].m, m);
      lse[tid] = (double)m + log((double)s);
      if (!isfinite(lse[tid])) k = 2;
    }
    kind[tid] = k;
  }
  __syncthreads();
  // item i of a list
  auto item = [&](int list, int i) {
    const int k = list / parts;
    Item it{-INFINITY, 0ull, k};
    if (kind[k] == 0) {
      it.key = keys[list * K + i];
      if (it.key) it.value = (double)p.scores[prompt * K + k] + ((double)logit_of(it.key) - lse[k]);
    } else if (list % parts == 0) {  // one list: eos first, then the other tokens
      int token = i;
      if (kind[k] == 1) {
        token = i == 0 ? p.eos : i - 1 + (i - 1 >= p.eos);
        if (i == 0) it.value = p.scores[prompt * K + k];
      }
      if (token < p.V) it.key = (unsigned)~(unsigned)token | (Key)(i == 0 && kind[k] == 1) << 32;
    }
    return it;
  };
  // the K-th of the lists' first items bounds what can be among the K best
  if (tid < L) heads[tid] = item(tid, 0);
  __syncthreads();
  for (int i = warp; i < L; i += kWarps) {
    const bool is = lane < L && lane != i && (ahead(heads[lane], heads[i]) || (lane < i && !ahead(heads[i], heads[lane])));
    if (__popc(__ballot_sync(0xffffffffu, is)) == K - 1 && lane == 0) limit = heads[i];
  }
  __syncthreads();
  for (int i = tid; i < L * K; i += kThreads) {
    const Item it = item(i / K, i % K);
    if (it.key && !ahead(limit, it)) kept[atomicAdd(&n, 1)] = it;
  }
  __syncthreads();
  for (int i = warp; i < n; i += kWarps) {
    const Item mine = kept[i];
    int r = 0;
    for (int j = lane; j - lane < n; j += 32) r += __popc(__ballot_sync(0xffffffffu, j < n && ahead(kept[j], mine)));
    if (lane == 0 && r < K) {
      const int o = prompt * K + r;
      p.out_scores[o] = (float)mine.value;
      p.out_tokens[o] = token_of(mine.key);
      p.out_rows[o] = prompt * K + mine.beam;
    }
  }
}

template <int DT, int NV>
cudaError_t launch(const BeamP& p, int parts, int blocks, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.N * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, beam_select<DT, NV>, p, parts);
}

template <int DT>
cudaError_t launch(const BeamP& p, int sms, cudaStream_t st) {
  constexpr int tile = kThreads * Vec<DT>::N;  // a piece a thread
  // a row is shared out where there are fewer rows than SMs, while every thread has a piece
  int parts = 1;
  while (parts * 2 * p.K <= kCluster && p.N * p.K * parts * 2 <= sms && p.V > parts * tile) parts *= 2;
  const int blocks = std::min(p.K * parts, kCluster);
  return p.V / parts <= 2 * tile ? launch<DT, 2>(p, parts, blocks, st) : launch<DT, 8>(p, parts, blocks, st);
}

}  // namespace

cudaError_t launch_beam(const BeamP& p, int sms, cudaStream_t st) {
  switch (p.dt) {
    case BOZO_DT_F32: return launch<BOZO_DT_F32>(p, sms, st);
    case BOZO_DT_BF16: return launch<BOZO_DT_BF16>(p, sms, st);
    default: return launch<BOZO_DT_F16>(p, sms, st);
  }
}

}  // namespace bozo
