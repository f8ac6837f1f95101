// beam.cu — the best continuations of a beam search's hypotheses (bozo_beam_select).
//
// A continuation is worth score + logit − log Σ exp(logits); within one row the logits
// alone order them.  One cluster a prompt, each block a row, a part of one, or (more
// than kCluster hypotheses) a few rows, and one pass over the logits:
//   * the row's largest value and Σ exp(x − largest), 32 logits a thread at a time;
//   * its K best: the K-th largest of 64 groups of threads' maxima is a bound that at least
//     K elements reach, and for unequal logits few more.  The threads that hold them read
//     theirs once more, and only those elements are compared with one another (many equal
//     ones: the best are taken out one after the other).  Keeping a row in registers
//     instead left one block an SM (64 prompts' eight hypotheses: 43 µs);
//   * every block's K best keys and sum go to the first block's shared memory, which
//     finds the prompt's best among them in 64 bits.
// Bound by the logits' bytes where rows are many, by the chain of these steps where
// they are few: 64 prompts × 8 hypotheses × 32768 tokens in bf16 14.3 µs in a graph (29.4
// MB without the ended ones, 4.5 µs; the loop over them 6), 1 × 4 × 8192 in fp32 5.3.  Rows
// that are not all aligned to 16 bytes take a kernel of their own, 20.0 µs for the former
// with 32767 tokens (as branches of one kernel they cost aligned rows 1.2 µs).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "beam.cuh"

namespace bozo {
namespace {

namespace cg = cooperative_groups;
using Key = unsigned long long;
constexpr int kGroups = 64, kCluster = 16;
constexpr int kParts = 8;  // blocks that share a prompt's rows out in parts, at most
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
// two that are (the second is the neighbour's first, out of the L1).  AL: every row is.
template <int DT, bool AL> struct Row {
  const char* at;
  int from16, V, pieces;  // bytes from a multiple of 16
  static constexpr int N = Vec<DT>::N, size = 16 / N;
  __device__ __forceinline__ Row(const BeamP& p, int row) {
    at = static_cast<const char*>(p.logits) + (long long)row * p.stride * size;
    from16 = AL ? 0 : (int)(reinterpret_cast<uintptr_t>(at) & 15);
    V = p.V;
    pieces = (V + N - 1) / N;
  }
  __device__ __forceinline__ int off() const { return AL ? 0 : from16; }
  // the 16 bytes that begin off() bytes into v's and y's 32
  __device__ __forceinline__ void shift(Vec<DT>& v, const uint4& y) const {
    unsigned u[8] = {v.w[0], v.w[1], v.w[2], v.w[3], y.x, y.y, y.z, y.w};
    if (off() & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) u[i] = u[i + 2];
    }
    if (off() & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) u[i] = u[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = __funnelshift_r(u[i], u[i + 1], 8 * (off() & 3));
  }
  __device__ __forceinline__ Vec<DT> load(int q, int end) const {
    Vec<DT> v;
    const int f = q * N;
    if (off() == 0 ? q < end && f + N <= V : q < end && q > 0 && f + 2 * N <= V) {
      const uint4* from = reinterpret_cast<const uint4*>(at - off()) + q;
      const uint4 x = __ldg(from);
      v.w[0] = x.x; v.w[1] = x.y; v.w[2] = x.z; v.w[3] = x.w;
      if (off()) shift(v, __ldg(from + 1));
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

// Items in order: value, then the lower hypothesis, then the key.  The value is a double
// as an integer in its order; 0 is no item.
__device__ __forceinline__ Key ordered(double x) {
  const Key u = (Key)__double_as_longlong(x + 0.);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double value_of(Key o) {
  return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o));
}
struct Item {
  Key value, key;
  int beam;
};
__device__ __forceinline__ bool ahead(const Item& a, const Item& b) {
  if (a.value != b.value) return a.value > b.value;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}

template <int kThreads> struct Scratch {
  float top[kGroups], wm[32], ws[32];
  Key list[kList], cur[32], wbest[32];
  float bound, m, s;
  unsigned short holds[kThreads];
  int n, held;
};

// The warp's largest; NaN are passed over.
__device__ __forceinline__ float warp_most(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// log s to about 1e-9 for a sum of exponentials of which the largest is 1: with s = 2^e · f,
// f in [√½, √2), log f = 2·atanh z, z = (f − 1) / (f + 1); z in 64 bits, the series' further
// terms, a hundredth of the first, in 32.  (The library's function takes a few times as long,
// which every selection waits for.)
__device__ __forceinline__ double log_sum(float s) {
  if (!(s >= 0.5f && s < 3e38f)) return log((double)s);  // nothing, or not finite
  int e = (int)(__float_as_uint(s) >> 23) - 127;
  float f = __uint_as_float((__float_as_uint(s) & 0x7fffffu) | 0x3f800000u);
  if (f > 1.41421356f) {
    f *= 0.5f;
    ++e;
  }
  const double n = (double)f - 1., d = (double)f + 1.;
  const float r = __frcp_rn(f + 1.f), z0 = (f - 1.f) * r, w = z0 * z0;
  const double z = fma(fma(-(double)z0, d, n), (double)r, (double)z0);
  const float p = w * fmaf(w, fmaf(w, fmaf(w, fmaf(w, fmaf(w, 1.f / 13, 1.f / 11), 1.f / 9), 1.f / 7), 1.f / 5), 1.f / 3);
  return fma((double)e, 0.69314718055994530942, fma(2. * z, (double)p, 2. * z));
}

// Two exponentials relative to m, added to (a, b).
__device__ __forceinline__ void add_pow2(float& a, float& b, float x, float y, float m) {
  asm("{.reg .b64 p, q; .reg .f32 x, y; mov.b64 p, {%2, %3}; mov.b64 q, {%4, %4}; add.rn.f32x2 p, p, q;"
      " mov.b64 q, {%5, %5}; mul.rn.f32x2 p, p, q; mov.b64 {x, y}, p; ex2.approx.ftz.f32 x, x;"
      " ex2.approx.ftz.f32 y, y; mov.b64 p, {x, y}; mov.b64 q, {%0, %1}; add.rn.f32x2 p, p, q; mov.b64 {%0, %1}, p;}"
      : "+f"(a), "+f"(b) : "f"(x), "f"(y), "f"(-m), "f"(kLog2e));
}

// put(i, how many of the n items come before item i), eight threads an item.
template <int kThreads, typename B, typename P>
__device__ __forceinline__ void for_ranks(int n, B is_before, P put) {
  const int sub = threadIdx.x & 7;
  for (int i0 = 0; i0 < n; i0 += kThreads / 8) {  // the same for all threads
    const int i = i0 + (threadIdx.x >> 3), me = min(i, n - 1);
    int r = 0;
#pragma unroll 4
    for (int j = sub; j < n; j += 8) r += is_before(me, j);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    if (sub == 0 && i < n) put(i, r);
  }
}

// A thread's largest logit m, and s + rest = Σ exp(x − ref): what adding a batch to s leaves over
// is kept, so that the error does not grow with the row (128 rows of 2^20 fp32 logits: 2e-7,
// without it 1.5e-5; 64 × 8 × 32768 in bf16 14.7 µs for 14.4, with doubles 15.1).  The
// reference follows m in steps of kStep or more: what is rescaled, to 2^-22, is then at most
// exp(−kStep) of itself, and however often m rises that adds up to 4.5 · 2^-22.  In all
// log Σ exp is off by (79 + 2.3 ln V) · 2^-24 at most: exponentials of 2^-22, a batch's
// additions, and those of warps, blocks and parts.
constexpr float kStep = 0.25f;
struct Sum {
  float m = -INFINITY, ref = -INFINITY, s = 0.f, rest = 0.f;
};
template <int DT, int U>
__device__ __forceinline__ void take(const Vec<DT>* v, Sum& t) {
  constexpr int N = Vec<DT>::N;
#pragma unroll
  for (int j = 0; j < U; ++j) t.m = fmaxf(t.m, v[j].most());
  const float to = t.m >= t.ref + kStep ? t.m : t.ref, ref = finite_or_0(to);
  float a[2] = {0.f, 0.f}, b[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int i = 0; i < N; i += 2) add_pow2(a[i / 2 % 2], b[i / 2 % 2], v[j].at(i), v[j].at(i + 1), ref);
  const float f = rescale(t.ref, to), s = t.s * f, x = (a[0] + a[1]) + (b[0] + b[1]);
  t.s = __fadd_rn(s, x);
  const float y = __fsub_rn(t.s, s);  // of x; the rest of it and of s (Knuth's sum of two)
  t.rest = t.rest * f + (__fsub_rn(s, __fsub_rn(t.s, y)) + __fsub_rn(x, y));
  t.ref = to;
}

// A thread's batch of pieces q, q + kThreads, … below q1: whole pieces are nothing but loads,
// all in flight together (and shifts).
constexpr int kBatch = 8;
template <int DT, int kThreads, int U = kBatch, bool AL>
__device__ __forceinline__ void batch(const Row<DT, AL>& row, int q, int q1, Vec<DT>* v) {
  const int last = q + (U - 1) * kThreads;
  if (row.off() == 0 ? last < min(q1, row.V / Vec<DT>::N) : q > 0 && last < q1 && (last + 2) * Vec<DT>::N <= row.V) {
    const uint4* from = reinterpret_cast<const uint4*>(row.at - row.off()) + q;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const uint4 x = __ldg(from + j * kThreads);
      v[j].w[0] = x.x; v[j].w[1] = x.y; v[j].w[2] = x.z; v[j].w[3] = x.w;
    }
    if (row.off()) {
#pragma unroll
      for (int j = 0; j < U; ++j) row.shift(v[j], __ldg(from + j * kThreads + 1));
    }
  } else {
#pragma unroll
    for (int j = 0; j < U; ++j) v[j] = row.load(q + j * kThreads, q1);
  }
}
// The first one of pieces [q0, q1): half of one where that is all there is.
template <int DT, int kThreads, bool AL>
__device__ __forceinline__ void first_batch(const Row<DT, AL>& row, int q0, int q1, Vec<DT>* v) {
  if (q1 - q0 <= kBatch / 2 * kThreads) batch<DT, kThreads, kBatch / 2>(row, q0 + threadIdx.x, q1, v);
  else batch<DT, kThreads>(row, q0 + threadIdx.x, q1, v);
}

// The K best of pieces [q0, q1) of a row, sorted, into sc.cur, its largest logit and sum (to all
// threads), and the two's logarithm (to the first of the last warp).  v: the first batch.
template <int DT, int kThreads, bool AL>
__device__ __forceinline__ void scan(const Row<DT, AL>& row, int q0, int q1, int K, Scratch<kThreads>& sc, Vec<DT>* v,
                                     float& M, float& S, double& lse) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kWarps = kThreads / 32, N = Vec<DT>::N;
  Sum sum;
  if (q1 - q0 <= kBatch / 2 * kThreads) {
    take<DT, kBatch / 2>(v, sum);
  } else {
    for (int q = q0 + tid;;) {
      take<DT, kBatch>(v, sum);
      q += kBatch * kThreads;
      if (q >= q1) break;
      batch<DT, kThreads>(row, q, q1, v);
    }
  }
  const float m = sum.m;
  float g = m;
#pragma unroll
  for (int o = 1; o < kThreads / kGroups; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
  const float wm = warp_most(m);
  if (tid % (kThreads / kGroups) == 0) sc.top[tid / (kThreads / kGroups)] = g;
  const float s = warp_sum((sum.s + sum.rest) * rescale(sum.ref, wm));
  if (lane == 0) {
    sc.wm[warp] = wm;
    sc.ws[warp] = s;
  }
  if (tid == 0) sc.n = sc.held = 0;
  __syncthreads();
  // the K-th largest group: each has kThreads / kGroups threads that compare it with a share
  constexpr int kEach = kThreads / kGroups;
  {
    const int me = tid / kEach;
    const float x = sc.top[me];
    int r = 0;
#pragma unroll
    for (int i = 0; i < kGroups / kEach; ++i) {
      const int j = i * kEach + tid % kEach;
      const float y = sc.top[j];
      r += y > x || (y == x && j < me);
    }
#pragma unroll
    for (int o = 1; o < kEach; o <<= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    if (r == K - 1 && tid % kEach == 0) sc.bound = x;
  }
  if (warp == kWarps - 1) {
    const float y = lane < kWarps ? sc.wm[lane] : -INFINITY;
    M = warp_most(y);
    S = warp_sum(lane < kWarps ? sc.ws[lane] * rescale(y, M) : 0.f);
    if (lane == 0) {
      sc.m = M;
      sc.s = S;
    }
  }
  __syncthreads();
  M = sc.m;
  S = sc.s;
  const float bound = sc.bound;
  // the few threads that hold such logits have theirs read again, by all threads at once
  if (m >= bound) sc.holds[atomicAdd(&sc.held, 1)] = (unsigned short)tid;
  __syncthreads();
  const int held = sc.held, each = (q1 - q0 + kThreads - 1) / kThreads;
  for (int i = tid; i < held * each; i += kThreads) {
    const int q = q0 + sc.holds[i / each] + i % each * kThreads, f = q * N;
    if (q >= q1) continue;
    const Vec<DT> v = row.load(q, q1);
    if (v.most() < bound) continue;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = v.at(j);
      if (x >= bound && f + j < row.V) {
        const int at = atomicAdd(&sc.n, 1);
        if (at < kList) sc.list[at] = key_of(x, f + j);
      }
    }
  }
  if (tid == kThreads - 32) lse = (double)M + log_sum(S);
  __syncthreads();
  const int n = sc.n;
  if (n <= kList) {
    for_ranks<kThreads>(n, [&](int i, int j) { return sc.list[j] > sc.list[i]; },
                        [&](int i, int r) { if (r < K) sc.cur[r] = sc.list[i]; });
    if (tid >= n && tid < K) sc.cur[tid] = 0;  // a part with fewer tokens
    __syncthreads();
  } else {
    // many equal logits: the largest key below the last, K times
    Key last = ~0ull;
    for (int k = 0; k < K; ++k) {
      Key best = 0;
#pragma unroll 1
      for (int q = q0 + tid; q < q1; q += kThreads) {
        const Vec<DT> u = row.load(q, q1);
        const int f = q * N;
        if (u.most() < bound) continue;
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

// Parts of a row and blocks of a cluster: parts · K blocks, or (K > kCluster) blocks that
// take every so many-th row.
template <int DT, int kThreads, bool AL>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) beam_select(BeamP p, int log_parts) {
  constexpr int kWarps = kThreads / 32;
  __shared__ Scratch<kThreads> sc;
  // of the first block: every list, and what is left of them
  __shared__ Key keys[32 * 32];
  __shared__ Best sums[32];
  __shared__ Item kept[32 * 32];
  __shared__ Item heads[32], limit;
  __shared__ double lse[32];
  __shared__ float score[32];
  __shared__ int kind[32], n;  // 0: scanned, 1: ended, 2: nothing but −infinity
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), blocks = (int)cl.num_blocks();
  const int prompt = blockIdx.x / blocks, K = p.K, parts = 1 << log_parts, L = K << log_parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (blocks > 1) cl.barrier_arrive();
  // this block's pieces of a list's row
  auto part_of = [&](const Row<DT, AL>& row, int list, int& q0, int& q1) {
    const int each = (row.pieces + parts - 1) >> log_parts;
    q0 = min(row.pieces, each * (list & (parts - 1)));
    q1 = min(row.pieces, q0 + each);
  };
  // the first one's first logits are fetched beside the scores (L ≥ blocks)
  Vec<DT> v[kBatch];
  {
    const Row<DT, AL> row(p, prompt * K + (rank >> log_parts));
    int q0, q1;
    part_of(row, rank, q0, q1);
    first_batch<DT, kThreads>(row, q0, q1, v);
  }
  if (tid < K) {
    score[tid] = p.scores[prompt * K + tid];
    const bool ended = p.done && p.done[prompt * K + tid];
    kind[tid] = !isfinite(score[tid]) ? 2 : ended ? 1 : 0;
  }
  if (tid == 0) n = 0;
  const int my_list = tid / K, my_item = tid - my_list * K;
  __syncthreads();
  bool there = blocks == 1;  // the first block is
  for (int list = rank; list < L; list += blocks) {
    const int r = prompt * K + (list >> log_parts);
    if (kind[list >> log_parts]) continue;
    const Row<DT, AL> row(p, r);
    int q0, q1;
    part_of(row, list, q0, q1);
    if (list != rank) first_batch<DT, kThreads>(row, q0, q1, v);
    float M, S;
    double one;
    scan<DT, kThreads>(row, q0, q1, K, sc, v, M, S, one);
    if (!there) cl.barrier_wait();
    there = true;
    Key* to = cl.map_shared_rank(keys, 0) + list * K;
    if (tid < K) to[tid] = sc.cur[tid];
    if (tid == kThreads - 32) {
      *(cl.map_shared_rank(sums, 0) + list) = Best{M, S};
      if (parts == 1) *(cl.map_shared_rank(lse, 0) + list) = one;
    }
    __syncthreads();
  }
  if (!there) cl.barrier_wait();
  if (blocks > 1) cl.sync();
  if (rank != 0) return;

  // log Σ exp of hypothesis k's logits, from its parts' sums
  auto log_of = [&](int k) {
    if (parts == 1) return lse[k];
    float m = -INFINITY, s = 0.f;
    for (int i = 0; i < parts; ++i) m = fmaxf(m, sums[k * parts + i].m);
    for (int i = 0; i < parts; ++i) s += sums[k * parts + i].s * rescale(sums[k * parts + i].m, m);
    return (double)m + log_sum(s);
  };
  // item i of a list, whose hypothesis' logarithm is `log`
  auto item = [&](int list, int i, double log) {
    const int k = list >> log_parts;
    Item it{0ull, 0ull, k};
    if (kind[k] == 0 && isfinite(log)) {
      it.key = keys[list * K + i];
      if (it.key) it.value = ordered((double)score[k] + ((double)logit_of(it.key) - log));
    } else if ((list & (parts - 1)) == 0) {  // one list: eos first, then the other tokens
      const bool ended = kind[k] == 1;
      const int token = !ended ? i : i == 0 ? p.eos : i - 1 + (i - 1 >= p.eos);
      it.value = ordered(ended && i == 0 ? score[k] : -INFINITY);
      it.key = (unsigned)~(unsigned)token | (Key)(ended && i == 0) << 32;
    }
    return it;
  };
  if (L * K <= 256) {  // one a thread
    if (tid < L * K) kept[tid] = item(my_list, my_item, kind[my_list >> log_parts] ? 0. : log_of(my_list >> log_parts));
    if (tid == 0) n = L * K;
  } else {
    // of many items, of hypotheses that are not shared out in parts, those that the K-th of
    // the lists' first ones does not come before
    static_assert(kParts * kParts <= 256, "up to kParts lists of as many items");
    if (tid < K) heads[tid] = item(tid, 0, lse[tid]);
    __syncthreads();
    for_ranks<kThreads>(K, [&](int i, int j) { return ahead(heads[j], heads[i]) || (j < i && !ahead(heads[i], heads[j])); },
                        [&](int i, int r) { if (r == K - 1) limit = heads[i]; });
    __syncthreads();
    for (int i = tid; i < K * K; i += kThreads) {
      const Item it = item(i / K, i % K, lse[i / K]);
      if (it.key && !ahead(limit, it)) kept[atomicAdd(&n, 1)] = it;
    }
  }
  __syncthreads();
  for_ranks<kThreads>(n, [&](int i, int j) { return ahead(kept[j], kept[i]); },
                      [&](int i, int r) {
                        if (r >= K || !kept[i].key) return;
                        const int o = prompt * K + r;
                        p.out_scores[o] = (float)value_of(kept[i].value);
                        p.out_tokens[o] = token_of(kept[i].key);
                        p.out_rows[o] = prompt * K + kept[i].beam;
                      });
}

template <int DT, int kThreads, bool AL>
cudaError_t launch(const BeamP& p, int log_parts, int blocks, cudaStream_t st) {
  if (blocks > 8) {
    static std::atomic<unsigned long long> allowed{0};  // devices where clusters of more than 8 are
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
      e = cudaFuncSetAttribute(beam_select<DT, kThreads, AL>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
      if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.N * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, beam_select<DT, kThreads, AL>, p, log_parts);
}

template <int DT, bool AL>
cudaError_t launch(const BeamP& p, int sms, cudaStream_t st) {
  // A row is shared out where there are fewer rows than SMs; rows up to 32 KB are not worth the
  // larger cluster.  In a graph, µs, whole | parts:
  // bf16 1 × 1 × 8192 4.4 | 5.6, 1 × 4 × 16384 5.6 | 5.7, 1 × 4 × 32768 7.6 | 6.4, 1 × 1 × 32768
  // 6.3 | 5.6; fp32 1 × 1 × 8192 4.6 | 5.3, 1 × 4 × 16384 6.8 | 5.9.
  int parts = 1, log_parts = 0;
  while (p.V > 2048 * Vec<DT>::N && parts * 2 * p.K <= kParts && p.N * p.K * parts * 2 <= sms) parts *= 2, ++log_parts;
  const int blocks = std::min(p.K * parts, kCluster);
  // Long rows in few blocks: more threads, which also share the elements above the bound out,
  // many with many hypotheses.  256 | 1024 threads, bf16: 1 × 8 × 32768 7.2 | 8.0, × 98304
  // 11.3 | 12.4, × 131072 13.2 | 11.8; 1 × 16 × 32768 15.9 | 11.3, 1 × 32 × 16384 15.3 | 15.2;
  // 4 × 4 × 131072 in two parts 9.0 | 9.8, × 262144 15.7 | 13.0; in 64 blocks (16 × 4 × 32768) 7.0 | 14.3.
  if (2 * p.N * blocks <= sms && p.V / parts >= (p.K > 8 ? 4096 : 16384) * Vec<DT>::N) return launch<DT, 1024, AL>(p, log_parts, blocks, st);
  return launch<DT, 256, AL>(p, log_parts, blocks, st);
}

}  // namespace

template <int DT>
static cudaError_t launch_type(const BeamP& p, int sms, cudaStream_t st) {
  const bool aligned = !((reinterpret_cast<uintptr_t>(p.logits) | (p.stride * (16 / Vec<DT>::N))) & 15);
  return aligned ? launch<DT, true>(p, sms, st) : launch<DT, false>(p, sms, st);
}

cudaError_t launch_beam(const BeamP& p, int sms, cudaStream_t st) {
  switch (p.dt) {
    case BOZO_DT_F32: return launch_type<BOZO_DT_F32>(p, sms, st);
    case BOZO_DT_BF16: return launch_type<BOZO_DT_BF16>(p, sms, st);
    default: return launch_type<BOZO_DT_F16>(p, sms, st);
  }
}

}  // namespace bozo
