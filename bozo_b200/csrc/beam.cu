// beam.cu — the best continuations of a beam search's hypotheses (bozo_beam_select).
//
// A continuation is worth score + logit − log Σ exp(logits).  Of one row the logits
// alone order them, so a first kernel goes over the logits once: a block takes a chunk
// of a row into registers, keeps its largest value and Σ exp(x − largest), and sorts
// out its K best.  No chunk holds a place among the K best of a row that has K better
// groups of lanes: the K-th largest of the groups' maxima is a bound that at most
// K groups reach, so few elements are ever compared with one another.  A second kernel
// joins the chunks' sums and finds each prompt's best among what is left, in 64 bits.
#include "beam.cuh"

namespace bozo {
namespace {

constexpr int kThreads = 256, kGroups = 64;
constexpr int kEach = 32;                      // logits of a thread
constexpr int kChunk = kThreads * kEach;

// Larger keys come first: the logit, then the lower token.
__device__ __forceinline__ unsigned long long key_of(float x, unsigned token) {
  const unsigned u = __float_as_uint(x + 0.f);  // −0 is 0
  const unsigned o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (unsigned long long)o << 32 | (unsigned)~token;
}
__device__ __forceinline__ unsigned token_of(unsigned long long k) { return ~(unsigned)k; }
__device__ __forceinline__ float logit_of(unsigned long long k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// One block per (chunk, row): its part of ws.
template <int DT>
__global__ void __launch_bounds__(kThreads) beam_scan(BeamP p) {
  __shared__ unsigned long long top[kGroups], list[32 * kEach * kThreads / kGroups];
  __shared__ float wmax[kThreads / 32], wsum[kThreads / 32];
  __shared__ unsigned long long bound;
  __shared__ int n;
  const int S = gridDim.x, chunk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((p.done && p.done[row]) || !isfinite(p.scores[row])) return;
  const int lo = chunk * kChunk, K = p.K;
  float x[kEach], m = -INFINITY;
  unsigned long long best = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int v = lo + i * kThreads + tid;
    x[i] = v < p.V ? ldf(p.logits, (long long)row * p.stride + v, DT) : -INFINITY;
    m = fmaxf(m, x[i]);
    if (v < p.V) best = max(best, key_of(x[i], v));
  }
  float s = 0.f;
  const float m0 = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (lo + i * kThreads + tid < p.V) s += pow2((x[i] - m0) * kLog2e);
  float M = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) wmax[warp] = M;
  unsigned long long g = best;
#pragma unroll
  for (int o = 1; o < kThreads / kGroups; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
  if (tid % (kThreads / kGroups) == 0) top[tid / (kThreads / kGroups)] = g;
  if (tid == 0) n = 0, bound = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) M = fmaxf(M, wmax[w]);
  s = warp_sum(m == -INFINITY ? s : s * pow2((m - M) * kLog2e));  // s is NaN where the row has one, 0 of nothing
  if (lane == 0) wsum[warp] = s;
  // the K-th largest group
  if (tid < kGroups) {
    const unsigned long long mine = top[tid];
    int before = 0;
    for (int i = 0; i < kGroups; ++i) before += top[i] > mine || (top[i] == mine && i < tid);
    if (before == K - 1) bound = mine;
  }
  __syncthreads();
  const unsigned long long t = max(bound, 1ull);
  if (best >= t) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int v = lo + i * kThreads + tid;
      if (v >= p.V) continue;
      const unsigned long long k = key_of(x[i], v);
      if (k >= t) list[atomicAdd(&n, 1)] = k;
    }
  }
  __syncthreads();
  unsigned long long* keys = p.keys + ((size_t)row * S + chunk) * K;
  for (int i = tid; i < n; i += kThreads) {
    int before = 0;
    for (int j = 0; j < n; ++j) before += list[j] > list[i];
    if (before < K) keys[before] = list[i];
  }
  for (int i = n + tid; i < K; i += kThreads) keys[i] = 0;  // fewer tokens than that
  if (tid == 0) {
    float total = 0.f;
    for (int w = 0; w < kThreads / 32; ++w) total += wsum[w];
    p.sums[(size_t)row * S + chunk] = make_float2(M, total);
  }
}

struct Item {
  double value;
  unsigned long long key;
  int beam;
};
__device__ __forceinline__ bool before(const Item& a, const Item& b) {
  if (a.value != b.value) return a.value > b.value;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}

// One block per prompt.
__global__ void __launch_bounds__(kThreads) beam_join(BeamP p, int S) {
  extern __shared__ Item items[];  // the heads of all lists [K·S], or what reaches the bound [≤ K·K]
  __shared__ double lse[32], bound;
  __shared__ int kind[32], n;      // 0: scanned, 1: ended, 2: nothing but −infinity
  const int prompt = blockIdx.x, K = p.K, tid = threadIdx.x, H = K * S;
  Item* kept = items + H;
  __shared__ Item limit;
  if (tid == 0) n = 0;
  for (int k = tid; k < K; k += kThreads) {
    const int row = prompt * K + k;
    const float score = p.scores[row];
    kind[k] = !isfinite(score) ? 2 : p.done && p.done[row] ? 1 : 0;
    if (kind[k]) continue;
    float m = -INFINITY;
    for (int c = 0; c < S; ++c) m = fmaxf(m, p.sums[(size_t)row * S + c].x);
    double s = 0.;
    for (int c = 0; c < S; ++c) {
      const float2 u = p.sums[(size_t)row * S + c];
      s += u.x == -INFINITY && u.y == 0.f ? 0. : (double)u.y * exp((double)u.x - (double)m);
    }
    lse[k] = (double)m + log(s);
    if (!isfinite(lse[k])) kind[k] = 2;
  }
  __syncthreads();
  // item i of list c of hypothesis k
  auto item = [&](int k, int c, int i) {
    const int row = prompt * K + k;
    Item it{-INFINITY, 0ull, k};
    if (kind[k] == 0) {
      it.key = p.keys[((size_t)row * S + c) * K + i];
      if (it.key) it.value = (double)p.scores[row] + ((double)logit_of(it.key) - lse[k]);
    } else if (c == 0) {  // one list: eos first, then the other tokens
      int token = i;
      if (kind[k] == 1) {
        token = i == 0 ? p.eos : i - 1 + (i - 1 >= p.eos);
        if (i == 0) it.value = p.scores[row];
      }
      if (token < p.V) it.key = (unsigned)~(unsigned)token | (unsigned long long)(i == 0 && kind[k] == 1) << 32;
    }
    return it;
  };
  for (int h = tid; h < H; h += kThreads) items[h] = item(h / S, h % S, 0);
  __syncthreads();
  for (int h = tid; h < H; h += kThreads) {
    const Item mine = items[h];
    int ahead = 0;
    for (int j = 0; j < H; ++j) ahead += before(items[j], mine) || (!before(mine, items[j]) && j < h);
    if (ahead == K - 1) limit = mine;
  }
  __syncthreads();
  for (int h = tid; h < H; h += kThreads) {
    if (before(limit, items[h]) || !items[h].key) continue;
    for (int i = 0; i < K; ++i) {
      const Item it = i ? item(h / S, h % S, i) : items[h];
      if (before(limit, it) || !it.key) break;
      kept[atomicAdd(&n, 1)] = it;
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const Item mine = kept[i];
    int ahead = 0;
    for (int j = 0; j < n; ++j) ahead += before(kept[j], mine);
    if (ahead < K) {
      const int o = prompt * K + ahead;
      p.out_scores[o] = (float)mine.value;
      p.out_tokens[o] = token_of(mine.key);
      p.out_rows[o] = prompt * K + mine.beam;
    }
  }
}

}  // namespace

int beam_chunks(const BeamP& p) { return (p.V + kChunk - 1) / kChunk; }

size_t beam_bytes(const BeamP& p) {
  const size_t lists = (size_t)p.N * p.K * beam_chunks(p);
  return lists * (p.K * sizeof(unsigned long long) + sizeof(float2));
}

cudaError_t launch_beam(BeamP p, void* ws, cudaStream_t st) {
  const int S = beam_chunks(p);
  p.keys = static_cast<unsigned long long*>(ws);
  p.sums = reinterpret_cast<float2*>(p.keys + (size_t)p.N * p.K * S * p.K);
  const dim3 grid((unsigned)S, (unsigned)(p.N * p.K));
  switch (p.dt) {
    case BOZO_DT_F32: beam_scan<BOZO_DT_F32><<<grid, kThreads, 0, st>>>(p); break;
    case BOZO_DT_BF16: beam_scan<BOZO_DT_BF16><<<grid, kThreads, 0, st>>>(p); break;
    default: beam_scan<BOZO_DT_F16><<<grid, kThreads, 0, st>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const size_t smem = ((size_t)p.K * S + p.K * p.K) * sizeof(Item);
  if (smem > 48 * 1024 && (e = cudaFuncSetAttribute(beam_join, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess)
    return e;
  beam_join<<<p.N, kThreads, smem, st>>>(p, S);
  return cudaGetLastError();
}

}  // namespace bozo
