// paged_decode.cu — one decode step of the tension operator over a paged cache
// (bozo_paged_decode).
//
// With t = lengths[b]: τ_s = σ(R(t)q·k_s / scale) over the keys s in reach,
// out = Σ τ_s·v_s / (max(Σ τ_s, 1e-6) | max(n, 1) | 1).  Both sums are plain
// sums over keys, so a long row is cut into pieces that are summed on their own
// and joined by adding, in the order of the pieces.
#include <algorithm>

#include "paged.cuh"

namespace bozo {
namespace {

constexpr int kThreads = 128;
constexpr int kMinPiece = 128;      // keys of a piece, at least
constexpr int kMaxPiece = 8192;     // and at most: τ of a piece is held in shared memory
constexpr int kResident = 8;        // blocks an SM is given, counted over whole rows

// Keys in reach of a sequence's query: [lo, lo + n), or false where it is inactive.
__device__ __forceinline__ bool reach(const PagedP& p, int b, int& t, unsigned& lo, unsigned& n) {
  t = __ldg(p.len + b);
  n = lo = 0;
  if (t < 0) return false;
  if (p.cos && t >= p.rope_len) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, kErrPaged | 1);
    return false;
  }
  const unsigned end = (unsigned)t + (p.mode == BOZO_MODE_GLOBAL ? 1u : 0u);
  n = min(end, p.mode == BOZO_MODE_GLOBAL ? p.cap : (unsigned)p.W);
  lo = end - n;
  return true;
}

// A row of n keys is cut into `count` pieces of `size` keys (the last one less).
__device__ __forceinline__ void cut(unsigned n, unsigned S, unsigned& count, unsigned& size) {
  count = max(1u, min(S, (n + kMinPiece - 1) / kMinPiece));
  size = ((n + count - 1) / count + 15) & ~15u;
  if (size) count = (n + size - 1) / size;
}

__device__ __forceinline__ float norm_divisor(const PagedP& p, float mass, unsigned n) {
  return p.norm == BOZO_NORM_MASS ? fmaxf(mass, kMassEps)
                                  : p.norm == BOZO_NORM_COUNT ? (float)max(n, 1u) : 1.f;
}

// One block per (b, h, piece), one warp per key: any head width and types.
__global__ void __launch_bounds__(kThreads) paged_decode_any(PagedP p, int S) {
  extern __shared__ float sm[];
  float* sq = sm;             // rotated q [HD]
  float* stau = sm + p.HD;    // τ of the piece's keys
  __shared__ float red[kThreads / 32];
  const int piece = blockIdx.x % S, bh = blockIdx.x / S;
  const int b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const int HD = p.HD, half = HD / 2, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int t;
  unsigned lo, n, count, size;
  const bool active = reach(p, b, t, lo, n);
  cut(n, S, count, size);
  if ((unsigned)piece >= count) return;
  const unsigned j0 = piece * size, j1 = min(n, j0 + size);
  const long long qo = (long long)b * p.q.sb + (long long)h * p.q.sh;
  if (active) {
    for (int i = threadIdx.x; i < HD; i += kThreads) {
      float x = ldf(p.q.p, qo + i * p.q.sd, p.q.dt);
      if (p.cos) {
        const int f = i < half ? i : i - half;
        const float c = p.cos[(size_t)t * half + f], s = p.sin[(size_t)t * half + f];
        const float y = ldf(p.q.p, qo + (i < half ? i + half : f) * p.q.sd, p.q.dt);
        x = i < half ? x * c - y * s : y * s + x * c;
      }
      sq[i] = x;
    }
  }
  __syncthreads();
  for (unsigned j = j0 + warp; j < j1; j += kThreads / 32) {
    const unsigned row0 = paged_row(p, b, lo + j);
    const size_t row = row0 + (size_t)hk * p.page;
    float dot = 0.f;
    if (row0 != kNoRow)
      for (int d = lane; d < HD; d += 32) dot = fmaf(sq[d], ld_page(p.k, row * HD + d, p.dt), dot);
    dot = warp_sum(dot);
    if (lane == 0) {
      if (row0 != kNoRow && p.ks) dot *= p.ks[row];
      stau[j - j0] = row0 == kNoRow ? 0.f : sigmoid_exact(dot * p.inv_scale);
    }
  }
  __syncthreads();
  float m = 0.f;
  for (unsigned j = j0 + threadIdx.x; j < j1; j += kThreads) m += stau[j - j0];
  m = warp_sum(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = 0.f;
  for (int w = 0; w < kThreads / 32; ++w) m += red[w];
  for (int d = threadIdx.x; d < HD; d += kThreads) {
    float acc = 0.f;
    for (unsigned j = j0; j < j1; ++j) {
      const unsigned row0 = paged_row(p, b, lo + j);
      if (row0 == kNoRow) continue;
      const size_t row = row0 + (size_t)hk * p.page;
      float x = ld_page(p.v, row * HD + d, p.dt);
      acc = fmaf(p.vs ? stau[j - j0] * p.vs[row] : stau[j - j0], x, acc);
    }
    if (count == 1)
      stf(p.out, (long long)bh * HD + d, p.out_dt, acc / norm_divisor(p, m, n));
    else
      p.ws[((size_t)bh * S + piece) * (HD + 1) + d] = acc;
  }
  if (count > 1 && threadIdx.x == 0) p.ws[((size_t)bh * S + piece) * (HD + 1) + HD] = m;
  if (p.tau) {
    // LOCAL slot c holds key j = n − (W − c), GLOBAL column c key j = n − 1 − c;
    // the first piece also clears the slots without a key
    for (int c = threadIdx.x; c < p.tw; c += kThreads) {
      const long long j = p.mode == BOZO_MODE_LOCAL ? (long long)n - (p.W - c) : (long long)n - 1 - c;
      const long long at = (long long)bh * p.tw + c;
      if (j >= (long long)j0 && j < (long long)j1) stf(p.tau, at, p.tau_dt, stau[j - j0]);
      else if (j < 0 && piece == 0) stf(p.tau, at, p.tau_dt, 0.f);
    }
  }
}

// Rows cut into more than one piece: one block per (b, h).
__global__ void __launch_bounds__(kThreads) paged_join(PagedP p, int S) {
  const int bh = blockIdx.x, HD = p.HD;
  int t;
  unsigned lo, n, count, size;
  reach(p, bh / p.H, t, lo, n);
  cut(n, S, count, size);
  if (count < 2) return;
  const float* w = p.ws + (size_t)bh * S * (HD + 1);
  for (int d = threadIdx.x; d < HD; d += kThreads) {
    float acc = 0.f, m = 0.f;
    for (unsigned i = 0; i < count; ++i) {
      acc += w[i * (HD + 1) + d];
      m += w[i * (HD + 1) + HD];
    }
    stf(p.out, (long long)bh * HD + d, p.out_dt, acc / norm_divisor(p, m, n));
  }
}

int pieces(const PagedP& p, int sms) {
  const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
  const long long rows = (long long)p.B * p.H;
  long long s = (sms * kResident + rows - 1) / rows;
  s = std::min(s, (keys + kMinPiece - 1) / kMinPiece);
  return (int)std::max({s, (keys + kMaxPiece - 1) / kMaxPiece, 1LL});
}

}  // namespace

size_t paged_decode_bytes(const PagedP& p, int sms) {
  const int S = pieces(p, sms);
  return S < 2 ? 0 : ((size_t)p.B * p.H * S * (p.HD + 1) * sizeof(float) + 255) & ~(size_t)255;
}

cudaError_t launch_paged_decode(const PagedP& p, int sms, cudaStream_t st, int* launches) {
  *launches = 0;
  if (p.kn.p) {
    cudaError_t e = launch_paged_write(p, st);
    if (e != cudaSuccess) return e;
    ++*launches;
  }
  const int S = pieces(p, sms);
  const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
  const size_t smem = (size_t)(p.HD + std::min<long long>(keys, kMaxPiece) + 16) * sizeof(float);
  paged_decode_any<<<(unsigned)(p.B * p.H * S), kThreads, smem, st>>>(p, S);
  ++*launches;
  if (S > 1) {
    paged_join<<<(unsigned)(p.B * p.H), kThreads, 0, st>>>(p, S);
    ++*launches;
  }
  return cudaGetLastError();
}

}  // namespace bozo
