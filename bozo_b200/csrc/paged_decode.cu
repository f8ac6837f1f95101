// paged_decode.cu — one decode step of the tension operator over a paged cache
// (bozo_paged_decode).
//
// With t = lengths[b]: τ_s = σ(R(t)q·k_s / scale) over the keys s in reach,
// out = Σ τ_s·v_s / (max(Σ τ_s, 1e-6) | max(n, 1) | 1).  Both sums are plain
// sums over keys, so a long row is cut into pieces that are summed on their own
// and joined by adding, in the order of the pieces.
#include <algorithm>

#include "paged_decode.cuh"

namespace bozo {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxPiece = 8192;     // positions of a piece of paged_decode_any, which holds their τ in shared memory
constexpr int kCluster = 8;         // pieces that are joined inside a cluster

// One block per (b, h, piece), one warp per key: any head width and types.
__global__ void __launch_bounds__(kThreads) paged_decode_any(PagedP p, int S) {
  extern __shared__ float sm[];
  float* sq = sm;             // rotated q [HD]
  float* stau = sm + p.HD;    // τ of the piece's keys
  __shared__ float red[kThreads / 32];
  const int piece = blockIdx.x % S, bh = blockIdx.x / S;
  const int b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const int HD = p.HD, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Reach r = reach(p, b, S);
  if ((unsigned)piece >= r.count) return;
  const unsigned j0 = max(r.first(piece), r.lo), j1 = r.last(piece);
  if (r.active)
    for (int i = threadIdx.x; i < HD; i += kThreads) sq[i] = query(p, b, h, r.t, i);
  if (writes_row(p, r, piece, h % (p.H / p.Hk) == 0)) append_row(p, b, hk, r.t, warp, lane);
  __syncthreads();
  for (unsigned j = j0 + warp; j < j1; j += kThreads / 32) {
    const unsigned row0 = paged_row(p, b, j);
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
      const unsigned row0 = paged_row(p, b, j);
      if (row0 == kNoRow) continue;
      const size_t row = row0 + (size_t)hk * p.page;
      float x = ld_page(p.v, row * HD + d, p.dt);
      acc = fmaf(p.vs ? stau[j - j0] * p.vs[row] : stau[j - j0], x, acc);
    }
    if (r.count == 1)
      stf(p.out, (long long)bh * HD + d, p.out_dt, acc / norm_divisor(p, m, r.n));
    else
      p.ws[((size_t)bh * S + piece) * HD + d] = acc;
  }
  if (r.count > 1 && threadIdx.x == 0) piece_mass(p, S)[(size_t)bh * S + piece] = m;
  if (p.tau) {
    for (unsigned j = j0 + threadIdx.x; j < j1; j += kThreads) put_tau(p, bh, r.t, j, stau[j - j0]);
    if (piece == 0) clear_tau(p, bh, r.n, threadIdx.x, kThreads);
  }
}

// Rows cut into more than one piece: one block per (b, h).
__global__ void __launch_bounds__(kThreads) paged_join(PagedP p, int S) {
  const int bh = blockIdx.x, HD = p.HD;
  const Reach r = reach(p, bh / p.H, S);
  if (r.count < 2) return;
  const float* w = p.ws + (size_t)bh * S * HD;
  const float* wm = piece_mass(p, S) + (size_t)bh * S;
  for (int d = threadIdx.x; d < HD; d += kThreads) {
    float acc = 0.f, m = 0.f;
    for (unsigned i = 0; i < r.count; ++i) {
      acc += w[i * HD + d];
      m += wm[i];
    }
    stf(p.out, (long long)bh * HD + d, p.out_dt, acc / norm_divisor(p, m, r.n));
  }
}

bool mma_path(const PagedP& p) {
  return p.dt != BOZO_DT_F32 && (p.HD == 32 || p.HD == 64 || p.HD == 128);
}

PagedPlan plan(const PagedP& p, int sms) {
  const bool mma = mma_path(p);
  const long long keys = (p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap) + 15;
  const int G = p.H / p.Hk;
  const long long rows = (long long)p.B * (mma ? (long long)p.Hk * ((G + kHeads - 1) / kHeads) : p.H);
  long long s = (sms * (mma ? 16 : 8) + rows - 1) / rows;
  s = std::min(s, (keys + kMinPiece - 1) / kMinPiece);
  if (!mma) s = std::max(s, (keys + kMaxPiece - 1) / kMaxPiece);
  s = std::max(s, 1LL);
  return {(int)s, mma && s > 1 && s <= kCluster};
}

}  // namespace

size_t paged_decode_bytes(const PagedP& p, int sms) {
  const PagedPlan pl = plan(p, sms);
  if (pl.S < 2 || pl.clustered) return 0;
  return ((size_t)p.B * p.H * pl.S * (p.HD + 1) * sizeof(float) + 255) & ~(size_t)255;
}

cudaError_t launch_paged_decode(const PagedP& p, int sms, cudaStream_t st, int* launches) {
  const PagedPlan pl = plan(p, sms);
  cudaError_t e;
  if (mma_path(p)) {
    switch (p.dt) {
      case BOZO_DT_BF16: e = launch_paged_mma_bf16(p, pl, st); break;
      case BOZO_DT_F16: e = launch_paged_mma_f16(p, pl, st); break;
      case BOZO_DT_F8E4M3: e = launch_paged_mma_f8(p, pl, st); break;
      default: e = launch_paged_mma_i8(p, pl, st);
    }
  } else {
    const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
    const size_t smem = (size_t)(p.HD + std::min<long long>(keys, kMaxPiece) + 16) * sizeof(float);
    paged_decode_any<<<(unsigned)(p.B * p.H * pl.S), kThreads, smem, st>>>(p, pl.S);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  *launches = 1;
  if (pl.S > 1 && !pl.clustered) {
    paged_join<<<(unsigned)(p.B * p.H), kThreads, 0, st>>>(p, pl.S);
    *launches = 2;
  }
  return cudaGetLastError();
}

}  // namespace bozo
