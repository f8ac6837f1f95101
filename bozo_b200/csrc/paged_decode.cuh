// paged_decode.cuh — what the kernels of a decode step over a paged cache share:
// the keys in reach and their cut into pieces, the new token's row, the query,
// the exported τ row.
#pragma once

#include "paged.cuh"

namespace bozo {

constexpr int kMinPiece = 128;  // positions of a piece, at least (where there are two)
constexpr int kHeads = 8;       // query heads of a block in the tensor-core kernel, at most

// A join that is launched before its pieces are done waits for them here; a block
// that has no more to start lets it be launched.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct PagedPlan {
  int S;           // pieces a row may be cut into
  bool clustered;  // joined inside a cluster, else by a second kernel from the workspace
};

// The tensor-core kernel, by page type (paged_mma_*.cu).
cudaError_t launch_paged_mma_bf16(const PagedP& p, const PagedPlan& pl, cudaStream_t st);
cudaError_t launch_paged_mma_f16(const PagedP& p, const PagedPlan& pl, cudaStream_t st);
cudaError_t launch_paged_mma_f8(const PagedP& p, const PagedPlan& pl, cudaStream_t st);
cudaError_t launch_paged_mma_i8(const PagedP& p, const PagedPlan& pl, cudaStream_t st);

// Keys that a sequence's query reaches: the n positions [lo, end); none where it
// is inactive.  They are cut into `count` pieces of `size` positions counted from
// `base`, the multiple of 16 at or before lo, so that 16 positions of a piece lie
// in one page wherever the page size is a multiple of 16.
struct Reach {
  int t;
  unsigned lo, end, n, base, count, size;
  bool active;
  __device__ unsigned first(unsigned piece) const { return base + piece * size; }
  __device__ unsigned last(unsigned piece) const { return min(end, base + (piece + 1) * size); }
};
__device__ __forceinline__ Reach reach(const PagedP& p, int b, unsigned S) {
  Reach r;
  r.t = __ldg(p.len + b);
  r.active = r.t >= 0;
  if (r.active && p.cos && r.t >= p.rope_len) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, kErrPaged | 1);
    r.active = false;
  }
  r.end = r.active ? (unsigned)r.t + (p.mode == BOZO_MODE_GLOBAL ? 1u : 0u) : 0u;
  r.n = min(r.end, p.mode == BOZO_MODE_GLOBAL ? p.cap : (unsigned)p.W);
  r.lo = r.end - r.n;
  r.base = r.lo & ~15u;
  const unsigned len = r.end - r.base;
  r.count = 1;
  r.size = max(16u, (len + 15) & ~15u);
  if (S > 1) {
    r.count = max(1u, min(S, (len + kMinPiece - 1) / kMinPiece));
    r.size = max(16u, ((len + r.count - 1) / r.count + 15) & ~15u);
    r.count = max(1u, (len + r.size - 1) / r.size);
  }
  return r;
}

__device__ __forceinline__ float norm_divisor(const PagedP& p, float mass, unsigned n) {
  return p.norm == BOZO_NORM_MASS ? fmaxf(mass, kMassEps)
                                  : p.norm == BOZO_NORM_COUNT ? (float)max(n, 1u) : 1.f;
}

// Workspace: Σ τ·v of every piece [B·H][S][HD], then their masses [B·H][S].
__device__ __forceinline__ float* piece_mass(const PagedP& p, int S) {
  return p.ws + (size_t)p.B * p.H * S * p.HD;
}

// The new token's key and value go into their row before it is read: the blocks
// whose keys end with the new token's write it (each the same bytes; a local
// window does not hold it, so there the first block of a key head does).
__device__ __forceinline__ bool writes_row(const PagedP& p, const Reach& r, unsigned piece, bool first) {
  return p.kn.p && r.active && (p.mode == BOZO_MODE_GLOBAL ? piece == r.count - 1 : piece == 0 && first);
}
__device__ __forceinline__ void append_part(const PagedP& p, int b, int hk, int t, bool key, int lane) {
  const NewRow x(p, key ? p.kn : p.vn, b, hk, (unsigned)t, key && p.cos, lane);
  const unsigned row0 = paged_row(p, b, (unsigned)t);
  if (row0 != kNoRow)
    x.put(p, key ? p.k : p.v, key ? p.ks : p.vs, (size_t)row0 + (size_t)hk * p.page, lane);
}
__device__ __forceinline__ void append_row(const PagedP& p, int b, int hk, int t, int lane) {  // by one warp
  const NewRow k(p, p.kn, b, hk, (unsigned)t, p.cos != nullptr, lane), v(p, p.vn, b, hk, (unsigned)t, false, lane);
  const unsigned row0 = paged_row(p, b, (unsigned)t);
  if (row0 == kNoRow) return;
  const size_t row = (size_t)row0 + (size_t)hk * p.page;
  k.put(p, p.k, p.ks, row, lane);
  v.put(p, p.v, p.vs, row, lane);
}

// Rotated query element i of head h.
__device__ __forceinline__ float query(const PagedP& p, int b, int h, int t, int i) {
  const int half = p.HD / 2;
  const long long qo = (long long)b * p.q.sb + (long long)h * p.q.sh;
  const float x = ldf(p.q.p, qo + i * p.q.sd, p.q.dt);
  if (!p.cos) return x;
  const int f = i < half ? i : i - half;
  const float c = __ldg(p.cos + (size_t)t * half + f), s = __ldg(p.sin + (size_t)t * half + f);
  const float y = ldf(p.q.p, qo + (i < half ? i + half : f) * p.q.sd, p.q.dt);
  return i < half ? x * c - y * s : y * s + x * c;
}

// τ of the key at `pos` into its slot of the exported row: LOCAL slot
// W − (t − pos), GLOBAL column t − pos.
__device__ __forceinline__ void put_tau(const PagedP& p, size_t bh, int t, unsigned pos, float tau) {
  const unsigned back = (unsigned)t - pos;
  const unsigned slot = p.mode == BOZO_MODE_LOCAL ? (unsigned)p.W - back : back;
  if (slot < (unsigned)p.tw) stf(p.tau, (long long)(bh * p.tw + slot), p.tau_dt, tau);
}
// Slots without a key.
__device__ __forceinline__ void clear_tau(const PagedP& p, size_t bh, unsigned n, int i, int step) {
  const unsigned first = p.mode == BOZO_MODE_LOCAL ? 0u : min(n, (unsigned)p.tw);
  const unsigned last = p.mode == BOZO_MODE_LOCAL ? (unsigned)p.W - n : (unsigned)p.tw;
  for (unsigned s = first + i; s < last; s += step) stf(p.tau, (long long)(bh * p.tw + s), p.tau_dt, 0.f);
}

}  // namespace bozo
