// paged.cu — writing keys and values into a paged cache and reading them back
// (bozo_paged_write, bozo_paged_read).
//
// A row is one token's key or value of one head.  Written keys are rotated,
// k'[i] = k[i]·cos − k[i+HD/2]·sin, k'[i+HD/2] = k[i]·sin + k[i+HD/2]·cos, each
// product and sum rounded on its own in fp32 (the plain formula's bits, so a
// code does not depend on how the compiler contracts it), then rounded once to
// the page's type, or quantised with the row's own scale.
#include "paged.cuh"

namespace bozo {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ unsigned warp_max(unsigned v) { return __reduce_max_sync(0xffffffffu, v); }

// One warp per (row, head): any head width, types and strides.
__global__ void __launch_bounds__(kThreads) paged_write_any(PagedP p) {
  const int lane = threadIdx.x & 31;
  const long long g = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (g >= p.rows * p.Hk) return;
  const int n = (int)(g / p.Hk), h = (int)(g - (long long)n * p.Hk);
  int b;
  unsigned pos, end;
  if (!paged_place(p, n, b, pos, end)) return;
  if (end > p.cap && pos < end - p.cap) return;  // overwritten by a later row of this call
  if (p.cos && pos >= (unsigned)p.rope_len) {
    if (lane == 0) atomicCAS(p.err, 0, kErrPaged | 1);
    return;
  }
  const unsigned row0 = paged_row(p, b, pos);
  if (row0 == kNoRow) return;
  const size_t row = row0 + (size_t)h * p.page, at = row * p.HD;
  const int HD = p.HD, half = HD / 2;
  const long long ko = n * p.kn.sb + h * p.kn.sh, vo = n * p.vn.sb + h * p.vn.sh;
  const float* c = p.cos + (size_t)pos * half;
  const float* s = p.sin + (size_t)pos * half;
  auto key = [&](int d) {
    const float x = ldf(p.kn.p, ko + d * p.kn.sd, p.kn.dt);
    if (!p.cos) return x;
    if (d < half) {
      const float y = ldf(p.kn.p, ko + (d + half) * p.kn.sd, p.kn.dt);
      return __fsub_rn(__fmul_rn(x, c[d]), __fmul_rn(y, s[d]));
    }
    const float y = ldf(p.kn.p, ko + (d - half) * p.kn.sd, p.kn.dt);
    return __fadd_rn(__fmul_rn(y, s[d - half]), __fmul_rn(x, c[d - half]));
  };
  auto val = [&](int d) { return ldf(p.vn.p, vo + d * p.vn.sd, p.vn.dt); };
  if (p.dt <= BOZO_DT_F16) {
    for (int d = lane; d < HD; d += 32) {
      stf(p.k, (long long)(at + d), p.dt, key(d));
      stf(p.v, (long long)(at + d), p.dt, val(d));
    }
    return;
  }
  const float top = p.dt == BOZO_DT_I8 ? 127.f : 448.f;
  unsigned ka = 0, va = 0;
  for (int d = lane; d < HD; d += 32) {
    ka = max(ka, __float_as_uint(key(d)) & 0x7fffffffu);
    va = max(va, __float_as_uint(val(d)) & 0x7fffffffu);
  }
  float ksc, kinv, vsc, vinv;
  quant_scale(warp_max(ka), top, ksc, kinv);
  quant_scale(warp_max(va), top, vsc, vinv);
  for (int d = lane; d < HD; d += 32) {
    static_cast<unsigned char*>(p.k)[at + d] = quant_code(key(d), kinv, p.dt);
    static_cast<unsigned char*>(p.v)[at + d] = quant_code(val(d), vinv, p.dt);
  }
  if (lane == 0) {
    p.ks[row] = ksc;
    p.vs[row] = vsc;
  }
}

// One warp per (row, head).
__global__ void __launch_bounds__(kThreads) paged_read_any(PagedP p) {
  const int lane = threadIdx.x & 31;
  const long long g = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (g >= p.rows * p.Hk) return;
  const int n = (int)(g / p.Hk), h = (int)(g - (long long)n * p.Hk);
  int b;
  unsigned pos, end, row0 = kNoRow;
  if (paged_place(p, n, b, pos, end)) row0 = paged_row(p, b, pos);
  const size_t row = row0 + (size_t)h * p.page, at = row * p.HD;
  for (int d = lane; d < p.HD; d += 32) {
    float k = 0.f, v = 0.f;
    if (row0 != kNoRow) {
      k = ld_page(p.k, at + d, p.dt);
      v = ld_page(p.v, at + d, p.dt);
      if (p.ks) {
        k = __fmul_rn(k, p.ks[row]);
        v = __fmul_rn(v, p.vs[row]);
      }
    }
    stf(p.k_out, g * p.HD + d, p.out_dt, k);
    stf(p.v_out, g * p.HD + d, p.out_dt, v);
  }
}

}  // namespace

cudaError_t launch_paged_write(const PagedP& p, cudaStream_t st) {
  const long long warps = p.rows * p.Hk;
  paged_write_any<<<(unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_paged_read(const PagedP& p, cudaStream_t st) {
  const long long warps = p.rows * p.Hk;
  paged_read_any<<<(unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace bozo
