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
  const size_t row = row0 + (size_t)h * p.page;
  put_row(p, p.kn, p.k, p.ks, n, h, pos, row, p.cos != nullptr, lane);
  put_row(p, p.vn, p.v, p.vs, n, h, pos, row, false, lane);
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

// ─────────────── vector path: HD 32, 64, 128, unit element stride, aligned rows ───────────────
// HD/8 lanes hold one row: of a key the dimensions 4l … 4l+3 and HD/2 + 4l …, so a
// lane has both halves of its rotations, of a value 8l … 8l+7.  A group of lanes
// takes NH heads of its token: their loads are in flight together and the
// token's place is looked up once for all of them.
template <int DT> struct PageT;
template <> struct PageT<BOZO_DT_F32> { using type = float; };
template <> struct PageT<BOZO_DT_BF16> { using type = __nv_bfloat16; };
template <> struct PageT<BOZO_DT_F16> { using type = __half; };
template <> struct PageT<BOZO_DT_F8E4M3> { using type = unsigned char; };
template <> struct PageT<BOZO_DT_I8> { using type = unsigned char; };

template <int BYTES> struct Bytes;
template <> struct Bytes<4> { using type = unsigned; };
template <> struct Bytes<8> { using type = uint2; };
template <> struct Bytes<16> { using type = uint4; };

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f(float& y, float x) { y = x; }
__device__ __forceinline__ void from_f(__nv_bfloat16& y, float x) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f(__half& y, float x) { y = __float2half_rn(x); }

// N elements of type T, N·sizeof(T) bytes aligned to themselves (at most 16)
template <typename T, int N> struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack { T e[N]; };

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> ld_pack(const T* p) {
  Pack<T, N> x;
  constexpr int B = N * sizeof(T) < 16 ? N * sizeof(T) : 16;
  using V = typename Bytes<B>::type;
#pragma unroll
  for (int i = 0; i < (int)(N * sizeof(T)) / B; ++i)
    reinterpret_cast<V*>(&x)[i] = __ldg(reinterpret_cast<const V*>(p) + i);
  return x;
}
template <typename T, int N>
__device__ __forceinline__ void st_pack(T* p, const Pack<T, N>& x) {
  constexpr int B = N * sizeof(T) < 16 ? N * sizeof(T) : 16;
  using V = typename Bytes<B>::type;
#pragma unroll
  for (int i = 0; i < (int)(N * sizeof(T)) / B; ++i)
    reinterpret_cast<V*>(p)[i] = reinterpret_cast<const V*>(&x)[i];
}

// N fp32 numbers as a page holds them (for codes: times inv; |x·inv| ≤ top up to
// rounding, which no code passes)
template <int DT, int N>
__device__ __forceinline__ void st_page(typename PageT<DT>::type* p, const float* x, float inv) {
  using T = typename PageT<DT>::type;
  Pack<T, N> y;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (DT == BOZO_DT_F8E4M3 || DT == BOZO_DT_I8) y.e[i] = quant_code(x[i], inv, DT);
    else from_f(y.e[i], x[i]);
  }
  st_pack(p, y);
}

template <int DT, typename I, int NH>
__global__ void __launch_bounds__(kThreads) paged_write_vec(PagedP p, int lanes, FastDiv units) {
  using T = typename PageT<DT>::type;
  constexpr bool Q = DT == BOZO_DT_F8E4M3 || DT == BOZO_DT_I8;
  const int L = 1 << lanes, l = threadIdx.x & (L - 1);
  const unsigned nu = (unsigned)(p.Hk + NH - 1) / NH;  // units of a token
  const unsigned g = (blockIdx.x * kThreads + threadIdx.x) >> lanes;
  const unsigned n = fast_div(g, units);
  const int h0 = (int)(g - n * nu) * NH;
  int b = 0;
  unsigned pos = 0, end = 0, row0 = kNoRow;
  if (n < (unsigned)p.rows && paged_place(p, (int)n, b, pos, end) && !(end > p.cap && pos < end - p.cap)) {
    if (p.cos && pos >= (unsigned)p.rope_len) {
      if (l == 0) atomicCAS(p.err, 0, kErrPaged | 1);
    } else {
      row0 = paged_row(p, b, pos);
    }
  }
  const bool live = row0 != kNoRow;
  const int HD = L * 8, half = L * 4;
  Pack<I, 4> ka[NH], kb[NH];
  Pack<I, 8> va[NH];
  float4 cs{}, sn{};
#pragma unroll
  for (int i = 0; i < NH; ++i)
    if (live && h0 + i < p.Hk) {
      const I* k = static_cast<const I*>(p.kn.p) + n * p.kn.sb + (h0 + i) * p.kn.sh;
      const I* v = static_cast<const I*>(p.vn.p) + n * p.vn.sb + (h0 + i) * p.vn.sh;
      ka[i] = ld_pack<I, 4>(k + 4 * l);
      kb[i] = ld_pack<I, 4>(k + half + 4 * l);
      va[i] = ld_pack<I, 8>(v + 8 * l);
    }
  if (live && p.cos) {
    cs = __ldg(reinterpret_cast<const float4*>(p.cos + (size_t)pos * half) + l);
    sn = __ldg(reinterpret_cast<const float4*>(p.sin + (size_t)pos * half) + l);
  }
  const float c[4] = {cs.x, cs.y, cs.z, cs.w}, s[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const bool on = live && h0 + i < p.Hk;
    float k[8], v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = to_f(ka[i].e[e]), y = to_f(kb[i].e[e]);
      k[e] = p.cos ? __fsub_rn(__fmul_rn(x, c[e]), __fmul_rn(y, s[e])) : x;
      k[4 + e] = p.cos ? __fadd_rn(__fmul_rn(x, s[e]), __fmul_rn(y, c[e])) : y;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f(va[i].e[e]);
    const size_t row = (size_t)row0 + (size_t)(h0 + i) * p.page;
    float kinv = 1.f, vinv = 1.f;
    if constexpr (Q) {
      constexpr float top = DT == BOZO_DT_I8 ? 127.f : 448.f;
      unsigned km = 0, vm = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        km = max(km, __float_as_uint(k[e]) & 0x7fffffffu);
        vm = max(vm, __float_as_uint(v[e]) & 0x7fffffffu);
      }
      for (int o = L / 2; o; o >>= 1) {
        km = max(km, __shfl_xor_sync(0xffffffffu, km, o));
        vm = max(vm, __shfl_xor_sync(0xffffffffu, vm, o));
      }
      float ksc, vsc;
      quant_scale(km, top, ksc, kinv);
      quant_scale(vm, top, vsc, vinv);
      if (on && l == 0) {
        p.ks[row] = ksc;
        p.vs[row] = vsc;
      }
    }
    if (on) {
      T* kp = static_cast<T*>(p.k) + row * HD;
      st_page<DT, 4>(kp + 4 * l, k, kinv);
      st_page<DT, 4>(kp + half + 4 * l, k + 4, kinv);
      st_page<DT, 8>(static_cast<T*>(p.v) + row * HD + 8 * l, v, vinv);
    }
  }
}

template <int DT, typename O, int NH>
__global__ void __launch_bounds__(kThreads) paged_read_vec(PagedP p, int lanes, FastDiv units) {
  using T = typename PageT<DT>::type;
  constexpr bool Q = DT == BOZO_DT_F8E4M3 || DT == BOZO_DT_I8;
  const int L = 1 << lanes, l = threadIdx.x & (L - 1), HD = L * 8;
  const unsigned nu = (unsigned)(p.Hk + NH - 1) / NH;
  const unsigned g = (blockIdx.x * kThreads + threadIdx.x) >> lanes;
  const unsigned n = fast_div(g, units);
  const int h0 = (int)(g - n * nu) * NH;
  if (n >= (unsigned)p.rows) return;
  int b = 0;
  unsigned pos = 0, end = 0, row0 = kNoRow;
  if (paged_place(p, (int)n, b, pos, end)) row0 = paged_row(p, b, pos);
  Pack<T, 8> k[NH], v[NH];
  float ks[NH], vs[NH];
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    ks[i] = vs[i] = 1.f;
    if (row0 != kNoRow && h0 + i < p.Hk) {
      const size_t row = (size_t)row0 + (size_t)(h0 + i) * p.page;
      k[i] = ld_pack<T, 8>(static_cast<const T*>(p.k) + row * HD + 8 * l);
      v[i] = ld_pack<T, 8>(static_cast<const T*>(p.v) + row * HD + 8 * l);
      if constexpr (Q) {
        ks[i] = __ldg(p.ks + row);
        vs[i] = __ldg(p.vs + row);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    if (h0 + i >= p.Hk) break;
    Pack<O, 8> x, y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a = 0.f, d = 0.f;
      if (row0 != kNoRow) {
        if constexpr (Q) {
          a = __fmul_rn(code_value(k[i].e[e], DT), ks[i]);
          d = __fmul_rn(code_value(v[i].e[e], DT), vs[i]);
        } else {
          a = to_f(k[i].e[e]);
          d = to_f(v[i].e[e]);
        }
      }
      from_f(x.e[e], a);
      from_f(y.e[e], d);
    }
    const size_t at = ((size_t)n * p.Hk + h0 + i) * HD + 8 * l;
    st_pack(static_cast<O*>(p.k_out) + at, x);
    st_pack(static_cast<O*>(p.v_out) + at, y);
  }
}

// log2 of the lanes a row takes, or −1 where the vector kernels do not apply
int vec_lanes(const PagedP& p) { return p.HD == 32 ? 2 : p.HD == 64 ? 3 : p.HD == 128 ? 4 : -1; }

bool vec_input(const DevT4& t, int dt) {
  const long long e = dt == BOZO_DT_F32 ? 4 : 2;
  return t.dt == dt && t.sd == 1 && !((reinterpret_cast<uintptr_t>(t.p) | (t.sb * e) | (t.sh * e)) & 15);
}

// Heads of a group: one while the rows do not fill the device, else four
constexpr int kGroupHeads = 4;
bool few_rows(const PagedP& p, int lanes) { return ((p.rows * p.Hk) << lanes) <= 148LL * 2048; }

template <typename F>
cudaError_t launch_vec(const PagedP& p, int lanes, int nh, cudaStream_t st, F kern) {
  const unsigned nu = (unsigned)((p.Hk + nh - 1) / nh);
  const long long groups = p.rows * nu;
  const long long per = kThreads >> lanes;
  kern<<<(unsigned)((groups + per - 1) / per), kThreads, 0, st>>>(p, lanes, make_fastdiv(nu));
  return cudaGetLastError();
}

template <int DT, typename I>
cudaError_t write_vec(const PagedP& p, int lanes, cudaStream_t st) {
  if (few_rows(p, lanes)) return launch_vec(p, lanes, 1, st, paged_write_vec<DT, I, 1>);
  return launch_vec(p, lanes, kGroupHeads, st, paged_write_vec<DT, I, kGroupHeads>);
}
template <int DT>
cudaError_t write_vec(const PagedP& p, int lanes, cudaStream_t st) {
  switch (p.kn.dt) {
    case BOZO_DT_F32: return write_vec<DT, float>(p, lanes, st);
    case BOZO_DT_BF16: return write_vec<DT, __nv_bfloat16>(p, lanes, st);
    default: return write_vec<DT, __half>(p, lanes, st);
  }
}
template <int DT, typename O>
cudaError_t read_vec(const PagedP& p, int lanes, cudaStream_t st) {
  if (few_rows(p, lanes)) return launch_vec(p, lanes, 1, st, paged_read_vec<DT, O, 1>);
  return launch_vec(p, lanes, kGroupHeads, st, paged_read_vec<DT, O, kGroupHeads>);
}
template <int DT>
cudaError_t read_vec(const PagedP& p, int lanes, cudaStream_t st) {
  switch (p.out_dt) {
    case BOZO_DT_F32: return read_vec<DT, float>(p, lanes, st);
    case BOZO_DT_BF16: return read_vec<DT, __nv_bfloat16>(p, lanes, st);
    default: return read_vec<DT, __half>(p, lanes, st);
  }
}

}  // namespace

cudaError_t launch_paged_write(const PagedP& p, cudaStream_t st) {
  const int lanes = vec_lanes(p);
  const bool tables = !p.cos || !((reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin)) & 15);
  // groups are numbered in 32 bits
  if (lanes >= 0 && tables && vec_input(p.kn, p.kn.dt) && vec_input(p.vn, p.kn.dt) &&
      ((p.rows * p.Hk) << lanes) < (1LL << 31)) {
    switch (p.dt) {
      case BOZO_DT_F32: return write_vec<BOZO_DT_F32>(p, lanes, st);
      case BOZO_DT_BF16: return write_vec<BOZO_DT_BF16>(p, lanes, st);
      case BOZO_DT_F16: return write_vec<BOZO_DT_F16>(p, lanes, st);
      case BOZO_DT_F8E4M3: return write_vec<BOZO_DT_F8E4M3>(p, lanes, st);
      default: return write_vec<BOZO_DT_I8>(p, lanes, st);
    }
  }
  const long long warps = p.rows * p.Hk;
  paged_write_any<<<(unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_paged_read(const PagedP& p, cudaStream_t st) {
  const int lanes = vec_lanes(p);
  if (lanes >= 0 && !((reinterpret_cast<uintptr_t>(p.k_out) | reinterpret_cast<uintptr_t>(p.v_out)) & 15) &&
      ((p.rows * p.Hk) << lanes) < (1LL << 31)) {
    switch (p.dt) {
      case BOZO_DT_F32: return read_vec<BOZO_DT_F32>(p, lanes, st);
      case BOZO_DT_BF16: return read_vec<BOZO_DT_BF16>(p, lanes, st);
      case BOZO_DT_F16: return read_vec<BOZO_DT_F16>(p, lanes, st);
      case BOZO_DT_F8E4M3: return read_vec<BOZO_DT_F8E4M3>(p, lanes, st);
      default: return read_vec<BOZO_DT_I8>(p, lanes, st);
    }
  }
  const long long warps = p.rows * p.Hk;
  paged_read_any<<<(unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace bozo
