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

constexpr int kThreads = 128;

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
  NewRow(p, p.kn, n, h, pos, p.cos != nullptr, lane).put(p, p.k, p.ks, row, lane);
  NewRow(p, p.vn, n, h, pos, false, lane).put(p, p.v, p.vs, row, lane);
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
// A block takes `rows` consecutive rows.  Their sequence is found by all its threads
// at once (one of B compares holds), each row's place by one thread; then groups of
// HD/16 lanes go through the heads' keys and values of one row, sixteen elements a
// lane: dimensions 8l … 8l+7 of either half of the row, so a lane has both halves of
// its rotations, whose cosines and sines it loads once for all heads.  A head's key
// and value are in flight together.
template <int DT> struct PageT;
template <> struct PageT<BOZO_DT_F32> { using type = float; };
template <> struct PageT<BOZO_DT_BF16> { using type = __nv_bfloat16; };
template <> struct PageT<BOZO_DT_F16> { using type = __half; };
template <> struct PageT<BOZO_DT_F8E4M3> { using type = unsigned char; };
template <> struct PageT<BOZO_DT_I8> { using type = unsigned char; };

// Eight elements of type T: 8, 16 or 32 bytes, moved in pieces of up to 16.
template <typename T> struct Eight {
  static constexpr int words = 8 * sizeof(T) / 4;
  unsigned w[words];
};
template <typename T>
__device__ __forceinline__ Eight<T> ld8(const T* p) {
  Eight<T> x;
  if constexpr (sizeof(T) == 1) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    x.w[0] = v.x; x.w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < Eight<T>::words / 4; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      x.w[4 * i] = v.x; x.w[4 * i + 1] = v.y; x.w[4 * i + 2] = v.z; x.w[4 * i + 3] = v.w;
    }
  }
  return x;
}
template <typename T>
__device__ __forceinline__ void st8(T* p, const Eight<T>& x) {
  if constexpr (sizeof(T) == 1) {
    *reinterpret_cast<uint2*>(p) = make_uint2(x.w[0], x.w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < Eight<T>::words / 4; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(x.w[4 * i], x.w[4 * i + 1], x.w[4 * i + 2], x.w[4 * i + 3]);
  }
}
__device__ __forceinline__ void widen(const Eight<float>& x, float* y) {
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(x.w[i]);
}
__device__ __forceinline__ void widen(const Eight<__nv_bfloat16>& x, float* y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = __uint_as_float(x.w[i] << 16);
    y[2 * i + 1] = __uint_as_float(x.w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void widen(const Eight<__half>& x, float* y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x.w[i]));
    y[2 * i] = f.x;
    y[2 * i + 1] = f.y;
  }
}
template <int DT>
__device__ __forceinline__ void widen_codes(const Eight<unsigned char>& x, float* y) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (DT == BOZO_DT_F8E4M3) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x.w[i] >> (16 * j)), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        y[4 * i + 2 * j] = f.x;
        y[4 * i + 2 * j + 1] = f.y;
      }
    } else {
      // 2^23 + (code + 128) has those low bits
      const unsigned u = x.w[i] ^ 0x80808080u;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        y[4 * i + j] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 + j)) - 8388736.f;
    }
  }
}
__device__ __forceinline__ void narrow(Eight<float>& x, const float* y) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x.w[i] = __float_as_uint(y[i]);
}
__device__ __forceinline__ void narrow(Eight<__nv_bfloat16>& x, const float* y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
    x.w[i] = *reinterpret_cast<const unsigned*>(&h);
  }
}
__device__ __forceinline__ void narrow(Eight<__half>& x, const float* y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
    x.w[i] = *reinterpret_cast<const unsigned*>(&h);
  }
}
// Two products (sums) in one instruction, each rounded as on its own.  A pair of
// products must not run into a pair of sums, which would contract them: where one
// follows, the products are single instructions.
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b, float c, float d) {
  asm("{.reg .b64 p, q; mov.b64 p, {%2, %3}; mov.b64 q, {%4, %5}; mul.rn.f32x2 p, p, q; mov.b64 {%0, %1}, p;}"
      : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b, float c, float d) {
  asm("{.reg .b64 p, q; mov.b64 p, {%2, %3}; mov.b64 q, {%4, %5}; add.rn.f32x2 p, p, q; mov.b64 {%0, %1}, p;}"
      : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d));
}

// Codes of y · inv (|y·inv| ≤ top up to a rounding that no code passes); all zero
// where inv is.
template <int DT>
__device__ __forceinline__ void narrow_codes(Eight<unsigned char>& x, const float* y, float inv) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    unsigned w;
    float z[4];
    if constexpr (DT == BOZO_DT_F8E4M3) {
      mul2(z[0], z[1], y[4 * i], y[4 * i + 1], inv, inv);
      mul2(z[2], z[3], y[4 * i + 2], y[4 * i + 3], inv, inv);
      const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(z[0], z[1]), __NV_SATFINITE, __NV_E4M3);
      const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(z[2], z[3]), __NV_SATFINITE, __NV_E4M3);
      w = lo | hi << 16;
    } else {
      // 1.5·2^23 + z: the low byte is z rounded to even
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = __fmul_rn(y[4 * i + j], inv);
      add2(z[0], z[1], z[0], z[1], 12582912.f, 12582912.f);
      add2(z[2], z[3], z[2], z[3], 12582912.f, 12582912.f);
      w = __byte_perm(__byte_perm(__float_as_uint(z[0]), __float_as_uint(z[1]), 0x0040),
                      __byte_perm(__float_as_uint(z[2]), __float_as_uint(z[3]), 0x0040), 0x5410);
    }
    x.w[i] = inv == 0.f ? 0u : w;
  }
}
__device__ __forceinline__ float max_abs(float a, float b) {  // ± max(|a|, |b|); a NaN stays
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The places of a block's rows n0 … n0 + rows − 1: row numbers (head 0) and
// positions in shared memory.
template <bool WRITE>
__device__ __forceinline__ void block_places(const PagedP& p, unsigned n0, int rows, unsigned* srow, unsigned* spos) {
  __shared__ int found;
  if (p.cu) {
    // the sequence of the block's first row, or the first one if that row comes before it
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < p.B; i += kThreads) {
      const int lo = __ldg(p.cu + i), hi = __ldg(p.cu + i + 1);
      if (((i == 0) | (lo <= (int)n0)) & ((int)n0 < hi)) found = i;
    }
    __syncthreads();
  }
  for (int r = threadIdx.x; r < rows; r += kThreads) {
    const unsigned n = n0 + r;
    unsigned row = kNoRow, pos = 0;
    if (n < (unsigned)p.rows) {
      int b = (int)n, first = (int)n, next = (int)n + 1;
      if (p.cu) {
        b = found;
        if (b >= 0) {
          while (b < p.B && (next = __ldg(p.cu + b + 1)) <= (int)n) ++b;
          if (b < p.B) first = __ldg(p.cu + b);
          if (b == p.B || first > (int)n) b = -1;
        }
      }
      const int t = b < 0 ? -1 : __ldg(p.len + b);
      if (t >= 0) {
        pos = (unsigned)t + (n - (unsigned)first);
        const unsigned end = (unsigned)t + (unsigned)(next - first);
        if (pos <= 0x7fffffffu && !(WRITE && end > p.cap && pos < end - p.cap)) {
          if (WRITE && p.cos && pos >= (unsigned)p.rope_len) atomicCAS(p.err, 0, kErrPaged | 1);
          else row = paged_row(p, b, pos);
        }
      }
    }
    srow[r] = row;
    if (WRITE) spos[r] = pos;
  }
  __syncthreads();
}

constexpr int kMaxRows = kThreads / 2;  // rows of a block, at most
// What hides the chain from a sequence's offset to its rows is other blocks, so the
// kernels keep to the registers that let this many stay on an SM (42136 rows of
// 16 heads from bf16 to e4m3 and back: 101 µs; with 16 reading blocks 104, with six
// writing ones 110; a head's key and value one after the other 109).
constexpr int kWriteBlocks = 9, kReadBlocks = 12;

// Sixteen elements a lane of one key (KEY) or value into its row.
template <int DT, typename I, bool KEY>
__device__ __forceinline__ void write_head(const PagedP& p, const Eight<I>& xl, const Eight<I>& xh, unsigned row, int L,
                                           int l, unsigned group, const float* c, const float* s) {
  using T = typename PageT<DT>::type;
  constexpr bool Q = sizeof(T) == 1;
  const int half = L * 8, HD = half * 2;
  float x[16];
  widen(xl, x);
  widen(xh, x + 8);
  if (KEY && p.cos) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float d0 = __fmul_rn(x[i], s[i]), d1 = __fmul_rn(x[i + 1], s[i + 1]);
      const float e0 = __fmul_rn(x[8 + i], c[i]), e1 = __fmul_rn(x[9 + i], c[i + 1]);
      add2(x[i], x[i + 1], __fmul_rn(x[i], c[i]), __fmul_rn(x[i + 1], c[i + 1]), __fmul_rn(x[8 + i], -s[i]),
           __fmul_rn(x[9 + i], -s[i + 1]));
      add2(x[8 + i], x[9 + i], d0, d1, e0, e1);
    }
  }
  Eight<T> yl, yh;
  if constexpr (Q) {
    float a = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) a = max_abs(a, x[i]);
    for (int o = L / 2; o; o >>= 1) a = max_abs(a, __shfl_xor_sync(group, a, o));
    float scale, inv;
    quant_scale(__float_as_uint(a) & 0x7fffffffu, DT == BOZO_DT_I8 ? 127.f : 448.f, scale, inv);
    if (l == 0) (KEY ? p.ks : p.vs)[row] = scale;
    narrow_codes<DT>(yl, x, inv);
    narrow_codes<DT>(yh, x + 8, inv);
  } else {
    narrow(yl, x);
    narrow(yh, x + 8);
  }
  T* to = static_cast<T*>(KEY ? p.k : p.v) + (size_t)row * HD + 8 * l;
  st8(to, yl);
  st8(to + half, yh);
}

template <int DT, typename I>
__global__ void __launch_bounds__(kThreads, kWriteBlocks) paged_write_vec(PagedP p, int lanes, int rows) {
  __shared__ unsigned srow[kMaxRows], spos[kMaxRows];
  const int L = 1 << lanes, l = threadIdx.x & (L - 1), half = L * 8;
  const int per = (kThreads >> lanes) / rows;  // groups of a row
  const int g = threadIdx.x >> lanes, r = g / per, sub = g - r * per;
  const unsigned n0 = blockIdx.x * rows, n = n0 + r;
  block_places<true>(p, n0, rows, srow, spos);
  const unsigned row0 = srow[r];
  if (row0 == kNoRow) return;
  float c[8], s[8];
  if (p.cos && sub < p.Hk) {
    const size_t at = (size_t)spos[r] * half + 8 * l;
    widen(ld8(p.cos + at), c);
    widen(ld8(p.sin + at), s);
  }
  const I* kf = static_cast<const I*>(p.kn.p) + n * p.kn.sb + sub * p.kn.sh + 8 * l;
  const I* vf = static_cast<const I*>(p.vn.p) + n * p.vn.sb + sub * p.vn.sh + 8 * l;
  unsigned row = row0 + (unsigned)sub * (unsigned)p.page;  // rows are numbered in 32 bits
  const long long ks = per * p.kn.sh, vs = per * p.vn.sh;
  const unsigned group = ((1u << L) - 1u) << (threadIdx.x & 31 & ~(L - 1));
#pragma unroll 1
  for (int h = sub; h < p.Hk; h += per, kf += ks, vf += vs, row += (unsigned)(per * p.page)) {
    const Eight<I> kl = ld8(kf), kh = ld8(kf + half), vl = ld8(vf), vh = ld8(vf + half);
    write_head<DT, I, true>(p, kl, kh, row, L, l, group, c, s);
    write_head<DT, I, false>(p, vl, vh, row, L, l, group, c, s);
  }
}

template <int DT, typename O>
__global__ void __launch_bounds__(kThreads, kReadBlocks) paged_read_vec(PagedP p, int lanes, int rows) {
  using T = typename PageT<DT>::type;
  constexpr bool Q = sizeof(T) == 1;
  __shared__ unsigned srow[kMaxRows];
  const int L = 1 << lanes, l = threadIdx.x & (L - 1), half = L * 8, HD = half * 2;
  const int per = (kThreads >> lanes) / rows;
  const int g = threadIdx.x >> lanes, r = g / per, sub = g - r * per;
  const unsigned n0 = blockIdx.x * rows, n = n0 + r;
  block_places<false>(p, n0, rows, srow, nullptr);
  const unsigned row0 = srow[r];
  if (n >= (unsigned)p.rows) return;
  O* to[2] = {static_cast<O*>(p.k_out) + ((size_t)n * p.Hk + sub) * HD + 8 * l,
              static_cast<O*>(p.v_out) + ((size_t)n * p.Hk + sub) * HD + 8 * l};
  unsigned row = row0 + (unsigned)sub * (unsigned)p.page;
#pragma unroll 1
  for (int h = sub; h < p.Hk; h += per, row += (unsigned)(per * p.page)) {
    Eight<T> lo[2], hi[2];
    float scale[2] = {1.f, 1.f};
    if (row0 != kNoRow) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const T* at = static_cast<const T*>(j ? p.v : p.k) + (size_t)row * HD + 8 * l;
        lo[j] = ld8(at);
        hi[j] = ld8(at + half);
        if constexpr (Q) scale[j] = __ldg((j ? p.vs : p.ks) + row);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float x[16];
      if (row0 != kNoRow) {
        if constexpr (Q) {
          widen_codes<DT>(lo[j], x);
          widen_codes<DT>(hi[j], x + 8);
#pragma unroll
          for (int i = 0; i < 16; i += 2) mul2(x[i], x[i + 1], x[i], x[i + 1], scale[j], scale[j]);
        } else {
          widen(lo[j], x);
          widen(hi[j], x + 8);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.f;
      }
      Eight<O> yl, yh;
      narrow(yl, x);
      narrow(yh, x + 8);
      st8(to[j], yl);
      st8(to[j] + half, yh);
      to[j] += per * HD;
    }
  }
}

// log2 of the lanes a row takes, or −1 where the vector kernels do not apply
int vec_lanes(const PagedP& p) { return p.HD == 32 ? 1 : p.HD == 64 ? 2 : p.HD == 128 ? 3 : -1; }

bool vec_input(const DevT4& t, int dt) {
  const long long e = dt == BOZO_DT_F32 ? 4 : 2;
  return t.dt == dt && t.sd == 1 && !((reinterpret_cast<uintptr_t>(t.p) | (t.sb * e) | (t.sh * e)) & 15);
}

// Rows of a block: as many as leave each group at most 8 keys and values, fewer
// where that gives less than six blocks an SM, down to one (the same prompts: 101 µs
// at 8, 105 at 4; reading 79868 rows out of e4m3 86 at 8 and 90 at 16).
constexpr int kGroupHeads = 8;
int block_rows(const PagedP& p, int lanes, int sms) {
  const int groups = kThreads >> lanes;
  int per = 1;
  while (per < groups && per < 2 * p.Hk && (per * kGroupHeads < 2 * p.Hk || p.rows * per < 6LL * sms * groups)) per *= 2;
  return groups / per;
}

template <typename F>
cudaError_t launch_vec(const PagedP& p, int lanes, int sms, cudaStream_t st, F kern) {
  const int rows = block_rows(p, lanes, sms);
  kern<<<(unsigned)((p.rows + rows - 1) / rows), kThreads, 0, st>>>(p, lanes, rows);
  return cudaGetLastError();
}

template <int DT>
cudaError_t write_vec(const PagedP& p, int lanes, int sms, cudaStream_t st) {
  switch (p.kn.dt) {
    case BOZO_DT_F32: return launch_vec(p, lanes, sms, st, paged_write_vec<DT, float>);
    case BOZO_DT_BF16: return launch_vec(p, lanes, sms, st, paged_write_vec<DT, __nv_bfloat16>);
    default: return launch_vec(p, lanes, sms, st, paged_write_vec<DT, __half>);
  }
}
template <int DT>
cudaError_t read_vec(const PagedP& p, int lanes, int sms, cudaStream_t st) {
  switch (p.out_dt) {
    case BOZO_DT_F32: return launch_vec(p, lanes, sms, st, paged_read_vec<DT, float>);
    case BOZO_DT_BF16: return launch_vec(p, lanes, sms, st, paged_read_vec<DT, __nv_bfloat16>);
    default: return launch_vec(p, lanes, sms, st, paged_read_vec<DT, __half>);
  }
}

}  // namespace

cudaError_t launch_paged_write(const PagedP& p, int sms, cudaStream_t st) {
  const int lanes = vec_lanes(p);
  const bool tables = !p.cos || !((reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin)) & 15);
  if (lanes >= 0 && tables && vec_input(p.kn, p.kn.dt) && vec_input(p.vn, p.kn.dt)) {
    switch (p.dt) {
      case BOZO_DT_F32: return write_vec<BOZO_DT_F32>(p, lanes, sms, st);
      case BOZO_DT_BF16: return write_vec<BOZO_DT_BF16>(p, lanes, sms, st);
      case BOZO_DT_F16: return write_vec<BOZO_DT_F16>(p, lanes, sms, st);
      case BOZO_DT_F8E4M3: return write_vec<BOZO_DT_F8E4M3>(p, lanes, sms, st);
      default: return write_vec<BOZO_DT_I8>(p, lanes, sms, st);
    }
  }
  const long long blocks = (p.rows * p.Hk + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  paged_write_any<<<(unsigned)blocks, kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_paged_read(const PagedP& p, int sms, cudaStream_t st) {
  const int lanes = vec_lanes(p);
  if (lanes >= 0 && !((reinterpret_cast<uintptr_t>(p.k_out) | reinterpret_cast<uintptr_t>(p.v_out)) & 15)) {
    switch (p.dt) {
      case BOZO_DT_F32: return read_vec<BOZO_DT_F32>(p, lanes, sms, st);
      case BOZO_DT_BF16: return read_vec<BOZO_DT_BF16>(p, lanes, sms, st);
      case BOZO_DT_F16: return read_vec<BOZO_DT_F16>(p, lanes, sms, st);
      case BOZO_DT_F8E4M3: return read_vec<BOZO_DT_F8E4M3>(p, lanes, sms, st);
      default: return read_vec<BOZO_DT_I8>(p, lanes, sms, st);
    }
  }
  const long long blocks = (p.rows * p.Hk + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  paged_read_any<<<(unsigned)blocks, kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace bozo
