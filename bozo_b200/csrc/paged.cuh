// paged.cuh — parameter block and launchers of the paged-cache kernels
// (paged.cu, paged_decode.cu) and the device helpers they share.
#pragma once

#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace bozo {

constexpr int kErrPaged = 0x900;  // device error codes: | 1 position, | 2 page

struct PagedP {
  // cache
  void* k;
  void* v;
  float* ks;
  float* vs;
  unsigned char* kg;  // 4-bit rows: e4m3 scales of 16 elements
  unsigned char* vg;
  int dt, P, Hk, page, HD, B, M;
  unsigned cap;             // C = M·page
  FastDiv div_cap, div_page;
  const int* table;
  long long ts;
  const int* len;
  // rows of a write or a read
  long long rows;
  const int* cu;
  int rope_len;
  const float* cos;
  const float* sin;
  DevT4 kn, vn;             // new keys / values as [rows, 1, Hk, HD] views
  void* k_out;
  void* v_out;
  int out_dt;
  // decode
  int H, mode, W, norm, tw, tau_dt;
  float inv_scale;
  DevT4 q;
  void* out;
  void* tau;
  float* ws;
  int* err;
};

inline PagedP paged_params(const bozo_paged_cache& c, unsigned char* kg, unsigned char* vg) {
  PagedP p{};
  p.kg = kg; p.vg = vg;
  p.k = c.k_pages; p.v = c.v_pages; p.ks = c.k_scale; p.vs = c.v_scale;
  p.dt = c.dtype; p.P = c.pages; p.Hk = c.kv_heads; p.page = c.page_size; p.HD = c.HD;
  p.B = c.batch; p.M = c.width;
  p.cap = (unsigned)c.width * (unsigned)c.page_size;
  p.div_cap = make_fastdiv(p.cap);
  p.div_page = make_fastdiv((unsigned)c.page_size);
  p.table = c.table; p.ts = c.table_stride; p.len = c.lengths;
  return p;
}

cudaError_t launch_paged_write(const PagedP& p, int sms, cudaStream_t st);
cudaError_t launch_paged_read(const PagedP& p, int sms, cudaStream_t st);
size_t paged_decode_bytes(const PagedP& p, int sms);
cudaError_t launch_paged_decode(const PagedP& p, int sms, cudaStream_t st, int* launches, int* path);

constexpr unsigned kNoRow = 0xffffffffu;

// Row number of position `pos` of sequence b for head 0 (head h: + h·page), or
// kNoRow (and the error word set) where the table names no page of the pool.
__device__ __forceinline__ unsigned paged_row(const PagedP& p, int b, unsigned pos) {
  const unsigned s = pos - fast_div(pos, p.div_cap) * p.cap;
  const unsigned j = fast_div(s, p.div_page);
  const int pid = __ldg(p.table + b * p.ts + j);
  if ((unsigned)pid >= (unsigned)p.P) {
    atomicCAS(p.err, 0, kErrPaged | 2);
    return kNoRow;
  }
  return (unsigned)pid * (unsigned)p.Hk * (unsigned)p.page + (s - j * (unsigned)p.page);
}

// Sequence and position of row n of a write or a read; false for padding and
// inactive sequences.  `end`: the position after the sequence's last row.
__device__ __forceinline__ bool paged_place(const PagedP& p, int n, int& b, unsigned& pos,
                                            unsigned& end) {
  int first = n, next = n + 1;
  b = n;
  if (p.cu) {
    // the last b with cu[b] ≤ n
    int lo = 0, hi = p.B;
    if (n < __ldg(p.cu) || n >= __ldg(p.cu + p.B)) return false;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.cu + mid) <= n) lo = mid; else hi = mid;
    }
    b = lo;
    first = __ldg(p.cu + b);
    next = __ldg(p.cu + b + 1);
  }
  const int t = __ldg(p.len + b);
  if (t < 0) return false;
  pos = (unsigned)t + (unsigned)(n - first);
  end = (unsigned)t + (unsigned)(next - first);
  return pos <= 0x7fffffffu;
}

// 8-bit rows: scale = a / top and code = round(x · inv), inv = top / a.  The scale
// is at most FLT_MAX / top rounded down, so that top · scale is finite (at top 127
// the rounded quotient of FLT_MAX itself is one unit above).
constexpr float kTinyRow = 0x1p-100f;
// a / top, correctly rounded: a product with the rounded 1 / top and one correction
// by its exact remainder (Markstein, "Computation of elementary functions on the
// IBM RISC System/6000", 1990; checked for every significand at both tops).
__device__ __forceinline__ float div_top(float a, float top) {
  const float r = top == 127.f ? 0x1.020408p-7f : 0x1.24924ap-9f;
  const float q = __fmul_rn(a, r);
  return __fmaf_rn(__fmaf_rn(-q, top, a), r, q);
}
__device__ __forceinline__ void quant_scale(unsigned abs_bits, float top, float& scale, float& inv) {
  const float a = __uint_as_float(abs_bits);
  if (abs_bits >= 0x7f800000u) {  // an infinity or a NaN in the row
    scale = __uint_as_float(0x7fc00000u);
    inv = 0.f;
  } else if (a < kTinyRow) {
    scale = inv = 0.f;
  } else {
    scale = fminf(div_top(a, top), top == 127.f ? 0x1.020406p+121f : 0x1.249248p+119f);
    inv = __fdiv_rn(top, a);
  }
}
__device__ __forceinline__ unsigned char quant_code(float x, float inv, int dt) {
  const float y = inv == 0.f ? 0.f : __fmul_rn(x, inv);
  if (dt == BOZO_DT_I8) return (unsigned char)(signed char)max(-127, min(127, __float2int_rn(y)));
  return (unsigned char)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float code_value(unsigned char c, int dt) {
  if (dt == BOZO_DT_I8) return (float)(signed char)c;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}

// 4-bit rows.  The row's scale is a power of two, so the group scale is a correctly
// rounded sixth and the code a correctly rounded quotient by a few bits: both are a
// product with a reciprocal and one correction by its exact remainder, as in div_top
// (checked for every significand by 6 and by 8 … 15, those of an e4m3, with reciprocals
// up to two units off: the approximate one is at most one).
constexpr float kTinyRow4 = 0x1p-80f;  // below it the remainders would lose bits
struct Row4 {
  float scale, inv, most;  // the row's scale, its inverse, the largest group scale
  bool bad;
  __device__ __forceinline__ explicit Row4(unsigned abs_bits) {
    bad = abs_bits >= 0x7f800000u;  // an infinity or a NaN in the row
    scale = bad ? __uint_as_float(0x7fc00000u) : 0.f;
    inv = 0.f;
    most = 448.f;
    if (!bad && __uint_as_float(abs_bits) >= kTinyRow4) {
      // 2688 = 1.3125 · 2^11
      const unsigned e = (abs_bits >> 23) - 11u + ((abs_bits & 0x7fffffu) > 0x280000u ? 1u : 0u);
      scale = __uint_as_float(e << 23);
      inv = __uint_as_float((254u - e) << 23);
      if (e == 127u + 117u) most = 320.f;  // 6 · 352 · 2^117 is past the largest float
    }
  }
  // Scale of 16 elements with the largest magnitude a, as e4m3; unit: what a code of 1 stands for.
  __device__ __forceinline__ unsigned char group(float a, float& unit, float& recip) const {
    unsigned char c = 0;
    unit = recip = 0.f;
    if (inv != 0.f) {
      const float q = __fmul_rn(a, 0x1.555556p-3f);
      const float sixth = __fmaf_rn(__fmaf_rn(-q, 6.f, a), 0x1.555556p-3f, q);
      c = (unsigned char)__nv_cvt_float_to_fp8(fminf(__fmul_rn(sixth, inv), most), __NV_SATFINITE, __NV_E4M3);
      if (c) {
        unit = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3))) * scale;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(recip) : "f"(unit));
      }
    }
    return c;
  }
  // x / unit, anything in a bad row
  __device__ __forceinline__ float in_units(float x, float unit, float recip) const {
    const float q = __fmul_rn(x, recip);
    return __fmaf_rn(__fmaf_rn(q, unit, -x), -recip, q);  // in this order −0 stays −0
  }
};
// Two elements as a byte, the first in the low bits; and back (exact).
__device__ __forceinline__ unsigned pack4(float x, float y) {
  return __nv_cvt_float2_to_fp4x2(make_float2(x, y), __NV_E2M1, cudaRoundNearest);
}
__device__ __forceinline__ float2 unpack4(unsigned char c) {
  return __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)c, __NV_E2M1)));
}
__device__ __forceinline__ float e4m3(unsigned char c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}

// Element i of a page, without its row's scale; `groups` for 4-bit pages.
__device__ __forceinline__ float ld_page(const void* p, const unsigned char* groups, size_t i, int dt) {
  if (dt <= BOZO_DT_F16) return ldf(p, (long long)i, dt);
  if (dt == BOZO_DT_F4E2M1) {
    const float2 x = unpack4(static_cast<const unsigned char*>(p)[i >> 1]);
    return (i & 1 ? x.y : x.x) * e4m3(groups[i >> 4]);
  }
  return code_value(static_cast<const unsigned char*>(p)[i], dt);
}

// One warp holds a new row in its registers: element lane + 32·i of key (turned at
// `pos`) or value h of input row n; any head width up to 128, types and strides.
struct NewRow {
  float x[4];
  __device__ __forceinline__ NewRow(const PagedP& p, const DevT4& src, int n, int h, unsigned pos, bool turn,
                                    int lane) {
    const int half = p.HD / 2;
    const long long o = (long long)n * src.sb + (long long)h * src.sh;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      x[i] = 0.f;
      if (d >= p.HD) continue;
      x[i] = ldf(src.p, o + d * src.sd, src.dt);
      if (!turn) continue;
      const int f = d < half ? d : d - half;
      const float c = __ldg(p.cos + (size_t)pos * half + f), s = __ldg(p.sin + (size_t)pos * half + f);
      const float y = ldf(src.p, o + (d < half ? d + half : f) * src.sd, src.dt);
      x[i] = d < half ? __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(y, s))
                      : __fadd_rn(__fmul_rn(y, s), __fmul_rn(x[i], c));
    }
  }
  // … into row `row` of the pages, whose type is DT where it is known.
  template <int DT = -1>
  __device__ __forceinline__ void put(const PagedP& p, void* pages, float* scales, unsigned char* groups, size_t row,
                                      int lane) const {
    const int dt = DT >= 0 ? DT : p.dt;
    float inv = 1.f;
    unsigned a = 0;
    if (dt > BOZO_DT_F16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a = max(a, __float_as_uint(x[i]) & 0x7fffffffu);
      a = __reduce_max_sync(0xffffffffu, a);
    }
    if (dt == BOZO_DT_F4E2M1) {
      const Row4 r(a);
      if (lane == 0) scales[row] = r.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (32 * i >= p.HD) break;  // the same for all lanes
        const int d = lane + 32 * i;
        float m = fabsf(x[i]), unit, recip;
#pragma unroll
        for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const unsigned char c = r.group(m, unit, recip);
        const float y = r.bad ? 0.f : r.in_units(x[i], unit, recip), z = __shfl_down_sync(0xffffffffu, y, 1);
        if (d >= p.HD) continue;
        if (lane % 16 == 0) groups[row * (p.HD / 16) + d / 16] = c;
        if (lane % 2 == 0) static_cast<unsigned char*>(pages)[(row * p.HD + d) / 2] = (unsigned char)pack4(y, z);
      }
      return;
    }
    if (dt > BOZO_DT_F16) {
      float scale;
      quant_scale(a, dt == BOZO_DT_I8 ? 127.f : 448.f, scale, inv);
      if (lane == 0) scales[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      if (d >= p.HD) continue;
      if (dt <= BOZO_DT_F16) stf(pages, (long long)(row * p.HD + d), dt, x[i]);
      else static_cast<unsigned char*>(pages)[row * p.HD + d] = quant_code(x[i], inv, dt);
    }
  }
};

}  // namespace bozo
