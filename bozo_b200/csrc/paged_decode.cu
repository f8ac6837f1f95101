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

// Workspace: Σ τ·v of every piece [B·H][S][HD], then their masses [B·H][S].
__device__ __forceinline__ float* piece_mass(const PagedP& p, int S) {
  return p.ws + (size_t)p.B * p.H * S * p.HD;
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
      p.ws[((size_t)bh * S + piece) * HD + d] = acc;
  }
  if (count > 1 && threadIdx.x == 0) piece_mass(p, S)[(size_t)bh * S + piece] = m;
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
  const float* w = p.ws + (size_t)bh * S * HD;
  const float* wm = piece_mass(p, S) + (size_t)bh * S;
  for (int d = threadIdx.x; d < HD; d += kThreads) {
    float acc = 0.f, m = 0.f;
    for (unsigned i = 0; i < count; ++i) {
      acc += w[i * HD + d];
      m += wm[i];
    }
    stf(p.out, (long long)bh * HD + d, p.out_dt, acc / norm_divisor(p, m, n));
  }
}

// ─────────────── tensor-core kernel: 16- and 8-bit pages, HD 32, 64, 128 ───────────────
// One block per (b, key head, up to 8 of its query heads, piece); a warp takes 16
// keys at a time, straight from memory into mma.m16n8k16 operands:
//   S = Q·Kᵀ  A: rows 0-7 the heads' q rounded to 16 bits, rows 8-15 what that
//             rounding left, so the sum of an accumulator's two halves (both in
//             one lane) has q to 16 bits and more at the price of one product;
//             B: lane (g, c) = (lane/4, lane%4) holds key g, a quarter of each
//             row in 16-byte pieces — the order of the dot product's terms is
//             free, so the dimensions go to the k index as the loads bring them;
//   O = P·V   A: τ (· the row's scale), high and low parts in the same way: S's
//             accumulator layout is P's operand layout; B: lane (g, c) holds the
//             keys 2c, 2c+1, 8+2c, 9+2c and every 8th part of their rows, pairs
//             of keys put together by byte permutes.
// Nothing goes through shared memory but row numbers, scales and the final sum
// over the block's warps.
constexpr int kWarps = 4;
constexpr int kHeads = 8;
constexpr int kMmaPiece = 4096;  // keys of a piece, at most

template <int DT> struct Fmt;
template <> struct Fmt<BOZO_DT_BF16> { static constexpr int size = 2; static constexpr bool bf = true, scaled = false; };
template <> struct Fmt<BOZO_DT_F16> { static constexpr int size = 2; static constexpr bool bf = false, scaled = false; };
template <> struct Fmt<BOZO_DT_F8E4M3> { static constexpr int size = 1; static constexpr bool bf = false, scaled = true; };
template <> struct Fmt<BOZO_DT_I8> { static constexpr int size = 1; static constexpr bool bf = false, scaled = true; };

template <bool BF>
__device__ __forceinline__ void mma16816(float* d, const unsigned* a, unsigned b0, unsigned b1) {
  if constexpr (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x, y as a pair of 16-bit numbers and the pair of what that left of them
template <bool BF>
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - __low2float(h), y - __high2float(h));
    hi = *reinterpret_cast<const unsigned*>(&h);
    lo = *reinterpret_cast<const unsigned*>(&l);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    const __half2 l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    hi = *reinterpret_cast<const unsigned*>(&h);
    lo = *reinterpret_cast<const unsigned*>(&l);
  }
}

// Four 8-bit codes as two pairs of halfs (exact).
template <int DT>
__device__ __forceinline__ void widen4(unsigned x, unsigned& p01, unsigned& p23) {
  if constexpr (DT == BOZO_DT_F8E4M3) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x >> 16), __NV_E4M3);
    p01 = *reinterpret_cast<const unsigned*>(&a);
    p23 = *reinterpret_cast<const unsigned*>(&b);
  } else {
    // 1024 + (code + 128) is the half with those low bits; less 1152 it is the code
    const unsigned u = x ^ 0x80808080u;
    unsigned a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 hb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    p01 = *reinterpret_cast<const unsigned*>(&ha);
    p23 = *reinterpret_cast<const unsigned*>(&hb);
  }
}

template <int N>  // N 32-bit words from an address aligned to them
__device__ __forceinline__ void ld_words(const char* p, unsigned* w) {
  if constexpr (N == 4) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const unsigned*>(p));
  }
}

template <int DT, int HD>
__global__ void __launch_bounds__(kWarps * 32) paged_decode_mma(PagedP p, int S, int HG) {
  using F = Fmt<DT>;
  constexpr bool BF = F::bf;
  constexpr int kRow = HD * F::size;                       // bytes of a row
  constexpr int kKB = kRow / 4 < 16 ? kRow / 4 : 16;       // bytes of a key load
  constexpr int kKL = kRow / (4 * kKB), kKE = kKB / F::size, kKW = kKB / 4;
  constexpr int kVB = kRow / 8 < 16 ? kRow / 8 : 16;       // bytes of a value load
  constexpr int kVL = kRow / (8 * kVB), kVE = kVB / F::size, kVW = kVB / 4;
  constexpr int kSteps = HD / 16, kTiles = HD / 8;
  extern __shared__ unsigned smu[];
  __shared__ float sq[kHeads][HD + 4];
  __shared__ float smass[kWarps][kHeads];
  const int G = p.H / p.Hk;
  int x = blockIdx.x;
  const int piece = x % S;
  x /= S;
  const int hg = x % HG;
  x /= HG;
  const int hk = x % p.Hk, b = x / p.Hk;
  const int h0 = hk * G + hg * kHeads, Gh = min(kHeads, G - hg * kHeads);  // query heads h0 … h0+Gh−1
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  int t;
  unsigned lo, n, count, size;
  const bool active = reach(p, b, t, lo, n);
  cut(n, S, count, size);
  if ((unsigned)piece >= count) return;
  const unsigned j0 = piece * size, nk = min(n, j0 + size) - j0;  // this block's keys
  const unsigned np = (nk + 15) & ~15u;
  unsigned* srow = smu;
  float* ssc = reinterpret_cast<float*>(smu + size);  // key scales [size], value scales [size]
  for (unsigned i = tid; i < np; i += kWarps * 32) {
    unsigned r = kNoRow;
    if (i < nk) {
      r = paged_row(p, b, lo + j0 + i);
      if (r != kNoRow) r += (unsigned)hk * p.page;
    }
    srow[i] = r;
    if constexpr (F::scaled) {
      ssc[i] = r == kNoRow ? 0.f : __ldg(p.ks + r) * p.inv_scale;
      ssc[size + i] = r == kNoRow ? 0.f : __ldg(p.vs + r);
    }
  }
  if (active) {
    constexpr int half = HD / 2;
    for (int i = tid; i < kHeads * half; i += kWarps * 32) {
      const int h = i / half, f = i - h * half;
      float u = 0.f, v = 0.f;
      if (h < Gh) {
        const long long qo = (long long)b * p.q.sb + (long long)(h0 + h) * p.q.sh;
        u = ldf(p.q.p, qo + f * p.q.sd, p.q.dt);
        v = ldf(p.q.p, qo + (f + half) * p.q.sd, p.q.dt);
        if (p.cos) {
          const float cs = p.cos[(size_t)t * half + f], sn = p.sin[(size_t)t * half + f];
          const float r = u * cs - v * sn;
          v = u * sn + v * cs;
          u = r;
        }
      }
      sq[h][f] = u;
      sq[h][f + half] = v;
    }
  }
  __syncthreads();

  float acc[kTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  float mass = 0.f, unit = 1.f, lim = 0.f;  // P operand: p · unit, renewed where p passes lim (halfs)
  if (active) {
    // A operand of S: q of head g, as halfs brought near 1 by a power of two
    unsigned qa[kSteps][4];
    float sscale = F::scaled ? 1.f : p.inv_scale;
    {
      float qs = 1.f;
      if constexpr (!BF) {
        float m = 0.f;
        for (int d = c; d < HD; d += 4) m = fmaxf(m, fabsf(sq[g][d]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = min(126, max(-126, (int)(__float_as_uint(m) >> 23) - 127));
        if (m > 0.f) {
          qs = __uint_as_float((unsigned)(127 - e) << 23);
          sscale *= __uint_as_float((unsigned)(127 + e) << 23);
        }
      }
#pragma unroll
      for (int l = 0; l < kKL; ++l)
#pragma unroll
        for (int u = 0; u < kKE / 4; ++u) {
          const float* s = &sq[g][l * 4 * kKE + c * kKE + 4 * u];
          unsigned* a = qa[l * (kKE / 4) + u];
          split2<BF>(s[0] * qs, s[1] * qs, a[0], a[1]);
          split2<BF>(s[2] * qs, s[3] * qs, a[2], a[3]);
        }
    }
    const char* kbase = static_cast<const char*>(p.k) + c * kKB;
    const char* vbase = static_cast<const char*>(p.v) + g * kVB;
    unsigned kw[2][kKL * kKW], vw[4][kVL * kVW];
    auto load_k = [&](unsigned i) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned r = srow[i + 8 * u + g];
#pragma unroll
        for (int l = 0; l < kKL; ++l) {
          if (r != kNoRow) {
            ld_words<kKW>(kbase + (size_t)r * kRow + l * 4 * kKB, &kw[u][l * kKW]);
          } else {
#pragma unroll
            for (int w = 0; w < kKW; ++w) kw[u][l * kKW + w] = 0u;
          }
        }
      }
    };
    auto load_v = [&](unsigned i) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned r = srow[i + 8 * (u >> 1) + 2 * c + (u & 1)];
#pragma unroll
        for (int l = 0; l < kVL; ++l) {
          if (r != kNoRow) {
            ld_words<kVW>(vbase + (size_t)r * kRow + l * 8 * kVB, &vw[u][l * kVW]);
          } else {
#pragma unroll
            for (int w = 0; w < kVW; ++w) vw[u][l * kVW + w] = 0u;
          }
        }
      }
    };
    unsigned i = warp * 16;
    if (i < np) {
      load_k(i);
      load_v(i);
    }
    for (; i < np; i += kWarps * 16) {
      const unsigned next = i + kWarps * 16;
      float s[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
#pragma unroll
        for (int l = 0; l < kKL; ++l) {
          if constexpr (F::size == 2) {
#pragma unroll
            for (int w = 0; w < kKW / 2; ++w)
              mma16816<BF>(s[u], qa[l * (kKE / 4) + w], kw[u][l * kKW + 2 * w], kw[u][l * kKW + 2 * w + 1]);
          } else {
#pragma unroll
            for (int w = 0; w < kKW; ++w) {
              unsigned b0, b1;
              widen4<DT>(kw[u][l * kKW + w], b0, b1);
              mma16816<BF>(s[u], qa[l * (kKE / 4) + w], b0, b1);
            }
          }
        }
      }
      if (next < np) load_k(next);
      // τ of head g and the keys 2c, 2c+1, 8+2c, 9+2c
      float pr[4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned at = i + 8 * u + 2 * c + e;
          float z = (s[u][e] + s[u][2 + e]) * sscale;
          if constexpr (F::scaled) z *= ssc[at];
          float tau = __fdividef(1.f, 1.f + __expf(-z));
          tau = srow[at] == kNoRow ? 0.f : tau;
          mass += tau;
          if (p.tau && g < Gh && at < nk) {
            const long long j = (long long)j0 + at;
            const long long slot = p.mode == BOZO_MODE_LOCAL ? p.W - (long long)n + j : (long long)n - 1 - j;
            if (slot < p.tw) stf(p.tau, ((long long)b * p.H + h0 + g) * p.tw + slot, p.tau_dt, tau);
          }
          pr[2 * u + e] = F::scaled ? tau * ssc[size + at] : tau;
        }
      unsigned pa[4];
      if constexpr (!BF) {
        // halfs reach from 2^-24 to 65504: keep the largest p of a head between 1
        // and 4096 by a power of two, what was summed before following it
        const float pm = fmaxf(fmaxf(pr[0], pr[1]), fmaxf(pr[2], pr[3]));
        if (__any_sync(0xffffffffu, pm > lim)) {
          float m = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          if (m > lim) {
            const int e = min(113, max(-126, (int)(__float_as_uint(m) >> 23) - 127));
            const float nu = __uint_as_float((unsigned)(127 - e) << 23);
            const float f = lim == 0.f ? 0.f : nu / unit;
#pragma unroll
            for (int j = 0; j < kTiles; ++j)
#pragma unroll
              for (int e2 = 0; e2 < 4; ++e2) acc[j][e2] *= f;
            unit = nu;
            lim = __uint_as_float((unsigned)(127 + e + 12) << 23);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] *= unit;
      }
      split2<BF>(pr[0], pr[1], pa[0], pa[1]);
      split2<BF>(pr[2], pr[3], pa[2], pa[3]);
#pragma unroll
      for (int l = 0; l < kVL; ++l)
#pragma unroll
        for (int w = 0; w < kVW; ++w) {
          const int at = l * kVW + w;
          if constexpr (F::size == 2) {
            const int j = l * kVE + 2 * w;
            mma16816<BF>(acc[j], pa, __byte_perm(vw[0][at], vw[1][at], 0x5410),
                         __byte_perm(vw[2][at], vw[3][at], 0x5410));
            mma16816<BF>(acc[j + 1], pa, __byte_perm(vw[0][at], vw[1][at], 0x7632),
                         __byte_perm(vw[2][at], vw[3][at], 0x7632));
          } else {
            const int j = l * kVE + 4 * w;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const unsigned sel = e ? 0x7362 : 0x5140;  // keys' codes side by side
              unsigned a0, a1, b0, b1;
              widen4<DT>(__byte_perm(vw[0][at], vw[1][at], sel), a0, a1);
              widen4<DT>(__byte_perm(vw[2][at], vw[3][at], sel), b0, b1);
              mma16816<BF>(acc[j + 2 * e], pa, a0, b0);
              mma16816<BF>(acc[j + 2 * e + 1], pa, a1, b1);
            }
          }
        }
      if (next < np) load_v(next);
    }
  }

  // the warps' sums, added in order
  __syncthreads();  // the row numbers are no longer needed
  float* part = reinterpret_cast<float*>(smu);  // [warps][Gh][HD]
  mass += __shfl_xor_sync(0xffffffffu, mass, 1);
  mass += __shfl_xor_sync(0xffffffffu, mass, 2);
  if (c == 0) smass[warp][g] = mass;
  if (g < Gh) {
    const float back = 1.f / unit;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = (j / kVE) * 8 * kVE + (2 * c + e) * kVE + j % kVE;
        part[(warp * Gh + g) * HD + d] = (acc[j][e] + acc[j][2 + e]) * back;
      }
  }
  __syncthreads();
  for (int i = tid; i < Gh * HD; i += kWarps * 32) {
    const int h = i / HD, d = i - h * HD;
    float o = 0.f, m = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      o += part[w * Gh * HD + i];
      m += smass[w][h];
    }
    const size_t bh = (size_t)b * p.H + h0 + h;
    if (count == 1) {
      stf(p.out, (long long)(bh * HD + d), p.out_dt, o / norm_divisor(p, m, n));
    } else {
      p.ws[(bh * S + piece) * HD + d] = o;
      if (d == 0) piece_mass(p, S)[bh * S + piece] = m;
    }
  }
  if (p.tau && piece == 0) {  // slots without a key
    const int first = p.mode == BOZO_MODE_LOCAL ? 0 : (int)min(n, (unsigned)p.tw);
    const int last = p.mode == BOZO_MODE_LOCAL ? p.W - (int)n : p.tw;
    for (int h = warp; h < Gh; h += kWarps)
      for (int s = first + lane; s < last; s += 32)
        stf(p.tau, ((long long)b * p.H + h0 + h) * p.tw + s, p.tau_dt, 0.f);
  }
}

bool mma_path(const PagedP& p) {
  return p.dt != BOZO_DT_F32 && (p.HD == 32 || p.HD == 64 || p.HD == 128);
}

int pieces(const PagedP& p, int sms) {
  const bool mma = mma_path(p);
  const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
  const int G = p.H / p.Hk;
  const long long rows = (long long)p.B * (mma ? (long long)p.Hk * ((G + kHeads - 1) / kHeads) : p.H);
  const int most = mma ? kMmaPiece : kMaxPiece;
  long long s = (sms * (mma ? 16 : kResident) + rows - 1) / rows;
  s = std::min(s, (keys + kMinPiece - 1) / kMinPiece);
  return (int)std::max({s, (keys + most - 1) / most, 1LL});
}

template <int DT>
cudaError_t launch_mma(const PagedP& p, int S, cudaStream_t st) {
  const int G = p.H / p.Hk, HG = (G + kHeads - 1) / kHeads;
  const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
  const size_t per = DT == BOZO_DT_F8E4M3 || DT == BOZO_DT_I8 ? 12 : 4;
  const long long size = std::min<long long>(((keys + S - 1) / S + 15) & ~15LL, kMmaPiece);
  // a short row is cut into fewer pieces, each at most kMinPiece and the rounding
  const size_t idx = (size_t)std::max<long long>(size, kMinPiece + 16) * per;
  const size_t part = (size_t)kWarps * std::min(G, kHeads) * p.HD * sizeof(float);
  const size_t smem = std::max(idx, part);
  auto go = [&](auto kern) {
    if (smem > 40 * 1024) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return e;
    }
    kern<<<(unsigned)((long long)p.B * p.Hk * HG * S), kWarps * 32, smem, st>>>(p, S, HG);
    return cudaGetLastError();
  };
  switch (p.HD) {
    case 32: return go(paged_decode_mma<DT, 32>);
    case 64: return go(paged_decode_mma<DT, 64>);
    default: return go(paged_decode_mma<DT, 128>);
  }
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
  cudaError_t e;
  if (mma_path(p)) {
    switch (p.dt) {
      case BOZO_DT_BF16: e = launch_mma<BOZO_DT_BF16>(p, S, st); break;
      case BOZO_DT_F16: e = launch_mma<BOZO_DT_F16>(p, S, st); break;
      case BOZO_DT_F8E4M3: e = launch_mma<BOZO_DT_F8E4M3>(p, S, st); break;
      default: e = launch_mma<BOZO_DT_I8>(p, S, st);
    }
  } else {
    const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
    const size_t smem = (size_t)(p.HD + std::min<long long>(keys, kMaxPiece) + 16) * sizeof(float);
    paged_decode_any<<<(unsigned)(p.B * p.H * S), kThreads, smem, st>>>(p, S);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  ++*launches;
  if (S > 1) {
    paged_join<<<(unsigned)(p.B * p.H), kThreads, 0, st>>>(p, S);
    ++*launches;
  }
  return cudaGetLastError();
}

}  // namespace bozo
