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
constexpr int kMaxPiece = 8192;     // and at most in paged_decode_any, which holds their τ in shared memory
constexpr int kHeads = 8;           // query heads of a block in the tensor-core kernel
constexpr int kCluster = 8;         // pieces that are joined inside a cluster

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

// The new token's key and value go into their row before it is read: the blocks
// whose keys end with the new token's write it (each the same bytes; a local
// window does not hold it, so there the first block of a key head does).
__device__ __forceinline__ bool writes_row(const PagedP& p, bool active, unsigned piece, unsigned count, bool first) {
  return p.kn.p && active && (p.mode == BOZO_MODE_GLOBAL ? piece == count - 1 : piece == 0 && first);
}
__device__ __forceinline__ void append_row(const PagedP& p, int b, int hk, int t, int warp, int lane) {
  if (warp > 1) return;
  const unsigned row0 = paged_row(p, b, (unsigned)t);
  if (row0 == kNoRow) return;
  const size_t row = (size_t)row0 + (size_t)hk * p.page;
  if (warp == 0) put_row(p, p.kn, p.k, p.ks, b, hk, (unsigned)t, row, p.cos != nullptr, lane);
  else put_row(p, p.vn, p.v, p.vs, b, hk, (unsigned)t, row, false, lane);
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

// τ of key j (of the n in reach) into its slot of the exported row: LOCAL slot
// W − n + j, GLOBAL column n − 1 − j.
__device__ __forceinline__ void put_tau(const PagedP& p, size_t bh, unsigned n, unsigned j, float tau) {
  const unsigned slot = p.mode == BOZO_MODE_LOCAL ? (unsigned)p.W - n + j : n - 1 - j;
  if (slot < (unsigned)p.tw) stf(p.tau, (long long)(bh * p.tw + slot), p.tau_dt, tau);
}
// Slots without a key.
__device__ __forceinline__ void clear_tau(const PagedP& p, size_t bh, unsigned n, int i, int step) {
  const unsigned first = p.mode == BOZO_MODE_LOCAL ? 0u : min(n, (unsigned)p.tw);
  const unsigned last = p.mode == BOZO_MODE_LOCAL ? (unsigned)p.W - n : (unsigned)p.tw;
  for (unsigned s = first + i; s < last; s += step) stf(p.tau, (long long)(bh * p.tw + s), p.tau_dt, 0.f);
}

// One block per (b, h, piece), one warp per key: any head width and types.
__global__ void __launch_bounds__(kThreads) paged_decode_any(PagedP p, int S) {
  extern __shared__ float sm[];
  float* sq = sm;             // rotated q [HD]
  float* stau = sm + p.HD;    // τ of the piece's keys
  __shared__ float red[kThreads / 32];
  const int piece = blockIdx.x % S, bh = blockIdx.x / S;
  const int b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const int HD = p.HD, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int t;
  unsigned lo, n, count, size;
  const bool active = reach(p, b, t, lo, n);
  cut(n, S, count, size);
  if ((unsigned)piece >= count) return;
  const unsigned j0 = piece * size, j1 = min(n, j0 + size);
  if (active)
    for (int i = threadIdx.x; i < HD; i += kThreads) sq[i] = query(p, b, h, t, i);
  if (writes_row(p, active, piece, count, h % (p.H / p.Hk) == 0)) append_row(p, b, hk, t, warp, lane);
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
    for (unsigned j = j0 + threadIdx.x; j < j1; j += kThreads) put_tau(p, bh, n, j, stau[j - j0]);
    if (piece == 0) clear_tau(p, bh, n, threadIdx.x, kThreads);
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
// One block per (b, key head, up to 8 of its query heads, piece).  Each warp walks
// tiles of its own through a ring in shared memory that 16-byte asynchronous
// copies fill a few tiles ahead (rows out of reach are filled with zeros), and
// feeds mma.m16n8k16 from it; nothing is shared between warps before the end.
//   S = Q·Kᵀ  A: rows 0-7 the heads' q rounded to 16 bits, rows 8-15 what that
//             rounding left, so the sum of an accumulator's two halves (both in
//             one lane) has q to 16 bits and more at the price of one product;
//             B: lane (g, c) = (lane/4, lane%4) takes key g, a quarter of each
//             row in 16-byte pieces — the order of the dot product's terms is
//             free, so the dimensions go to the k index as the loads bring them;
//   O = P·V   A: τ (· the row's scale), high and low parts in the same way: S's
//             accumulator layout is P's operand layout; B: lane (g, c) takes the
//             keys 2c, 2c+1, 8+2c, 9+2c and every 8th part of their rows, pairs
//             of keys put together by byte permutes.
// The 16-byte pieces of a 128-byte line are permuted (K: by the row's low bit, V:
// by the next two) so that both access patterns are free of bank conflicts.
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

template <int N>  // N 32-bit words from shared memory
__device__ __forceinline__ void lds_words(const char* p, unsigned* w) {
  if constexpr (N == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const unsigned*>(p);
  }
}

// Asynchronous copies to shared memory; `bytes` 0 fills with zeros.
__device__ __forceinline__ void copy16(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_peer(unsigned addr, unsigned rank) {
  unsigned a;
  float x;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
  return x;
}

// Geometry of the kernel for one page type and head width.
template <int DT, int HD> struct Geo {
  static constexpr int size = Fmt<DT>::size;
  static constexpr int row = HD * size;                      // bytes of a row
  static constexpr int keys = row >= 128 ? 16 : 2048 / row;  // keys of a tile: 4 KB of K and V (8 KB at 256-byte rows)
  static constexpr int kv = keys * row;                      // bytes of a tile's K (or V)
  static constexpr int scales = Fmt<DT>::scaled ? 2 * keys * 4 : 0;
  static constexpr int slot = 2 * kv + scales + 16;          // and the mask of its live keys
};
constexpr int kWarps = 4;
constexpr int kStages = 4;

// Byte offset of 16-byte piece ch of row r of a K / V tile with R-byte rows.
template <int R> __device__ __forceinline__ int k_at(int r, int ch) {
  return r * R + ((R >= 128 ? ch ^ ((r & 1) << 2) : ch) << 4);
}
template <int R> __device__ __forceinline__ int v_at(int r, int ch) {
  if constexpr (R >= 128) return r * R + ((ch ^ (((r >> 1) & 3) << 1)) << 4);
  // rows share 128-byte lines
  constexpr int per = 128 / R;
  const int line = r / per, c8 = (r % per) * (R / 16) + ch;
  return line * 128 + ((c8 ^ (R == 64 ? (line & 3) << 1 : (line & 1) << 1)) << 4);
}

template <int DT, int HD>
__global__ void __launch_bounds__(kWarps * 32) paged_decode_mma(PagedP p, int S, int HG, bool clustered) {
  using F = Fmt<DT>;
  using Z = Geo<DT, HD>;
  constexpr bool BF = F::bf;
  constexpr int R = Z::row, KT = Z::keys, NCH = R / 16;
  constexpr int kKB = R / 4 < 16 ? R / 4 : 16;             // bytes of a lane's key load
  constexpr int kKL = R / (4 * kKB), kKE = kKB / F::size, kKW = kKB / 4;
  constexpr int kVB = R / 8 < 16 ? R / 8 : 16;             // bytes of a lane's value load
  constexpr int kVL = R / (8 * kVB), kVE = kVB / F::size, kVW = kVB / 4;
  constexpr int kSteps = HD / 16, kTiles = HD / 8;
  extern __shared__ __align__(128) char smb[];
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
  const bool mine = (unsigned)piece < count;
  if (!mine && !clustered) return;
  const unsigned j0 = piece * size, nk = mine ? min(n, j0 + size) - j0 : 0u;  // this block's keys
  float mass = 0.f, unit = 1.f, lim = 0.f;  // P operand: p · unit, renewed where p passes lim (halfs)
  float acc[kTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;

  if (mine) {
    if (active)
      for (int i = tid; i < kHeads * HD; i += kWarps * 32) {
        const int h = i / HD, d = i - h * HD;
        sq[h][d] = h < Gh ? query(p, b, h0 + h, t, d) : 0.f;
      }
    if (writes_row(p, active, piece, count, hg == 0)) append_row(p, b, hk, t, warp, lane);
    __syncthreads();
  }
  if (nk) {
    char* ring = smb + warp * kStages * Z::slot;
    const char* kpages = static_cast<const char*>(p.k);
    const char* vpages = static_cast<const char*>(p.v);
    constexpr unsigned step = kWarps * KT;
    // row numbers of the tile from key i on, in lane key % 32 (KT 16: twice)
    constexpr int RR = KT > 32 ? KT / 32 : 1;
    auto find = [&](unsigned i, unsigned* rows) {
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const unsigned j = i + r * 32 + (KT < 32 ? lane % KT : lane);
        rows[r] = kNoRow;
        if (j < nk) {
          const unsigned row = paged_row(p, b, lo + j0 + j);
          if (row != kNoRow) rows[r] = row + (unsigned)hk * p.page;
        }
      }
    };
    auto fill = [&](int slot, const unsigned* rows) {
      char* at = ring + slot * Z::slot;
      const unsigned kd = smem_u32(at), vd = kd + Z::kv;
#pragma unroll
      for (int it = 0; it < KT * NCH / 32; ++it) {
        const int r = (it * 32 + lane) / NCH, ch = lane % NCH;
        const unsigned row = __shfl_sync(0xffffffffu, rows[(it * 32 / NCH) / 32], r % 32);
        const bool on = row != kNoRow;
        const size_t off = on ? (size_t)row * R + ch * 16 : 0;
        copy16(kd + k_at<R>(r, ch), kpages + off, on ? 16 : 0);
        copy16(vd + v_at<R>(r, ch), vpages + off, on ? 16 : 0);
      }
      if constexpr (F::scaled) {
        const unsigned sd = vd + Z::kv;
        if constexpr (KT == 16) {
          const bool on = rows[0] != kNoRow;
          copy4(sd + lane * 4, (lane < 16 ? p.ks : p.vs) + (on ? rows[0] : 0u), on ? 4 : 0);
        } else {
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            const bool on = rows[r] != kNoRow;
            copy4(sd + (r * 32 + lane) * 4, p.ks + (on ? rows[r] : 0u), on ? 4 : 0);
            copy4(sd + (KT + r * 32 + lane) * 4, p.vs + (on ? rows[r] : 0u), on ? 4 : 0);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const unsigned m = __ballot_sync(0xffffffffu, rows[r] != kNoRow);
        if (lane == 0) reinterpret_cast<unsigned*>(at + 2 * Z::kv + Z::scales)[r] = m;
      }
    };

    unsigned i = warp * KT;
    unsigned rows[kStages - 1][RR], next[RR];
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) find(i + s * step, rows[s]);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      if (i + s * step < nk) fill(s, rows[s]);
      copy_commit();
    }
    find(i + (kStages - 1) * step, next);

    // A operand of S: q of head g, as halfs brought near 1 by a power of two
    unsigned qa[kSteps][4];
    float sscale = p.inv_scale;
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

    int slot = 0;
#pragma unroll 1
    for (; i < nk; i += step) {
      copy_wait<kStages - 2>();
      __syncwarp();
      {  // the slot of the tile before this one takes the tile kStages − 1 ahead
        const unsigned f = i + (kStages - 1) * step;
        if (f < nk) fill((slot + kStages - 1) % kStages, next);
        copy_commit();
        find(f + step, next);
      }
      const char* at = ring + slot * Z::slot;
      slot = (slot + 1) % kStages;
#pragma unroll
      for (int sub = 0; sub < KT / 16; ++sub) {
        float s[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
          const int r = sub * 16 + 8 * u + g;
#pragma unroll
          for (int l = 0; l < kKL; ++l) {
            unsigned kw[kKW];
            const int byte = l * 4 * kKB + c * kKB;
            lds_words<kKW>(at + k_at<R>(r, byte >> 4) + (byte & 15), kw);
            if constexpr (F::size == 2) {
#pragma unroll
              for (int w = 0; w < kKW / 2; ++w)
                mma16816<BF>(s[u], qa[l * (kKE / 4) + w], kw[2 * w], kw[2 * w + 1]);
            } else {
#pragma unroll
              for (int w = 0; w < kKW; ++w) {
                unsigned b0, b1;
                widen4<DT>(kw[w], b0, b1);
                mma16816<BF>(s[u], qa[l * (kKE / 4) + w], b0, b1);
              }
            }
          }
        }
        // τ of head g and the keys 2c, 2c+1, 8+2c, 9+2c
        const unsigned live = reinterpret_cast<const unsigned*>(at + 2 * Z::kv + Z::scales)[sub >> 1] >> ((sub & 1) * 16);
        const float* sc = reinterpret_cast<const float*>(at + 2 * Z::kv) + sub * 16;
        float pr[4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int k = 8 * u + 2 * c + e;
            float z = (s[u][e] + s[u][2 + e]) * sscale;
            if constexpr (F::scaled) z *= sc[k];
            float tau = __fdividef(1.f, 1.f + __expf(-z));
            const bool on = (live >> k) & 1;
            tau = on ? tau : 0.f;
            mass += tau;
            if (p.tau && g < Gh && on) put_tau(p, (size_t)b * p.H + h0 + g, n, j0 + i + sub * 16 + k, tau);
            pr[2 * u + e] = F::scaled ? tau * sc[KT + k] : tau;
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
        for (int l = 0; l < kVL; ++l) {
          unsigned vw[4][kVW];
          const int byte = l * 8 * kVB + g * kVB;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            lds_words<kVW>(at + Z::kv + v_at<R>(sub * 16 + 8 * (u >> 1) + 2 * c + (u & 1), byte >> 4) + (byte & 15),
                           vw[u]);
#pragma unroll
          for (int w = 0; w < kVW; ++w) {
            if constexpr (F::size == 2) {
              const int j = l * kVE + 2 * w;
              mma16816<BF>(acc[j], pa, __byte_perm(vw[0][w], vw[1][w], 0x5410),
                           __byte_perm(vw[2][w], vw[3][w], 0x5410));
              mma16816<BF>(acc[j + 1], pa, __byte_perm(vw[0][w], vw[1][w], 0x7632),
                           __byte_perm(vw[2][w], vw[3][w], 0x7632));
            } else {
              const int j = l * kVE + 4 * w;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const unsigned sel = e ? 0x7362 : 0x5140;  // keys' codes side by side
                unsigned a0, a1, b0, b1;
                widen4<DT>(__byte_perm(vw[0][w], vw[1][w], sel), a0, a1);
                widen4<DT>(__byte_perm(vw[2][w], vw[3][w], sel), b0, b1);
                mma16816<BF>(acc[j + 2 * e], pa, a0, b0);
                mma16816<BF>(acc[j + 2 * e + 1], pa, a1, b1);
              }
            }
          }
        }
      }
    }
    copy_wait<0>();
  }

  // the warps' sums, added in order
  __syncthreads();  // the rings are done with
  float* part = reinterpret_cast<float*>(smb);        // [warps][Gh][HD], then the block's [Gh][HD]
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
  float* sum = part + kWarps * Gh * HD;
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
      if (piece == 0) stf(p.out, (long long)(bh * HD + d), p.out_dt, o / norm_divisor(p, m, n));
    } else if (clustered) {
      sum[i] = o;
      if (d == 0) sq[0][h] = m;  // the queries are done with
    } else {
      p.ws[(bh * S + piece) * HD + d] = o;
      if (d == 0) piece_mass(p, S)[bh * S + piece] = m;
    }
  }
  if (p.tau && piece == 0)
    for (int h = warp; h < Gh; h += kWarps) clear_tau(p, (size_t)b * p.H + h0 + h, n, lane, 32);
  if (clustered) {
    // the pieces' sums through the cluster's shared memory, each block a part of
    // the elements, in the order of the pieces
    cluster_sync();
    if (count > 1)
      for (int i = tid + piece * kWarps * 32; i < Gh * HD; i += S * kWarps * 32) {
        const int h = i / HD, d = i - h * HD;
        float o = 0.f, m = 0.f;
        for (unsigned r = 0; r < count; ++r) {
          o += ld_peer(smem_u32(sum + i), r);
          m += ld_peer(smem_u32(&sq[0][h]), r);
        }
        const size_t bh = (size_t)b * p.H + h0 + h;
        stf(p.out, (long long)(bh * HD + d), p.out_dt, o / norm_divisor(p, m, n));
      }
    cluster_sync();
  }
}

bool mma_path(const PagedP& p) {
  return p.dt != BOZO_DT_F32 && (p.HD == 32 || p.HD == 64 || p.HD == 128);
}

struct Plan {
  int S;           // pieces a row may be cut into
  bool clustered;  // joined inside a cluster, else by a second kernel from the workspace
};

Plan plan(const PagedP& p, int sms) {
  const bool mma = mma_path(p);
  const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
  const int G = p.H / p.Hk;
  const long long rows = (long long)p.B * (mma ? (long long)p.Hk * ((G + kHeads - 1) / kHeads) : p.H);
  long long s = (sms * (mma ? 16 : 8) + rows - 1) / rows;
  s = std::min(s, (keys + kMinPiece - 1) / kMinPiece);
  if (!mma) s = std::max(s, (keys + kMaxPiece - 1) / kMaxPiece);
  s = std::max(s, 1LL);
  return {(int)s, mma && s > 1 && s <= kCluster};
}

template <int DT, int HD>
cudaError_t launch_mma(const PagedP& p, const Plan& pl, cudaStream_t st) {
  const int G = p.H / p.Hk, HG = (G + kHeads - 1) / kHeads;
  const size_t ring = (size_t)kWarps * kStages * Geo<DT, HD>::slot;
  const size_t part = (size_t)(kWarps + 1) * std::min(G, kHeads) * HD * sizeof(float);
  const size_t smem = std::max(ring, part);
  auto kern = paged_decode_mma<DT, HD>;
  if (smem > 32 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((long long)p.B * p.Hk * HG * pl.S));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)pl.S, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = pl.clustered ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p, pl.S, HG, pl.clustered);
}
template <int DT>
cudaError_t launch_mma(const PagedP& p, const Plan& pl, cudaStream_t st) {
  switch (p.HD) {
    case 32: return launch_mma<DT, 32>(p, pl, st);
    case 64: return launch_mma<DT, 64>(p, pl, st);
    default: return launch_mma<DT, 128>(p, pl, st);
  }
}

}  // namespace

size_t paged_decode_bytes(const PagedP& p, int sms) {
  const Plan pl = plan(p, sms);
  if (pl.S < 2 || pl.clustered) return 0;
  return ((size_t)p.B * p.H * pl.S * (p.HD + 1) * sizeof(float) + 255) & ~(size_t)255;
}

cudaError_t launch_paged_decode(const PagedP& p, int sms, cudaStream_t st, int* launches) {
  const Plan pl = plan(p, sms);
  cudaError_t e;
  if (mma_path(p)) {
    switch (p.dt) {
      case BOZO_DT_BF16: e = launch_mma<BOZO_DT_BF16>(p, pl, st); break;
      case BOZO_DT_F16: e = launch_mma<BOZO_DT_F16>(p, pl, st); break;
      case BOZO_DT_F8E4M3: e = launch_mma<BOZO_DT_F8E4M3>(p, pl, st); break;
      default: e = launch_mma<BOZO_DT_I8>(p, pl, st);
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
