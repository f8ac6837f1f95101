// paged_mma.cuh — the tensor-core kernel of a decode step over a paged cache:
// 16- and 8-bit pages, head widths 32, 64 and 128.
//
// One block per (b, key head, up to 8 of its query heads, piece).  Each warp walks
// tiles of its own through a ring in shared memory that 16-byte asynchronous
// copies fill a few tiles ahead (rows out of reach are filled with zeros), and
// feeds mma.m16n8k16 from it; nothing is shared between warps before the end.
//   Sᵀ = K·Qᵀ  16 keys by 8 columns: a column is a query head's q in 16 bits or
//              what that left of it, side by side, so the sum of neighbouring
//              accumulators has both.  Where there are few heads, the columns
//              repeat them and each group of lanes takes its scores from a tile
//              of its own, so that every lane computes different τ.
//   O  = P·V   rows 0-7 the heads' τ (· the value row's scale) in 16 bits, rows
//              8-15 what that left; τ goes from lanes to operands through a few
//              words of shared memory.
// Scores, τ, both sums and what is joined are fp32.  Two halfs keep q and τ to 2^-22
// of the largest, which a power of two brings near one.  A bf16 has 8 of fp32's 24
// bits: q and τ go in as three, cut off one after the other, and are exact (two parts
// keep 2^-17 of each, which an fp32 output showed as twenty times fp32's error).  The
// three parts of q are
//   up to 2 heads: four columns (one empty); two lanes share a sum and take a key each,
//   4 heads:       two columns and, in a product of its own, the first one again,
//   8 heads:       a column for each head, three products;
// those of τ rows of their own with up to 4 heads; with 8, O is turned round, Oᵀ =
// Vᵀ·Pᵀ, a column for each head and three products.  That costs 0.05 µs in the
// shortest step, nothing measurable with a head or two of 64 or 128 elements (up to
// 6 % at 32), 3-4 % with four heads and 3-12 % with eight (309 MB, 64 wide: 68.4 µs,
// with two parts 66.2; 128 wide 73.6 and 67.7, with half-filled second products 82).
//
// What bounds it: 1 flop a byte for 16-bit rows of a head of their own (memory),
// instructions for 8-bit rows of shared heads.  4 warps with 3 tiles of 4 KB each and
// 3-4 blocks an SM keep 100-130 KB under way.  Measured: 64 sequences of up to 8192
// keys × 16 heads, bf16: 164 µs for 1084 MB, the rate of a copy; one row set of 120002
// keys 75.6 µs (0.99); e4m3, 128 wide, four heads a key head: 189 µs for 1106 MB
// (0.89).  Tiles of 8 KB and half the blocks: 193 µs for the first.
#pragma once

#include <algorithm>
#include <atomic>
#include <utility>

#include "paged_decode.cuh"

namespace bozo {
namespace {

template <int DT> struct Fmt;
template <> struct Fmt<BOZO_DT_BF16> { static constexpr int size = 2; static constexpr bool bf = true, scaled = false; };
template <> struct Fmt<BOZO_DT_F16> { static constexpr int size = 2; static constexpr bool bf = false, scaled = false; };
template <> struct Fmt<BOZO_DT_F8E4M3> { static constexpr int size = 1; static constexpr bool bf = false, scaled = true; };
template <> struct Fmt<BOZO_DT_I8> { static constexpr int size = 1; static constexpr bool bf = false, scaled = true; };

template <bool BF>
__device__ __forceinline__ void mma16816(float* d, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                         unsigned b1) {
  if constexpr (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// x as a half (high half) and what that left of it (low half)
__device__ __forceinline__ unsigned split(float x) {
  unsigned w;
  const float h = __half2float(__float2half_rn(x));
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(x), "f"(x - h));
  return w;
}
// x = its first bf16 + the rest, exactly; the first bf16 of x and of y
__device__ __forceinline__ float less_top(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ unsigned tops(float x, float y) {
  return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
}

// Four 8-bit codes as two pairs of halfs (exact).
template <int DT>
__device__ __forceinline__ void widen4(unsigned x, unsigned& p01, unsigned& p23) {
  if constexpr (DT == BOZO_DT_F8E4M3) {
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}"
        : "=r"(p01), "=r"(p23) : "r"(x));
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

// σ(z) from −z·log2 e: one exponential and one reciprocal, each with a relative
// error of about 2^-22; results below 2^-126 are zero.
__device__ __forceinline__ float sigmoid_exp2(float y) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
template <int N, int OFF>  // N 32-bit words at a + OFF
__device__ __forceinline__ void lds_words(unsigned a, unsigned* w) {
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4 + %5];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a), "n"(OFF) : "memory");
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2 + %3];" : "=r"(w[0]), "=r"(w[1]) : "r"(a), "n"(OFF) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(w[0]) : "r"(a), "n"(OFF) : "memory");
}
// f(0), f(1), … f(N − 1) with the number as a constant
template <int... I, typename F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  each_of(std::make_integer_sequence<int, N>{}, f);
}
template <bool T>
__device__ __forceinline__ void ldmatrix4(unsigned a, unsigned* w) {
  if constexpr (T)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
}

// Asynchronous copies to shared memory; `bytes` 0 fills with zeros.
template <int DST, int SRC>
__device__ __forceinline__ void copy16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
}
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

constexpr int kWarps = 4;
constexpr int kStages = 3;

// Geometry of the kernel for one page type, head width and count of heads.
template <int DT, int HD, int GP> struct Geo {
  static constexpr int row = HD * Fmt<DT>::size;             // bytes of a row
  static constexpr int keys = row >= 128 ? 16 : 2048 / row;  // keys of a tile of the ring
  static constexpr int kv = keys * row;                      // bytes of its K (or V): 2 KB, 4 KB at 256-byte rows
  static constexpr int scales = Fmt<DT>::scaled ? 2 * keys * 4 : 0;
  static constexpr int meta = scales + 16;                   // scales, and 16 bits a 16 keys: which are in reach
  static constexpr int pstride = keys + 8;                   // words of a head's τ
  // Blocks an SM whose registers have to fit: two leave the compiler what it wants
  // (e4m3 128 wide, 616 MB: 113 µs, with three 118; e4m3 32 wide 146 against 153),
  // but 64 wide 8-bit rows are faster under the tighter bound (e4m3, 634 MB: 113
  // against 119), and so are 64 wide bf16 rows, which else take a few registers too
  // many for a third block (a head each, 617 MB: 96.7 against 99.7; eight heads, 309 MB:
  // 68.4 against 74).
  static constexpr int blocks = HD == 64 && (Fmt<DT>::scaled || Fmt<DT>::bf) ? 3 : 2;
  static constexpr bool fold = Fmt<DT>::bf && GP <= 4;  // τ's second parts have rows 4-7 of P
  static constexpr int parts = (fold ? 2 : 1) * kWarps;  // sums that are added at the end
  static constexpr int warp = kStages * (2 * kv + meta) + GP * pstride * (Fmt<DT>::bf ? 6 : 4);
};

// Byte offset of 16-byte piece ch of row r of a K or V tile with R-byte rows.  The
// pieces of a 128-byte line are permuted so that reading is free of bank
// conflicts: 16-bit rows are read as 8×8 matrices (8 rows' pieces of one number),
// 8-bit K rows two at a time, 8-bit V rows four at a time in steps of two.
template <int SIZE, int R, bool V> __device__ __forceinline__ int ring_at(int r, int ch) {
  if constexpr (SIZE == 2) {
    if constexpr (R >= 128) return r * R + ((ch ^ (r & 7)) << 4);
    else return (r >> 1) * 128 + (((((r & 1) << 2) | ch) ^ ((r >> 1) & 3)) << 4);
  } else if constexpr (R >= 128) {
    return r * R + ((ch ^ (V ? ((r >> 1) & 3) << 1 : (r & 1) << 2)) << 4);
  } else if constexpr (V) {
    constexpr int per = 128 / R;  // rows of a line
    const int line = r / per, c8 = (r % per) * (R / 16) + ch;
    return line * 128 + ((c8 ^ (R == 64 ? (line & 3) << 1 : (line & 1) << 1)) << 4);
  } else {
    return r * R + (ch << 4);
  }
}

// Block x: piece x mod S of key head hk's head group hg, (b·Hk + hk)·HG + hg = x / S.
struct MmaGrid {
  int S, G, HG;  // pieces, query heads of a key head, groups of them
  FastDiv div_s, div_hg, div_hk;
  bool clustered;
};

// GR: positions from a multiple of GR on that lie in one page (16, 8 or 1).
template <int DT, int HD, int GP, int GR>
__global__ void __launch_bounds__(kWarps * 32 + 32, Geo<DT, HD, GP>::blocks) paged_decode_mma(PagedP p, MmaGrid grid) {
  using F = Fmt<DT>;
  using Z = Geo<DT, HD, GP>;
  constexpr bool BF = F::bf;
  constexpr int R = Z::row, KT = Z::keys, NT = KT / 16, NCH = R / 16, SZ = F::size;
  constexpr bool QUAD = BF && GP <= 2, WIDE = BF && GP == 8;       // four columns of S a head, one
  constexpr int GQ = GP < 4 ? GP : 4;                              // heads whose columns repeat
  constexpr int NS = GP == 8 ? 2 : 1;                              // heads of a lane
  constexpr int NA = WIDE ? 1 : NS, NB = QUAD ? 1 : WIDE ? 3 : BF ? 2 : NS;  // accumulators, operands
  constexpr int kCopies = (QUAD ? 2 : 4) / GQ;                     // groups of lanes with the same columns
  constexpr int T = NT < kCopies ? NT : kCopies;                   // 16-key tiles whose scores they share out
  constexpr int kSteps = HD / 16, kTiles = HD / 8;
  // sums that a score's products run in side by side
  constexpr int NC = NA == 1 && kSteps * (BF ? NB : 1) >= 4 ? 2 : 1;
  constexpr int NK = QUAD ? 1 : 2;      // keys of a lane, of a tile's 16
  constexpr bool FOLD = Z::fold;
  // 8-bit rows: lane (g, c) reads a quarter of key rows g, g + 8 and an eighth of four value rows
  constexpr int kKB = R / 4 < 16 ? R / 4 : 16, kKL = R / (4 * kKB), kKW = kKB / 4;
  constexpr int kVB = R / 8 < 16 ? R / 8 : 16, kVL = R / (8 * kVB), kVW = kVB / 4;
  extern __shared__ __align__(256) char smb[];
  __shared__ float sq[BF ? 1 : kHeads][HD + 4];
  __shared__ __align__(4) unsigned short scut[BF ? GP : 1][3][HD + 8];  // the three bf16 of each q element
  __shared__ float sback[kHeads];  // what undoes the power of two that q was multiplied by (halfs)
  __shared__ float smass[kWarps][kHeads];
  const int S = grid.S, G = grid.G;
  const bool clustered = grid.clustered;
  const unsigned row = fast_div(blockIdx.x, grid.div_s), head = fast_div(row, grid.div_hg);
  const int piece = blockIdx.x - row * S, hg = row - head * grid.HG;
  const int b = fast_div(head, grid.div_hk), hk = head - b * p.Hk;
  const int h0 = hk * G + hg * kHeads, Gh = min(kHeads, G - hg * kHeads);  // query heads h0 … h0+Gh−1
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const Reach rc = reach(p, b, S);
  const bool mine = (unsigned)piece < rc.count;
  if (!mine && !clustered) return;
  const unsigned p0 = rc.first(piece), p1 = mine ? rc.last(piece) : p0;  // this block's positions
  const unsigned nk = p1 > p0 ? p1 - p0 : 0u;
  float mass[NS], unit[NS], lim[NS];  // P operand: p · unit, renewed where p passes lim (halfs)
  constexpr int kAcc = WIDE ? HD / 16 : kTiles;
  float acc[kAcc][4];
#pragma unroll
  for (int s = 0; s < NS; ++s) mass[s] = lim[s] = 0.f, unit[s] = 1.f;
#pragma unroll
  for (int j = 0; j < kAcc; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;

  const unsigned ring = smem_u32(smb) + warp * kStages * 2 * Z::kv;
  char* meta = smb + kWarps * kStages * 2 * Z::kv + warp * kStages * Z::meta;
  unsigned* ps = reinterpret_cast<unsigned*>(smb + kWarps * kStages * (2 * Z::kv + Z::meta)) + warp * GP * Z::pstride;
  char* lo = smb + kWarps * (kStages * (2 * Z::kv + Z::meta) + GP * Z::pstride * 4) + warp * GP * Z::pstride * 2;  // τ's third parts
  const char* kpages = static_cast<const char*>(p.k);
  const char* vpages = static_cast<const char*>(p.v);
  // Row numbers.  GR > 1: a look-up for GR keys, 32 of them at once, kBatch tiles'
  // worth; else one for each key of the next tile.
  constexpr bool AL = GR > 1;
  constexpr int RR = AL ? 1 : (KT > 32 ? KT / 32 : 1), kUnits = AL ? KT / GR : 1, kBatch = 32 / kUnits;
  unsigned cur[RR], nxt[RR];
  auto start = [&](int k) { return (unsigned)(warp + k * kWarps) * KT; };  // first key of the warp's tile k
  auto find = [&](int k, unsigned* rows) {
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const unsigned j =
          AL ? start(k + lane / kUnits) + lane % kUnits * GR : start(k) + r * 32 + (KT < 32 ? lane % KT : lane);
      rows[r] = kNoRow;
      // none for positions wholly before the reach: their pages may be gone
      if (j < nk && p0 + j + GR > rc.lo) {
        const unsigned row = paged_row(p, b, p0 + j);
        if (row != kNoRow) rows[r] = row + (unsigned)hk * p.page;
      }
    }
  };
  auto fill = [&](int slot, int k) {
    const unsigned kd = ring + slot * 2 * Z::kv, vd = kd + Z::kv;
    char* md = meta + slot * Z::meta;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      // rows of these 16 keys: from r0 on, and with GR 8 from r1 on the last eight
      const int src = AL ? k % kBatch * kUnits + u * 16 / GR : 0;
      const unsigned r0 = AL ? __shfl_sync(0xffffffffu, cur[0], src) : 0u;
      const unsigned r1 = GR == 8 ? __shfl_sync(0xffffffffu, cur[0], src + 1) : r0;
      const unsigned pos = p0 + start(k) + u * 16;
      auto whole = [&](int r) { return GR == 8 && r >= 8 ? r1 + r - 8 : r0 + r; };
      // the row of key r, or kNoRow
      auto row_of = [&](int r) {
        if constexpr (AL) return (r < 8 ? r0 : r1) == kNoRow || pos + r < rc.lo || pos + r >= p1 ? kNoRow : whole(r);
        else return __shfl_sync(0xffffffffu, cur[u / 2], (u * 16 + r) % 32);
      };
      if (AL && r0 != kNoRow && r1 != kNoRow && pos >= rc.lo && pos + 16 <= p1) {
        // rows that follow each other: from the first on 512 bytes a round
        const size_t at = (size_t)r0 * R + lane * 16, at1 = (size_t)r1 * R + lane * 16;
        // a round's place in the ring: the permutation repeats every 8 rows
        constexpr int kSame = 8 * NCH / 32 < 1 ? 1 : 8 * NCH / 32;  // rounds of 8 rows
        const char *ka = kpages + at, *va = vpages + at, *kb = kpages + at1, *vb = vpages + at1;
        each<(NCH + 1) / 2>([&](auto i) {
          constexpr int it = i, first = it % kSame, back = (it - first) * 512;
          const int r = (first * 32 + lane) / NCH, ch = lane % NCH;
          const bool second = GR == 8 && (it * 32 + lane) / NCH >= 8;
          copy16<back, it * 512>(kd + u * 16 * R + ring_at<SZ, R, false>(r, ch), second ? kb - 8 * R : ka);
          copy16<back, it * 512>(vd + u * 16 * R + ring_at<SZ, R, true>(r, ch), second ? vb - 8 * R : va);
        });
        if (F::scaled) copy4(smem_u32(md) + ((u * 16 + (lane & 15)) << 3) + (lane >> 4) * 4,
                             (lane < 16 ? p.ks : p.vs) + whole(lane & 15), 4);
        if (lane == 0) reinterpret_cast<unsigned short*>(md + Z::scales)[u] = 0xffffu;
      } else {
#pragma unroll
        for (int it = 0; it < (NCH + 1) / 2; ++it) {
          const int r = (it * 32 + lane) / NCH, ch = lane % NCH;
          const unsigned rr = row_of(r);
          const size_t at = rr == kNoRow ? 0 : (size_t)rr * R + ch * 16;
          copy16(kd + ring_at<SZ, R, false>(u * 16 + r, ch), kpages + at, rr == kNoRow ? 0 : 16);
          copy16(vd + ring_at<SZ, R, true>(u * 16 + r, ch), vpages + at, rr == kNoRow ? 0 : 16);
        }
        const unsigned rr = row_of(lane & 15);
        if (F::scaled) copy4(smem_u32(md) + ((u * 16 + (lane & 15)) << 3) + (lane >> 4) * 4,
                             (lane < 16 ? p.ks : p.vs) + (rr == kNoRow ? 0u : rr), rr == kNoRow ? 0 : 4);
        const unsigned m = __ballot_sync(0xffffffffu, rr != kNoRow);
        if (lane == 0) reinterpret_cast<unsigned short*>(md + Z::scales)[u] = (unsigned short)m;
      }
    }
  };
  // Fills the ring with tile k, if there is one, and looks ahead for the next rows.
  auto feed = [&](int slot, int k) {
    if (start(k) < nk) fill(slot, k);
    copy_commit();
    if (!AL) {
#pragma unroll
      for (int r = 0; r < RR; ++r) cur[r] = nxt[r];
      find(k + 2, nxt);
    } else if ((k + 1) % kBatch == 0) {
      cur[0] = nxt[0];
      find(k + 1 + kBatch, nxt);
    }
  };
  // A warp beyond the others writes the new token's row.  Keys that end with it are
  // read after a barrier: the one before the first tile is worked on, or if the
  // row's tile is among those that are fetched before that, one of their own.
  const bool writes = writes_row(p, rc, piece, hg == 0);
  const bool early = writes && p.mode == BOZO_MODE_GLOBAL && nk <= (kStages - 1) * kWarps * KT;
  if (warp == kWarps) {
    if (writes) append_row(p, b, hk, rc.t, lane);
    if (early) __syncthreads();
    __syncthreads();
  } else {
    // columns of S: lane (g, c) holds k-pairs of column g.  Of halfs that is head
    // (g/2) mod GQ of each operand, its 16-bit part (g even) or the rest.
    unsigned qb[NB][kSteps][2];
    float back[NS];
    // the heads, the tile (of T) and the keys whose τ this lane computes; one of the
    // lanes with the same
    auto head_of = [&](int e) { return QUAD ? (c >> 1) % GQ : WIDE ? 2 * c + e : e * 4 + c % GQ; };
    auto key_of = [&](int o) { return g + (QUAD ? 8 * (c & 1) : 8 * o); };
    const int copy = WIDE ? 0 : (QUAD ? c >> 1 : c) / GQ, tsel = copy % T;
    const bool once = copy < T;
    const int mrow = (lane & 7) + (lane & 8), mch = lane >> 4;  // row and piece of an 8×8 matrix's row

    find(0, cur);
    nxt[0] = kNoRow;
    if (!AL || start(kBatch) < nk) find(AL ? kBatch : 1, nxt);
    if (mine && rc.active)
      for (int i = tid; i < GP * HD; i += kWarps * 32) {
        const int h = i / HD, d = i - h * HD;
        const float x = h < Gh ? query(p, b, h0 + h, rc.t, d) : 0.f;
        if constexpr (BF) {
          const float x1 = less_top(x), x2 = less_top(x1);
          scut[h][0][d] = (unsigned short)(__float_as_uint(x) >> 16);
          scut[h][1][d] = (unsigned short)(__float_as_uint(x1) >> 16);
          scut[h][2][d] = (unsigned short)(__float_as_uint(x2) >> 16);
        } else {
          sq[h][d] = x;
        }
      }
    if (early) __syncthreads();
#pragma unroll 1
    for (int k = 0; k < kStages - 1; ++k) feed(k, k);
    __syncthreads();
    if (start(0) < nk) {
      if constexpr (BF) {
        const int h = QUAD ? (g >> 2) % GQ : WIDE ? g : g >> 1;
        auto pair = [&](int part, int d) { return *reinterpret_cast<const unsigned*>(&scut[h][part][d]); };
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int d = 16 * i + 8 * j + 2 * c;
            if constexpr (QUAD) {
              qb[0][i][j] = (g & 3) == 3 ? 0u : pair(g & 3, d);
            } else if constexpr (WIDE) {
#pragma unroll
              for (int e = 0; e < 3; ++e) qb[e][i][j] = pair(e, d);
            } else {
              qb[0][i][j] = pair(g & 1, d);
              qb[1][i][j] = g & 1 ? 0u : pair(2, d);
            }
          }
      } else {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const int h = s * 4 + (g >> 1) % GQ;
          // as halfs, brought near 1 by a power of two
          float m = 0.f;
          for (int d = c; d < HD; d += 4) m = fmaxf(m, fabsf(sq[h][d]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const int e = m > 0.f ? min(126, max(-126, (int)(__float_as_uint(m) >> 23) - 127)) : 0;
          const float qs = __uint_as_float((unsigned)(127 - e) << 23);
          if (c == 0) sback[h] = __uint_as_float((unsigned)(127 + e) << 23);  // every warp the same
          auto pair = [&](int d) {
            const unsigned u = split(sq[h][d] * qs), v = split(sq[h][d + 1] * qs);
            return __byte_perm(u, v, g & 1 ? 0x5410 : 0x7632);
          };
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            if constexpr (SZ == 2) {
              qb[s][i][0] = pair(16 * i + 2 * c);
              qb[s][i][1] = pair(16 * i + 8 + 2 * c);
            } else {
              const int d = i / kKW * 4 * kKB + c * kKB + i % kKW * 4;
              qb[s][i][0] = pair(d);
              qb[s][i][1] = pair(d + 2);
            }
          }
        }
      }
      __syncwarp();
      // exponent of the sigmoid: −log2 e · score
#pragma unroll
      for (int s = 0; s < NS; ++s)
        back[s] = (BF ? 1.f : sback[s * 4 + c % GQ]) * p.inv_scale * -1.4426950408889634f;
    }
    int slot = 0;
#pragma unroll 1
    for (int k = 0; start(k) < nk; ++k) {
      copy_wait<kStages - 2>();
      __syncwarp();
      feed(slot == 0 ? kStages - 1 : slot - 1, k + kStages - 1);
      const unsigned kt = ring + slot * 2 * Z::kv, vt = kt + Z::kv;
      const char* md = meta + slot * Z::meta;
      const float2* sc = reinterpret_cast<const float2*>(md);
      slot = slot == kStages - 1 ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < NT / T; ++q) {
        float s[T][NA][NC][4];
#pragma unroll
        for (int u = 0; u < T; ++u) {
#pragma unroll
          for (int e = 0; e < NA; ++e)
#pragma unroll
            for (int i = 0; i < NC; ++i) s[u][e][i][0] = s[u][e][i][1] = s[u][e][i][2] = s[u][e][i][3] = 0.f;
          const int r0 = (q * T + u) * 16;
          if constexpr (SZ == 2) {
            const unsigned a = kt + ring_at<SZ, R, false>(r0 + mrow, mch);
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
              unsigned w[4];
              ldmatrix4<false>(a ^ (st << 5), w);
#pragma unroll
              for (int e = 0; e < NB; ++e)
                mma16816<BF>(s[u][BF ? 0 : e][(BF ? st * NB + e : st) % NC], w[0], w[1], w[2], w[3], qb[e][st][0],
                             qb[e][st][1]);
            }
          } else {
            // 8 rows on the permutation is the same, and where a row is longer than a
            // line two 16-byte pieces on it is that with another bit turned over
            const int byte0 = c * kKB;
            const unsigned a0_ = kt + r0 * R + ring_at<SZ, R, false>(g, byte0 >> 4) + (byte0 & 15);
#pragma unroll
            for (int l = 0; l < kKL; ++l) {
              unsigned ka[kKW], kb[kKW];
              const unsigned at = a0_ ^ (l * 4 * kKB);
              lds_words<kKW, 0>(at, ka);
              lds_words<kKW, 8 * R>(at, kb);
#pragma unroll
              for (int w = 0; w < kKW; ++w) {
                unsigned a0, a1, a2, a3;
                widen4<DT>(ka[w], a0, a2);
                widen4<DT>(kb[w], a1, a3);
#pragma unroll
                for (int e = 0; e < NS; ++e)
                  mma16816<BF>(s[u][e][(l * kKW + w) % NC], a0, a1, a2, a3, qb[e][l * kKW + w][0],
                               qb[e][l * kKW + w][1]);
              }
            }
          }
        }
        const int tile = q * T + tsel;
        const unsigned live = reinterpret_cast<const unsigned short*>(md + Z::scales)[tile];
        float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
        if constexpr (F::scaled) {
          const float2 a = sc[tile * 16 + g], c2 = sc[tile * 16 + g + 8];  // a key's and a value's
          ks[0] = a.x, vs[0] = a.y, ks[1] = c2.x, vs[1] = c2.y;
        }
        // the score of key g + 8·o: a column's sums, or two columns'
        auto score = [&](int e, int o) {
          float z = 0.f;
#pragma unroll
          for (int u = 0; u < T; ++u) {
            float y = 0.f;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
              const float x = WIDE ? s[u][0][i][2 * o + e] : s[u][e][i][2 * o] + s[u][e][i][2 * o + 1];
              y = i == 0 ? x : y + x;
            }
            z = u == 0 || tsel == u ? y : z;
          }
          return z;
        };
#pragma unroll
        for (int e = 0; e < NS; ++e) {
          float pr[NK];
#pragma unroll
          for (int o = 0; o < NK; ++o) {
            float z;
            if constexpr (QUAD) {  // two lanes have two columns each: they swap halves of the keys
              const float z0 = score(e, 0), z1 = score(e, 1);
              const bool odd = c & 1;
              z = (odd ? z1 : z0) + __shfl_xor_sync(0xffffffffu, odd ? z0 : z1, 1);
            } else {
              z = score(e, o);
            }
            z *= back[e];
            if constexpr (F::scaled) z *= ks[o];
            const int key = key_of(o);
            const bool on = (live >> key) & 1;
            const float tau = on ? sigmoid_exp2(z) : 0.f;
            mass[e] += tau;
            // zero where a key in reach has no page
            const unsigned pos = p0 + start(k) + tile * 16 + key;
            if (p.tau && once && pos >= rc.lo && pos < p1 && head_of(e) < Gh)
              put_tau(p, (size_t)b * p.H + h0 + head_of(e), rc.t, pos, tau);
            pr[o] = F::scaled ? tau * vs[o] : tau;
          }
          if constexpr (!BF) {
            // halfs reach from 2^-24 to 65504: keep the largest p of a head between 1
            // and 4096 by a power of two, what was summed before following it
            const float pm = fmaxf(pr[0], pr[1]);
            if (__any_sync(0xffffffffu, pm > lim[e])) {
              float m = pm;
#pragma unroll
              for (int o = GQ; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
              float f = 1.f;
              if (m > lim[e]) {
                const int ex = min(113, max(-126, (int)(__float_as_uint(m) >> 23) - 127));
                const float nu = __uint_as_float((unsigned)(127 - ex) << 23);
                f = lim[e] == 0.f ? 0.f : nu / unit[e];
                unit[e] = nu;
                lim[e] = __uint_as_float((unsigned)(127 + ex + 12) << 23);
              }
              f = __shfl_sync(0xffffffffu, f, g % 4 % GQ);  // of this lane's row of O
              if (g / 4 == e || GP <= 4) {
#pragma unroll
                for (int j = 0; j < kTiles; ++j)
#pragma unroll
                  for (int i = 0; i < 4; ++i) acc[j][i] *= f;
              }
            }
            pr[0] *= unit[e];
            pr[1] *= unit[e];
          }
#pragma unroll
          for (int o = 0; o < NK; ++o) {
            const int at = head_of(e) * Z::pstride + tile * 16 + key_of(o);
            if constexpr (BF) {
              const float rest = less_top(pr[o]);
              ps[at] = tops(rest, pr[o]);
              reinterpret_cast<unsigned short*>(lo)[at] = (unsigned short)(__float_as_uint(less_top(rest)) >> 16);
            } else {
              ps[at] = split(pr[o]);
            }
          }
        }
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        unsigned a0 = 0, a1 = 0, a2 = 0, a3 = 0, l0 = 0, l2 = 0;
        const int h = FOLD ? g & 3 : g;  // the head of rows g and g + 8
        if (h < GP) {
          const int i = h * Z::pstride + u * 16 + 2 * c;
          unsigned x[2], y[2];
          lds_words<2, 0>(smem_u32(ps + i), x);
          lds_words<2, 32>(smem_u32(ps + i), y);
          if constexpr (BF) {
            lds_words<1, 0>(smem_u32(lo) + 2 * i, &l0);
            lds_words<1, 16>(smem_u32(lo) + 2 * i, &l2);
          }
          if constexpr (FOLD) {  // rows 0-3 and 8-11: first and third parts, rows 4-7: second parts
            a0 = __byte_perm(x[0], x[1], g < 4 ? 0x7632 : 0x5410);
            a2 = __byte_perm(y[0], y[1], g < 4 ? 0x7632 : 0x5410);
            a1 = g < 4 ? l0 : 0u;
            a3 = g < 4 ? l2 : 0u;
          } else {
            a0 = __byte_perm(x[0], x[1], 0x7632);
            a1 = __byte_perm(x[0], x[1], 0x5410);
            a2 = __byte_perm(y[0], y[1], 0x7632);
            a3 = __byte_perm(y[0], y[1], 0x5410);
          }
        }
        if constexpr (SZ == 2) {
          const unsigned a = vt + ring_at<SZ, R, true>(u * 16 + mrow, mch);
          if constexpr (WIDE) {  // Oᵀ = Vᵀ·Pᵀ: a product for each of the eight heads' parts
            constexpr int N = kAcc < 4 ? kAcc : 4;  // side by side
#pragma unroll
            for (int j = 0; j < kAcc; j += N) {
              unsigned w[N][4];
#pragma unroll
              for (int i = 0; i < N; ++i) ldmatrix4<true>(a ^ ((j + i) << 5), w[i]);
#pragma unroll
              for (int i = 0; i < N; ++i) mma16816<BF>(acc[j + i], w[i][0], w[i][2], w[i][1], w[i][3], a0, a2);
#pragma unroll
              for (int i = 0; i < N; ++i) mma16816<BF>(acc[j + i], w[i][0], w[i][2], w[i][1], w[i][3], a1, a3);
#pragma unroll
              for (int i = 0; i < N; ++i) mma16816<BF>(acc[j + i], w[i][0], w[i][2], w[i][1], w[i][3], l0, l2);
            }
          } else {
#pragma unroll
            for (int j = 0; j < kTiles; j += 2) {
              unsigned w[4];
              ldmatrix4<true>(a ^ (j << 4), w);
              mma16816<BF>(acc[j], a0, a1, a2, a3, w[0], w[1]);
              mma16816<BF>(acc[j + 1], a0, a1, a2, a3, w[2], w[3]);
            }
          }
        } else {
#pragma unroll
          for (int l = 0; l < kVL; ++l) {
            unsigned vw[4][kVW];
            const int byte = l * 8 * kVB + g * kVB;
            // rows 2c and 2c + 1 of each eight
            const unsigned v0 = vt + u * 16 * R + ring_at<SZ, R, true>(2 * c, byte >> 4) + (byte & 15);
            const unsigned v1 = vt + u * 16 * R + ring_at<SZ, R, true>(2 * c + 1, byte >> 4) + (byte & 15);
            lds_words<kVW, 0>(v0, vw[0]);
            lds_words<kVW, 0>(v1, vw[1]);
            lds_words<kVW, 8 * R>(v0, vw[2]);
            lds_words<kVW, 8 * R>(v1, vw[3]);
#pragma unroll
            for (int w = 0; w < kVW; ++w)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const unsigned sel = i ? 0x7362 : 0x5140;  // two keys' codes side by side
                unsigned x0, x1, y0, y1;
                widen4<DT>(__byte_perm(vw[0][w], vw[1][w], sel), x0, x1);
                widen4<DT>(__byte_perm(vw[2][w], vw[3][w], sel), y0, y1);
                const int j = l * kVB + 4 * w + 2 * i;
                mma16816<BF>(acc[j], a0, a1, a2, a3, x0, y0);
                mma16816<BF>(acc[j + 1], a0, a1, a2, a3, x1, y1);
              }
          }
        }
      }
    }
    copy_wait<0>();
  }

  // the warps' sums, added in order
  grid_release();
  __syncthreads();  // the rings and the queries are done with
  float* part = reinterpret_cast<float*>(smb);  // [parts][Gh][HD], then the block's [Gh][HD]
#pragma unroll
  for (int e = 0; e < NS; ++e) {
    // over all lanes but those of other heads
    float m = mass[e];
    if constexpr (QUAD) {
      m = (c >> 1) / GQ < T ? m : 0.f;
      m += __shfl_xor_sync(0xffffffffu, m, 1);
      if (GQ == 1) m += __shfl_xor_sync(0xffffffffu, m, 2);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      if (lane < 2 * GQ && warp < kWarps) smass[warp][lane >> 1] = m;
    } else {
      m = c / GQ < T ? m : 0.f;
#pragma unroll
      for (int o = GQ; o < 32; o <<= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      if (lane < GQ && warp < kWarps) smass[warp][WIDE ? 2 * lane + e : e * 4 + lane] = m;
    }
  }
  float un = 1.f;  // of head g
  if constexpr (!BF) {
    un = __shfl_sync(0xffffffffu, unit[0], g % 4 % GQ);
    if constexpr (NS == 2) {
      const float u1 = __shfl_sync(0xffffffffu, unit[1], g % 4);
      un = g < 4 ? un : u1;
    }
  }
  // rows of O: head g, or with FOLD head g mod 4 in two parts
  const int hrow = FOLD ? g & 3 : g;
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < kAcc; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)  // head 2c or 2c + 1, element g or g + 8
        if (2 * c + (e & 1) < Gh && warp < kWarps)
          part[(warp * Gh + 2 * c + (e & 1)) * HD + 16 * j + g + 8 * (e >> 1)] = acc[j][e];
  } else if (hrow < Gh && warp < kWarps) {
    const float back = 1.f / un;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = SZ == 2 ? 8 * j + 2 * c + e : j / kVB * 8 * kVB + (2 * c + e) * kVB + j % kVB;
        part[((FOLD ? 2 * warp + (g >> 2) : warp) * Gh + hrow) * HD + d] = (acc[j][e] + acc[j][2 + e]) * back;
      }
  }
  __syncthreads();
  float* sum = part + Z::parts * Gh * HD;
  for (int i = tid; i < Gh * HD && warp < kWarps; i += kWarps * 32) {
    const int h = i / HD, d = i - h * HD;
    float o = 0.f, m = 0.f;
#pragma unroll
    for (int w = 0; w < Z::parts; ++w) o += part[w * Gh * HD + i];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m += smass[w][h];
    const size_t bh = (size_t)b * p.H + h0 + h;
    if (rc.count == 1) {
      if (piece == 0) stf(p.out, (long long)(bh * HD + d), p.out_dt, o / norm_divisor(p, m, rc.n));
    } else if (clustered) {
      sum[i] = o;
      if (d == 0) sq[0][h] = m;
    } else {
      p.ws[(bh * S + piece) * HD + d] = o;
      if (d == 0) piece_mass(p, S)[bh * S + piece] = m;
    }
  }
  if (p.tau && piece == 0)
    for (int h = warp; h < Gh && warp < kWarps; h += kWarps) clear_tau(p, (size_t)b * p.H + h0 + h, rc.n, lane, 32);
  if (clustered) {
    // the pieces' sums through the cluster's shared memory, each block a part of
    // the elements, in the order of the pieces
    cluster_sync();
    if (rc.count > 1 && warp < kWarps)
      for (int i = tid + piece * kWarps * 32; i < Gh * HD; i += S * kWarps * 32) {
        const int h = i / HD, d = i - h * HD;
        float o = 0.f, m = 0.f;
        for (unsigned r = 0; r < rc.count; ++r) {
          o += ld_peer(smem_u32(sum + i), r);
          m += ld_peer(smem_u32(&sq[0][h]), r);
        }
        const size_t bh = (size_t)b * p.H + h0 + h;
        stf(p.out, (long long)(bh * HD + d), p.out_dt, o / norm_divisor(p, m, rc.n));
      }
    cluster_sync();
  }
}

template <int DT, int HD, int GP, int GR>
cudaError_t launch_paged_mma(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  const int G = p.H / p.Hk, HG = (G + kHeads - 1) / kHeads;
  using Z = Geo<DT, HD, GP>;
  const size_t ring = (size_t)kWarps * Z::warp;
  const size_t part = (size_t)(Z::parts + 1) * std::min(G, kHeads) * HD * sizeof(float);
  const size_t smem = std::max(ring, part);
  auto kern = paged_decode_mma<DT, HD, GP, GR>;
  static std::atomic<unsigned long long> allowed{0};  // devices where the kernel may use that much
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
    const int most = (int)std::max(ring, (size_t)(Z::parts + 1) * kHeads * HD * sizeof(float));
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
    if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((long long)p.B * p.Hk * HG * pl.S));
  cfg.blockDim = dim3(kWarps * 32 + (p.kn.p ? 32 : 0));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)pl.S, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = pl.clustered ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p, MmaGrid{pl.S, G, HG, make_fastdiv(pl.S), make_fastdiv(HG), make_fastdiv(p.Hk), pl.clustered});
}
template <int DT, int HD, int GP>
cudaError_t launch_paged_mma(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  if (p.page % 16 == 0) return launch_paged_mma<DT, HD, GP, 16>(p, pl, st);
  return p.page % 8 == 0 ? launch_paged_mma<DT, HD, GP, 8>(p, pl, st) : launch_paged_mma<DT, HD, GP, 1>(p, pl, st);
}
template <int DT, int HD>
cudaError_t launch_paged_mma(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  const int G = p.H / p.Hk;
  if (G == 1) return launch_paged_mma<DT, HD, 1>(p, pl, st);
  if (G == 2) return launch_paged_mma<DT, HD, 2>(p, pl, st);
  if (G <= 4) return launch_paged_mma<DT, HD, 4>(p, pl, st);
  return launch_paged_mma<DT, HD, 8>(p, pl, st);
}
template <int DT>
cudaError_t launch_paged_mma(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  switch (p.HD) {
    case 32: return launch_paged_mma<DT, 32>(p, pl, st);
    case 64: return launch_paged_mma<DT, 64>(p, pl, st);
    default: return launch_paged_mma<DT, 128>(p, pl, st);
  }
}

}  // namespace
}  // namespace bozo
