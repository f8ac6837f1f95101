// paged_mma.cuh — the tensor-core kernel of a decode step over a paged cache:
// 16-, 8- and 4-bit pages, head widths 32, 64 and 128.
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
// 4-bit rows: a code (e2m1) times its group's scale (e4m3) is a half exactly, so a product
// goes as for 8 bits, and O is turned round up to four heads (half the products, and half
// the accumulators).  With a head each the scales of groups are not multiplied into the
// codes at all.  Of S's eight columns two belong to each quarter of the elements, which
// are those of one lane of four, with scales of its own: its sums take them, and the four
// lanes add up theirs.  Of O's, two belong to each group (128 wide: of either half): τ times
// the key's scale of that group, as a half and the rest of it; of the products those of an
// element's own group are kept.
//
// What bounds it: 1 flop a byte for 16-bit rows of a head of their own (memory),
// instructions for 8-bit rows of shared heads.  4 warps with 3 tiles of 4 KB each and
// 3-4 blocks an SM keep 100-130 KB under way.  Measured: 64 sequences of up to 8192
// keys × 16 heads, bf16: 164 µs for 1084 MB, the rate of a copy; one row set of 120002
// keys 75.6 µs (0.99); e4m3, 128 wide, four heads a key head: 189 µs for 1106 MB
// (0.89).  Tiles of 8 KB and half the blocks: 193 µs for the first.  4-bit rows: 180
// instructions for 16 keys of 1.3 KB, many of them conversions and selections that run at
// half rate, bound them (a head each, 64 ragged sequences × 16 heads: 77 µs for 337 MB, 0.67
// of a copy; before the last steps 79, then 66 with no page read at all, 83 with scaled codes;
// 91 where the new rows are written).  128 wide, four heads: 178 µs for 658 MB.
#pragma once

#include <limits.h>

#include <algorithm>
#include <atomic>
#include <utility>

#include "paged_decode.cuh"

namespace bozo {
namespace {

// size: bytes of an element, 0: half a byte
template <int DT> struct Fmt;
template <> struct Fmt<BOZO_DT_BF16> { static constexpr int size = 2; static constexpr bool bf = true, scaled = false; };
template <> struct Fmt<BOZO_DT_F16> { static constexpr int size = 2; static constexpr bool bf = false, scaled = false; };
template <> struct Fmt<BOZO_DT_F8E4M3> { static constexpr int size = 1; static constexpr bool bf = false, scaled = true; };
template <> struct Fmt<BOZO_DT_I8> { static constexpr int size = 1; static constexpr bool bf = false, scaled = true; };
template <> struct Fmt<BOZO_DT_F4E2M1> { static constexpr int size = 0; static constexpr bool bf = false, scaled = true; };

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

// Eight 4-bit codes as pairs of halfs.
__device__ __forceinline__ void codes8(unsigned x, unsigned* w) {
  asm("{.reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %4; cvt.rn.f16x2.e2m1x2 %0, a; cvt.rn.f16x2.e2m1x2 %1, b;"
      " cvt.rn.f16x2.e2m1x2 %2, c; cvt.rn.f16x2.e2m1x2 %3, d;}"
      : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(x));
}
// … times the scales s (two halfs): exact, since the product has 6 significant bits and
// lies between 2^-10 and 2688.
__device__ __forceinline__ void widen8(unsigned x, unsigned s, unsigned* w) {
  codes8(x, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&w[i]), *reinterpret_cast<const __half2*>(&s));
    w[i] = *reinterpret_cast<const unsigned*>(&y);
  }
}
// The two e4m3 in the low half of x as halfs.
__device__ __forceinline__ unsigned group_pair(unsigned x) {
  unsigned w;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(w) : "r"(x));
  return w;
}
__device__ __forceinline__ float2 halves(unsigned x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
// τ · unit · kGroupUnit times a group's scale (≤ 448) stays under 65504.  Its rest beside
// the half goes in times kRest, in a column of its own: with the smallest group scale, 2^-9,
// the largest τ of a head gives at least 2^-15, which is then held to 2^-36 (without kRest to
// 2^-25: columns whose groups are far below their rows' largest were off by up to 2^-10).
constexpr float kGroupUnit = 0x1p-6f, kRest = 0x1p11f;
__device__ __forceinline__ unsigned two_halves(float x, float y) {
  unsigned w;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
  return w;
}
template <int N> __device__ __forceinline__ unsigned lds_part(unsigned a) {  // 1 or 2 bytes
  unsigned short x;
  if constexpr (N == 1) asm volatile("ld.shared.u8 %0, [%1];" : "=h"(x) : "r"(a) : "memory");
  else asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(a) : "memory");
  return x;
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
__device__ __forceinline__ void copy8(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
// Windows up to here take tiles of 32 4-bit rows, for more of the warps (16 sequences × 12
// heads that write their new rows, as a model's step does, in a graph: 64 keys 6.3 µs, with
// tiles of 64 rows 7.1; 128 keys 6.8 and 7.2, 256 8.1 and 8.8, 512 9.8 and 9.7; without new rows
// 4.8 and 5.6, 5.7 and 5.5, 6.6 and 7.3, 8.7 and 8.3).
constexpr int kShortWindow = 256;


// Geometry of the kernel for one page type, head width and count of heads.
// KEYS: of a tile, where it is not the usual count.
template <int DT, int HD, int GP, int KEYS = 0> struct Geo {
  static constexpr bool four = Fmt<DT>::size == 0;
  static constexpr int row = four ? HD / 2 : HD * Fmt<DT>::size;  // bytes of a row
  static constexpr int keys = KEYS ? KEYS : row >= 128 ? 16 : row >= 32 ? 2048 / row : 64;  // keys of a tile of the ring
  static constexpr int kv = keys * row;                      // bytes of its K (or V): 1 or 2 KB, 4 KB at 256-byte rows
  static constexpr int scales = Fmt<DT>::scaled ? 2 * keys * 4 : 0;
  static constexpr int gr = four ? HD / 16 : 0;              // bytes of a row's group scales
  static constexpr int live = scales + 2 * keys * gr;        // offset of the 16 bits a 16 keys: which are in reach
  static constexpr int meta = live + 16;                     // scales, K's and V's group scales, those bits
  static constexpr int pstride = keys + 8;                   // words of a head's τ
  // Blocks an SM whose registers have to fit: two leave the compiler what it wants
  // (e4m3 128 wide, 616 MB: 113 µs, with three 118; e4m3 32 wide 146 against 153),
  // but 64 wide 8-bit rows are faster under the tighter bound (e4m3, 634 MB: 113
  // against 119), and so are 64 wide bf16 rows, which else take a few registers too
  // many for a third block (a head each, 617 MB: 96.7 against 99.7; eight heads, 309 MB:
  // 68.4 against 74).
  static constexpr bool lone = four && GP == 1;  // a head each: group scales go to the scores and to τ
  static constexpr bool turned = four && GP <= 4;  // O turned round: a column for each head's two halfs
  // 4-bit rows (64 ragged sequences): 64 wide four (a head each 87 µs, with three 91, two 98),
  // 128 wide three (four heads 141, with four 150, two 152); eight heads one less (157 to 139).
  static constexpr int blocks = four ? (HD == 128 ? 3 : 4) - (GP == 8) : HD == 64 && (Fmt<DT>::scaled || Fmt<DT>::bf) ? 3 : 2;
  static constexpr bool fold = Fmt<DT>::bf && GP <= 4;  // τ's second parts have rows 4-7 of P
  static constexpr int parts = (fold ? 2 : 1) * kWarps;  // sums that are added at the end
  static constexpr int stages = four && !KEYS ? 2 : 3;                // tiles of the ring; 4-bit rows' take so long that
                                                             // two do (64 ragged sequences 104 µs, with three 114)
  static constexpr int warp = stages * (2 * kv + meta) + GP * pstride * (Fmt<DT>::bf ? 6 : 4);
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
    if constexpr (R < 32) return r * R + (ch << 4);
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
  bool sorted;   // the longest sequences' blocks first
};

// The sequence with `rank` longer ones, of up to kSorted.  With the longest first the
// blocks that start last are short (64 sequences of up to 8192 keys, 4-bit pages: 94 µs,
// in their own order 105).
constexpr int kSortedBlocks = 600;  // more than one wave
__device__ __forceinline__ int by_length(const PagedP& p, int rank) {
  __shared__ __align__(16) int len[kSorted];
  __shared__ int found;
  const int t = threadIdx.x;
  if (t < kSorted) len[t] = t < p.B ? __ldg(p.len + t) : INT_MIN;
  __syncthreads();
  if (t < p.B) {
    const int mine = len[t];
    int before = 0;
    for (int i = 0; i < p.B; i += 4) {
      const int4 x = *reinterpret_cast<const int4*>(len + i);
      before += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
      before += (x.x == mine && i < t) + (x.y == mine && i + 1 < t) + (x.z == mine && i + 2 < t) + (x.w == mine && i + 3 < t);
    }
    if (before == rank) found = t;
  }
  __syncthreads();
  return found;
}

// GR: positions from a multiple of GR on that lie in one page (16, 8 or 1).
template <int DT, int HD, int GP, int GR, int KEYS = 0>
__global__ void __launch_bounds__(kWarps * 32 + 32, Geo<DT, HD, GP, KEYS>::blocks) paged_decode_mma(PagedP p, MmaGrid grid) {
  using F = Fmt<DT>;
  using Z = Geo<DT, HD, GP, KEYS>;
  constexpr bool BF = F::bf;
  constexpr int R = Z::row, KT = Z::keys, NT = KT / 16, NCH = R / 16, SZ = F::size, RS = Z::four ? 1 : SZ, GB = Z::gr;
  constexpr bool QUAD = BF && GP <= 2, WIDE = BF && GP == 8;       // four columns of S a head, one
  constexpr bool LONE = Z::lone, TURN = Z::turned;
  constexpr int GQ = GP < 4 ? GP : 4;                              // heads whose columns repeat
  constexpr int NS = GP == 8 ? 2 : 1;                              // heads of a lane
  constexpr int NA = WIDE ? 1 : NS, NB = QUAD ? 1 : WIDE ? 3 : BF ? 2 : NS;  // accumulators, operands
  constexpr int kCopies = (QUAD ? 2 : 4) / GQ;                     // groups of lanes with the same columns
  constexpr int T = NT < kCopies ? NT : kCopies;                   // 16-key tiles whose scores they share out
  constexpr int kSteps = HD / 16, kTiles = HD / 8;
  // sums that a score's products run in side by side
  constexpr int NC = NA == 1 && kSteps * (BF ? NB : 1) >= 4 ? 2 : 1;
  constexpr bool ONE = QUAD || (LONE && T == 2);
  constexpr int NK = ONE ? 1 : 2;       // keys of a lane, of a tile's 16
  constexpr bool FOLD = Z::fold;
  // 8-bit rows: lane (g, c) reads a quarter of key rows g, g + 8 and an eighth of four value rows
  constexpr int kKB = R / 4 < 16 ? R / 4 : 16, kKL = R / (4 * kKB), kKW = kKB / 4;
  constexpr int kVB = R / 8 < 16 ? R / 8 : 16, kVL = R / (8 * kVB), kVW = kVB < 4 ? 1 : kVB / 4;
  extern __shared__ __align__(256) char smb[];
  __shared__ float sq[BF ? 1 : kHeads][HD + 4];
  __shared__ __align__(4) unsigned short scut[BF ? GP : 1][3][HD + 8];  // the three bf16 of each q element
  __shared__ float sback[kHeads];  // what undoes the power of two that q was multiplied by (halfs)
  __shared__ float smass[kWarps][kHeads];
  const int S = grid.S, G = grid.G;
  const bool clustered = grid.clustered;
  const unsigned row = fast_div(blockIdx.x, grid.div_s), head = fast_div(row, grid.div_hg);
  const int piece = blockIdx.x - row * S, hg = row - head * grid.HG;
  int b = fast_div(head, grid.div_hk);
  const int hk = head - b * p.Hk;
  if constexpr (Z::four) {
    if (grid.sorted) b = by_length(p, b);
  }
  const int h0 = hk * G + hg * kHeads, Gh = min(kHeads, G - hg * kHeads);  // query heads h0 … h0+Gh−1
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  // a short table's row (a window's ring) is fetched beside the length
  const bool ring_row = Z::four && p.M <= 32;
  const int my_page = ring_row && lane < p.M ? __ldg(p.table + b * p.ts + lane) : 0;
  const Reach rc = reach(p, b, S);
  const bool mine = (unsigned)piece < rc.count;
  if (!mine && !clustered) return;
  const unsigned p0 = rc.first(piece), p1 = mine ? rc.last(piece) : p0;  // this block's positions
  const unsigned nk = p1 > p0 ? p1 - p0 : 0u;
  float mass[NS], unit[NS], lim[NS];  // P operand: p · unit, renewed where p passes lim (halfs)
  constexpr int kAcc = WIDE || TURN ? HD / 16 : kTiles;
  float acc[kAcc][4];
#pragma unroll
  for (int s = 0; s < NS; ++s) mass[s] = lim[s] = 0.f, unit[s] = 1.f;
#pragma unroll
  for (int j = 0; j < kAcc; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;

  const unsigned ring = smem_u32(smb) + warp * Z::stages * 2 * Z::kv;
  char* meta = smb + kWarps * Z::stages * 2 * Z::kv + warp * Z::stages * Z::meta;
  unsigned* ps = reinterpret_cast<unsigned*>(smb + kWarps * Z::stages * (2 * Z::kv + Z::meta)) + warp * GP * Z::pstride;
  char* lo = smb + kWarps * (Z::stages * (2 * Z::kv + Z::meta) + GP * Z::pstride * 4) + warp * GP * Z::pstride * 2;  // τ's third parts
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
      if (Z::four && ring_row) {
        const unsigned pos = p0 + j, s = pos - fast_div(pos, p.div_cap) * p.cap, col = fast_div(s, p.div_page);
        const unsigned pid = (unsigned)__shfl_sync(0xffffffffu, my_page, col & 31);
        if (j < nk && pos + GR > rc.lo) {
          if (pid < (unsigned)p.P) rows[r] = (pid * (unsigned)p.Hk + (unsigned)hk) * (unsigned)p.page + (s - col * (unsigned)p.page);
          else atomicCAS(p.err, 0, kErrPaged | 2);
        }
        continue;
      }
      // none for positions wholly before the reach: their pages may be gone
      if (j < nk && p0 + j + GR > rc.lo) {
        const unsigned row = paged_row(p, b, p0 + j);
        if (row != kNoRow) rows[r] = row + (unsigned)hk * p.page;
      }
    }
  };
  // The group scales of key u·16 + lane mod 16 (K's by the first 16 lanes, V's by the others)
  // from row rr; zeros without one, as its codes: a product with what a page holds there
  // could be NaN.
  // (offset of a key's scale, of K and of V: side by side, or for 4 bits all of K's first)
  auto scale_at = [](int key, int v) { return Z::four ? (v * KT + key) * 4 : key * 8 + v * 4; };
  auto put_groups = [&](char* md, int u, unsigned rr) {
    const unsigned to = smem_u32(md) + Z::scales + (lane >> 4) * KT * GB + (u * 16 + (lane & 15)) * GB;
    const unsigned char* from = (lane < 16 ? p.kg : p.vg) + (rr == kNoRow ? 0 : (size_t)rr * GB);
    if constexpr (GB == 8) copy8(to, from, rr == kNoRow ? 0 : 8);
    else if constexpr (GB == 4) copy4(to, from, rr == kNoRow ? 0 : 4);
    else if constexpr (GB == 2) {  // too short for an asynchronous copy; only at the ends of the reach and of odd pages
      const unsigned short x = rr == kNoRow ? 0 : *reinterpret_cast<const unsigned short*>(from);
      asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(x) : "memory");
    }
  };
  auto fill = [&](int slot, int k) {
    const unsigned kd = ring + slot * 2 * Z::kv, vd = kd + Z::kv;
    char* md = meta + slot * Z::meta;
    if constexpr (Z::four && GR == 16) {
      // a tile of whole pages' parts: rows and both kinds of scales 16 bytes at a time
      const int at = k % kBatch * kUnits;
      const unsigned pos = p0 + start(k), have = __ballot_sync(0xffffffffu, cur[0] != kNoRow) >> at;
      if (pos >= rc.lo && pos + KT <= p1 && (have & ((1u << NT) - 1u)) == (1u << NT) - 1u) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const size_t r0 = (size_t)__shfl_sync(0xffffffffu, cur[0], at + u) * R;
          if constexpr (NCH == 1) {
            copy16((lane < 16 ? kd : vd) + u * 16 * R + (lane & 15) * R, (lane < 16 ? kpages : vpages) + r0 + (lane & 15) * R, 16);
          } else {
            const char *ka = kpages + r0 + lane * 16, *va = vpages + r0 + lane * 16;
            each<NCH / 2>([&](auto i) {
              constexpr int it = i;  // the permutation repeats every 8 rows: the places of all rounds are alike
              copy16<0, it * 512>(kd + (u * 16 + it * 32 / NCH) * R + ring_at<RS, R, false>(lane / NCH, lane % NCH), ka);
              copy16<0, it * 512>(vd + (u * 16 + it * 32 / NCH) * R + ring_at<RS, R, true>(lane / NCH, lane % NCH), va);
            });
          }
        }
        constexpr int NS4 = NT * 4, NG4 = NT * GB;  // 16-byte pieces of a tile's scales, group scales
        const unsigned to = smem_u32(md) + lane * 16;
        const unsigned rs = __shfl_sync(0xffffffffu, cur[0], at + lane % NS4 / 4);
        if (lane < 2 * NS4) copy16(to, (lane < NS4 ? p.ks : p.vs) + rs + lane % 4 * 4, 16);
        const unsigned rg = __shfl_sync(0xffffffffu, cur[0], at + lane % NG4 / GB);
        if (lane < 2 * NG4) copy16(to + Z::scales, (lane < NG4 ? p.kg : p.vg) + (size_t)rg * GB + lane % GB * 16, 16);
        if (lane < NT) reinterpret_cast<unsigned short*>(md + Z::live)[lane] = 0xffffu;
        return;
      }
    }
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
        if constexpr (NCH == 1) {  // a piece a row: 16 lanes for K, 16 for V
          const int r = lane & 15;
          copy16((lane < 16 ? kd : vd) + u * 16 * R + r * R, (lane < 16 ? kpages : vpages) + (size_t)whole(r) * R, 16);
        } else each<(NCH + 1) / 2>([&](auto i) {
          constexpr int it = i, first = it % kSame, back = (it - first) * 512;
          const int r = (first * 32 + lane) / NCH, ch = lane % NCH;
          const bool second = GR == 8 && (it * 32 + lane) / NCH >= 8;
          copy16<back, it * 512>(kd + u * 16 * R + ring_at<RS, R, false>(r, ch), second ? kb - 8 * R : ka);
          copy16<back, it * 512>(vd + u * 16 * R + ring_at<RS, R, true>(r, ch), second ? vb - 8 * R : va);
        });
        if (F::scaled) copy4(smem_u32(md) + scale_at(u * 16 + (lane & 15), lane >> 4),
                             (lane < 16 ? p.ks : p.vs) + whole(lane & 15), 4);
        if constexpr (GB == 2) {  // two rows' at a time, which begin at an even one
          const int r = 2 * (lane & 7);
          if (lane < 16)
            copy4(smem_u32(md) + Z::scales + (lane >> 3) * KT * GB + (u * 16 + r) * GB,
                  (lane < 8 ? p.kg : p.vg) + (size_t)whole(r) * GB, 4);
        } else if constexpr (GB > 0) {
          put_groups(md, u, whole(lane & 15));
        }
        if (lane == 0) reinterpret_cast<unsigned short*>(md + Z::live)[u] = 0xffffu;
      } else {
        if constexpr (NCH == 1) {
          const int r = lane & 15;
          const unsigned rr = row_of(r);
          copy16((lane < 16 ? kd : vd) + (u * 16 + r) * R,
                 (lane < 16 ? kpages : vpages) + (rr == kNoRow ? 0 : (size_t)rr * R), rr == kNoRow ? 0 : 16);
        } else {
#pragma unroll
          for (int it = 0; it < (NCH + 1) / 2; ++it) {
            const int r = (it * 32 + lane) / NCH, ch = lane % NCH;
            const unsigned rr = row_of(r);
            const size_t at = rr == kNoRow ? 0 : (size_t)rr * R + ch * 16;
            copy16(kd + ring_at<RS, R, false>(u * 16 + r, ch), kpages + at, rr == kNoRow ? 0 : 16);
            copy16(vd + ring_at<RS, R, true>(u * 16 + r, ch), vpages + at, rr == kNoRow ? 0 : 16);
          }
        }
        const unsigned rr = row_of(lane & 15);
        if (F::scaled) copy4(smem_u32(md) + scale_at(u * 16 + (lane & 15), lane >> 4),
                             (lane < 16 ? p.ks : p.vs) + (rr == kNoRow ? 0u : rr), rr == kNoRow ? 0 : 4);
        if constexpr (GB > 0) put_groups(md, u, rr);
        const unsigned m = __ballot_sync(0xffffffffu, rr != kNoRow);
        if (lane == 0) reinterpret_cast<unsigned short*>(md + Z::live)[u] = (unsigned short)m;
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
  const bool early = writes && p.mode == BOZO_MODE_GLOBAL && nk <= (Z::stages - 1) * kWarps * KT;
  if (warp == kWarps) {
    if (writes) append_row<DT>(p, b, hk, rc.t, lane);
    if (early) __syncthreads();
    __syncthreads();
  } else {
    // columns of S: lane (g, c) holds k-pairs of column g.  Of halfs that is head
    // (g/2) mod GQ of each operand, its 16-bit part (g even) or the rest.
    unsigned qb[NB][kSteps][2];
    float back[NS];
    // the heads, the tile (of T) and the keys whose τ this lane computes; one of the
    // lanes with the same
    auto head_of = [&](int e) { return LONE ? 0 : QUAD ? (c >> 1) % GQ : WIDE ? 2 * c + e : e * 4 + c % GQ; };
    auto key_of = [&](int o) { return g + (QUAD ? 8 * (c & 1) : ONE ? 8 * (c >> 1) : 8 * o); };
    const int copy = WIDE ? 0 : (QUAD ? c >> 1 : c) / GQ, tsel = copy % T;
    const bool once = LONE || copy < T;
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
    for (int k = 0; k < Z::stages - 1; ++k) feed(k, k);
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
          const int h = LONE ? 0 : s * 4 + (g >> 1) % GQ;
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
            // a head each: two columns for each quarter of the elements, which have scales of their own
            return LONE && c != g >> 1 ? 0u : __byte_perm(u, v, g & 1 ? 0x5410 : 0x7632);
          };
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            if constexpr (SZ == 2) {
              qb[s][i][0] = pair(16 * i + 2 * c);
              qb[s][i][1] = pair(16 * i + 8 + 2 * c);
            } else {
              const int d = SZ == 0 ? c * 2 * kKB + 4 * i : i / kKW * 4 * kKB + c * kKB + i % kKW * 4;
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
      copy_wait<Z::stages - 2>();
      __syncwarp();
      feed(slot == 0 ? Z::stages - 1 : slot - 1, k + Z::stages - 1);
      const unsigned kt = ring + slot * 2 * Z::kv, vt = kt + Z::kv;
      const char* md = meta + slot * Z::meta;
      const float2* sc = reinterpret_cast<const float2*>(md);
      slot = slot == Z::stages - 1 ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < NT / T; ++q) {
        float s[T][NA][NC][4], y[LONE ? T : 1][2];
#pragma unroll
        for (int u = 0; u < T; ++u) {
#pragma unroll
          for (int e = 0; e < NA; ++e)
#pragma unroll
            for (int i = 0; i < NC; ++i) s[u][e][i][0] = s[u][e][i][1] = s[u][e][i][2] = s[u][e][i][3] = 0.f;
          const int r0 = (q * T + u) * 16;
          if constexpr (SZ == 2) {
            const unsigned a = kt + ring_at<RS, R, false>(r0 + mrow, mch);
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
              unsigned w[4];
              ldmatrix4<false>(a ^ (st << 5), w);
#pragma unroll
              for (int e = 0; e < NB; ++e)
                mma16816<BF>(s[u][BF ? 0 : e][(BF ? st * NB + e : st) % NC], w[0], w[1], w[2], w[3], qb[e][st][0],
                             qb[e][st][1]);
            }
          } else if constexpr (SZ == 0) {
            // lane (g, c): a quarter of rows g and g + 8, 8, 16 or 32 elements from c·HD/4 on
            const unsigned at = kt + (r0 + g) * R + c * kKB;
            const unsigned gs = smem_u32(md) + Z::scales + (r0 + g) * GB + c * GB / 4;
            unsigned ka[kKW], kb[kKW];
            lds_words<kKW, 0>(at, ka);
            lds_words<kKW, 8 * R>(at, kb);
            constexpr int NG = GB == 8 ? 2 : 1;  // groups of a lane's elements
            const unsigned ga = lds_part<NG>(gs), gb = lds_part<NG>(gs + 8 * GB);
            if constexpr (LONE) {
              // the codes as they are; this lane's two columns are those of its quarter, so
              // its sums take the quarter's scales (128 wide: two sums, of a group each)
              static_assert(NC >= NG, "a sum for each group");
#pragma unroll
              for (int w = 0; w < kKW; ++w) {
                const int i = NG == 2 ? w / (kKW / 2) : 0;
                unsigned x[4], z[4];
                codes8(ka[w], x);
                codes8(kb[w], z);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  mma16816<BF>(s[u][0][i], x[2 * h], z[2 * h], x[2 * h + 1], z[2 * h + 1], qb[0][2 * w + h][0],
                               qb[0][2 * w + h][1]);
              }
              const float2 fa = halves(group_pair(ga)), fb = halves(group_pair(gb));
              y[u][0] = (s[u][0][0][0] + s[u][0][0][1]) * fa.x;
              y[u][1] = (s[u][0][0][2] + s[u][0][0][3]) * fb.x;
              if constexpr (NG == 2) {
                y[u][0] = fmaf(s[u][0][NG - 1][0] + s[u][0][NG - 1][1], fa.y, y[u][0]);
                y[u][1] = fmaf(s[u][0][NG - 1][2] + s[u][0][NG - 1][3], fb.y, y[u][1]);
              }
              continue;
            }
#pragma unroll
            for (int w = 0; w < kKW; ++w) {
              const unsigned sel = NG == 2 && w >= kKW / 2 ? 0x1111 : 0x0000;
              unsigned x[4], y[4];
              widen8(ka[w], group_pair(__byte_perm(ga, 0, sel)), x);
              widen8(kb[w], group_pair(__byte_perm(gb, 0, sel)), y);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < NS; ++e)
                  mma16816<BF>(s[u][e][(2 * w + h) % NC], x[2 * h], y[2 * h], x[2 * h + 1], y[2 * h + 1],
                               qb[e][2 * w + h][0], qb[e][2 * w + h][1]);
            }
          } else {
            // 8 rows on the permutation is the same, and where a row is longer than a
            // line two 16-byte pieces on it is that with another bit turned over
            const int byte0 = c * kKB;
            const unsigned a0_ = kt + r0 * R + ring_at<RS, R, false>(g, byte0 >> 4) + (byte0 & 15);
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
        float z4[2];
        if constexpr (LONE) {
          // the four quarters' sums: each lane is left with its tile's keys
          if constexpr (T == 4) {
            const bool up = c & 2, odd = c & 1;
            float h[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int o = 0; o < 2; ++o)
                h[i][o] = (up ? y[i + 2][o] : y[i][o]) + __shfl_xor_sync(0xffffffffu, up ? y[i][o] : y[i + 2][o], 2);
#pragma unroll
            for (int o = 0; o < 2; ++o)
              z4[o] = (odd ? h[1][o] : h[0][o]) + __shfl_xor_sync(0xffffffffu, odd ? h[0][o] : h[1][o], 1);
          } else {  // two tiles: one key each
            const bool up = c & 2, odd = c & 1;
            float h[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              h[i] = (up ? y[i][1] : y[i][0]) + __shfl_xor_sync(0xffffffffu, up ? y[i][0] : y[i][1], 2);
            z4[0] = (odd ? h[1] : h[0]) + __shfl_xor_sync(0xffffffffu, odd ? h[0] : h[1], 1);
          }
        }
        const int tile = q * T + tsel;
        const unsigned live = reinterpret_cast<const unsigned short*>(md + Z::live)[tile];
        float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
        if constexpr (F::scaled) {
          if constexpr (Z::four) {
            const float* f = reinterpret_cast<const float*>(md) + tile * 16 + g;
            ks[0] = f[0], ks[1] = f[8], vs[0] = f[KT], vs[1] = f[KT + 8];
          } else {
            const float2 a = sc[tile * 16 + g], c2 = sc[tile * 16 + g + 8];  // a key's and a value's
            ks[0] = a.x, vs[0] = a.y, ks[1] = c2.x, vs[1] = c2.y;
          }
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
            if constexpr (LONE) {
              z = z4[o];
            } else if constexpr (QUAD) {  // two lanes have two columns each: they swap halves of the keys
              const float z0 = score(e, 0), z1 = score(e, 1);
              const bool odd = c & 1;
              z = (odd ? z1 : z0) + __shfl_xor_sync(0xffffffffu, odd ? z0 : z1, 1);
            } else {
              z = score(e, o);
            }
            z *= back[e];
            if constexpr (F::scaled) z *= ONE ? (c & 2 ? ks[1] : ks[0]) : ks[o];
            const int key = key_of(o);
            const bool on = (live >> key) & 1;
            const float tau = on ? sigmoid_exp2(z) : 0.f;
            mass[e] += tau;
            // zero where a key in reach has no page
            const unsigned pos = p0 + start(k) + tile * 16 + key;
            if (p.tau && once && pos >= rc.lo && pos < p1 && head_of(e) < Gh)
              put_tau(p, (size_t)b * p.H + h0 + head_of(e), rc.t, pos, tau);
            pr[o] = F::scaled ? tau * (ONE ? (c & 2 ? vs[1] : vs[0]) : vs[o]) : tau;
          }
          if constexpr (!BF) {
            // halfs reach from 2^-24 to 65504: keep the largest p of a head between 1
            // and 4096 by a power of two, what was summed before following it
            const float pm = fmaxf(pr[0], pr[NK - 1]);
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
              if (!TURN) f = __shfl_sync(0xffffffffu, f, g % 4 % GQ);  // of this lane's row of O; else its columns' own
              if (g / 4 == e || GP <= 4) {
#pragma unroll
                for (int j = 0; j < kAcc; ++j)
#pragma unroll
                  for (int i = 0; i < 4; ++i) acc[j][i] *= f;
              }
            }
#pragma unroll
            for (int o = 0; o < NK; ++o) pr[o] *= LONE ? unit[e] * kGroupUnit : unit[e];
          }
#pragma unroll
          for (int o = 0; o < NK; ++o) {
            const int at = head_of(e) * Z::pstride + tile * 16 + key_of(o);
            if constexpr (BF) {
              const float rest = less_top(pr[o]);
              ps[at] = tops(rest, pr[o]);
              reinterpret_cast<unsigned short*>(lo)[at] = (unsigned short)(__float_as_uint(less_top(rest)) >> 16);
            } else {
              ps[at] = LONE ? __float_as_uint(pr[o]) : split(pr[o]);
            }
          }
        }
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        unsigned a0 = 0, a1 = 0, a2 = 0, a3 = 0, l0 = 0, l2 = 0;
        const int h = FOLD ? g & 3 : g;  // the head of rows g and g + 8
        if (!TURN && h < GP) {
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
          const unsigned a = vt + ring_at<RS, R, true>(u * 16 + mrow, mch);
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
        } else if constexpr (TURN) {
          // Oᵀ = Vᵀ·Pᵀ.  Lane (g, c): elements 8g … 8g + 7 (32 wide: 4g …) of rows 2c, 2c + 1,
          // 2c + 8, 2c + 9, and column g: of a head the half of τ or the rest of it.  With a head
          // each there is a column pair for each group, τ times the group's scale, and of the
          // products the ones of an element's own group count; else the values are scaled.
          const bool odd = g & 1;
          const unsigned pa = smem_u32(ps + (LONE ? 0 : (g >> 1) % GP * Z::pstride) + u * 16 + 2 * c);
          unsigned pk[4];
          if constexpr (LONE) {
            lds_words<2, 0>(pa + (odd ? 32 : 0), pk);
          } else {
            lds_words<2, 0>(pa, pk);
            lds_words<2, 32>(pa, pk + 2);
          }
          constexpr int kHalves = GB == 8 ? 2 : 1;  // of four groups
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) {
            const int grp = LONE ? (GB == 2 ? (g >> 1) & 1 : hf * 4 + (g >> 1)) : GB == 2 ? g >> 2 : hf * 4 + (g >> 1);
            const unsigned gs = smem_u32(md) + Z::scales + KT * GB + (u * 16 + 2 * c) * GB + grp;
            unsigned b0, b1, s01 = 0, s89 = 0;
            if constexpr (LONE) {
              // a column's halfs or rests of two of the four keys, and of the other two from the
              // lane that has the column beside it, which has made both
              const unsigned at = gs + (odd ? 8 * GB : 0);
              const float2 f = halves(group_pair(lds_part<1>(at) | lds_part<1>(at + GB) << 8));
              const float x = __uint_as_float(pk[0]) * f.x, y = __uint_as_float(pk[1]) * f.y;
              const unsigned hi = two_halves(x, y);
              const float2 h = halves(hi);
              const unsigned lo = two_halves((x - h.x) * kRest, (y - h.y) * kRest);
              const unsigned got = __shfl_xor_sync(0xffffffffu, odd ? hi : lo, 4);
              b0 = odd ? got : hi;
              b1 = odd ? lo : got;
            } else {
              s01 = group_pair(lds_part<1>(gs) | lds_part<1>(gs + GB) << 8);
              s89 = group_pair(lds_part<1>(gs + 8 * GB) | lds_part<1>(gs + 9 * GB) << 8);
              b0 = __byte_perm(pk[0], pk[1], odd ? 0x5410 : 0x7632);
              b1 = __byte_perm(pk[2], pk[3], odd ? 0x5410 : 0x7632);
            }
            constexpr int kBytes = GB == 2 ? 2 : 4;  // of a row: two elements each
            const int byte = hf * (R / 2) + g * kBytes;
            const unsigned v0 = vt + u * 16 * R + ring_at<RS, R, true>(2 * c, byte >> 4) + (byte & 15);
            const unsigned v1 = vt + u * 16 * R + ring_at<RS, R, true>(2 * c + 1, byte >> 4) + (byte & 15);
            unsigned w[4];
            if constexpr (kBytes == 2) {
              w[0] = lds_part<2>(v0), w[1] = lds_part<2>(v1), w[2] = lds_part<2>(v0 + 8 * R), w[3] = lds_part<2>(v1 + 8 * R);
            } else {
              lds_words<1, 0>(v0, w), lds_words<1, 0>(v1, w + 1), lds_words<1, 8 * R>(v0, w + 2), lds_words<1, 8 * R>(v1, w + 3);
            }
            unsigned a[4][4];  // even and odd elements of the first two rows, and of the others
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const unsigned even = (w[2 * i] & 0x0f0f0f0fu) | (w[2 * i + 1] << 4 & 0xf0f0f0f0u);
              const unsigned odds = (w[2 * i] >> 4 & 0x0f0f0f0fu) | (w[2 * i + 1] & 0xf0f0f0f0u);
              if constexpr (LONE) {
                codes8(even, a[2 * i]);
                codes8(odds, a[2 * i + 1]);
              } else {
                widen8(even, i ? s89 : s01, a[2 * i]);
                widen8(odds, i ? s89 : s01, a[2 * i + 1]);
              }
            }
#pragma unroll
            for (int m = 0; m < kBytes; ++m)
              mma16816<BF>(acc[hf * 4 + m], a[0][m], a[1][m], a[2][m], a[3][m], b0, b1);
          }
        } else if constexpr (SZ == 0) {
          // lane (g, c): an eighth of rows 2c, 2c + 1, 2c + 8, 2c + 9: HD/8 elements from g·HD/8 on
          const int byte = g * kVB;
          const unsigned v0 = vt + u * 16 * R + ring_at<RS, R, true>(2 * c, byte >> 4) + (byte & 15);
          const unsigned v1 = vt + u * 16 * R + ring_at<RS, R, true>(2 * c + 1, byte >> 4) + (byte & 15);
          unsigned vw[4][kVB < 4 ? 1 : kVB / 4];
          if constexpr (kVB < 4) {
            vw[0][0] = lds_part<2>(v0);
            vw[1][0] = lds_part<2>(v1);
            vw[2][0] = lds_part<2>(v0 + 8 * R);
            vw[3][0] = lds_part<2>(v1 + 8 * R);
          } else {
            lds_words<kVW, 0>(v0, vw[0]);
            lds_words<kVW, 0>(v1, vw[1]);
            lds_words<kVW, 8 * R>(v0, vw[2]);
            lds_words<kVW, 8 * R>(v1, vw[3]);
          }
          // the two rows' scales of that group, side by side
          const unsigned gs = smem_u32(md) + Z::scales + KT * GB + (u * 16 + 2 * c) * GB + g * GB / 8;
          const unsigned s01 = group_pair(lds_part<1>(gs) | lds_part<1>(gs + GB) << 8);
          const unsigned s89 = group_pair(lds_part<1>(gs + 8 * GB) | lds_part<1>(gs + 9 * GB) << 8);
#pragma unroll
          for (int w = 0; w < (kVB < 4 ? 1 : kVB / 4); ++w)
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // even, odd elements: two keys' codes in a byte
              const unsigned a = vw[0][w], b2 = vw[1][w], d = vw[2][w], f = vw[3][w];
              unsigned x[4], y[4];
              widen8(i ? (a >> 4 & 0x0f0f0f0fu) | (b2 & 0xf0f0f0f0u) : (a & 0x0f0f0f0fu) | (b2 << 4 & 0xf0f0f0f0u), s01, x);
              widen8(i ? (d >> 4 & 0x0f0f0f0fu) | (f & 0xf0f0f0f0u) : (d & 0x0f0f0f0fu) | (f << 4 & 0xf0f0f0f0u), s89, y);
#pragma unroll
              for (int h = 0; h < (kVB < 4 ? kVB : 4); ++h)
                mma16816<BF>(acc[8 * w + 2 * h + i], a0, a1, a2, a3, x[h], y[h]);
            }
        } else {
#pragma unroll
          for (int l = 0; l < kVL; ++l) {
            unsigned vw[4][kVW];
            const int byte = l * 8 * kVB + g * kVB;
            // rows 2c and 2c + 1 of each eight
            const unsigned v0 = vt + u * 16 * R + ring_at<RS, R, true>(2 * c, byte >> 4) + (byte & 15);
            const unsigned v1 = vt + u * 16 * R + ring_at<RS, R, true>(2 * c + 1, byte >> 4) + (byte & 15);
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
      m = LONE || c / GQ < T ? m : 0.f;
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
  } else if constexpr (TURN) {
    // this lane's columns: of these elements' group, or of head c
    if ((LONE ? c == (GB == 2 ? g >> 2 : g >> 1) : c < Gh) && warp < kWarps) {
      const float back = 1.f / (LONE ? unit[0] * kGroupUnit : unit[0]), rest = LONE ? 1.f / kRest : 1.f;
      constexpr int kBytes = GB == 2 ? 2 : 4;
#pragma unroll
      for (int j = 0; j < kAcc; ++j) {
        const int d = j / kBytes * 64 + 2 * kBytes * g + 2 * (j % kBytes);
        float* to = part + (warp * Gh + (LONE ? 0 : c)) * HD + d;
        to[0] = fmaf(acc[j][1], rest, acc[j][0]) * back;
        to[1] = fmaf(acc[j][3], rest, acc[j][2]) * back;
      }
    }
  } else if (hrow < Gh && warp < kWarps) {
    const float back = 1.f / un;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = SZ == 2 ? 8 * j + 2 * c + e : SZ == 0 ? (2 * c + e) * (HD / 8) + j : j / kVB * 8 * kVB + (2 * c + e) * kVB + j % kVB;
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

template <int DT, int HD, int GP, int GR, int KEYS = 0>
cudaError_t launch_paged_mma(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  const int G = p.H / p.Hk, HG = (G + kHeads - 1) / kHeads;
  using Z = Geo<DT, HD, GP, KEYS>;
  const size_t ring = (size_t)kWarps * Z::warp;
  const size_t part = (size_t)(Z::parts + 1) * std::min(G, kHeads) * HD * sizeof(float);
  const size_t smem = std::max(ring, part);
  auto kern = paged_decode_mma<DT, HD, GP, GR, KEYS>;
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
  const bool sorted = Z::four && p.mode == BOZO_MODE_GLOBAL && p.B > 1 && p.B <= kSorted && !pl.clustered &&
                      (long long)p.B * p.Hk * HG * pl.S > kSortedBlocks;
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
  return cudaLaunchKernelEx(&cfg, kern, p, MmaGrid{pl.S, G, HG, make_fastdiv(pl.S), make_fastdiv(HG), make_fastdiv(p.Hk), pl.clustered, sorted});
}
template <int DT, int HD, int GP>
cudaError_t launch_paged_mma(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  // short windows: tiles of half the keys, for more of the warps
  if constexpr (Geo<DT, HD, GP>::lone && Geo<DT, HD, GP>::keys == 64)
    if (p.page % 16 == 0 && p.mode == BOZO_MODE_LOCAL && p.W <= kShortWindow)
      return launch_paged_mma<DT, HD, GP, 16, 32>(p, pl, st);
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
