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
constexpr int kRowWarps = 8;        // warps of a block of paged_decode_rows
constexpr int kRowHeads = 4;        // and its query heads, at most

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
  if (warp < 2 && writes_row(p, r, piece, h % (p.H / p.Hk) == 0)) append_part(p, b, hk, r.t, warp == 0, lane);
  __syncthreads();
  for (unsigned j = j0 + warp; j < j1; j += kThreads / 32) {
    const unsigned row0 = paged_row(p, b, j);
    const size_t row = row0 + (size_t)hk * p.page;
    float dot = 0.f;
    if (row0 != kNoRow)
      for (int d = lane; d < HD; d += 32) dot = fmaf(sq[d], ld_page(p.k, p.kg, row * HD + d, p.dt), dot);
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
      float x = ld_page(p.v, p.vg, row * HD + d, p.dt);
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

// Four consecutive elements of a page (at a multiple of 4).
template <int DT>
__device__ __forceinline__ void ld4(const void* pages, const unsigned char* groups, size_t at, float* x) {
  if constexpr (DT == BOZO_DT_F32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(pages) + at);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else if constexpr (DT == BOZO_DT_BF16) {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(pages) + at);
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
  } else if constexpr (DT == BOZO_DT_F16) {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __half*>(pages) + at);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    x[0] = a.x; x[1] = a.y; x[2] = c.x; x[3] = c.y;
  } else if constexpr (DT == BOZO_DT_F4E2M1) {
    const unsigned v = *reinterpret_cast<const unsigned short*>(static_cast<const unsigned char*>(pages) + at / 2);
    const float2 a = unpack4((unsigned char)v), c = unpack4((unsigned char)(v >> 8));
    const float g = e4m3(groups[at / 16]);
    x[0] = a.x * g; x[1] = a.y * g; x[2] = c.x * g; x[3] = c.y * g;
  } else {
    const unsigned v = *reinterpret_cast<const unsigned*>(static_cast<const unsigned char*>(pages) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = code_value((unsigned char)(v >> (8 * i)), DT);
  }
}

// fp32 pages, and head widths without a tensor-core kernel (multiples of 4): one
// block per (b, key head, NH of its query heads, piece).  A row is held by L = 4, 8
// or 16 lanes, eight elements each (the 4-element pieces l and l + L); a warp takes
// 8, 4 or 2 rows at a time and has kUnroll such steps' keys and values in flight.
// τ with the exact sigmoid, in fp32 throughout.
template <int DT, int NH>
__global__ void __launch_bounds__(kRowWarps * 32, 2) paged_decode_rows(PagedP p, int S, int HG, int lanes) {
  constexpr int kUnroll = NH == 1 ? 4 : 2;
  __shared__ float sq[NH][132];
  __shared__ float part[kRowWarps][NH][132];
  __shared__ float smass[kRowWarps][NH];
  const int G = p.H / p.Hk, HD = p.HD;
  int x = blockIdx.x;
  const int piece = x % S;
  x /= S;
  const int hg = x % HG;
  x /= HG;
  const int hk = x % p.Hk, b = x / p.Hk;
  const int h0 = hk * G + hg * NH, Gh = min(NH, G - hg * NH);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int L = 1 << lanes, l = lane & (L - 1), per = 32 >> lanes;  // rows of a warp's step
  const Reach rc = reach(p, b, S);
  if ((unsigned)piece >= rc.count) return;
  const unsigned j0 = max(rc.first(piece), rc.lo), j1 = rc.last(piece);
  if (rc.active)
    for (int i = tid; i < NH * HD; i += kRowWarps * 32) {
      const int h = i / HD, d = i - h * HD;
      sq[h][d] = h < Gh ? query(p, b, h0 + h, rc.t, d) : 0.f;
    }
  // the last two warps: the first ones fetch the query
  if (warp >= kRowWarps - 2 && writes_row(p, rc, piece, hg == 0))
    append_part<DT>(p, b, hk, rc.t, warp == kRowWarps - 1, lane);
  __syncthreads();
  const bool on[2] = {4 * l < HD, 4 * (l + L) < HD};
  const int own = NH == 1 ? 0 : l / (L / 4);  // the head whose τ this lane computes
  float q[NH][8], acc[NH][8], mass = 0.f;
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[h][i] = rc.active && on[i / 4] ? sq[h][4 * (l + i / 4 * L) + i % 4] : 0.f;
      acc[h][i] = 0.f;
    }
  }
  const unsigned step = kRowWarps * per;
  for (unsigned j = j0 + warp * per + (lane >> lanes); j - (lane >> lanes) < j1; j += kUnroll * step) {
    float k[kUnroll][8], v[kUnroll][8], ks[kUnroll], vs[kUnroll];
    bool live[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned pos = j + u * step;
      const unsigned row0 = pos < j1 ? paged_row(p, b, pos) : kNoRow;
      const size_t row = (size_t)row0 + (size_t)hk * p.page;
      live[u] = row0 != kNoRow;
      ks[u] = vs[u] = 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) k[u][i] = v[u][i] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (live[u] && on[i]) {
          ld4<DT>(p.k, p.kg, row * HD + 4 * (l + i * L), k[u] + 4 * i);
          ld4<DT>(p.v, p.vg, row * HD + 4 * (l + i * L), v[u] + 4 * i);
        }
      if (live[u] && DT > BOZO_DT_F16) {
        ks[u] = p.ks[row];
        vs[u] = p.vs[row];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float z[NH];
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        z[h] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) z[h] = fmaf(q[h][i], k[u][i], z[h]);
      }
      // over the row's lanes; of four heads each lane keeps one, head `own`
      float y = z[0];
      int o = L / 2;
      if constexpr (NH == 4) {
        const bool up = l & o, odd = l & (o / 2);
        const float a = (up ? z[2] : z[0]) + __shfl_xor_sync(0xffffffffu, up ? z[0] : z[2], o);
        const float c = (up ? z[3] : z[1]) + __shfl_xor_sync(0xffffffffu, up ? z[1] : z[3], o);
        o /= 2;
        y = (odd ? c : a) + __shfl_xor_sync(0xffffffffu, odd ? a : c, o);
        o /= 2;
      }
      for (; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      const float tau = live[u] ? sigmoid_exact(y * ks[u] * p.inv_scale) : 0.f;
      mass += tau;
      if (p.tau && j + u * step < j1 && (l & (L / NH - 1)) == 0 && own < Gh)  // zero where a key has no page
        put_tau(p, (size_t)b * p.H + h0 + own, rc.t, j + u * step, tau);
      const float w = tau * vs[u];
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const float wh = NH == 1 ? w : __shfl_sync(0xffffffffu, w, (lane & ~(L - 1)) + h * (L / 4));
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[h][i] = fmaf(wh, v[u][i], acc[h][i]);
      }
    }
  }
  grid_release();
  // the warp's rows, then the warps, each in a fixed order
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    for (int o = L; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[h][i] += __shfl_xor_sync(0xffffffffu, acc[h][i], o);
    if (lane < L)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (on[i / 4]) part[warp][h][4 * (l + i / 4 * L) + i % 4] = acc[h][i];
  }
  for (int o = L; o < 32; o <<= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
  if (lane < L && (l & (L / NH - 1)) == 0) smass[warp][own] = mass;
  __syncthreads();
  for (int i = tid; i < Gh * HD; i += kRowWarps * 32) {
    const int h = i / HD, d = i - h * HD;
    float o = 0.f, m = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      o += part[w][h][d];
      m += smass[w][h];
    }
    const size_t bh = (size_t)b * p.H + h0 + h;
    if (rc.count == 1) {
      stf(p.out, (long long)(bh * HD + d), p.out_dt, o / norm_divisor(p, m, rc.n));
    } else {
      p.ws[(bh * S + piece) * HD + d] = o;
      if (d == 0) piece_mass(p, S)[bh * S + piece] = m;
    }
  }
  if (p.tau && piece == 0)
    for (int h = warp; h < Gh; h += kRowWarps) clear_tau(p, (size_t)b * p.H + h0 + h, rc.n, lane, 32);
}

// Rows cut into more than one piece: one block per (b, h).  Groups of HD/4 threads
// take every so many-th piece, so that all pieces' loads are in flight together,
// and their sums are added in the groups' order.
__global__ void __launch_bounds__(kThreads) paged_join(PagedP p, int S) {
  __shared__ float part[kThreads * 4], smass[kThreads];
  const int bh = blockIdx.x, HD = p.HD;
  const Reach r = reach(p, bh / p.H, S);
  grid_wait();
  if (r.count < 2) return;
  const float* w = p.ws + (size_t)bh * S * HD;
  const float* wm = piece_mass(p, S) + (size_t)bh * S;
  const int each = HD % 4 ? 1 : 4, width = HD / each;  // elements of a thread, threads of a group
  const int groups = kThreads / width, g = threadIdx.x / width, d = (threadIdx.x - g * width) * each;
  if (g < groups) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, m = 0.f;
#pragma unroll 4
    for (unsigned i = g; i < r.count; i += groups) {
      if (each == 4) {
        const float4 x = *reinterpret_cast<const float4*>(w + (size_t)i * HD + d);
        acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w;
      } else {
        acc[0] += w[(size_t)i * HD + d];
      }
      m += wm[i];
    }
    for (int e = 0; e < each; ++e) part[g * HD + d + e] = acc[e];
    if (d == 0) smass[g] = m;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < HD; i += kThreads) {
    float acc = 0.f, m = 0.f;
    for (int k = 0; k < groups; ++k) {
      acc += part[k * HD + i];
      m += smass[k];
    }
    stf(p.out, (long long)bh * HD + i, p.out_dt, acc / norm_divisor(p, m, r.n));
  }
}

bool mma_path(const PagedP& p) {
  return p.dt != BOZO_DT_F32 && (p.HD == 32 || p.HD == 64 || p.HD == 128);
}

bool rows_path(const PagedP& p) { return p.HD % 4 == 0; }

// Blocks of a row's heads.
int head_groups(const PagedP& p) {
  const int G = p.H / p.Hk;
  return mma_path(p) ? (G + kHeads - 1) / kHeads : rows_path(p) ? (G + kRowHeads - 1) / kRowHeads : G;
}

// Pieces of a row.  About three blocks an SM keep the memory busy (16 rows of
// 120002 keys: 76.4 µs at 18 pieces, 75.3 at 24, 75.9 at 28, 78.5 at 37; four of 4-bit
// pages, 42.9 µs at 18, 38.2 at 27, 37.3 at 37, 37.7 at 46, 44.2 at 92).  Sequences
// of different lengths want smaller pieces to even out — twelve an SM, of 2048 keys
// at least (1024 rows of up to 8192 keys: 164 µs in two to four; 512 rows of up to
// 16384 keys in e4m3: 199 µs in three, 192 in four, 190 in six, 195 in eight).  4-bit
// pages' blocks take the longest sequences first, which evens them out by itself: six an
// SM (two draws of lengths: 1024 rows of up to 8192 keys 81 and 75 µs in one piece or two,
// 88 and 82 in three; 512 rows of up to 16384, 128 wide with four heads, 184 and 141 in two,
// 169 and 152 in four, 264 in one; 64 wide 120 and 93 in two, 114 and 104 in four).
// Up to eight pieces are joined inside a cluster, which saves a second kernel's
// 2-3 µs of a call, where the clusters all find their place at once (12 rows of 1024
// keys in eight: 5.9 µs and 8.2 a call, 6.1 and 10.1 with a second kernel; 192 rows of up
// to 1000 keys in two 9.7 against 10.4, in four 14.5 against 13.6; 300 rows of 4192 keys
// in two 60.1 against 58.9, 1600 such rows 266 against 255, 1024 rows of up to 8191
// keys 163.0 against 163.9); so a few pieces more than eight become eight, and
// whatever is asked for where that leaves 256 keys (12 rows of 2048 keys: 6.5
// against 6.7 µs in sixteen; of 8192 keys 11.2 against 8.7).  Short rows stay whole
// (48 rows of 256 keys: 5.2 µs, 5.9 in two).
PagedPlan plan(const PagedP& p, int sms) {
  constexpr int kCluster = 8;
  const bool mma = mma_path(p);
  const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
  const long long rows = (long long)p.B * p.Hk * head_groups(p);
  const bool four = mma && p.dt == BOZO_DT_F4E2M1;
  long long s = (four ? 4LL : 3LL) * sms / rows;
  const long long per_sm = four && p.B <= kSorted && p.mode == BOZO_MODE_GLOBAL ? 6 : 12;
  if (p.B > 1) s = std::max(s, std::min((per_sm * sms + rows - 1) / rows, keys / 2048));
  s = std::min(s, keys <= (mma ? 256 : 512) ? 1 : (keys + 15 + kMinPiece - 1) / kMinPiece);
  if (mma && s > kCluster && (s <= kCluster + 4 || keys <= 256 * kCluster)) s = kCluster;
  if (!mma && !rows_path(p)) s = std::max(s, (keys + 15 + kMaxPiece - 1) / kMaxPiece);
  s = std::max(s, 1LL);
  return {(int)s, mma && s > 1 && s <= kCluster && rows * s <= 3LL * sms};
}

template <int DT>
cudaError_t launch_rows(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  const int lanes = p.HD <= 32 ? 2 : p.HD <= 64 ? 3 : 4, HG = head_groups(p);
  const unsigned grid = (unsigned)((long long)p.B * p.Hk * HG * pl.S);
  if (p.H == p.Hk) paged_decode_rows<DT, 1><<<grid, kRowWarps * 32, 0, st>>>(p, pl.S, HG, lanes);
  else paged_decode_rows<DT, kRowHeads><<<grid, kRowWarps * 32, 0, st>>>(p, pl.S, HG, lanes);
  return cudaGetLastError();
}

cudaError_t launch_join(const PagedP& p, const PagedPlan& pl, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.B * p.H));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join, p, pl.S);
}

}  // namespace

size_t paged_decode_bytes(const PagedP& p, int sms) {
  const PagedPlan pl = plan(p, sms);
  if (pl.S < 2 || pl.clustered) return 0;
  return ((size_t)p.B * p.H * pl.S * (p.HD + 1) * sizeof(float) + 255) & ~(size_t)255;
}

cudaError_t launch_paged_decode(const PagedP& p, int sms, cudaStream_t st, int* launches, int* path) {
  const PagedPlan pl = plan(p, sms);
  cudaError_t e;
  if ((long long)p.B * p.Hk * head_groups(p) * pl.S > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  if (mma_path(p)) {
    switch (p.dt) {
      case BOZO_DT_BF16: e = launch_paged_mma_bf16(p, pl, st); break;
      case BOZO_DT_F16: e = launch_paged_mma_f16(p, pl, st); break;
      case BOZO_DT_F8E4M3: e = launch_paged_mma_f8(p, pl, st); break;
      case BOZO_DT_F4E2M1: e = launch_paged_mma_f4(p, pl, st); break;
      default: e = launch_paged_mma_i8(p, pl, st);
    }
  } else if (rows_path(p)) {
    switch (p.dt) {
      case BOZO_DT_F32: e = launch_rows<BOZO_DT_F32>(p, pl, st); break;
      case BOZO_DT_BF16: e = launch_rows<BOZO_DT_BF16>(p, pl, st); break;
      case BOZO_DT_F16: e = launch_rows<BOZO_DT_F16>(p, pl, st); break;
      case BOZO_DT_F8E4M3: e = launch_rows<BOZO_DT_F8E4M3>(p, pl, st); break;
      case BOZO_DT_F4E2M1: e = launch_rows<BOZO_DT_F4E2M1>(p, pl, st); break;
      default: e = launch_rows<BOZO_DT_I8>(p, pl, st);
    }
  } else {
    const long long keys = p.mode == BOZO_MODE_LOCAL ? p.W : (long long)p.cap;
    const size_t smem = (size_t)(p.HD + std::min<long long>(keys, kMaxPiece) + 16) * sizeof(float);
    paged_decode_any<<<(unsigned)(p.B * p.H * pl.S), kThreads, smem, st>>>(p, pl.S);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  *path = mma_path(p) ? BOZO_PATH_MMA : BOZO_PATH_SIMT;
  *launches = 1;
  if (pl.S > 1 && !pl.clustered) {
    e = launch_join(p, pl, st);
    *launches = 2;
  }
  return e;
}

}  // namespace bozo
