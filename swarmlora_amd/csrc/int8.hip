// Products in 8-bit integers: rows with a scale each, times a weight with a scale
// for each output channel.
//
//   q_ik = round(x_ik 127 / max_k |x_ik|), s_i = max_k |x_ik| / 127
//   y_ij = bf16(s_i s_j sum_k q_ik q_jk + b_j)
//
// Sums are int32: exact, in any order.  The weight is held as the A operands of the
// 16x16x64 MFMA: 16 rows (output channels) x 64 k are a block of 1 KiB, lane l's 16
// bytes row l % 16, k 16 (l / 16) .. + 15; a tile's blocks follow one another
// along k, tiles along n; rows past n and k past its end (a multiple of 128) are
// zeros, so what the rows of x hold past k does not matter.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <cmath>

#include "dev_util.h"
#include "swl.h"
#include "swl_common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 128;   // k of a step (two blocks)
constexpr int kCus = 256;    // of an MI355X
constexpr int64_t kMaxChannels = (int64_t)1 << 26;  // (packed by 64 threads each)
static_assert(swl::grid_fits((kMaxChannels - 1) / 16, 1024), "");

__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x16 mfma_i8(u32x4 a, u32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// ------------------------------------------------------------- rows, weight ---
// Eight bf16 of a row from index i; past its end zeros.
__device__ __forceinline__ u32x4 row8(const bf16* row, int64_t i, int64_t k) {
  if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && i + 8 <= k) return ldg16(row + i);
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
  u32x4 q = {0u, 0u, 0u, 0u};
#pragma unroll 1
  for (int e = 0; e < 8; e += 2, i += 2) {
    const uint32_t lo = i < k ? p[i] : 0u, hi = i + 1 < k ? p[i + 1] : 0u;
    q = u32x4{q[1], q[2], q[3], lo | hi << 16};
  }
  return q;
}
__device__ __forceinline__ uint32_t top8(u32x4 q, uint32_t top) {  // the largest magnitude's bits (bf16 << 16)
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(max(top, (q[e] & 0x7fffu) << 16), q[e] & 0x7fff0000u);
  return top;
}
// What a row's elements are multiplied by, first (exact) and then, and its scale,
// from the bits of its largest magnitude.  A row with an infinity or a NaN: codes
// of 0 and a NaN scale.
struct RowScale {
  float top, up, inv, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  const float m = __uint_as_float(top);
  if (top >= 0x7f800000u) return RowScale{0.f, 0.f, 0.f, NAN};
  if (top == 0) return RowScale{0.f, 0.f, 0.f, 0.f};
  // (127 over a largest under 2^-121 is no number: that times 2^64)
  const float up = top < 0x20000000u ? 0x1p64f : 1.f;
  return RowScale{m, up, 127.f / (m * up), m / 127.f};
}
// Codes of eight elements: x 127 / max to the nearest, halves to even.  It is half
// way where 254 x = odd max: where max has the bits of 127 (127 / max is exact then),
// or x is half of max, 63.5 itself.  Elsewhere it is at least 2^-17 from half way (8
// bits in x and max), far more than the two roundings here are off.
__device__ __forceinline__ u32x2 codes8(u32x4 q, const RowScale& s) {
  float f[8];
  unpack8(q, f);
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v = rintf(f[e] * s.up * s.inv);
    v = fabsf(f[e]) * 2.f == s.top ? copysignf(64.f, f[e]) : v;
    c[e] = s.inv == 0.f ? 0u : (uint32_t)(int)v & 255u;
  }
  return u32x2{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
}

// A row of x a workgroup: its largest, then its codes, the row in registers between
// (rows over 8 NV THREADS, or not in whole 16-byte pieces, are read twice).
template <int NV, int THREADS>
__global__ __launch_bounds__(THREADS) void int8_rows_kernel(const bf16* x, int64_t ldx, int64_t k, int8_t* q, int64_t ldq,
                                                            float* scale) {
  __shared__ uint32_t sh[THREADS / 64];
  const int64_t row = blockIdx.x;
  const bf16* src = x + row * ldx;
  int8_t* dst = q + row * ldq;
  const bool held = (reinterpret_cast<uintptr_t>(src) & 15) == 0 && k % 8 == 0 && k <= 8 * NV * THREADS;
  u32x4 v[NV];
  uint32_t top = 0;
  if (held) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * THREADS + threadIdx.x) * 8;
      v[j] = u32x4{0u, 0u, 0u, 0u};
      if (i < k) v[j] = ldg16(src + i);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) top = top8(v[j], top);
  } else {
#pragma unroll 1
    for (int64_t i = threadIdx.x * 8; i < k; i += THREADS * 8) top = top8(row8(src, i, k), top);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) top = max(top, sh[i]);
  const RowScale s = row_scale(top);
  if (threadIdx.x == 0) scale[row] = s.scale;
  const int64_t kp = (k + 15) / 16 * 16;  // (the bytes behind the last code are zeros)
  if (held) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (j * THREADS + threadIdx.x) * 8;
      if (i < kp) *(__attribute__((address_space(1))) u32x2*)(dst + i) = codes8(v[j], s);
    }
  } else {
#pragma unroll 1
    for (int64_t i = threadIdx.x * 8; i < kp; i += THREADS * 8)
      *(__attribute__((address_space(1))) u32x2*)(dst + i) = codes8(row8(src, i, k), s);
  }
}

// A tile of 16 rows of a weight a workgroup of 16 waves: each wave its row's
// largest, then the tile's blocks.  Made once for a weight.
__global__ __launch_bounds__(1024) void int8_pack_kernel(const bf16* w, int64_t ldw, int64_t n, int64_t k, int64_t steps,
                                                         u32x4* data, float* scale) {
  __shared__ uint32_t sh[16];
  const int lane = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int64_t row = blockIdx.x * 16 + r;
  const bf16* src = w + min(row, n - 1) * ldw;
  uint32_t top = 0;
  for (int64_t i = lane * 8; i < k; i += 512) top = top8(row8(src, i, k), top);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if (lane == 0) {
    sh[r] = row < n ? top : 0;
    if (row < n) scale[row] = row_scale(top).scale;
  }
  __syncthreads();
  const int64_t pieces = steps * 128;  // 16 bytes each
  for (int64_t p = threadIdx.x; p < pieces; p += 1024) {
    const int l = (int)(p & 63), rr = l & 15;
    const int64_t i = (p >> 6) * 64 + 16 * (l >> 4), at = blockIdx.x * 16 + rr;
    const RowScale s = row_scale(sh[rr]);
    const bf16* from = w + min(at, n - 1) * ldw;
    u32x4 o = {0u, 0u, 0u, 0u};
    if (at < n && i < k) {
      const u32x2 a = codes8(row8(from, i, k), s);
      const u32x2 b = i + 8 < k ? codes8(row8(from, i + 8, k), s) : u32x2{0u, 0u};
      o = u32x4{a[0], a[1], b[0], b[1]};
    }
    data[blockIdx.x * pieces + p] = o;
  }
}

// ------------------------------------------------------------------ product ---
struct Int8Args {
  const int8_t* x;      // [m, k] codes, row stride ldx
  const float* xs;      // [m]
  const int8_t* w;      // tiles
  const float* ws;      // [n]
  const bf16* bias;     // [n] or null
  bf16* y;              // [m, n], row stride ldy
  int32_t* part;        // [splits][m][n] sums, or null
  int64_t m, n, ldx, ldy;
  int32_t klast;        // byte offset of a row's last 16
  int32_t steps;        // of 128 k
  int32_t tiles;        // of 16 channels
  int32_t splits;
};

// y of four channels n0 .. + 3 of a row
__device__ __forceinline__ bf16x2 two(float a, float b) { return bf16x2{f2bf(a), f2bf(b)}; }
__device__ __forceinline__ void finish4(const Int8Args& a, i32x4 c, int64_t m, int64_t n0, float (&o)[4]) {
  const float xs = a.xs[m];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = min(n0 + i, a.n - 1);
    o[i] = (float)c[i] * (xs * a.ws[n]) + (a.bias ? bf2f(a.bias[n]) : 0.f);
  }
}
__device__ __forceinline__ void store4(const Int8Args& a, const float (&o)[4], int64_t m, int64_t n0) {
  bf16* dst = a.y + m * a.ldy + n0;
  if ((a.ldy & 3) == 0 && n0 + 4 <= a.n) {  // (y is 8-byte aligned)
    stg(dst, u32x2{__builtin_bit_cast(uint32_t, two(o[0], o[1])), __builtin_bit_cast(uint32_t, two(o[2], o[3]))});
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n0 + i < a.n) stg(dst + i, f2bf(o[i]));
}

// Few rows (at most 16 MT): a workgroup of W waves per TPW tiles of 16 channels;
// wave w takes the steps of 128 k w, w + W, ... of all of them, the weight straight
// into registers past the caches, the rows from L2, and the waves' sums meet in
// LDS: no partial sums in memory, one launch.
template <int MT, int TPW, int W, int D>
__global__ __launch_bounds__(64 * W) void int8_rows_product_kernel(Int8Args a) {
  __shared__ __attribute__((aligned(16))) i32x4 sh[W][TPW * MT * 64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = blockIdx.x * TPW;
  const int8_t* wp[TPW];
#pragma unroll
  for (int t = 0; t < TPW; ++t) wp[t] = a.w + (int64_t)min(t0 + t, a.tiles - 1) * a.steps * 2048 + lane * 16;
  const int8_t* xp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xp[t] = a.x + min<int64_t>(16 * t + (lane & 15), a.m - 1) * a.ldx;
  const int ko = 16 * (lane >> 4);
  i32x4 acc[TPW][MT];
#pragma unroll
  for (int i = 0; i < TPW; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  u32x4 wf[D][TPW][2], xf[D][MT][2];
  auto load = [&](int d, int s) {
    s = min(s, a.steps - 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < TPW; ++t) wf[d][t][h] = ldg16_nt(wp[t] + (int64_t)s * 2048 + 1024 * h);
      const int at = min(s * kStep + 64 * h + ko, a.klast);
#pragma unroll
      for (int t = 0; t < MT; ++t) xf[d][t][h] = ldg16(xp[t] + at);
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(d, w + d * W);
  for (int s0 = w; s0 < a.steps; s0 += D * W) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (s0 + d * W < a.steps) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] = mfma_i8(wf[d][i][h], xf[d][j][h], acc[i][j]);
        load(d, s0 + (d + D) * W);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TPW; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) sh[w][(i * MT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int p = threadIdx.x; p < TPW * MT * 64; p += 64 * W) {
    const int i = p / (MT * 64), j = p / 64 % MT, l = p & 63;
    const int64_t m = 16 * j + (l & 15), n0 = (int64_t)(t0 + i) * 16 + 4 * (l >> 4);
    if (m >= a.m || n0 >= a.n) continue;
    i32x4 c = sh[0][p];
#pragma unroll
    for (int v = 1; v < W; ++v) c += sh[v][p];
    float o[4];
    finish4(a, c, m, n0, o);
    store4(a, o, m, n0);
  }
}

// Many rows: 64 NI channels x 32 WM NJ rows a workgroup of 2 WM waves, a wave
// NI x NJ tiles of the 32x32x32 MFMA (the weight as A: a lane ends up with four
// consecutive channels of one row).  Stages of 128 k through SLOTS places in LDS,
// filled by LDS-DMA a stage (or more) ahead, fragments read two k-steps ahead of
// their MFMAs into four register sets, one barrier a stage, requests and reads in a
// fixed order between the MFMAs.  The weight's blocks lie in LDS as in memory
// (reads of 16 rows are 256 contiguous bytes); a row of x is 128 bytes, its piece c
// at c ^ (r % 8) ^ (r / 8 % 2).  Tiles are numbered so that an XCD walks a
// contiguous run of them.
template <int NI, int NJ, int WM, int SLOTS>
struct TileGeom {
  static constexpr int NT = 64 * NI, MT = 32 * WM * NJ;
  static constexpr int STAGE = (NT + MT) * kStep;
  static constexpr int TPW = 32 * NJ, CPW = 32 * NI;        // rows, channels of a wave
  static constexpr int OROW = CPW * 2 + 16;                 // bytes of an output row of a wave in LDS
  static constexpr int EPI = 2 * WM * TPW * OROW;
  static constexpr int LDS = SLOTS * STAGE > EPI ? SLOTS * STAGE : EPI;
};

template <int NI, int NJ, int WM, int SLOTS>
__global__ __launch_bounds__(128 * WM, 1) void int8_tile_kernel(Int8Args a, int tiles_m, int tiles, int per_xcd, int gm) {
  using Geo = TileGeom<NI, NJ, WM, SLOTS>;
  constexpr int WAVES = 2 * WM;
  constexpr int NT = Geo::NT, MT = Geo::MT, CPW = Geo::CPW, TPW = Geo::TPW;
  constexpr int XR = MT / WAVES, WR = NT / WAVES;  // rows, channels a wave moves of a stage
  constexpr int MF = NI * NJ, NR = NI + NJ;
  constexpr int QW = WR / 8, NREQ = QW + XR / 8;
  constexpr int RPM = (NR + MF - 1) / MF;
  static_assert(WR % 16 == 0 && XR % 16 == 0 && NREQ * (SLOTS - 1) < 64 && NREQ <= 2 * MF, "");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wv >> 1, wn = wv & 1;
  const int lin = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (lin >= tiles) return;  // uniform over the workgroup
  // groups of gm row tiles, each walking its channel tiles with the rows fastest
  const int gsz = gm * (tiles / tiles_m), grp = lin / gsz, gl = lin - grp * gsz;
  const int gr = min(gm, tiles_m - grp * gm);
  const int64_t m0 = (int64_t)(grp * gm + gl % gr) * MT, n0 = (int64_t)(gl / gr) * NT;
  const int sp = blockIdx.y, kt0 = (int)((int64_t)a.steps * sp / a.splits);
  const int nk = (int)((int64_t)a.steps * (sp + 1) / a.splits) - kt0;

  i32x16 acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  const int fr = lane & 31, fh = lane >> 5;
  auto mfma_at = [&](u32x4 (&a0)[NI], u32x4 (&b0)[NJ], u32x4 (&a1)[NI], u32x4 (&b1)[NJ], int t) {
    const int i = (t % MF) / NJ, j = t % NJ;
    acc[i][j] = t < MF ? mfma_i8(a0[i], b0[j], acc[i][j]) : mfma_i8(a1[i], b1[j], acc[i][j]);
  };
  // wave w moves channels WR w .. (a tile's two blocks an instruction each) and rows
  // XR w .. (8 rows of 128 bytes an instruction)
  const int dr = lane >> 3;
  const int8_t* wsrc[QW];
  const int8_t* xsrc[XR / 8];
  int xo[XR / 8];
#pragma unroll
  for (int i = 0; i < QW; ++i) {
    const int tile = (int)min<int64_t>(n0 / 16 + WR / 16 * wv + (i >> 1), a.tiles - 1);
    wsrc[i] = a.w + ((int64_t)tile * a.steps + kt0) * 2048 + (i & 1) * 1024 + lane * 16;
  }
#pragma unroll
  for (int i = 0; i < XR / 8; ++i) {
    xsrc[i] = a.x + min<int64_t>(m0 + XR * wv + 8 * i + dr, a.m - 1) * a.ldx;
    xo[i] = 16 * ((lane & 7) ^ dr ^ (i & 1));
  }
  auto request_at = [&](int kt, int s, int q) {
    char* st = lds + s * Geo::STAGE;
    if (q < QW)
      __builtin_amdgcn_global_load_lds((gbl_ptr)(wsrc[q] + (int64_t)kt * 2048),
                                       (lds_ptr)(st + (WR / 16 * wv + (q >> 1)) * 2048 + (q & 1) * 1024), 16, 0, 0);
    else
      __builtin_amdgcn_global_load_lds((gbl_ptr)(xsrc[q - QW] + min((kt0 + kt) * kStep + xo[q - QW], a.klast)),
                                       (lds_ptr)(st + NT * kStep + (XR * wv + 8 * (q - QW)) * kStep), 16, 0, 0);
  };
  const int sw = (fr & 7) ^ ((fr >> 3) & 1);
  auto read_at = [&](int s, int kk, u32x4 (&fa_)[NI], u32x4 (&fb_)[NJ], int idx) {
    const char* st = lds + s * Geo::STAGE;
    const int c = 2 * kk + fh;
    if (idx < NI)
      fa_[idx] = *reinterpret_cast<const u32x4*>(st + ((wn * CPW + 32 * idx) / 16 + (fr >> 4)) * 2048 + (kk >> 1) * 1024 +
                                                 (((fr & 15) + 16 * (c & 3)) << 4));
    else
      fb_[idx - NI] = *reinterpret_cast<const u32x4*>(st + NT * kStep + (wm * TPW + 32 * (idx - NI) + fr) * kStep + ((c ^ sw) << 4));
  };
  u32x4 fa[4][NI], fb[4][NJ];
#pragma unroll
  for (int i = 0; i < SLOTS; ++i)
#pragma unroll
    for (int q = 0; q < NREQ; ++q) request_at(min(i, nk - 1), i, q);
  __builtin_amdgcn_s_waitcnt(wait_vm_imm(NREQ * (SLOTS - 1)));
  lds_barrier();
  // live(j): whether the wave's 32 rows j hold a row of the batch (in its last row
  // tile the MFMAs and reads of those that do not are left out)
  auto main_loop = [&](auto live) {
    auto read_live = [&](int idx) { return idx < NI ? live(0) : live(idx - NI); };
#pragma unroll
    for (int idx = 0; idx < NR; ++idx)
      if (read_live(idx)) read_at(0, 0, fa[0], fb[0], idx);
#pragma unroll
    for (int idx = 0; idx < NR; ++idx)
      if (read_live(idx)) read_at(0, 1, fa[1], fb[1], idx);
    for (int kt = 0; kt < nk; ++kt) {
      const int s = kt & (SLOTS - 1), s1 = (kt + 1) & (SLOTS - 1);
#pragma unroll
      for (int t = 0; t < 2 * MF; ++t) {
        if (live(t % NJ)) mfma_at(fa[0], fb[0], fa[1], fb[1], t);
#pragma unroll
        for (int r = RPM * t; r < RPM * (t + 1); ++r) {
          if (r < NR) {
            if (read_live(r)) read_at(s, 2, fa[2], fb[2], r);
          } else if (r < 2 * NR) {
            if (read_live(r - NR)) read_at(s, 3, fa[3], fb[3], r - NR);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_waitcnt(wait_vm_imm(NREQ * (SLOTS - 2)));
      lds_barrier();  // stage kt + 1 is there, slot s read by every wave
      __builtin_amdgcn_sched_barrier(0);
      const int nx = min(kt + SLOTS, nk - 1);
#pragma unroll
      for (int t = 0; t < 2 * MF; ++t) {
        if (live(t % NJ)) mfma_at(fa[2], fb[2], fa[3], fb[3], t);
#pragma unroll
        for (int r = RPM * t; r < RPM * (t + 1); ++r) {
          if (r < NR) {
            if (read_live(r)) read_at(s1, 0, fa[0], fb[0], r);
          } else if (r < 2 * NR) {
            if (read_live(r - NR)) read_at(s1, 1, fa[1], fb[1], r - NR);
          }
        }
        if (t == 0 || (t * NREQ) / (2 * MF) != ((t - 1) * NREQ) / (2 * MF)) request_at(nx, s, (t * NREQ) / (2 * MF));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  const int jl = (int)min<int64_t>(NJ, max<int64_t>(0, (a.m - m0 - wm * TPW + 31) / 32));
  if (jl == NJ)
    main_loop([](int) { return true; });
  else
    main_loop([jl](int j) { return j < jl; });
  __builtin_amdgcn_s_waitcnt(wait_vm_imm(0));  // (the requests past the last stage)
  lds_barrier();

  const int64_t nw = n0 + wn * CPW, mw = m0 + wm * TPW;
  if (a.part) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int64_t m = mw + 32 * j + fr;
      if (m >= a.m) continue;
      int32_t* dst = a.part + (sp * a.m + m) * a.n;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int64_t n = nw + 32 * i + 2 * e + 4 * fh;
          if ((a.n & 3) == 0 && n + 4 <= a.n) {
            *(__attribute__((address_space(1))) i32x4*)(dst + n) = i32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (n + x < a.n) dst[n + x] = acc[i][j][e + x];
          }
        }
    }
    return;
  }
  // The wave's rows through LDS (its own part of it), whole rows a store.
  char* own = lds + wv * TPW * Geo::OROW;
  float xs[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) xs[j] = a.xs[min<int64_t>(mw + 32 * j + fr, a.m - 1)];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int c = 32 * i + 2 * e + 4 * fh;
      float ws[4], b[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int64_t n = min(nw + c + x, a.n - 1);
        ws[x] = a.ws[n];
        b[x] = a.bias ? bf2f(a.bias[n]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        float o[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] = (float)acc[i][j][e + x] * (xs[j] * ws[x]) + b[x];
        *reinterpret_cast<u32x2*>(own + (32 * j + fr) * Geo::OROW + 2 * c) =
            u32x2{__builtin_bit_cast(uint32_t, two(o[0], o[1])), __builtin_bit_cast(uint32_t, two(o[2], o[3]))};
      }
    }
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
  constexpr int LR = CPW / 8;  // lanes of a row
  const bool vec = (a.ldy & 7) == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
#pragma unroll 4
  for (int r = lane / LR; r < TPW; r += 64 / LR) {
    const int64_t m = mw + r;
    if (m >= a.m) break;
    const int c = 8 * (lane % LR);
    const u32x4 v = *reinterpret_cast<const u32x4*>(own + r * Geo::OROW + 2 * c);
    bf16* dst = a.y + m * a.ldy + nw + c;
    if (vec && nw + c + 8 <= a.n) {
      *(__attribute__((address_space(1))) u32x4*)(dst) = v;
    } else {
      const bf16x8 y = __builtin_bit_cast(bf16x8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (nw + c + e < a.n) stg(dst + e, y[e]);
    }
  }
}

// Adds the splits' sums and makes them y: four channels a thread.
__global__ __launch_bounds__(256) void int8_fold_kernel(Int8Args a) {
  const int64_t quads = (a.n + 3) / 4, p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p >= a.m * quads) return;
  const int64_t m = p / quads, n0 = (p - m * quads) * 4;
  i32x4 c = {0, 0, 0, 0};
  for (int s = 0; s < a.splits; ++s) {
    const int32_t* src = a.part + (s * a.m + m) * a.n + n0;
    if ((a.n & 3) == 0) {
      c += *(const __attribute__((address_space(1))) i32x4*)src;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n0 + e < a.n) c[e] += src[e];
    }
  }
  float o[4];
  finish4(a, c, m, n0, o);
  store4(a, o, m, n0);
}

// ---------------------------------------------------------------- launchers ---
// Which kernel takes a call (times of MI355X, the weight from memory, n x k by m):
//   at most 64 rows stream the weight, every workgroup reading all of x from L2; how
//   many tiles share that is the question: 28672 x 4096 by 28 rows 1 tile 41 us, 2
//   31, 4 22 (6.3 TB/s at 128256 x 4096), 8 26; by one row 21; but 6144 x 4096 by 28
//   rows, 2 tiles and 16 waves 8.5, 8 waves 9.1, 4 tiles 12.7, by one row 1 tile 6.1, 2
//   7.6.  More steps in flight a wave are slower (28672 by 28: one step 22, two 26,
//   three 27; the registers' cost in waves).
//   More rows, and 17 to 64 of a long k with few channels, take tiles of 128 x 128
//   with k split so that there are as many as CUs: 4096 x 14336 by 107 rows streamed 57,
//   8 splits 22.9 (by 60 16 splits 25.9).  17 to 64 rows streamed | by tiles:
//     k      n      17 rows      28           40           64
//     4096   4096   7.7 | 11.7   8.5 | 12.2   10.0 | 12.2  12.2 | 13.3
//            9216   12.2 | 14.4  13.6 | 14.6  17.6 | 15.0  22.2 | 16.2
//            12288  11.8 | 16.9  11.6 | 16.7  19.0 | 17.0  20.7 | 18.6
//            28672  21.3 | 26.3  22.1 | 26.6  26.0 | 26.9  28.6 | 27.5
//     8192   4096   13.0 | 15.0  14.6 | 14.9  16.4 | 15.3  21.5 | 16.2
//            8192   15.1 | 19.7  16.3 | 20.0  17.7 | 20.3  22.9 | 21.1
//            9216   21.1 | 20.5  24.3 | 20.7  31.6 | 21.1  41.0 | 22.5
//            12288  19.8 | 24.1  20.6 | 24.7  34.3 | 25.5  37.2 | 27.6
//            28672  41.3 | 45.5  41.9 | 46.0  48.3 | 46.5  52.3 | 48.1
//     14336  4096   22.1 | 20.2  24.2 | 20.0  28.6 | 19.7  36.4 | 20.4
//            8192   25.2 | 27.7  26.4 | 27.8  30.5 | 28.1  38.5 | 29.2
//            9216   36.0 | 29.3  41.4 | 29.5  54.4 | 30.4  71.4 | 32.3
//            12288  32.7 | 40.6  33.5 | 38.3  57.5 | 39.9  62.9 | 43.6
//            28672  69.4 | 78.4  74.0 | 72.9  79.0 | 73.4  88.5 | 77.2
//   The rule takes the slower side of 17 to 32 rows at k = 8192 with n of 6144 to 8192 (by
//   up to 1.3) and at n of 9216 and 10240 with k from 8192 (1.4), and of 33 to 64 rows by n
//   over 8192 (1.1 to 2.2).
constexpr int kFewRows = 64;

struct Int8Plan {
  bool few, big;
  int splits;
  int64_t bytes;
};
Int8Plan int8_plan(int64_t m, int64_t n, int64_t k) {
  Int8Plan p{};
  p.splits = 1;
  p.few = m <= kFewRows && (m <= 16 || k < 8192 || n > 8192);
  if (p.few) return p;
  const int64_t steps = (k + kStep - 1) / kStep;
  p.big = ((m + 255) / 256) * ((n + 255) / 256) >= 160;
  if (!p.big) {
    const int64_t tiles = ((m + 127) / 128) * ((n + 127) / 128);
    p.splits = (int)std::max<int64_t>(1, std::min({(int64_t)kCus / tiles, steps / 6, (int64_t)16}));
  }
  p.bytes = p.splits > 1 ? (int64_t)p.splits * m * n * 4 : 0;
  return p;
}

template <int NI, int NJ, int WM, int SLOTS>
int launch_tiles(const Int8Args& a, hipStream_t st) {
  using Geo = TileGeom<NI, NJ, WM, SLOTS>;
  const int tiles_m = (int)((a.m + Geo::MT - 1) / Geo::MT);
  const int64_t all = tiles_m * ((a.n + Geo::NT - 1) / Geo::NT);
  SWL_CHECK(swl::grid_fits(all + 8, 128 * WM), SWL_ERR_INVALID, "swl_int8_matmul_bf16: too many rows");
  const int tiles = (int)all, per_xcd = (tiles + 7) / 8;
  int gm = tiles_m;
  if (tiles <= kCus) {
    gm = 1;
    while ((gm + 1) * (gm + 1) <= per_xcd) ++gm;
    gm = std::min(gm, tiles_m);
  }
  auto kern = int8_tile_kernel<NI, NJ, WM, SLOTS>;  // (over the default 64 KiB of LDS: allowed a kernel)
  SWL_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, Geo::LDS));
  hipLaunchKernelGGL(kern, dim3((unsigned)(per_xcd * 8), (unsigned)a.splits), dim3(128 * WM), Geo::LDS, st, a, tiles_m, tiles,
                     per_xcd, gm);
  SWL_LAUNCH_CHECK("int8_tile_kernel launch");
  return SWL_OK;
}

template <int MT>
int launch_rows(const Int8Args& a, hipStream_t st) {
  auto go = [&](auto kern, int tpw, int waves) {
    hipLaunchKernelGGL(kern, dim3((unsigned)((a.tiles + tpw - 1) / tpw)), dim3(64 * waves), 0, st, a);
  };
  if (a.tiles >= 768)
    go(int8_rows_product_kernel<MT, 4, 4, 1>, 4, 4);
  else if (MT > 1 && a.tiles >= 192)
    go(int8_rows_product_kernel<MT, 2, 8, 1>, 2, 8);
  else
    go(int8_rows_product_kernel<MT, 1, 8, 1>, 1, 8);
  SWL_LAUNCH_CHECK("int8_rows_product_kernel launch");
  return SWL_OK;
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" int swl_int8_rows_bf16(const void* x, int64_t ldx, int64_t m, int64_t k, void* q, int64_t ldq, float* scale,
                                  void* stream) {
  SWL_CHECK(m >= 0 && m < ((int64_t)1 << 31) && k > 0 && k <= (1 << 17), SWL_ERR_INVALID,
            "swl_int8_rows_bf16: bad row count, or more than 131072 columns");
  if (m == 0) return SWL_OK;
  SWL_CHECK(x && q && scale, SWL_ERR_INVALID, "swl_int8_rows_bf16: null argument");
  SWL_CHECK(ldx >= k && ldq >= (k + 15) / 16 * 16, SWL_ERR_INVALID, "swl_int8_rows_bf16: row strides smaller than a row");
  SWL_CHECK(aligned(q, 16) && ldq % 16 == 0, SWL_ERR_INVALID, "swl_int8_rows_bf16: rows of q must be 16-byte aligned");
  // (threads with two vectors of 8 each up to 8192; 107 rows of 14336 7.5 us with 256 threads)
  constexpr int64_t kRowsLaunch = 1 << 22;
  static_assert(swl::grid_fits(kRowsLaunch, 512), "");
  auto rows = [&](auto kern, int threads) {
    for (int64_t r = 0; r < m; r += kRowsLaunch)
      hipLaunchKernelGGL(kern, dim3((unsigned)std::min(m - r, kRowsLaunch)), dim3(threads), 0, (hipStream_t)stream,
                         reinterpret_cast<const bf16*>(x) + r * ldx, ldx, k, reinterpret_cast<int8_t*>(q) + r * ldq, ldq,
                         scale + r);
  };
  if (k <= 4096)
    rows(int8_rows_kernel<2, 256>, 256);
  else
    rows(int8_rows_kernel<4, 512>, 512);
  SWL_LAUNCH_CHECK("int8_rows_kernel launch");
  return SWL_OK;
}

extern "C" int64_t swl_int8_weight_bytes(int64_t n, int64_t k) {
  if (n <= 0 || k <= 0) return 0;
  return (n + 15) / 16 * ((k + kStep - 1) / kStep) * 2048;
}

extern "C" int swl_int8_pack_bf16(const void* w, int64_t ldw, int64_t n, int64_t k, void* data, float* scale, void* stream) {
  SWL_CHECK(n > 0 && n < kMaxChannels && k > 0 && k <= (1 << 17), SWL_ERR_INVALID,
            "swl_int8_pack_bf16: bad channel count, or more than 131072 columns");
  SWL_CHECK(w && data && scale, SWL_ERR_INVALID, "swl_int8_pack_bf16: null argument");
  SWL_CHECK(ldw >= k, SWL_ERR_INVALID, "swl_int8_pack_bf16: row stride smaller than a row");
  SWL_CHECK(aligned(data, 16), SWL_ERR_INVALID, "swl_int8_pack_bf16: data must be 16-byte aligned");
  hipLaunchKernelGGL(int8_pack_kernel, dim3((unsigned)((n + 15) / 16)), dim3(1024), 0, (hipStream_t)stream,
                     reinterpret_cast<const bf16*>(w), ldw, n, k, (k + kStep - 1) / kStep, reinterpret_cast<u32x4*>(data), scale);
  SWL_LAUNCH_CHECK("int8_pack_kernel launch");
  return SWL_OK;
}

extern "C" int64_t swl_int8_matmul_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  return int8_plan(m, n, k).bytes;
}

extern "C" int swl_int8_matmul_bf16(const void* q, int64_t ldq, const float* q_scale, int64_t m, const void* w,
                                    const float* w_scale, int64_t n, int64_t k, const void* bias, void* y, int64_t ldy,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  SWL_CHECK(m >= 0 && m < ((int64_t)1 << 31) && n > 0 && n < kMaxChannels && k > 0 && k <= (1 << 17), SWL_ERR_INVALID,
            "swl_int8_matmul_bf16: bad sizes, or k over 131072");
  if (m == 0) return SWL_OK;
  SWL_CHECK(q && q_scale && w && w_scale && y, SWL_ERR_INVALID, "swl_int8_matmul_bf16: null argument");
  SWL_CHECK(ldq >= (k + 15) / 16 * 16 && ldy >= n, SWL_ERR_INVALID, "swl_int8_matmul_bf16: row strides smaller than a row");
  SWL_CHECK(aligned(q, 16) && ldq % 16 == 0 && aligned(w, 16) && aligned(y, 8), SWL_ERR_INVALID,
            "swl_int8_matmul_bf16: rows of q and w must be 16-byte aligned, y 8-byte");
  const Int8Plan p = int8_plan(m, n, k);
  SWL_CHECK(p.bytes == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= p.bytes), SWL_ERR_INVALID,
            "swl_int8_matmul_bf16: workspace smaller than swl_int8_matmul_workspace");
  Int8Args a{};
  a.x = reinterpret_cast<const int8_t*>(q);
  a.xs = q_scale;
  a.w = reinterpret_cast<const int8_t*>(w);
  a.ws = w_scale;
  a.bias = reinterpret_cast<const bf16*>(bias);
  a.y = reinterpret_cast<bf16*>(y);
  a.part = p.splits > 1 ? reinterpret_cast<int32_t*>(workspace) : nullptr;
  a.m = m;
  a.n = n;
  a.ldx = ldq;
  a.ldy = ldy;
  a.klast = (int32_t)((k + 15) / 16 * 16 - 16);
  a.steps = (int32_t)((k + kStep - 1) / kStep);
  a.tiles = (int32_t)((n + 15) / 16);
  a.splits = p.splits;
  const hipStream_t st = (hipStream_t)stream;
  if (p.few) {
    if (m <= 16) return launch_rows<1>(a, st);
    if (m <= 32) return launch_rows<2>(a, st);
    return launch_rows<4>(a, st);
  }
  if (p.big) return launch_tiles<4, 4, 2, 2>(a, st);
  if (int rc = launch_tiles<2, 2, 2, 4>(a, st)) return rc;
  if (p.splits > 1) {
    const int64_t quads = m * ((n + 3) / 4);
    hipLaunchKernelGGL(int8_fold_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, a);
    SWL_LAUNCH_CHECK("int8_fold_kernel launch");
  }
  return SWL_OK;
}
