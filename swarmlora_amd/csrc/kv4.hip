// The KV cache held in 4 bits: append with RoPE, read back, attention.
//
// A group of 32 dims of one token's key or value of one head is 32 codes
// (sign and 0 .5 1 1.5 2 3 4 6, e2m1) times 2^(b - 127), b one byte; these are
// the operands that gfx950's conversions and scaled MFMA take.  The cache is
// [num_blocks, hkv, block_size / 16] records of 16 tokens of one head (a
// "tile"), each laid out as the attention's MFMA operands read it:
//   0     key codes    64 t + d / 2 (token t of the tile, even dims low)
//   1024  value codes  256 (t / 4) + 16 (d / 8) + 4 (t % 4) + d % 8 / 2
//   2048  key scales   16 (d / 32) + t
//   2112  value scales 16 (t / 4) + 4 (d / 32) + t % 4
// Keys: lane (t, g) of a wave's 16-byte load holds token t's dims 32 g .. + 31,
// the A operand of the 16x16x128 MFMA with one scale per lane.  Values: lane
// (g, c) holds 8 dims 8 c .. + 7 of the four tokens 4 g .. + 3, which is what
// V^T as the A operand of a 16x16x32 MFMA needs of them, a token's scale per
// dword.  A tile is 2176 contiguous bytes, 17 lines of 128: one head's cache is
// read without its neighbours' (3.8 times fewer bytes than bf16).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dev_util.h"
#include "swl.h"
#include "swl_common.h"

namespace {

constexpr int kD = 128;          // head dim
constexpr int kTile = 16;        // tokens of a record
constexpr int kRec = 17 * kD;    // bytes of a record
constexpr int kRecV = 1024, kRecKs = 2048, kRecVs = 2112;

// Division by a number that the host knows, for dividends under 2^31.
struct FastDiv {
  uint32_t d, mul, shift;  // mul 0: d is 1
};
FastDiv fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  if (d > 1) {
    const int s = 32 - __builtin_clz(d - 1);  // 2^s >= d
    f.mul = (uint32_t)((((uint64_t)1 << (31 + s)) / d) + 1);
    f.shift = (uint32_t)(s - 1);
  }
  return f;
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const FastDiv& f) {
  return f.mul ? __umulhi(n, f.mul) >> f.shift : n;
}

struct Kv4Args {
  const bf16* q;            // [T, hq, 128], token stride qs
  const bf16* k;            // append: [T, hkv, 128]
  const bf16* v;
  int64_t qs, ks, vs;
  uint8_t* pages;
  const int32_t* bt;        // [nseq, max_blocks]
  const int32_t* seqlens;   // tokens before the new ones
  const int32_t* cu;        // [nseq + 1] token offsets, null: L tokens each
  const int64_t* pos;
  const bf16* cs;           // [max_pos, 128]
  bf16* out;                // append: rotated q; attention: [T, hq * 128]
  bf16* out2;               // read: values
  int64_t num_blocks, max_blocks, max_pos;
  int64_t T;
  int32_t kmax;             // keys of a table
  int32_t nseq, L, hq, hkv, G;
  int32_t tpp;              // tiles of a page
  FastDiv by_g, by_hkv, by_tpp, by_l;
  float scale;
  // attention: records of parts; workgroups that run at once
  float* part;
  int32_t slots, min_spp, row_lo, row_hi;
  int64_t max_rec;
};

__device__ __forceinline__ uint32_t ldg_u8(const uint8_t* p) {
  return *(const __attribute__((address_space(1))) uint8_t*)(p);
}
__device__ __forceinline__ uint32_t ldg_u32(const uint8_t* p) {
  return *(const __attribute__((address_space(1))) uint32_t*)(p);
}

__device__ __forceinline__ float max_groups(float v) {  // over the four lane groups
  const uint32_t x = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t y = __float_as_uint(v);
  auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The sequence of packed token t (the same for the whole wave): how many
// sequences end at or before it; nseq for a token behind the last one.
__device__ __forceinline__ int seq_of(const Kv4Args& a, int64_t t, int lane) {
  if (!a.cu) return (int)((uint32_t)t / a.by_l);
  int s = 0;
  for (int i0 = 0; i0 < a.nseq; i0 += 64) {
    const int i = i0 + lane;
    s += __popcll(__ballot(i < a.nseq && a.cu[i + 1] <= t));
  }
  return s;
}

// Record of the tile that holds token p of sequence s, head h; null where it
// has no page.
__device__ __forceinline__ uint8_t* tile_of(const Kv4Args& a, int s, int h, int64_t p) {
  if (p < 0) return nullptr;
  const int64_t tile = p / kTile;
  if (p >= a.kmax) return nullptr;
  const int64_t bi = (uint32_t)tile / a.by_tpp;
  const int32_t blk = a.bt[(int64_t)s * a.max_blocks + bi];
  if (blk < 0 || blk >= a.num_blocks) return nullptr;
  return a.pages + (((int64_t)blk * a.hkv + h) * a.tpp + (tile - bi * a.tpp)) * kRec;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, false);
}

// Scale byte of a group from the largest magnitude bits of its four lanes' 8
// dims: the largest / 2^(b - 127) in [3.5, 7), so that it rounds as if the grid
// went on to 8 (5 % less of its error than with [4, 8), where up to 8 would be
// cut to 6); [2, 252], so that every value held is a normal, finite bf16;
// 255 (read as NaN) for a group with an infinity or a NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  top = max(top, dpp_u<0xB1>(top));  // quad_perm [1, 0, 3, 2]
  top = max(top, dpp_u<0x4E>(top));  // quad_perm [2, 3, 0, 1]
  const int b = (int)((top + 0x200000u) >> 23) - 2;
  return top >= 0x7f800000u ? 255u : (uint32_t)min(max(b, 2), 252);
}

// Eight dims as codes under 2^(b - 127), dim i in bits 4 i.
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], uint32_t b) {
  const float s = __uint_as_float(min(b, 252u) << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
}

__device__ __forceinline__ uint32_t top8(const float (&x)[8]) {
  uint32_t t = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) t = max(t, __float_as_uint(x[e]) & 0x7fffffffu);
  return t;
}

// NeoX rotation of q and k at their positions; q to its output rows, k and v
// as 4-bit groups to the pages.  A 128-thread workgroup per (token, 16 heads),
// eight threads a head with 16-byte accesses: thread c has dims 8 c .. + 7 and
// the same of the other half, so that a quad of threads holds two whole groups
// of 32.  Keys are rounded once, from the fp32 rotation.  Bytes bound it where
// there are many tokens (10639 of 32 + 2 * 8 heads, 232 MB, 41 us: 5.7 TB/s),
// the launch and one trip to memory where there are few (28: 3.4 us).
__global__ __launch_bounds__(128) void kv4_append_kernel(Kv4Args a) {
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int nq = a.out ? a.hq : 0;
  const int h = blockIdx.y * 16 + (threadIdx.x >> 3);  // [0, nq): q, then k, then v heads
  const int s = seq_of(a, t, lane);
  if (s >= a.nseq || h >= nq + 2 * a.hkv) return;
  const int c = threadIdx.x & 7, d = 8 * c;
  const bool is_q = h < nq, is_k = !is_q && h < nq + a.hkv;
  const int kvh = is_k ? h - nq : h - nq - a.hkv;
  const bf16* row = (is_q ? a.q + t * a.qs + h * kD : is_k ? a.k + t * a.ks + kvh * kD : a.v + t * a.vs + kvh * kD) + d;
  const u32x4 w1 = ldg16(row), w2 = ldg16(row + 64);
  const int64_t pos = a.pos ? a.pos[t] : -1;
  const int64_t i = t - (a.cu ? (int64_t)a.cu[s] : (int64_t)s * a.L);
  const int64_t p = (int64_t)a.seqlens[s] + i;
  float x1[8], x2[8];
  unpack8(w1, x1);
  unpack8(w2, x2);
  if ((is_q || is_k) && pos >= 0 && pos < a.max_pos) {
    const bf16* cs = a.cs + pos * kD + d;
    float co[8], sn[8];
    unpack8(ldg16(cs), co);
    unpack8(ldg16(cs + 64), sn);
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // (products of two bf16 are exact: one rounding each)
      const float y1 = x1[e] * co[e] - x2[e] * sn[e];
      x2[e] = x2[e] * co[e] + x1[e] * sn[e];
      x1[e] = y1;
    }
  }
  if (is_q) {
    bf16x8 o1, o2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o1[e] = f2bf(x1[e]);
      o2[e] = f2bf(x2[e]);
    }
    bf16* dst = a.out + (t * a.hq + h) * kD + d;
    *reinterpret_cast<u32x4*>(dst) = __builtin_bit_cast(u32x4, o1);
    *reinterpret_cast<u32x4*>(dst + 64) = __builtin_bit_cast(u32x4, o2);
    return;
  }
  const uint32_t b1 = scale_byte(top8(x1)), b2 = scale_byte(top8(x2));
  const uint32_t q1 = codes8(x1, b1), q2 = codes8(x2, b2);
  uint8_t* rec = tile_of(a, s, kvh, p);
  if (!rec) return;
  const int tk = (int)(p & 15);
  uint8_t* dst = rec + (is_k ? 64 * tk + 4 * c : kRecV + 256 * (tk >> 2) + 4 * (tk & 3) + 16 * c);
  *reinterpret_cast<uint32_t*>(dst) = q1;
  *reinterpret_cast<uint32_t*>(dst + (is_k ? 32 : 128)) = q2;
  if ((c & 3) == 0) {
    uint8_t* sc = rec + (is_k ? kRecKs + 16 * (c >> 2) + tk : kRecVs + 16 * (tk >> 2) + 4 * (c >> 2) + (tk & 3));
    sc[0] = (uint8_t)b1;
    sc[is_k ? 32 : 8] = (uint8_t)b2;
  }
}

template <int J>
__device__ __forceinline__ uint32_t pair_bf16(uint32_t codes, float s) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, J));
}
__device__ __forceinline__ u32x4 values8(uint32_t codes, uint32_t b) {
  const float s = __uint_as_float(b << 23);  // (exponent 255: the conversion gives NaN)
  return u32x4{pair_bf16<0>(codes, s), pair_bf16<1>(codes, s), pair_bf16<2>(codes, s), pair_bf16<3>(codes, s)};
}

// (written once and not read here: kept out of the caches' way)
__device__ __forceinline__ void stg16_nt(bf16* p, u32x4 v) {
  __builtin_nontemporal_store(v, (__attribute__((address_space(1))) u32x4*)p);
}

// Cached tokens as bf16: sixteen lanes a (token, head) row of keys and of
// values (four tokens a wave at a time, sixteen in flight), so that a store
// covers whole rows.  Tokens without a page are zeros.  Its bytes bound it: 69
// thousand tokens of 8 heads, 358 MB, 55 us (6.5 TB/s; with stores through the
// caches and four tokens a wave 188 us); a request of 300 tokens 5.3 us.
constexpr int kReadTokens = 16;  // of a wave

__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Args a) {
  const int lane = threadIdx.x & 63, c = lane & 15, h = blockIdx.y;
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * kReadTokens;
  if (t0 >= a.T) return;
  constexpr int N = kReadTokens / 4;
  // sequences of the wave's tokens: how many end at or before each
  int seq[kReadTokens] = {};
  if (a.cu)
    for (int i0 = 0; i0 < a.nseq; i0 += 64) {
      const int i = i0 + lane;
      const int end = i < a.nseq ? a.cu[i + 1] : 0x7fffffff;
#pragma unroll
      for (int k = 0; k < kReadTokens; ++k) seq[k] += __popcll(__ballot(end <= t0 + k));
    }
  uint32_t kq[N], vq[N], kb[N], vb[N];
  bool in[N], there[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int64_t t = t0 + 4 * n + (lane >> 4);
    const int q = lane >> 4;
    int s = q == 0 ? seq[4 * n] : q == 1 ? seq[4 * n + 1] : q == 2 ? seq[4 * n + 2] : seq[4 * n + 3];
    if (!a.cu) s = (int)min<int64_t>((uint32_t)t / a.by_l, a.nseq);
    in[n] = t < a.T && s < a.nseq;
    const int64_t p = in[n] ? (int64_t)a.seqlens[s] + t - (a.cu ? (int64_t)a.cu[s] : (int64_t)s * a.L) : -1;
    const uint8_t* rec = tile_of(a, s, h, p);
    there[n] = rec != nullptr;
    if (!rec) rec = a.pages;
    const int tk = (int)(p & 15);
    kq[n] = ldg_u32(rec + 64 * tk + 4 * c);
    vq[n] = ldg_u32(rec + kRecV + 256 * (tk >> 2) + 16 * c + 4 * (tk & 3));
    kb[n] = ldg_u8(rec + kRecKs + 16 * (c >> 2) + tk);
    vb[n] = ldg_u8(rec + kRecVs + 16 * (tk >> 2) + 4 * (c >> 2) + (tk & 3));
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!in[n]) continue;
    const int64_t at = ((t0 + 4 * n + (lane >> 4)) * a.hkv + h) * kD + 8 * c;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    stg16_nt(a.out + at, there[n] ? values8(kq[n], kb[n]) : zero);
    stg16_nt(a.out2 + at, there[n] ? values8(vq[n], vb[n]) : zero);
  }
}

// ------------------------------------------------------------- attention ---
// Rows are (new token, query head) pairs of one kv head, row = token * G +
// head; a row sees the keys before its token and its own.  Work is cut into
// units (sequence, kv head, block of RB rows, part of the keys); every wave
// finds its unit by itself from the lengths (a scan over the sequences, 64 at
// a time), so that the host knows none of them and a captured call follows
// them.  A part is `spp` steps of KS keys, as many as make the whole call's
// units fit the GPU at once, so that units are equally long whatever the
// lengths are.  A block of one part writes its rows; others leave a record per
// part, merged by kv4_combine_kernel.
struct SeqInfo {
  int t0, n, rb;
  int len, steps;  // steps of the longest row
};

template <int RB, int KS>
__device__ __forceinline__ SeqInfo seq_info(const Kv4Args& a, int i) {
  SeqInfo r{0, 0, 0, 0, 0};
  if (i >= a.nseq) return r;
  r.t0 = a.cu ? a.cu[i] : i * a.L;
  r.n = a.cu ? a.cu[i + 1] - r.t0 : a.L;
  r.len = min(a.seqlens[i], 1 << 30);  // (tables end at 2^30)
  if (r.t0 < 0 || r.n < 0 || (int64_t)r.t0 + r.n > a.T) r.n = 0;  // offsets that are none
  const int rows = r.n * a.G;
  if (rows <= a.row_lo || rows > a.row_hi) return r;
  r.rb = (int)((uint32_t)(rows + RB - 1) / RB);
  const int kend = (int)min<int64_t>(max<int64_t>((int64_t)r.len + r.n, 0), a.kmax);
  r.steps = max((kend + KS - 1) / KS, 1);
  return r;
}

// Inclusive prefix over the wave's lanes, in six vector instructions (row
// shifts, then the row ends passed on).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_prefix(int v) {
  v += dpp_i<0x111, 0xF>(v);
  v += dpp_i<0x112, 0xF>(v);
  v += dpp_i<0x114, 0xF>(v);
  v += dpp_i<0x118, 0xF>(v);
  v += dpp_i<0x142, 0xA>(v);  // row_bcast 15
  return v + dpp_i<0x143, 0xC>(v);  // row_bcast 31
}
__device__ __forceinline__ float wave_sum(float v) {
  auto add = [&](int x) { v += __int_as_float(x); };
  add(dpp_i<0x111, 0xF>(__float_as_int(v)));
  add(dpp_i<0x112, 0xF>(__float_as_int(v)));
  add(dpp_i<0x114, 0xF>(__float_as_int(v)));
  add(dpp_i<0x118, 0xF>(__float_as_int(v)));
  add(dpp_i<0x142, 0xA>(__float_as_int(v)));
  add(dpp_i<0x143, 0xC>(__float_as_int(v)));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Steps of a part: the fewest (at least min_spp) that cut the call into no more
// units than `slots`, the workgroups that run at once: a second round of a few
// units costs as much as a whole one (28 sequences with 1 to 6 drafted tokens
// over 128 to 8192 keys 41 us, 44 with their steps shared out evenly).  With as
// many blocks as places, or more sequences than a wave's lanes, the steps are
// shared out evenly.  (Plans of several rounds are not looked at, though blocks
// between half and all of the places would gain by one: four chunks of 300
// tokens over 4000 keys, 320 blocks of 68 steps in 512 places, stay whole, 68
// steps a place, where three parts each would be two rounds of 23.)  Either way a part is at least steps / slots, so that there
// are at most `slots` full parts, `slots` + blocks units, `slots` blocks that
// are cut and 2 `slots` records, whatever the lengths.  r: seq_info of the
// lane's sequence.
template <int RB, int KS>
__device__ __forceinline__ int steps_per_part(const Kv4Args& a, int lane, const SeqInfo& r) {
  const float mine = (float)r.rb * (float)a.hkv, st = (float)r.steps;
  float sum = mine * st;
  for (int i = 64 + lane; i - lane < a.nseq; i += 64) {
    const SeqInfo x = seq_info<RB, KS>(a, i);
    sum += (float)x.rb * (float)a.hkv * (float)x.steps;
  }
  // (rounded up past what the sum's roundings may have lost)
  const float slots = (float)a.slots, all = wave_sum(sum) * 1.0001f;
  int lo = max(a.min_spp, (int)fminf(all / slots + 1.f, 1073741824.f));
  if (a.nseq > 64) return lo;
  auto units = [&](int spp) { return wave_sum(mine * ceilf(st / (float)spp)); };
  const float blocks = wave_sum(mine);
  if (blocks >= slots || units(lo) <= slots) return lo;
  int hi = max(lo, (int)fminf(all / (slots - blocks) + 1.f, 1073741824.f));  // enough: a block has under one part more
  while (hi - lo > max(1, lo >> 4)) {
    const int mid = (lo + hi) >> 1;
    if (units(mid) <= slots)
      hi = mid;
    else
      lo = mid;
  }
  return hi;
}

struct Unit {
  int s, h, b, p, parts, t0, n, len;
  int64_t rec;  // the block's first record (where parts > 1)
};

// ceil(n / d) for n >= 1 by a float reciprocal, off by one at most before it is
// put right (quotients under 2^22)
__device__ __forceinline__ int ceil_div(int n, int d, float inv) {
  int q = (int)((float)(n - 1) * inv);
  const int r = n - 1 - q * d;
  q += r >= d ? 1 : r < 0 ? -1 : 0;
  return q + 1;
}

__device__ __forceinline__ int64_t lane64(int64_t v, int l) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v & 0xffffffff), l) |
         ((int64_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32);
}

// The unit of a workgroup: u counts (block, part) pairs, or (CUT) the blocks
// that are cut.
template <int RB, int KS, bool CUT>
__device__ __forceinline__ bool find_unit(const Kv4Args& a, int64_t u, int lane, int& spp, Unit& o) {
  SeqInfo r = seq_info<RB, KS>(a, lane);
  spp = steps_per_part<RB, KS>(a, lane, r);
  const uint32_t uw = (uint32_t)u / a.by_hkv;
  o.h = (int)((uint32_t)u - uw * (uint32_t)a.hkv);
  const float inv = 1.f / (float)spp;
  const int want = (int)uw;
  int before = 0;
  int64_t rec = 0;
  for (int i0 = 0;;) {
    const int parts = ceil_div(max(r.steps, 1), spp, inv);
    const int units = r.rb * parts, recs = parts > 1 ? units : 0, mine = CUT ? (parts > 1 ? r.rb : 0) : units;
    const int inc = wave_prefix(mine), rinc = wave_prefix(recs);
    const uint64_t hit = __ballot(before + inc > want);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      o.s = i0 + l;
      o.parts = __builtin_amdgcn_readlane(parts, l);
      o.t0 = __builtin_amdgcn_readlane(r.t0, l);
      o.n = __builtin_amdgcn_readlane(r.n, l);
      o.len = __builtin_amdgcn_readlane(r.len, l);
      const int rb = __builtin_amdgcn_readlane(r.rb, l);
      const int local = want - before - __builtin_amdgcn_readlane(inc - mine, l);
      const int blk = CUT || o.parts == 1 ? local : local / o.parts;
      o.b = rb - 1 - blk;  // the blocks with the most keys first
      o.p = CUT ? 0 : local - blk * o.parts;
      if (local < 0 || o.b < 0 || o.p < 0) return false;  // (counts past 32 bits: offsets that are none)
      o.rec = (int64_t)(rec + __builtin_amdgcn_readlane(rinc - recs, l) + (int64_t)o.b * o.parts) * a.hkv + o.h;
      return true;
    }
    before += __builtin_amdgcn_readlane(inc, 63);
    rec += __builtin_amdgcn_readlane(rinc, 63);
    i0 += 64;
    if (i0 >= a.nseq) return false;
    r = seq_info<RB, KS>(a, i0 + lane);
  }
}

// Keys that row r of the unit's sequence sees.
__device__ __forceinline__ int last_key(const Kv4Args& a, const Unit& u, int r) {
  return min(max(u.len + (int)((uint32_t)r / a.by_g) + 1, 0), a.kmax);
}

// A record: 16 rows as [dim % 8][row-dim slot 256] sums, then the rows' maxima
// and sums of probabilities; slot (g * 16 + row) * 4 + i holds dim 32 g + 8 i +
// e in piece e.
constexpr int kRecF = 2048 + 32;

typedef int i32x8 __attribute__((ext_vector_type(8)));

// 16 rows of q as the B operand of the scaled MFMA: fp8 twice, the nearest and
// what is left of it, both exact but for elements under 2^-13 of their row's
// largest (off by 2^-21 of that at most: half of the second one's least step,
// 2^-13, where the largest is 2^7): a bf16 has 8 significant bits, e4m3 4.  The
// lane has dims 16 g .. + 15 and 64 + 16 g .. + 15, as the operand counts them.
struct QFrag {
  i32x8 hi, lo;
  int sb;  // scale byte of hi; lo's is 4 less
};
struct QRow {
  u32x4 x[4];
};
__device__ __forceinline__ QRow q_row(const bf16* row, int g) {
  QRow r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.x[j] = ldg16(row + 64 * (j >> 1) + 16 * g + 8 * (j & 1));
  return r;
}
__device__ __forceinline__ QFrag q_frag(const QRow& r) {
  float x[4][8];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unpack8(r.x[j], x[j]);
    top = max(top, top8(x[j]));
  }
  top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
  top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
  QFrag f;
  const int e = (int)(top >> 23);  // the largest / 2^(sb - 127) in [128, 256)
  f.sb = e == 255 ? 255 : max(e - 7, 5);
  const float s = __uint_as_float((uint32_t)min(f.sb, 250) << 23), s2 = s * 0.0625f;
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float* y = &x[j][4 * w];
      s16x2 h = {0, 0}, l = {0, 0};
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, y[0], y[1], s, false);
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, y[2], y[3], s, true);
      const int hw = __builtin_bit_cast(int, h);
      const f32x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, s, false);
      const f32x2 a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, s, true);
      l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, y[0] - a0[0], y[1] - a0[1], s2, false);
      l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, y[2] - a1[0], y[3] - a1[1], s2, true);
      f.hi[2 * j + w] = hw;
      f.lo[2 * j + w] = __builtin_bit_cast(int, l);
    }
  return f;
}

// scores of a 16-key tile (key 4 (lane / 16) + i) with 16 rows (lane % 16)
__device__ __forceinline__ f32x4 qk_hi(u32x4 k, int ks, const QFrag& q) {
  const i32x8 A = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, q.hi, f32x4{0.f, 0.f, 0.f, 0.f}, 4, 0, 0, ks, 0, q.sb);
}
__device__ __forceinline__ f32x4 qk_lo(u32x4 k, int ks, const QFrag& q, f32x4 c) {
  const i32x8 A = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, q.lo, c, 4, 0, 0, ks, 0, q.sb - 4);
}
__device__ __forceinline__ f32x4 scores(u32x4 k, int ks, const QFrag& q) { return qk_lo(k, ks, q, qk_hi(k, ks, q)); }

// A lane's dwords of a tile's values (8 dims of four tokens) as pairs of
// tokens: f[e][0], f[e][1] = tokens (0, 1), (2, 3) of dim 2 J + e.
template <int J>
__device__ __forceinline__ void v_pair(u32x4 v, uint32_t vs, uint32_t (&f)[2][2]) {
  const uint32_t w0 = pair_bf16<J>(v[0], __uint_as_float((vs & 0xffu) << 23));
  const uint32_t w1 = pair_bf16<J>(v[1], __uint_as_float((vs >> 8 & 0xffu) << 23));
  const uint32_t w2 = pair_bf16<J>(v[2], __uint_as_float((vs >> 16 & 0xffu) << 23));
  const uint32_t w3 = pair_bf16<J>(v[3], __uint_as_float((vs >> 24) << 23));
  f[0][0] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
  f[0][1] = __builtin_amdgcn_perm(w3, w2, 0x05040100u);
  f[1][0] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
  f[1][1] = __builtin_amdgcn_perm(w3, w2, 0x07060302u);
}
// All eight dims: f[e] of dim e.
__device__ __forceinline__ void v_pairs(u32x4 v, uint32_t vs, uint32_t (&f)[8][2]) {
  auto put = [&](int e, const uint32_t (&x)[2][2]) {
    f[e][0] = x[0][0];
    f[e][1] = x[0][1];
    f[e + 1][0] = x[1][0];
    f[e + 1][1] = x[1][1];
  };
  uint32_t x[2][2];
  v_pair<0>(v, vs, x);
  put(0, x);
  v_pair<1>(v, vs, x);
  put(2, x);
  v_pair<2>(v, vs, x);
  put(4, x);
  v_pair<3>(v, vs, x);
  put(6, x);
}

// Sums whose reference was not the largest score: outside [2^-60, 2^100), or
// not finite.
__device__ __forceinline__ bool bad_sums(float L, const f32x4 (&acc)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(acc[d][i]) & 0x7fffffffu);
  return !(L >= 0x1p-60f && L < 0x1p100f) || top >= 0x7f800000u;
}
// The factor that takes a sum L to [1, 2); m becomes the reference of that.
__device__ __forceinline__ float rebase(float L, float& m) {
  if (!(L > 0.f && L < INFINITY)) return 1.f;
  const int x = (int)(__float_as_uint(L) >> 23) - 127;  // (L at least 2^-60, or 1 with a running maximum)
  m = (m == -INFINITY ? 0.f : m) + (float)x;
  return __uint_as_float((uint32_t)(127 - x) << 23);
}

// Takes the NaN groups out of a tile's values where some row does not see
// their token (0 times a NaN is one); flags gets 0xff in the bytes of theirs.
__device__ __forceinline__ void take_nan(u32x4& v, uint32_t& vs, uint32_t& flags) {
  flags = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if ((vs >> (8 * k) & 0xffu) > 252u) {
      v[k] = 0;
      vs = (vs & ~(0xffu << (8 * k))) | 127u << (8 * k);
      flags |= 0xffu << (8 * k);
    }
}
// Whether the lane's row, which sees the first `see` keys of the step, sees one
// whose values of dims 32 g .. + 31 (the lane's) are a NaN group.  By the whole
// wave.
__device__ __forceinline__ bool sees_nan(const uint32_t (&flags)[2], int see, int g) {
  bool bad = false;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int qd = 0; qd < 4; ++qd) {
      const uint32_t f = (uint32_t)__shfl((int)flags[t], 16 * qd + 4 * g, 64);
#pragma unroll
      for (int k = 0; k < 4; ++k) bad |= (f >> (8 * k) & 1u) != 0 && 16 * t + 4 * qd + k < see;
    }
  return bad;
}

// e^(m - M) in powers of two; a side without a key (-inf) counts for nothing,
// one that has the maximum wholly (an infinite or NaN one too)
__device__ __forceinline__ float merge_factor(float m, float M) {
  return m == M ? (m == -INFINITY ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - M);
}

// dims 32 g + 8 i .. + 7 of a row; slot = (16 g + row % 16) * 4 + i
__device__ __forceinline__ void write_row(const Kv4Args& a, const Unit& u, int r, int slot, float L,
                                          const float (&o)[8]) {
  const int tok = (uint32_t)r / a.by_g, head = u.h * a.G + r - tok * a.G;
  // (L is 0 where the row sees no key, NaN where a score is)
  const float inv = L == 0.f ? 0.f : 1.f / L;
  bf16x8 y;
#pragma unroll
  for (int d = 0; d < 8; ++d) y[d] = f2bf(L == 0.f ? 0.f : o[d] * inv);
  bf16* dst = a.out + ((int64_t)(u.t0 + tok) * a.hq + head) * kD + 32 * (slot >> 6) + 8 * (slot & 3);
  *(__attribute__((address_space(1))) u32x4*)dst = __builtin_bit_cast(u32x4, y);
}

// Few rows, many keys (single and drafted tokens): a workgroup of four waves
// per unit of 16 SETS rows; wave w takes the part's steps of 32 keys (two
// tiles) w, w + 4, ... on its own, the operands straight from the pages into
// registers, each requested anew as soon as it has been used; the waves'
// results meet in LDS.  S^T = K Q^T (scaled MFMA, keys as stored) leaves in a
// lane the keys 4 g .. + 3 of both tiles of its row, which is the B operand of
// O^T = V^T P^T as it is.  The probabilities enter as one bf16 and are summed as
// they are, as in the kernel for many rows; a second bf16 of each would make the
// three cases below 135, 35 and 15 us.
//
// The cache's bytes bound it once they are many: 32 tokens over 8192 to 32767
// keys each (742 MB) take 124 us, 6.0 TB/s; 1 to 6 drafted tokens of 28 requests
// over 128 to 8192 keys (122 MB) 30 us, with a second step of loads in flight a
// wave 33.  Under that the chain of dependent loads (lengths, table, records)
// does: 7 us for four tokens over 300 keys, 14 for 28 over 128 to 2048.
constexpr int kSplitWaves = 4;

struct SplitLds {
  float mg[kSplitWaves][kRecF];
};

template <int SETS>
__device__ __forceinline__ void split_unit(const Kv4Args& a, uint32_t unit, SplitLds& sh) {
  constexpr int RB = 16 * SETS, KS = 32, W = kSplitWaves;
  auto& mg = sh.mg;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  int spp;
  Unit u;
  if (!find_unit<RB, KS, false>(a, unit, lane, spp, u)) return;  // the same for the whole workgroup
  const int rows = u.n * a.G, r0 = u.b * RB;
  const int kend = last_key(a, u, min(r0 + RB, rows) - 1);
  const int st0 = u.p * spp;                                // the part's first step
  const int nst = max(0, min(spp, (kend + KS - 1) / KS - st0));
  if (nst == 0 && u.p > 0) return;  // (the longest row's part; this block's end before it)
  const int nw = nst > w ? (nst - w + W - 1) / W : 0;  // this wave's steps: st0 + w + j W

  // lane 2 i + t: address of the record of tile t of this wave's step j0 + i
  // (the first record's where it is past the keys or has no page: `gone`
  // tells), a table of 32 steps; the pages of the next 32 are requested when a
  // table is made
  const int32_t* bt = a.bt + (int64_t)u.s * a.max_blocks;
  int64_t table = 0;
  uint64_t gone = 0;
  int32_t blk_next = -1;
  auto tile_of_lane = [&](int j) { return ((uint32_t)st0 + w + (j + (lane >> 1)) * W) * 2 + (lane & 1); };
  auto request = [&](int j) {
    const uint32_t tile = tile_of_lane(j);
    blk_next = tile * kTile < (uint32_t)kend ? bt[tile / a.by_tpp] : -1;
  };
  auto look = [&](int j) {
    const bool there = blk_next >= 0 && blk_next < a.num_blocks;
    gone = __ballot(!there);
    const uint32_t tile = tile_of_lane(j);
    table = (int64_t)a.pages + (there ? (((int64_t)blk_next * a.hkv + u.h) * a.tpp +
                                         (tile - tile / a.by_tpp * (uint32_t)a.tpp)) * kRec : 0);
    request(j + 32);
  };
  request(0);

  QRow raw[SETS];  // (made operands behind the first records' requests)
  int ctx[SETS];   // keys that the lane's rows see, from the part's first step
#pragma unroll
  for (int e = 0; e < SETS; ++e) {
    const int r = min(r0 + e * 16 + col, rows - 1), tok = (uint32_t)r / a.by_g;
    raw[e] = q_row(a.q + (u.t0 + tok) * a.qs + (int64_t)(u.h * a.G + r - tok * a.G) * kD, g);
    ctx[e] = min(max(u.len + tok + 1 - st0 * KS, 0), nst * KS);
  }
  const int all_see = min(max(last_key(a, u, r0) - st0 * KS, 0), nst * KS);  // keys that every row sees
  const int live = min(max(kend - st0 * KS, 0), nst * KS);                    // that any sees

  auto tile_at = [&](int j, int t) { return reinterpret_cast<const uint8_t*>(lane64(table, 2 * (j & 31) + t)); };
  uint32_t koff = 64 * col + 16 * g, soff = lane, voff = 16 * lane, xoff = 16 * g + (col & 12);
  u32x4 kc[2], vc[2];
  uint32_t ks[2], vs[2];
  auto load_k = [&](int j) {
    asm("" : "+v"(koff), "+v"(soff));  // (a scalar base and a 32-bit offset: not widened outside the loop)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* rec = tile_at(j, t);
      kc[t] = ldg16_nt(rec + koff);
      ks[t] = ldg_u8(rec + soff + kRecKs);
    }
  };
  auto load_v = [&](int j) {
    asm("" : "+v"(voff), "+v"(xoff));
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* rec = tile_at(j, t);
      vc[t] = ldg16_nt(rec + voff + kRecV);
      vs[t] = ldg_u32(rec + xoff + kRecVs);
    }
  };

  const float c2 = a.scale * 1.44269504088896340736f;  // scores in powers of two
  const u32x4 ones = u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  float m[SETS];
  bool nan_v[SETS];  // the row sees a NaN group of the lane's dims
  f32x4 acc[SETS][8], l[SETS];
#pragma unroll
  for (int e = 0; e < SETS; ++e) {
    m[e] = -INFINITY;
    nan_v[e] = false;
    l[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[e][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  look(0);
  load_k(0);
  load_v(0);
  QFrag q[SETS];
#pragma unroll
  for (int e = 0; e < SETS; ++e) q[e] = q_frag(raw[e]);
  auto walk = [&](auto sets) {  // the wave's steps, for the sets that have rows
    constexpr int NS = decltype(sets)::value;
    for (int j = 0; j < nw; ++j) {
      const int k0 = (w + j * W) * KS;  // from the part's first step
      const uint32_t none = (uint32_t)(gone >> (2 * (j & 31))) & 3u;  // bit t: tile t is not there
      // a row of the block ends inside the step, or a tile is missing
      const bool edge = k0 + KS > all_see || none;
      f32x4 sv[NS][2];
#pragma unroll
      for (int e = 0; e < NS; ++e)
#pragma unroll
        for (int t = 0; t < 2; ++t) sv[e][t] = scores(kc[t], (int)ks[t], q[e]);
      if (edge) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bool no = none >> t & 1;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (no || k0 + 16 * t + 4 * g + k >= live) {  // what is stored there is anything: 0 times a NaN is one
              vc[t][k] = 0;
              vs[t] = (vs[t] & ~(0xffu << (8 * k))) | 127u << (8 * k);
            }
#pragma unroll
          for (int e = 0; e < NS; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (no || k0 + 16 * t + 4 * g + k >= ctx[e]) sv[e][t][k] = -INFINITY;
        }
        uint32_t fl[2];  // NaN groups
        take_nan(vc[0], vs[0], fl[0]);
        take_nan(vc[1], vs[1], fl[1]);
        if (__ballot((fl[0] | fl[1]) != 0) != 0) {
#pragma unroll
          for (int e = 0; e < NS; ++e) nan_v[e] |= sees_nan(fl, ctx[e] - k0, g);
        }
      }
      if (((j + 1) & 31) == 0) look(j + 1);
      load_k(j + 1);  // (past the last step: the first record, or one of the next part's)
      u32x4 p[NS];
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        const float mx = c2 * max_groups(fmaxf(fmaxf(fmaxf(sv[e][0][0], sv[e][0][1]), fmaxf(sv[e][0][2], sv[e][0][3])),
                                               fmaxf(fmaxf(sv[e][1][0], sv[e][1][1]), fmaxf(sv[e][1][2], sv[e][1][3]))));
        // the reference the exponents are taken from moves only when the maximum
        // has grown by 2^8 since: any reference gives the same quotient.  (The
        // reference of the first step alone, as in the kernel for many rows, is
        // level or slower here: the cache's bytes are the bound.)
        if (__ballot(mx > m[e] + 8.f) != 0) {
          const float mn = fmaxf(m[e], mx);
          const float corr = mn == m[e] ? 1.f : __builtin_amdgcn_exp2f(m[e] - mn);
          m[e] = mn;
          l[e] *= corr;
#pragma unroll
          for (int d = 0; d < 8; ++d) acc[e][d] *= corr;
        }
        const float mr = m[e] == -INFINITY ? 0.f : m[e];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // tokens in pairs: one conversion for both
          const f32x4& y = sv[e][k >> 1];
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[2 * (k & 1)], c2, -mr));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[2 * (k & 1) + 1], c2, -mr));
          p[e][k] = __builtin_bit_cast(uint32_t, (bf16x2){f2bf(p0), f2bf(p1)});
        }
        l[e] = mfma16(ones, p[e], l[e]);
      }
      auto pv = [&](int d, const uint32_t (&f0)[2][2], const uint32_t (&f1)[2][2]) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < NS; ++e)
            acc[e][d + x] = mfma16(u32x4{f0[x][0], f0[x][1], f1[x][0], f1[x][1]}, p[e], acc[e][d + x]);
      };
      uint32_t f0[2][2], f1[2][2];
      v_pair<0>(vc[0], vs[0], f0);
      v_pair<0>(vc[1], vs[1], f1);
      pv(0, f0, f1);
      v_pair<1>(vc[0], vs[0], f0);
      v_pair<1>(vc[1], vs[1], f1);
      pv(2, f0, f1);
      v_pair<2>(vc[0], vs[0], f0);
      v_pair<2>(vc[1], vs[1], f1);
      pv(4, f0, f1);
      v_pair<3>(vc[0], vs[0], f0);
      v_pair<3>(vc[1], vs[1], f1);
      load_v(j + 1);
      pv(6, f0, f1);
    }
  };
  if (SETS > 1 && rows - r0 <= 16)
    walk(std::integral_constant<int, 1>{});
  else
    walk(std::integral_constant<int, SETS>{});

  // the waves' results in LDS, rows that there are; thread = (g, row, i): dims
  // 32 g + 8 i .. + 7
  const int row = threadIdx.x >> 2 & 15;
#pragma unroll
  for (int e = 0; e < SETS; ++e) {
    const int nr = rows - r0 - 16 * e;
    if (e > 0) {
      if (nr <= 0) return;  // the same for the whole workgroup
      __syncthreads();
    }
    if (col < nr) {
#pragma unroll
      for (int d = 0; d < 8; ++d)
        *reinterpret_cast<f32x4*>(&mg[w][d * 256 + lane * 4]) = nan_v[e] ? f32x4{NAN, NAN, NAN, NAN} : acc[e][d];
      if (g == 0) {
        mg[w][2048 + col] = m[e];
        mg[w][2064 + col] = l[e][0];
      }
    }
    __syncthreads();
    if (row >= nr) continue;
    float M = -INFINITY, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < W; ++v) M = fmaxf(M, mg[v][2048 + row]);
#pragma unroll
    for (int v = 0; v < W; ++v) {
      const float f = merge_factor(mg[v][2048 + row], M);
      L += mg[v][2064 + row] * f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] += mg[v][d * 256 + threadIdx.x] * f;
    }
    if (u.parts == 1) {
      write_row(a, u, r0 + e * 16 + row, threadIdx.x, L, o);
    } else {
      const int64_t at = u.rec + (int64_t)u.p * a.hkv;
      if (at >= a.max_rec) continue;  // (only where offsets overlap)
      float* rec = a.part + (at * SETS + e) * kRecF;
#pragma unroll
      for (int d = 0; d < 8; ++d) rec[d * 256 + threadIdx.x] = o[d];
      if ((threadIdx.x & 0xc3) == 0) {
        rec[2048 + row] = M;
        rec[2064 + row] = L;
      }
    }
  }
}

template <int SETS>
__global__ __launch_bounds__(64 * kSplitWaves, SETS == 1 ? 4 : 2) void kv4_split_kernel(Kv4Args a) {
  __shared__ __attribute__((aligned(16))) SplitLds sh;
  split_unit<SETS>(a, blockIdx.x, sh);
}

// Many rows (prompts and their chunks): a workgroup of four waves per unit of
// 128 rows, 32 a wave, all four over the same keys, 64 a step.  Keys go from
// the pages into every wave's registers as they are stored (the MFMA's 4-bit
// operand: no conversion, a quarter of bf16's bytes).  Values are made bf16
// once for the four waves: wave w turns tile w of the step into MFMA operand
// order and leaves it in LDS for the next step, one barrier a step.  The
// probabilities enter as one bf16 (off by 2^-8 of each at most, together 0.0014
// of the result, rms, less than its own rounding and a hundredth of what 4 bits
// cost; two would double the matrix work of PV: 760 us in place of 567 for the
// prompts below, both traced), and their sum is an MFMA row of ones over the
// same rounded values, so that the weights sum to 1 exactly.
//
// Exponents are taken from the row's largest score of its first 32 keys, and
// no maximum is kept after that: a reference too low makes all terms larger by
// one factor, which the quotient does not see, until a term passes the largest
// number.  That, an infinity or NaN, or a row without a key in its first 32
// leaves sums outside [2^-60, 2^100); the unit is then done again with a
// running maximum.
//
// Matrix and vector work bound it about alike: five prompts up to 8192 tokens
// (600 GFLOP of visible scores and sums, 32 heads) take 480 us, 1250 TFLOP/s
// (567 under a kernel trace, which holds the clock lower), the matrix units busy
// 54 % of the time; with a running maximum 656 us traced, with the compiler's
// own order as well 1171.  128 rows a workgroup: with 32 every record would be
// made bf16 four times as often.
constexpr int kPromptRows = 128, kPromptKeys = 64;

struct PromptLds {
  char vb[2][2 * 8 * 1024];  // values of a step: [32-key half][dim % 8][lane] 16 bytes
  uint32_t nanf[2][4][64];   // a tile's NaN groups, where some row does not see its keys
  uint32_t again[4];
};

__device__ __forceinline__ void prompt_unit(const Kv4Args& a, uint32_t unit, PromptLds& sh) {
  constexpr int RB = kPromptRows, KS = kPromptKeys;
  auto& vb = sh.vb;
  auto& nanf = sh.nanf;
  auto& again = sh.again;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  int spp;
  Unit u;
  if (!find_unit<RB, KS, false>(a, unit, lane, spp, u)) return;  // the same for the whole workgroup
  const int rows = u.n * a.G, r0 = u.b * RB, wr0 = r0 + 32 * w;
  const int kend = last_key(a, u, min(r0 + RB, rows) - 1);
  const int st0 = u.p * spp;
  const int nst = max(0, min(spp, (kend + KS - 1) / KS - st0));
  if (nst == 0 && u.p > 0) return;

  QFrag q[2];
  int ctx[2];  // keys that the lane's rows see, from the part's first step
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = min(wr0 + e * 16 + col, rows - 1), tok = (uint32_t)r / a.by_g;
    q[e] = q_frag(q_row(a.q + (u.t0 + tok) * a.qs + (int64_t)(u.h * a.G + r - tok * a.G) * kD, g));
    ctx[e] = min(max(u.len + tok + 1 - st0 * KS, 0), nst * KS);
  }
  const int all_see = min(max(last_key(a, u, r0) - st0 * KS, 0), nst * KS);  // by every row
  const int live = min(max(kend - st0 * KS, 0), nst * KS);                    // by any

  // lane 4 i + t: address of the record of tile t of step j0 + i (the first
  // record's where it is past the keys or has no page: `gone` tells), a table of
  // 16 steps; the pages of the next 16 are requested when a table is made
  const int32_t* bt = a.bt + (int64_t)u.s * a.max_blocks;
  int64_t table = 0;
  uint64_t gone = 0;
  int32_t blk_next = -1;
  auto request = [&](int j) {
    const uint32_t tile = (uint32_t)(st0 + j) * 4 + lane;  // (fewer than 2^26)
    blk_next = tile * kTile < (uint32_t)kend ? bt[tile / a.by_tpp] : -1;
  };
  auto look = [&](int j) {
    const uint32_t tile = (uint32_t)(st0 + j) * 4 + lane;
    const bool there = blk_next >= 0 && blk_next < a.num_blocks;
    gone = __ballot(!there);
    table = (int64_t)a.pages +
            (there ? (((int64_t)blk_next * a.hkv + u.h) * a.tpp + (tile - tile / a.by_tpp * (uint32_t)a.tpp)) * kRec : 0);
    request(j + 16);
  };
  auto tile_at = [&](int j, int t) { return reinterpret_cast<const uint8_t*>(lane64(table, 4 * (j & 15) + t)); };
  auto missing = [&](int j) { return (uint32_t)(gone >> (4 * (j & 15))) & 15u; };  // bit t: tile t is not there
  uint32_t koff = 64 * col + 16 * g, soff = lane, voff = 16 * lane, xoff = 16 * g + (col & 12);
  u32x4 kc[4], vn;
  uint32_t ks[4], vsn;
  // (scalar base, 32-bit lane offset: the offsets are kept from being widened
  // once, outside the loop, which costs a 64-bit addition per load)
  auto load_k = [&](int j, int t) {
    const uint8_t* rec = tile_at(j, t);
    asm("" : "+v"(koff), "+v"(soff));
    kc[t] = ldg16(rec + koff);
    ks[t] = ldg_u8(rec + soff + kRecKs);
  };
  auto load_v = [&](int j) {
    const uint8_t* rec = tile_at(j, w);
    asm("" : "+v"(voff), "+v"(xoff));
    vn = ldg16(rec + voff + kRecV);
    vsn = ldg_u32(rec + xoff + kRecVs);
  };
  // values of step j (in vn) to LDS; none: its missing tiles
  auto clean = [&](int j, uint32_t none) {
    if ((j + 1) * KS > all_see || none) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if ((none >> w & 1) || j * KS + 16 * w + 4 * g + k >= live) {  // what is stored there is anything
          vn[k] = 0;
          vsn = (vsn & ~(0xffu << (8 * k))) | 127u << (8 * k);
        }
      uint32_t fl;
      take_nan(vn, vsn, fl);
      nanf[j & 1][w][lane] = fl;
    }
  };
  auto stage = [&](int j) {
    uint32_t f[8][2];
    v_pairs(vn, vsn, f);
    char* dst = vb[j & 1] + (w >> 1) * 8192 + lane * 16 + (w & 1) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) *reinterpret_cast<u32x2*>(dst + e * 1024) = u32x2{f[e][0], f[e][1]};
  };

  const float c2 = a.scale * 1.44269504088896340736f;  // scores in powers of two
  const u32x4 ones = u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  float m[2];
  f32x4 acc[2][8], l[2];
  bool nan_v[2];  // the row sees a NaN group of the lane's dims

  auto pass = [&](auto running) {
    constexpr bool RUNNING = decltype(running)::value;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[e] = -INFINITY;
      nan_v[e] = false;
      l[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < 8; ++d) acc[e][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (nst == 0) return;
    // scores of tiles t0, t0 + 1 of step j (none: its missing tiles)
    f32x4 sv[2][2];
    auto qk = [&](f32x4 (&s)[2][2], int t0) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[e][t] = scores(kc[t0 + t], (int)ks[t0 + t], q[e]);
    };
    auto mask = [&](f32x4 (&s)[2][2], int j, int t0, uint32_t none) {
      if ((j + 1) * KS <= all_see && none == 0) return;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int see = ctx[e] - j * KS - 16 * t0 - 4 * g;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if ((none >> (t0 + t) & 1) || 16 * t + k >= see) s[e][t][k] = -INFINITY;
      }
    };
    auto top = [&](int e) {
      return max_groups(fmaxf(fmaxf(fmaxf(sv[e][0][0], sv[e][0][1]), fmaxf(sv[e][0][2], sv[e][0][3])),
                              fmaxf(fmaxf(sv[e][1][0], sv[e][1][1]), fmaxf(sv[e][1][2], sv[e][1][3])))) * c2;
    };
    request(0);
    look(0);
    uint32_t none = missing(0);
#pragma unroll
    for (int t = 0; t < 4; ++t) load_k(0, t);
    load_v(0);
    clean(0, none);
    stage(0);
    qk(sv, 0);
    mask(sv, 0, 0, none);
    load_k(1, 0);
    load_k(1, 1);
    if constexpr (!RUNNING) {
      m[0] = top(0);
      m[1] = top(1);
    }
    float mr[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
    lds_barrier();
    for (int j = 0; j < nst; ++j) {
      const uint32_t none_next = missing(j + 1);
      const char* vp = vb[j & 1] + lane * 16;
      load_v(j + 1);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        if constexpr (RUNNING) {
          const float mx[2] = {top(0), top(1)};
          if (__ballot(mx[0] > m[0] + 8.f || mx[1] > m[1] + 8.f) != 0) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float mn = fmaxf(m[e], mx[e]);
              const float corr = mn == m[e] ? 1.f : __builtin_amdgcn_exp2f(m[e] - mn);
              m[e] = mn;
              l[e] *= corr;
#pragma unroll
              for (int d = 0; d < 8; ++d) acc[e][d] *= corr;
              mr[e] = mn == -INFINITY ? 0.f : mn;
            }
          }
        }
        if (hf == 1) {
          clean(j + 1, none_next);
          if (((j + 2) & 15) == 0) look(j + 2);
        }
        // One block without branches: the half's values from LDS, the next
        // half's scores beside this one's exponentials, then PV beside the next
        // step's values.  The order is held by scheduling barriers: left to
        // itself the compiler puts all exponentials before the matrix
        // instructions, and one wave's matrix and vector units take turns.
        u32x4 vf[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) vf[d] = *reinterpret_cast<const u32x4*>(vp + hf * 8192 + d * 1024);
        f32x4 sn[2][2];
        u32x4 p[2];
        __builtin_amdgcn_sched_barrier(0);
        float x0 = 0.f, x1 = 0.f;  // exponentials of the pair before, rounded while the next are on their way
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = i >> 1 & 1, t = i & 1, kt = 2 - 2 * hf + t;
          sn[e][t] = i < 4 ? qk_hi(kc[kt], (int)ks[kt], q[e]) : qk_lo(kc[kt], (int)ks[kt], q[e], sn[e][t]);
          __builtin_amdgcn_sched_barrier(0);
          const int pe = i >> 2, k = i & 3;
          const f32x4& y = sv[pe][k >> 1];
          const float y0 = __builtin_fmaf(y[2 * (k & 1)], c2, -mr[pe]);
          const float y1 = __builtin_fmaf(y[2 * (k & 1) + 1], c2, -mr[pe]);
          __builtin_amdgcn_sched_barrier(0);
          if (i > 0) p[(i - 1) >> 2][(i - 1) & 3] = __builtin_bit_cast(uint32_t, (bf16x2){f2bf(x0), f2bf(x1)});
          x0 = __builtin_amdgcn_exp2f(y0);
          x1 = __builtin_amdgcn_exp2f(y1);
          __builtin_amdgcn_sched_barrier(0);
        }
        p[1][3] = __builtin_bit_cast(uint32_t, (bf16x2){f2bf(x0), f2bf(x1)});
        const int jn = hf == 0 ? j + 1 : j + 2;
        load_k(jn, 2 - 2 * hf);
        load_k(jn, 3 - 2 * hf);
        char* dst = vb[(j + 1) & 1] + (w >> 1) * 8192 + lane * 16 + (w & 1) * 8;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          acc[0][d] = mfma16(vf[d], p[0], acc[0][d]);
          acc[1][d] = mfma16(vf[d], p[1], acc[1][d]);
          if (hf == 1 && (d & 1) == 0) {
            __builtin_amdgcn_sched_barrier(0);
            uint32_t f[2][2];
            switch (d) {
              case 0: v_pair<0>(vn, vsn, f); break;
              case 2: v_pair<1>(vn, vsn, f); break;
              case 4: v_pair<2>(vn, vsn, f); break;
              default: v_pair<3>(vn, vsn, f); break;
            }
            *reinterpret_cast<u32x2*>(dst + d * 1024) = u32x2{f[0][0], f[0][1]};
            *reinterpret_cast<u32x2*>(dst + (d + 1) * 1024) = u32x2{f[1][0], f[1][1]};
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) l[e] = mfma16(ones, p[e], l[e]);
        if (hf == 0)
          mask(sn, j, 2, none);
        else
          mask(sn, j + 1, 0, none_next);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int t = 0; t < 2; ++t) sv[e][t] = sn[e][t];
      }
      if ((j + 1) * KS > all_see || none) {  // (as `clean` decided: the flags are there)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t fl[2] = {nanf[j & 1][2 * hf][lane], nanf[j & 1][2 * hf + 1][lane]};
          if (__ballot((fl[0] | fl[1]) != 0) == 0) continue;
#pragma unroll
          for (int e = 0; e < 2; ++e) nan_v[e] |= sees_nan(fl, ctx[e] - j * KS - 32 * hf, g);
        }
      }
      none = none_next;
      lds_barrier();  // the next step's values are there, and this one's read by all
    }
  };
  pass(std::false_type{});
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 2; ++e) bad |= bad_sums(l[e][0], acc[e]);
  const bool any = __ballot(bad) != 0;
  if (lane == 0) again[w] = any ? 1 : 0;
  __syncthreads();
  if (again[0] | again[1] | again[2] | again[3]) {  // the same for the whole workgroup
    __syncthreads();
    pass(std::true_type{});
  }

#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = wr0 + e * 16 + col;
    if (r >= rows) continue;
    const float f = rebase(l[e][0], m[e]), L = l[e][0] * f;
    if (nan_v[e])
#pragma unroll
      for (int d = 0; d < 8; ++d) acc[e][d] = f32x4{NAN, NAN, NAN, NAN};
    if (u.parts == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float o[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] = acc[e][d][i] * f;
        write_row(a, u, r, (g * 16 + col) * 4 + i, L, o);
      }
    } else {
      const int64_t at = u.rec + (int64_t)u.p * a.hkv;
      if (at >= a.max_rec) continue;  // (only where offsets overlap)
      float* rec = a.part + (at * (RB / 16) + 2 * w + e) * kRecF;
#pragma unroll
      for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(rec + d * 256 + lane * 4) = acc[e][d] * f;
      if (g == 0) {
        rec[2048 + col] = m[e];
        rec[2064 + col] = L;
      }
    }
  }
}

// A call with sequences of many rows: their units, then those of its sequences
// of few (none in a call of equal prompts).  One launch instead of two: 12 us
// less for prompts, level for a mixed batch (24 tokens and two chunks of 512,
// 124 us in four launches or two; the two kinds dealt out alternately, so that
// each CU has both at a time, 128).
__global__ __launch_bounds__(256, 2) void kv4_mixed_kernel(Kv4Args many, Kv4Args few, uint32_t n_many) {
  __shared__ __attribute__((aligned(16))) union {
    PromptLds prompt;
    SplitLds split;
  } sh;
  if (blockIdx.x < n_many)
    prompt_unit(many, blockIdx.x, sh.prompt);
  else
    split_unit<2>(few, blockIdx.x - n_many, sh.split);
}

// Merges the parts of the blocks that were cut: a workgroup per (block, kv head,
// combine_sets of 16 rows), thread (g, row, i) as above, parts in order.  Its
// launch, the unit's search and the records bound it: 4 us for 28 single tokens,
// 9 for the 34 MB of two prompt chunks of 512 cut in two (with one set a
// workgroup, and so four times the searches, 13.5; with all eight 12.5).
constexpr int combine_sets(int rb) { return rb == 128 ? 4 : 1; }

template <int RB, int KS>
__device__ __forceinline__ void combine_unit(const Kv4Args& a, uint32_t unit) {
  constexpr int SETS = RB / 16, EACH = combine_sets(RB);
  const int lane = threadIdx.x & 63;
  int spp;
  Unit u;
  if (!find_unit<RB, KS, true>(a, unit / (SETS / EACH), lane, spp, u)) return;
  const int rows = u.n * a.G, row = threadIdx.x >> 2 & 15;
  // the block's own parts: its last row may see fewer keys than the sequence's
  const int steps = (last_key(a, u, min((u.b + 1) * RB, rows) - 1) + KS - 1) / KS;
  const int parts = ceil_div(max(steps, 1), spp, 1.f / (float)spp);
  if (u.rec + (int64_t)(parts - 1) * a.hkv >= a.max_rec) return;
  const int64_t next = (int64_t)a.hkv * SETS * kRecF;
#pragma unroll 1
  for (int e = unit % (SETS / EACH) * EACH, e1 = e + EACH; e < e1; ++e) {
    const int r = u.b * RB + e * 16 + row;
    if (r >= rows) return;
    const float* rec = a.part + (u.rec * SETS + e) * kRecF;
    float M = -INFINITY, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    constexpr int B = 4;  // records in flight together
    for (int p0 = 0; p0 < parts; p0 += B) {
      float pm[B], pl[B], po[B][8];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (p0 + b >= parts) break;
        const float* rp = rec + (p0 + b) * next;
        pm[b] = rp[2048 + row];
        pl[b] = rp[2064 + row];
#pragma unroll
        for (int d = 0; d < 8; ++d) po[b][d] = rp[d * 256 + threadIdx.x];
      }
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (p0 + b >= parts) break;
        const float mn = fmaxf(M, pm[b]), fa = merge_factor(M, mn), fb = merge_factor(pm[b], mn);
        L = L * fa + pl[b] * fb;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] = o[d] * fa + po[b][d] * fb;
        M = mn;
      }
    }
    write_row(a, u, r, threadIdx.x, L, o);
  }
}

template <int RB, int KS>
__global__ __launch_bounds__(256) void kv4_combine_kernel(Kv4Args a) {
  combine_unit<RB, KS>(a, blockIdx.x);
}
__global__ __launch_bounds__(256) void kv4_combine_mixed_kernel(Kv4Args many, Kv4Args few, uint32_t n_many) {
  if (blockIdx.x < n_many)
    combine_unit<kPromptRows, kPromptKeys>(many, blockIdx.x);
  else
    combine_unit<32, 32>(few, blockIdx.x - n_many);
}

// ------------------------------------------------------------- launchers ---
// Geometry of one attention call, from shapes alone: bounds that hold for
// every set of lengths (steps_per_part).
struct Kv4Launch {
  bool on;
  int rb, slots, min_spp, row_lo, row_hi;
  int64_t blocks, units, recs, bytes;
};
struct Kv4Plan {
  Kv4Launch few, many;
};
// (Times of calls replayed in a graph, 8 kv heads of 4.)  Sequences of at most
// kSplitRows rows go to the kernel for few rows: 28 with 64 rows over 4000 keys
// 60 us there, 79 in the one for many; 8 with 96 over 16000 keys 98 and 83, over
// 4000 36 and 37.  So do all sequences of a call that cannot have more than
// kFewScores scores (tokens x keys of a table x query heads), for it starts
// sooner and is cut finer: one sequence of 512 tokens over 1500 keys (2^24.6
// scores) 30 and 42 us, 128 over 4000 (2^24) 27 and 40, 64 over 16000 (2^25) 36
// and 61; but 300 over 4000 (2^25.2) 51 and 47, two of 64 over 16000 (2^26) 56
// and 57.  (The host knows the table's width, not the lengths: 300 tokens alone
// in a table of 8192 keys take 15.6 us there, 13.2 here.)
constexpr int kSplitRows = 64;
constexpr double kFewScores = 0x1p25;
constexpr int kCus = 256;  // of an MI355X
// Workgroups of a CU (registers), and steps of a part at least.  16 of 32 keys,
// four a wave: 28 single tokens over 128 to 2048 keys 16.3 us, with 8 17.8; four
// over 300 7.0 and 9.6 (a second launch).  8 of 64 keys: 300 tokens in a table of
// 8192 keys 15.6 us, with 4 20.8; behind 500 others 27 and 29.5.
constexpr int kSplit1PerCu = 4, kSplit2PerCu = 2, kPromptPerCu = 2, kSplitSteps = 16, kPromptSteps = 8;

Kv4Launch kv4_launch(int64_t nseq, int64_t T, int G, int hkv, int64_t max_keys, int64_t max_rows, int rb, int ks,
                     int per_cu, int min_spp) {
  Kv4Launch p{};
  p.on = true;
  p.rb = rb;
  p.slots = per_cu * kCus;
  p.min_spp = min_spp;
  p.row_hi = 0x7fffffff;
  p.blocks = std::min({T * ((G + rb - 1) / rb), T * G / rb + nseq, nseq * ((max_rows + rb - 1) / rb)}) * hkv;
  const int64_t most = std::max<int64_t>(1, ((max_keys + ks - 1) / ks + min_spp - 1) / min_spp);
  p.units = std::min<int64_t>(p.blocks * most, p.blocks + p.slots);
  p.recs = most > 1 ? std::min<int64_t>(p.blocks * most, 2 * p.slots) : 0;
  p.bytes = p.recs * (rb / 16) * kRecF * (int64_t)sizeof(float);
  return p;
}

Kv4Plan kv4_plan(int64_t nseq, int64_t T, bool packed, int64_t max_q_len, int hq, int hkv, int64_t max_keys) {
  Kv4Plan p{};
  const int G = hq / hkv;
  const int64_t most = std::min(max_q_len, T) * G;
  const bool few = most <= kSplitRows || (double)T * (double)max_keys * hq <= kFewScores;
  if (few || packed)  // (a packed call's hint may be too small: its rows are bounded by T alone)
    p.few = kv4_launch(nseq, T, G, hkv, max_keys, !few ? kSplitRows : packed ? T * G : most, most <= 16 ? 16 : 32, 32,
                       most <= 16 ? kSplit1PerCu : kSplit2PerCu, kSplitSteps);
  if (!few) {
    p.many = kv4_launch(nseq, T, G, hkv, max_keys, T * G, kPromptRows, kPromptKeys, kPromptPerCu, kPromptSteps);
    p.few.row_hi = p.many.row_lo = packed ? kSplitRows : 0;
  }
  return p;
}

Kv4Args kv4_part_args(Kv4Args a, const Kv4Launch& p, void* ws) {
  a.part = reinterpret_cast<float*>(ws);
  a.max_rec = p.recs;
  a.slots = p.slots;
  a.min_spp = p.min_spp;
  a.row_lo = p.row_lo;
  a.row_hi = p.row_hi;
  return a;
}
// Workgroups of the combine: cut blocks, 16 rows each.
unsigned kv4_sets(const Kv4Launch& p) {
  return p.recs ? (unsigned)(std::min<int64_t>(p.blocks, p.slots) * (p.rb / 16 / combine_sets(p.rb))) : 0;
}

int kv4_launch_attention(const Kv4Args& a, const Kv4Plan& p, void* ws, hipStream_t st) {
  const Kv4Args few = kv4_part_args(a, p.few, ws);
  const unsigned few_units = (unsigned)p.few.units, few_sets = kv4_sets(p.few);
  if (p.many.on) {
    const Kv4Args many = kv4_part_args(a, p.many, reinterpret_cast<char*>(ws) + p.few.bytes);
    const unsigned units = (unsigned)p.many.units, sets = kv4_sets(p.many);
    hipLaunchKernelGGL(kv4_mixed_kernel, dim3(units + few_units), dim3(256), 0, st, many, few, units);
    SWL_LAUNCH_CHECK("kv4_mixed_kernel launch");
    if (sets + few_sets == 0) return SWL_OK;
    hipLaunchKernelGGL(kv4_combine_mixed_kernel, dim3(sets + few_sets), dim3(256), 0, st, many, few, sets);
    SWL_LAUNCH_CHECK("kv4_combine_mixed_kernel launch");
    return SWL_OK;
  }
  if (p.few.rb == 16)
    hipLaunchKernelGGL(kv4_split_kernel<1>, dim3(few_units), dim3(64 * kSplitWaves), 0, st, few);
  else
    hipLaunchKernelGGL(kv4_split_kernel<2>, dim3(few_units), dim3(64 * kSplitWaves), 0, st, few);
  SWL_LAUNCH_CHECK("kv4_split_kernel launch");
  if (few_sets == 0) return SWL_OK;
  if (p.few.rb == 16)
    hipLaunchKernelGGL((kv4_combine_kernel<16, 32>), dim3(few_sets), dim3(256), 0, st, few);
  else
    hipLaunchKernelGGL((kv4_combine_kernel<32, 32>), dim3(few_sets), dim3(256), 0, st, few);
  SWL_LAUNCH_CHECK("kv4_combine_kernel launch");
  return SWL_OK;
}

int kv4_check_pages(const char* what, const void* pages, int64_t num_blocks, int block_size,
                    const int32_t* block_table, int64_t max_blocks, const int32_t* cache_seqlens, int nseq, int64_t T,
                    const int32_t* cu, int hkv) {
  auto bad = [&](const char* m) { return swl::fail(SWL_ERR_INVALID, std::string(what) + ": " + m); };
  if (nseq < 0 || T < 0 || T >= ((int64_t)1 << 25)) return bad("bad sequence or token count");
  if (hkv < 1 || hkv > 4096) return bad("bad head counts");
  if (block_size < 16 || block_size % 16 != 0 || block_size > (1 << 20))
    return bad("block_size must be a multiple of 16");
  if (num_blocks < 1 || num_blocks >= ((int64_t)1 << 31) || max_blocks < 1 ||
      max_blocks > ((int64_t)1 << 30) / block_size)
    return bad("bad page geometry");
  if (nseq == 0 || T == 0) return SWL_OK;
  if (!pages || !block_table || !cache_seqlens) return bad("null argument");
  if (reinterpret_cast<uintptr_t>(pages) & 15) return bad("pages must be 16-byte aligned");
  if (!cu && T % nseq != 0) return bad("without cu_seqlens every sequence has as many tokens");
  return SWL_OK;
}

Kv4Args kv4_args(void* pages, int64_t num_blocks, int block_size, const int32_t* block_table, int64_t max_blocks,
                 const int32_t* cache_seqlens, int nseq, int64_t T, const int32_t* cu, int hkv) {
  Kv4Args a{};
  a.pages = reinterpret_cast<uint8_t*>(pages);
  a.num_blocks = num_blocks;
  a.tpp = block_size / kTile;
  a.bt = block_table;
  a.by_tpp = fast_div((uint32_t)a.tpp);
  a.by_hkv = fast_div((uint32_t)hkv);
  a.max_blocks = max_blocks;
  a.kmax = (int32_t)(max_blocks * block_size);  // (at most 2^30)
  a.seqlens = cache_seqlens;
  a.nseq = nseq;
  a.T = T;
  a.cu = cu;
  a.L = (int32_t)(nseq > 0 ? T / nseq : 0);
  a.by_l = fast_div((uint32_t)std::max(a.L, 1));
  a.hkv = hkv;
  return a;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" int64_t swl_kv4_record_bytes(void) { return kRec; }

extern "C" int swl_kv4_append_bf16(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                   int64_t v_stride, void* q_out, int nseq, int64_t ntok, const int32_t* cu_seqlens,
                                   int hq, int hkv, int d, void* pages, int64_t num_blocks, int block_size,
                                   const int32_t* block_table, int64_t max_blocks, const int32_t* cache_seqlens,
                                   const int64_t* positions, const void* cos_sin, int64_t max_pos, void* stream) {
  const char* what = "swl_kv4_append_bf16";
  int rc = kv4_check_pages(what, pages, num_blocks, block_size, block_table, max_blocks, cache_seqlens, nseq, ntok,
                           cu_seqlens, hkv);
  if (rc) return rc;
  SWL_CHECK(d == kD, SWL_ERR_INVALID, "swl_kv4_append_bf16: head_dim must be 128");
  SWL_CHECK((q == nullptr) == (q_out == nullptr), SWL_ERR_INVALID, "swl_kv4_append_bf16: q and q_out go together");
  SWL_CHECK(!q || (hq > 0 && hq <= 65536), SWL_ERR_INVALID, "swl_kv4_append_bf16: bad head counts");
  SWL_CHECK((positions == nullptr) == (cos_sin == nullptr) && (!positions || max_pos > 0), SWL_ERR_INVALID,
            "swl_kv4_append_bf16: positions and cos_sin go together");
  if (nseq == 0 || ntok == 0) return SWL_OK;
  SWL_CHECK(k && v, SWL_ERR_INVALID, "swl_kv4_append_bf16: null argument");
  SWL_CHECK((!q || q_stride >= (int64_t)hq * d) && k_stride >= (int64_t)hkv * d && v_stride >= (int64_t)hkv * d,
            SWL_ERR_INVALID, "swl_kv4_append_bf16: token strides smaller than a token row");
  SWL_CHECK(q != q_out || !q || q_stride == (int64_t)hq * d, SWL_ERR_INVALID,
            "swl_kv4_append_bf16: q_out may be q only where its rows are hq * 128 apart");
  SWL_CHECK(aligned16(k) && aligned16(v) && (k_stride & 7) == 0 && (v_stride & 7) == 0 &&
                (!q || (aligned16(q) && aligned16(q_out) && (q_stride & 7) == 0)) && aligned16(cos_sin),
            SWL_ERR_INVALID, "swl_kv4_append_bf16: q, k, v rows and cos_sin must be 16-byte aligned");
  Kv4Args a = kv4_args(pages, num_blocks, block_size, block_table, max_blocks, cache_seqlens, nseq, ntok, cu_seqlens,
                       hkv);
  a.q = reinterpret_cast<const bf16*>(q);
  a.k = reinterpret_cast<const bf16*>(k);
  a.v = reinterpret_cast<const bf16*>(v);
  a.qs = q_stride;
  a.ks = k_stride;
  a.vs = v_stride;
  a.out = reinterpret_cast<bf16*>(q_out);
  a.hq = hq;
  a.pos = positions;
  a.cs = reinterpret_cast<const bf16*>(cos_sin);
  a.max_pos = max_pos;
  const int heads = (q ? hq : 0) + 2 * hkv;
  hipLaunchKernelGGL(kv4_append_kernel, dim3((unsigned)ntok, (unsigned)((heads + 15) / 16)), dim3(128), 0,
                     (hipStream_t)stream, a);
  SWL_LAUNCH_CHECK("kv4_append_kernel launch");
  return SWL_OK;
}

extern "C" int swl_kv4_read_bf16(const void* pages, int64_t num_blocks, int block_size, const int32_t* block_table,
                                 int64_t max_blocks, const int32_t* starts, int nseq, int64_t ntok,
                                 const int32_t* cu_seqlens, int hkv, int d, void* k_out, void* v_out, void* stream) {
  int rc = kv4_check_pages("swl_kv4_read_bf16", pages, num_blocks, block_size, block_table, max_blocks, starts, nseq,
                           ntok, cu_seqlens, hkv);
  if (rc) return rc;
  SWL_CHECK(d == kD, SWL_ERR_INVALID, "swl_kv4_read_bf16: head_dim must be 128");
  if (nseq == 0 || ntok == 0) return SWL_OK;
  SWL_CHECK(k_out && v_out && aligned16(k_out) && aligned16(v_out), SWL_ERR_INVALID,
            "swl_kv4_read_bf16: k_out and v_out must be 16-byte aligned");
  Kv4Args a = kv4_args(const_cast<void*>(pages), num_blocks, block_size, block_table, max_blocks, starts, nseq, ntok,
                       cu_seqlens, hkv);
  a.out = reinterpret_cast<bf16*>(k_out);
  a.out2 = reinterpret_cast<bf16*>(v_out);
  hipLaunchKernelGGL(kv4_read_kernel, dim3((unsigned)((ntok + 4 * kReadTokens - 1) / (4 * kReadTokens)), (unsigned)hkv), dim3(256), 0,
                     (hipStream_t)stream, a);
  SWL_LAUNCH_CHECK("kv4_read_kernel launch");
  return SWL_OK;
}

extern "C" int64_t swl_kv4_attention_workspace(int nseq, int64_t ntok, int packed, int64_t max_q_len, int hq, int hkv,
                                               int64_t max_keys) {
  if (nseq <= 0 || ntok <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || max_keys <= 0 || max_q_len <= 0) return 0;
  const Kv4Plan p = kv4_plan(nseq, ntok, packed != 0, max_q_len, hq, hkv, max_keys);
  return p.few.bytes + p.many.bytes;
}

extern "C" int swl_kv4_attention_bf16(const void* q, int64_t q_stride, int nseq, int64_t ntok,
                                      const int32_t* cu_seqlens, int64_t max_q_len, int hq, int hkv, int d,
                                      const void* pages, int64_t num_blocks, int block_size,
                                      const int32_t* block_table, int64_t max_blocks, const int32_t* cache_seqlens,
                                      float softmax_scale, void* out, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
  int rc = kv4_check_pages("swl_kv4_attention_bf16", pages, num_blocks, block_size, block_table, max_blocks,
                           cache_seqlens, nseq, ntok, cu_seqlens, hkv);
  if (rc) return rc;
  SWL_CHECK(d == kD, SWL_ERR_INVALID, "swl_kv4_attention_bf16: head_dim must be 128");
  SWL_CHECK(hq > 0 && hq <= 65536 && hq % hkv == 0, SWL_ERR_INVALID, "swl_kv4_attention_bf16: bad head counts");
  SWL_CHECK(softmax_scale > 0.f && std::isfinite(softmax_scale), SWL_ERR_INVALID,
            "swl_kv4_attention_bf16: softmax_scale must be positive and finite");
  SWL_CHECK(max_q_len >= 1, SWL_ERR_INVALID, "swl_kv4_attention_bf16: max_q_len must be at least 1");
  if (nseq == 0 || ntok == 0) return SWL_OK;
  SWL_CHECK(ntok * (int64_t)(hq / hkv) < ((int64_t)1 << 31), SWL_ERR_INVALID,
            "swl_kv4_attention_bf16: too many rows");
  SWL_CHECK(q && out, SWL_ERR_INVALID, "swl_kv4_attention_bf16: null argument");
  SWL_CHECK(q != out, SWL_ERR_INVALID, "swl_kv4_attention_bf16: out must not be q");
  SWL_CHECK(q_stride >= (int64_t)hq * d && (q_stride & 7) == 0 && aligned16(q) && aligned16(out), SWL_ERR_INVALID,
            "swl_kv4_attention_bf16: q and out rows must be 16-byte aligned, a token's heads together");
  Kv4Args a = kv4_args(const_cast<void*>(pages), num_blocks, block_size, block_table, max_blocks, cache_seqlens, nseq,
                       ntok, cu_seqlens, hkv);
  a.q = reinterpret_cast<const bf16*>(q);
  a.qs = q_stride;
  a.hq = hq;
  a.G = hq / hkv;
  a.by_g = fast_div((uint32_t)a.G);
  a.scale = softmax_scale;
  a.out = reinterpret_cast<bf16*>(out);
  if (!cu_seqlens) max_q_len = ntok / nseq;
  const Kv4Plan p = kv4_plan(nseq, ntok, cu_seqlens != nullptr, max_q_len, hq, hkv, max_blocks * block_size);
  SWL_CHECK(p.few.units + p.many.units < ((int64_t)1 << 24), SWL_ERR_INVALID,
            "swl_kv4_attention_bf16: too many rows");
  const int64_t need = p.few.bytes + p.many.bytes;
  SWL_CHECK(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need), SWL_ERR_INVALID,
            "swl_kv4_attention_bf16: workspace smaller than swl_kv4_attention_workspace");
  return kv4_launch_attention(a, p, workspace, (hipStream_t)stream);
}
