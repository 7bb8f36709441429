// The next token of every row of logits from given random numbers: temperature,
// top-k, top-p, min-p.
//
// With w_i = e^((x_i - max) / temperature), the tokens in the order of falling
// logits (equal ones by index), the tokens kept are a beginning of that order: the
// shortest of the first top_k; of those the fewest whose weight reaches top_p of
// theirs; those with w_i >= min_p; at least one.  The token drawn is the first
// whose cumulative weight, in the order of indexes, exceeds u of all that is kept.
//
// Weights are 64-bit exponentials rounded to whole multiples of 2^-46 (fewer bits
// for vocabularies over 2^17), so every sum is one of integers: exact, the same in
// any order, whatever atomics and slices do.  Three launches of a workgroup per
// slice of a row:
//   1. the largest logit of every slice;
//   2. counts and weights of the row's tokens by their distance from the largest,
//      in bins of a 21st of a power of two (weights under 2^-48 are 0 and in
//      none); by the workgroup that ends last of a row, which bins are kept wholly,
//      and which hold the border of one of the filters;
//   3. the former's weight by slice, the latter's tokens as a list; by the workgroup
//      that ends last of a row the borders among the listed tokens, the slice that
//      the random number falls in, and its token.
// The kernels run once through their code: its fetching is much of their time where
// rows are few, so loops are kept rolled up.
//
// Measured on an MI355X, replayed in a graph (a reading of the logits at the rate of a
// large copy, 5.2 TB/s): one row of 32000, top-p 27.8 us (0.01): three launches, 3.7 + 7.6 +
// 14.0 traced, chains of loads, LDS atomics and prefixes that wait for one another; 28
// rows of 128256 that ask for different things 43.5 (1.4): 5 + 12 + 28; 256 rows with all
// filters 109 (12.7): 18 + 49 + 47, two readings weighed in 64 bits.
//
// Flat rows are slow: where more tokens are in the borders' bins than the list holds, the
// row's last workgroup goes through the whole row for every digit of a border.  A row of
// 128256 logits, top-p 0.9: normal ones of deviation 2 at a temperature of 1 36 us, 5 49,
// 20 469; three values 709, all equal 1695 (as much for top-k, both filters twice).
// 28 such rows 52, 70, 679, 1273, 3254; 256 164, 213, 1464, 2858, 6893.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "dev_util.h"
#include "swl.h"
#include "swl_common.h"

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kChunk = 4096;    // logits of a workgroup at a time, 8 a thread
constexpr int kBins = 1024;
constexpr double kPerPower = 21;  // bins of a power of two
constexpr int kOut = kBins - 1;   // the bin of what weighs nothing
constexpr int kListed = 4096;   // tokens of a row's list (of more than that, the row itself is gone through)
constexpr int kMaxSlices = 256;
constexpr int kGather = 1024;    // tokens that a slice can list
constexpr int kShort = 128;      // of rows that keep no more than so many tokens all are listed
// Slices in all, about (a row has at most kMaxSlices): 256 rows of 128256 logits 127 us
// at 512, 108 at 1024, 119 at 2048, 154 at 4096, where every slice's bins are added to
// the row's.  Fewer rows have slices of two chunks whatever this is.
constexpr int kWorkgroups = 1024;

// What the second launch finds of a row.
struct RowPlan {
  int32_t lo, hi;      // bins under lo are kept, those over hi are not
  int32_t bk, p_lo, p_hi;  // bins of top_k's border, and of what top_p's may be in (kBins: no such filter)
  uint32_t before_k;   // tokens in bins above bk
  uint32_t key_m;      // the least logit that has min_p (0x10000: none)
  uint32_t upto_hi;    // tokens in bins up to hi
  u64 above_k;         // weight in bins above bk
  u64 above_p;         // above p_lo
  u64 all;             // of all
};

struct DrawArgs {
  const bf16* logits;   // [n, vocab], row stride ld
  int64_t ld, vocab;
  const float* u;
  const float* temp;
  const int32_t* top_k; // or null, likewise the next two
  const float* top_p;
  const float* min_p;
  int64_t* tok;
  int32_t slices, chunks;
  double unit;          // 2^46, or less for large vocabularies
  u64* top;             // [n][slices] key of the slice's largest << 32 | ~index
  u64* bin_mass;        // [n][kBins]
  uint32_t* bin_count;  // [n][kBins]
  RowPlan* plan;        // [n]
  u64* mass;            // [n][slices] weight of the slice's tokens in wholly kept bins
  u64* list;            // [n][kListed]
  uint32_t* count;      // [n][4] listed tokens; slices that are done, by launch
};

// order-preserving map of a bf16's bits to 16 bits and back, a NaN of either
// sign above all, -0 the same as +0
__device__ __forceinline__ uint32_t vkey16(uint32_t bits) {
  if ((bits & 0x7fffu) > 0x7f80u) return 0xffffu;
  if (bits == 0x8000u) return 0x8000u;
  return (bits & 0x8000u) ? (~bits & 0xffffu) : (bits | 0x8000u);
}
__device__ __forceinline__ float vkey_value(uint32_t key) {
  return __uint_as_float(((key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu)) << 16);
}
// A token's place in the order: falling logits, then rising indexes.
__device__ __forceinline__ u64 place_of(uint32_t key, int64_t i) { return (u64)(0xffffu - key) << 32 | (uint32_t)i; }
__device__ __forceinline__ uint32_t place_key(u64 p) { return 0xffffu - (uint32_t)(p >> 32); }

// Eight logits of a row from index i (a multiple of 8): bits in pairs; past the
// row -inf.
__device__ __forceinline__ u32x4 logits8(const bf16* row, int64_t i, int64_t vocab) {
  if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && i + 8 <= vocab) return ldg16(row + i);
  u32x4 q = {0u, 0u, 0u, 0u};
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll 1
  for (int e = 0; e < 8; e += 2, i += 2) {
    const uint32_t lo = i < vocab ? p[i] : 0xff80u, hi = i + 1 < vocab ? p[i + 1] : 0xff80u;
    q = u32x4{q[1], q[2], q[3], lo | hi << 16};
  }
  return q;
}
__device__ __forceinline__ uint32_t bits_at(const u32x4& q, int e) {
  return (e & 1) ? q[e >> 1] >> 16 : q[e >> 1] & 0xffffu;
}
__device__ __forceinline__ float value_of(uint32_t bits) { return __uint_as_float(bits << 16); }

// What a row's weights and bins are taken by.
struct Row {
  float mx;      // the largest logit
  float by_bin;  // bins of two units of logits
  double rate;   // 256ths of a power of two of a unit
};
__device__ __forceinline__ Row row_of(float mx, float temp) {
  Row r;
  r.mx = mx;
  r.rate = 256.0 * 1.44269504088896340735992468100 / (double)temp;
  r.by_bin = fminf((float)(r.rate * (kPerPower / 128)), 1e30f);
  return r;
}
__device__ __forceinline__ int bin_of(const Row& r, float x) {
  // (by halves: two finite logits can be more than the largest number apart)
  return (int)fminf((0.5f * r.mx - 0.5f * x) * r.by_bin, (float)kOut);  // (-inf, and the NaN of a rate of 0 times it: kOut)
}
// unit 2^(k / 256), k = 0 .. 255, a thread each: the series of 2^f for |f| <= 1/2
// (the next term is under 2e-16 of it), times 2^(1/2)
__device__ __forceinline__ double power(int k, double unit) {
  const double f = (double)(k - 128) * (0.693147180559945309417232121458 / 256);
  double p = 1.0 / 479001600.0;
  p = fma(p, f, 1.0 / 39916800.0);
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return p * (1.41421356237309504880168872421 * unit);
}
// e^((x - mx) / temperature) in units: the table's power times the series of the
// rest |f| <= 1/512 of a power of two (the next term is under 4e-17).  -inf, and
// the NaN of a rate of 0 times it, give next to nothing.
__device__ __forceinline__ double weight(const Row& r, float x, const double* tab) {
  constexpr double c = 0.693147180559945309417232121458 / 256, c2 = c * c;
  const double y = fmax(((double)x - (double)r.mx) * r.rate, -65536.0), n = rint(y), f = y - n;
  const int k = (int)n;
  double p = c2 * c2 / 24;
  p = fma(p, f, c2 * c / 6);
  p = fma(p, f, c2 / 2);
  p = fma(p, f, c);
  p = fma(p, f, 1.0);
  return ldexp(p * tab[k & 255], k >> 8);
}
// as a whole number (at most 2^46: added to 2^52 it is the sum's low bits)
__device__ __forceinline__ u64 mass_of(const Row& r, float x, const double* tab) {
  return (u64)__double_as_longlong(weight(r, x, tab) + 0x1p52) - (u64)__double_as_longlong(0x1p52);
}

// Inclusive prefix over the wave's lanes by vector instructions (row shifts, then
// the row ends passed on).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t shifted(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 shifted(u64 v) {
  return (u64)shifted<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | shifted<CTRL, ROWS>((uint32_t)v);
}
template <typename T>
__device__ __forceinline__ T wave_prefix(T v) {
  v += shifted<0x111, 0xF>(v);
  v += shifted<0x112, 0xF>(v);
  v += shifted<0x114, 0xF>(v);
  v += shifted<0x118, 0xF>(v);
  v += shifted<0x142, 0xA>(v);  // row_bcast 15
  return v + shifted<0x143, 0xC>(v);  // row_bcast 31
}
template <typename T>
__device__ __forceinline__ T lane_of(T v, int lane) {
  if constexpr (sizeof(T) == 8)
    return (T)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(v & 0xffffffffu), lane);
  else
    return (T)__builtin_amdgcn_readlane((int)v, lane);
}
// Exclusive prefix over the threads, and the sum of all.
template <typename T>
__device__ __forceinline__ T block_prefix(T v, T* sh, T& all) {
  constexpr int W = kThreads / 64;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const T inc = wave_prefix(v);
  __syncthreads();
  if (lane == 63) sh[w] = inc;
  __syncthreads();
  const T waves = wave_prefix(lane < W ? sh[lane] : (T)0);
  all = lane_of(waves, W - 1);
  return inc - v + (w > 0 ? lane_of(waves, w - 1) : (T)0);
}

// Device-scope accesses, past the caches that other XCDs do not see.
template <typename T>
__device__ __forceinline__ void put(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T get(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the last of the row's to come here.  What it and the
// others wrote (device-scope stores and atomics) is in memory, for every XCD,
// before it is counted: every wave waits for its own.
__device__ __forceinline__ bool last_of_row(const DrawArgs& a, uint32_t* counter, int& sh) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) sh = (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return sh == a.slices - 1;
}

__global__ __launch_bounds__(kThreads) void draw_max_kernel(DrawArgs a) {
  __shared__ u64 sh[kThreads / 64];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, base = (int64_t)blockIdx.x * a.chunks * kChunk;
  const bf16* x = a.logits + row * a.ld;
  for (int b = blockIdx.x * kThreads + tid; b < kBins; b += a.slices * kThreads) {
    a.bin_mass[row * kBins + b] = 0;
    a.bin_count[row * kBins + b] = 0;
  }
  if (blockIdx.x == 0 && tid < 4) a.count[4 * row + tid] = 0;
  u64 best = 0;  // key << 32 | ~index
#pragma unroll 2
  for (int c = 0; c < a.chunks; ++c) {
    const int64_t from = base + (int64_t)c * kChunk + tid * 8;
    if (from >= a.vocab) break;
    const u32x4 q = logits8(x, from, a.vocab);
    uint32_t top = 0;  // key, then the thread's logits counted down
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (from + e < a.vocab) top = max(top, vkey16(bits_at(q, e)) << 3 | (uint32_t)(7 - e));
    best = max(best, (u64)(top >> 3) << 32 | (uint32_t)~(uint32_t)(from + 7 - (top & 7)));
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) best = max(best, (u64)__shfl_xor((long long)best, o, 64));
  if ((tid & 63) == 0) sh[tid >> 6] = best;
  __syncthreads();
  if (tid < 64) {
    best = tid < kThreads / 64 ? sh[tid] : 0;
#pragma unroll
    for (int o = kThreads / 128; o >= 1; o >>= 1) best = max(best, (u64)__shfl_xor((long long)best, o, 64));
    if (tid == 0) a.top[row * a.slices + blockIdx.x] = best;
  }
}

// The row's largest logit (key << 32 | ~index), by every wave for itself.
__device__ __forceinline__ u64 row_top(const DrawArgs& a, int64_t row) {
  u64 best = 0;
  for (int i = threadIdx.x & 63; i < a.slices; i += 64) best = max(best, a.top[row * a.slices + i]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) best = max(best, (u64)__shfl_xor((long long)best, o, 64));
  return best;
}
// Rows whose token is their largest logit: no temperature, or weights that are no
// numbers (a NaN, an infinity as the largest).
__device__ __forceinline__ bool row_greedy(uint32_t key, float temp) { return !(temp > 0.f) || key > 0xff7fu || key <= 0x007fu; }

struct Asked {
  bool k, p, m;
  int32_t top_k;
  double top_p, min_p;
};
__device__ __forceinline__ Asked asked_of(const DrawArgs& a, int64_t row) {
  Asked q;
  q.top_k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.f, m = a.min_p ? a.min_p[row] : 0.f;
  q.k = q.top_k > 0 && q.top_k < a.vocab;
  q.p = p < 1.f;
  q.m = m > 0.f;
  q.top_p = (double)p;
  q.min_p = (double)m;
  return q;
}

struct PlanLds {
  u64 sh64[kThreads / 64];
  uint32_t sh32[kThreads / 64];
  RowPlan plan;
  u64 bin_k;
  int key_m, last;
};

__global__ __launch_bounds__(kThreads) void draw_bins_kernel(DrawArgs a) {
  __shared__ u64 mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ double tab[256];
  __shared__ PlanLds l;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, base = (int64_t)blockIdx.x * a.chunks * kChunk;
  const Asked ask = asked_of(a, row);
  const float temp = a.temp[row];
  if (!ask.k && !ask.p && !ask.m) return;
  const bf16* x = a.logits + row * a.ld;
  const u64 top = row_top(a, row);
  const uint32_t top_key = (uint32_t)(top >> 32);
  if (row_greedy(top_key, temp)) return;
  const Row r = row_of(vkey_value(top_key), temp);
  if (tid < 256) tab[tid] = power(tid, a.unit);
  constexpr int E = kBins / kThreads;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    mass[e * kThreads + tid] = 0;
    count[e * kThreads + tid] = 0;
  }
  __syncthreads();
#pragma unroll 1
  for (int c = 0; c < a.chunks; ++c) {
    const int64_t from = base + (int64_t)c * kChunk + tid * 8;
    if (from >= a.vocab) break;
    const u32x4 q = logits8(x, from, a.vocab);
    int b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      b[e] = bin_of(r, value_of(bits_at(q, e)));
      if (b[e] < kOut) atomicAdd(&count[b[e]], 1u);
    }
    if (ask.p) {
      u64 w[8];  // (all of them before the branches: eight chains of 64-bit arithmetic side by side)
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = mass_of(r, value_of(bits_at(q, e)), tab);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (b[e] < kOut) atomicAdd(&mass[b[e]], w[e]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int b = e * kThreads + tid;
    if (b < kOut && count[b]) {
      atomicAdd(&a.bin_count[row * kBins + b], count[b]);
      if (ask.p) atomicAdd(&a.bin_mass[row * kBins + b], mass[b]);
    }
  }
  if (!last_of_row(a, &a.count[4 * row + 1], l.last)) return;

  // bins of the borders: two bins a thread, counts and weights above them
  static_assert(E == 2, "");
  if (tid == 0) {
    l.plan.bk = l.plan.p_lo = l.plan.p_hi = kBins;
    l.key_m = -1;
  }
  uint32_t n[E], nb[E], n_all;
  u64 m[E] = {0, 0}, mb[E] = {0, 0}, m_all = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    n[e] = get(&a.bin_count[row * kBins + E * tid + e]);
    if (ask.p) m[e] = get(&a.bin_mass[row * kBins + E * tid + e]);
  }
  nb[0] = block_prefix(n[0] + n[1], l.sh32, n_all);
  nb[1] = nb[0] + n[0];
  if (ask.p) mb[0] = block_prefix(m[0] + m[1], l.sh64, m_all);
  mb[1] = mb[0] + m[0];
  bool by_k = ask.k;
  if (ask.k) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (nb[e] < (uint32_t)ask.top_k && nb[e] + n[e] >= (uint32_t)ask.top_k) {
        l.plan.bk = E * tid + e;
        l.plan.above_k = mb[e];
        l.plan.before_k = nb[e];
        l.bin_k = m[e];
      }
    __syncthreads();
    by_k = l.plan.bk < kBins;  // (else all that weighs anything is among the first top_k)
  }
  if (ask.p) {  // the first bins whose weight and that above reaches top_p of what may be left by top_k
    const double lo = ask.top_p * (double)(by_k ? l.plan.above_k : m_all);
    const double hi = ask.top_p * (double)(by_k ? l.plan.above_k + l.bin_k : m_all);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (n[e] && (double)(mb[e] + m[e]) >= lo && ((double)mb[e] < lo || nb[e] == 0)) {
        l.plan.p_lo = E * tid + e;
        l.plan.above_p = mb[e];
      }
      if (n[e] && (double)(mb[e] + m[e]) >= hi && ((double)mb[e] < hi || nb[e] == 0)) l.plan.p_hi = E * tid + e;
    }
  }
  if (tid == 0) l.plan.all = m_all;
  __syncthreads();
  // the least logit of weight min_p: 128 keys apart, then each
  int bm = kBins;
  uint32_t key_m = 0;
  if (ask.m) {
    const double least = ask.min_p * a.unit;
    int step = 65536 / kThreads, from = (int)top_key;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      const int key = from - step * tid;
      if (key > 0x007f && weight(r, vkey_value((uint32_t)key), tab) >= least) atomicMax(&l.key_m, tid);
      __syncthreads();
      const int far = l.key_m;
      __syncthreads();
      if (far < 0) break;  // (over 1: none but the first token)
      if (tid == 0) l.key_m = -1;
      __syncthreads();
      from -= step * far;
      step = 1;
    }
    const bool met = step == 1;
    key_m = met ? (uint32_t)from : 0x10000u;
    bm = met ? bin_of(r, vkey_value(key_m)) : 0;
  }
  const int hi = min(min(l.plan.bk, l.plan.p_hi), bm);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (E * tid + e == min(hi, kOut)) l.plan.upto_hi = nb[e] + n[e];
  __syncthreads();
  if (tid == 0) {
    RowPlan o = l.plan;
    o.key_m = key_m;
    // (few tokens are all listed)
    o.lo = o.upto_hi <= kShort ? 0 : min(min(o.bk, o.p_lo), bm);
    o.hi = hi;
    a.plan[row] = o;
  }
}

// The token is the first with a cumulative weight above this: a whole number above
// floor(u all) is above u all, and the other way round.  (A u outside [0, 1) draws
// the first or the last that weighs anything.)
__device__ __forceinline__ u64 draw_goal(float u, u64 all) {
  const double want = (double)u * (double)all;
  return want > 0.0 ? (want < (double)all ? min((u64)want, all - 1) : all - 1) : 0;
}

struct Pair {
  u64 place, mass;  // (of a listed token; its bin in the mass's upper 16 bits)
};
__device__ __forceinline__ u64 other_lane(u64 v) {  // of a pair: quad_perm [1, 0, 3, 2]
  return (u64)(uint32_t)__builtin_amdgcn_mov_dpp((int)(v >> 32), 0xB1, 0xF, 0xF, false) << 32 |
         (uint32_t)__builtin_amdgcn_mov_dpp((int)(v & 0xffffffffu), 0xB1, 0xF, 0xF, false);
}

struct DrawLds {
  double tab[256];
  u64 sh64[kThreads / 64];
  uint32_t sh32[kThreads / 64];
  int last, at;
  u64 border, kept_k, goal;
  Pair pair[kThreads / 2];  // the list, where it is short
  u64 mass[256], most[256]; // digits of places
  uint32_t bin[256];
  int digit;
  u64 slice[kMaxSlices];
  u64 gather[kGather];
  uint32_t gathered;
};

// f(place) for the row's tokens whose bins are in question: the list, or where it
// is too short the row.
template <typename F>
__device__ __forceinline__ void for_listed(const DrawArgs& a, int64_t row, uint32_t listed, F f) {
  const bool whole = listed > kListed;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(a.logits + row * a.ld);
  const int64_t end = whole ? a.vocab : listed;
#pragma unroll 1
  for (int64_t i = threadIdx.x; i < end; i += kThreads) f(whole ? place_of(vkey16(x[i]), i) : get(&a.list[row * kListed + i]));
}

// The place of the goal-th token of bin b (by_mass: of the first whose cumulative
// weight reaches the goal), and the weight of the bin's tokens up to it: by digits
// of the place, eight bits at a time, the logit's first; a digit that one token
// has, or whose tokens are all wanted, ends it.  Tokens of one logit weigh the
// same: then weights are counts.  For lists over 256.
__device__ __forceinline__ u64 select_place(const DrawArgs& a, int64_t row, const Row& r, uint32_t listed, int b, bool by_mass,
                                         uint32_t goal, double goal_mass, DrawLds& l, u64& up_to) {
  u64 prefix = 0;
  up_to = 0;
  const int tid = threadIdx.x;
#pragma unroll 1
  for (int shift = 40;; shift -= 8) {
    __syncthreads();
    if (tid < 256) {
      l.mass[tid] = l.most[tid] = 0;
      l.bin[tid] = 0;
    }
    if (tid == 0) l.digit = -1;
    __syncthreads();
    for_listed(a, row, listed, [&](u64 p) {
      if (p >> (shift + 8) != prefix) return;
      const float v = vkey_value(place_key(p));
      if (bin_of(r, v) != b) return;
      const int d = (int)(p >> shift) & 255;
      atomicAdd(&l.bin[d], 1u);
      atomicAdd(&l.mass[d], mass_of(r, v, l.tab));
      atomicMax(&l.most[d], p);
    });
    __syncthreads();
    const uint32_t n = tid < 256 ? l.bin[tid] : 0;
    const u64 m = tid < 256 ? l.mass[tid] : 0;
    uint32_t n_all;
    u64 m_all;
    const uint32_t nb = block_prefix(n, l.sh32, n_all);
    const u64 mb = block_prefix(m, l.sh64, m_all);
    // the digit that holds the border (where a rounding has put the goal above
    // all, the last one)
    if (n > 0 && (by_mass ? ((double)(mb + m) >= goal_mass || nb + n == n_all) && (nb == 0 || (double)mb < goal_mass)
                          : nb < goal && nb + n >= min(goal, n_all)))
      atomicMax(&l.digit, tid);
    __syncthreads();
    const int d = l.digit;
    if (d < 0) return prefix << (shift + 8);  // (an empty bin: not reached)
    const uint32_t dn = l.bin[d];
    const u64 dm = l.mass[d];
    __syncthreads();
    if (tid == d) {
      l.goal = mb;
      l.sh32[0] = nb;
    }
    __syncthreads();
    const u64 before = l.goal;
    const uint32_t n_before = l.sh32[0];
    prefix = prefix << 8 | (u64)d;
    up_to += before;
    if (by_mass) {
      goal_mass -= (double)before;
      if (shift == 32) {  // one logit left: so many of it
        by_mass = false;
        const u64 each = dm / dn;
        const double want = each ? ceil(goal_mass / (double)each) : 1.0;
        goal = (uint32_t)fmin(fmax(want, 1.0), (double)dn);
      }
    } else {
      goal -= n_before;
    }
    if (dn == 1 || (!by_mass && goal >= dn) || shift == 0) {
      up_to += dm;
      return l.most[d];
    }
  }
}

__global__ __launch_bounds__(kThreads) void draw_token_kernel(DrawArgs a) {
  __shared__ DrawLds l;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, base = (int64_t)blockIdx.x * a.chunks * kChunk;
  const bf16* x = a.logits + row * a.ld;
  const Asked ask = asked_of(a, row);
  const float temp = a.temp[row];
  const u64 top = row_top(a, row);
  const uint32_t top_key = (uint32_t)(top >> 32);
  const int64_t first = (int64_t)(uint32_t)~(uint32_t)top;
  if (row_greedy(top_key, temp)) {
    if (blockIdx.x == 0 && tid == 0) a.tok[row] = first;
    return;
  }
  const Row r = row_of(vkey_value(top_key), temp);
  const bool some = ask.k || ask.p || ask.m;
  RowPlan plan;
  plan.lo = plan.hi = plan.bk = kBins;
  if (some) plan = a.plan[row];
  if (tid < 256) l.tab[tid] = power(tid, a.unit);
  if (tid == 0) l.gathered = 0;
  __syncthreads();

  u64 own = 0;
#pragma unroll 1
  for (int c = 0; c < a.chunks; ++c) {
    const int64_t start = base + (int64_t)c * kChunk, from = start + tid * 8;
    if (start >= a.vocab) break;
    const u32x4 q = logits8(x, from, a.vocab);
    uint32_t mask = 0, in = 0;  // of the thread's 8 tokens, the listed ones and those of bins that are kept wholly
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int b = bin_of(r, value_of(bits_at(q, e)));
      in |= (uint32_t)(b < plan.lo && b < kOut) << e;
      mask |= (uint32_t)(b >= plan.lo && b < kOut && (b <= plan.hi || b == plan.bk)) << e;
    }
    if (__ballot(in != 0) != 0) {
      u64 w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = mass_of(r, value_of(bits_at(q, e)), l.tab);
#pragma unroll
      for (int e = 0; e < 8; ++e) own += in >> e & 1u ? w[e] : 0;
    }
    if (mask) {
      uint32_t at = atomicAdd(&l.gathered, (uint32_t)__popc(mask));
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (mask >> e & 1u) {
          if (at < kGather) l.gather[at] = place_of(vkey16(bits_at(q, e)), from + e);
          ++at;
        }
    }
  }
  u64 all;
  block_prefix(own, l.sh64, all);
  if (tid == 0) put(&a.mass[row * a.slices + blockIdx.x], all);
  const uint32_t gathered = l.gathered;
  if (gathered) {  // (more than there is room for: the row itself will be gone through)
    if (tid == 0) l.at = (int)atomicAdd(&a.count[4 * row], gathered > kGather ? kListed + 1 : gathered);
    __syncthreads();
    const uint32_t at = (uint32_t)l.at;
    for (uint32_t i = tid; i < min(gathered, (uint32_t)kGather); i += kThreads)
      if (at + i < kListed) put(&a.list[row * kListed + at + i], l.gather[i]);
  }
  if (!last_of_row(a, &a.count[4 * row + 2], l.last)) return;

  // The row's last workgroup.  First the borders' places: a token of a short list
  // has two lanes, which take every other one of its pairs.
  const uint32_t listed = some ? get(&a.count[4 * row]) : 0;
  u64 place = get(&a.list[row * kListed + (tid >> 1)]);  // (before it is known to be one)
  if (tid < kMaxSlices) l.slice[tid] = tid < a.slices ? get(&a.mass[row * a.slices + tid]) : 0;
  const bool by_k = plan.bk < kBins;
  u64 border = ~(u64)0;
  if (some) {
    const bool small = listed <= kThreads / 2, there = (uint32_t)(tid >> 1) < listed;
    u64 mass = 0, mass_in = 0;  // the thread's token, the bin's before it
    uint32_t bin = kBins, count_in = 0;
    if (small) {
      if (there) {
        const float v = vkey_value(place_key(place));
        bin = (uint32_t)bin_of(r, v);
        mass = mass_of(r, v, l.tab);
      } else {
        place = ~(u64)0;
      }
      if ((tid & 1) == 0) l.pair[tid >> 1] = Pair{place, mass | (u64)bin << 48};
      __syncthreads();
      if ((ask.k || ask.p) && there) {
#pragma unroll 4
        for (int i = tid & 1; i < (int)listed; i += 2) {
          const Pair o = l.pair[i];
          const bool before = (uint32_t)(o.mass >> 48) == bin && o.place < place;
          mass_in += before ? o.mass & 0xffffffffffffull : 0;
          count_in += before ? 1 : 0;
        }
        mass_in += other_lane(mass_in);
        count_in += (uint32_t)__builtin_amdgcn_mov_dpp((int)count_in, 0xB1, 0xF, 0xF, false);
      }
    }
    u64 kept = plan.all;
    if (by_k) {
      u64 up_to = 0;
      const uint32_t goal = (uint32_t)ask.top_k - plan.before_k;
      if (small) {
        if (bin == (uint32_t)plan.bk && count_in + 1 == goal) {
          l.border = place;
          l.kept_k = mass_in + mass;
        }
        __syncthreads();
        border = l.border;
        up_to = l.kept_k;
      } else {
        border = select_place(a, row, r, listed, plan.bk, false, goal, 0.0, l, up_to);
      }
      kept = plan.above_k + up_to;
    }
    if (ask.p) {
      // the border's bin, one of p_lo .. p_hi: the first whose weight and that above reaches the goal
      const double goal = ask.top_p * (double)kept;
      u64 above = plan.above_p;
      int bp = plan.p_lo;
#pragma unroll 1
      for (; bp < plan.p_hi; ++bp) {
        const u64 m = a.bin_mass[row * kBins + bp];
        if (a.bin_count[row * kBins + bp] && (double)(above + m) >= goal) break;
        above += m;
      }
      if (bp <= plan.hi) {
        u64 up_to = 0, at;
        const double rest = goal - (double)above;
        if (small) {
          __syncthreads();
          if (tid == 0) l.border = ~(u64)0;
          __syncthreads();
          // (the first to reach it; by roundings none, then the bin's last: the largest place of all is no border)
          if (bin == (uint32_t)bp && (double)(mass_in + mass) >= rest) atomicMin(&l.border, place);
          __syncthreads();
          at = l.border;
          if (at == ~(u64)0) {
            __syncthreads();
            if (tid == 0) l.border = 0;
            __syncthreads();
            if (bin == (uint32_t)bp) atomicMax(&l.border, place);
            __syncthreads();
            at = l.border;
          }
        } else {
          at = select_place(a, row, r, listed, bp, true, 0, rest, l, up_to);
        }
        border = min(border, at);
      }
    }
    if (ask.m) border = min(border, plan.key_m > 0xffffu ? 0 : place_of(plan.key_m, 0xffffffffll));
    border = max(border, place_of(top_key, first));  // at least one
    if (small && plan.lo == 0) {
      // all that is kept is in the list: cumulative weights in the order of indexes
      // by all pairs
      __syncthreads();
      const uint32_t index = (uint32_t)place;
      const bool kept = place <= border && there;
      if (there && !kept) l.pair[tid >> 1].mass = 0;
      __syncthreads();
      if (!there) return;
      u64 before = 0, all = 0;
#pragma unroll 4
      for (int i = tid & 1; i < (int)listed; i += 2) {
        const Pair o = l.pair[i];
        const u64 m = o.mass & 0xffffffffffffull;
        all += m;
        before += (uint32_t)o.place < index ? m : 0;
      }
      all += other_lane(all);
      before += other_lane(before);
      const u64 goal = draw_goal(a.u[row], all);
      if (kept && mass > 0 && before <= goal && goal < before + mass) a.tok[row] = index;
      return;
    }
    // weights of the slices: what is kept wholly, and the listed tokens up to the border
    __syncthreads();
    const int64_t each = (int64_t)a.chunks * kChunk;
    if (small) {
      if ((tid & 1) == 0 && place <= border && bin >= (uint32_t)plan.lo && bin < (uint32_t)kOut)
        atomicAdd(&l.slice[(int64_t)(uint32_t)place / each], mass);
    } else {
      for_listed(a, row, listed, [&](u64 p) {
        if (p > border) return;
        const float v = vkey_value(place_key(p));
        const int b = bin_of(r, v);
        if (b >= plan.lo && b < kOut) atomicAdd(&l.slice[(int64_t)(uint32_t)p / each], mass_of(r, v, l.tab));
      });
    }
  }
  __syncthreads();
  const u64 mine = tid < kMaxSlices ? l.slice[tid] : 0;
  const u64 before = block_prefix(mine, l.sh64, all);
  const u64 goal = draw_goal(a.u[row], all);
  if (mine > 0 && before <= goal && goal < before + mine) {
    l.at = tid;
    l.goal = goal - before;
  }
  __syncthreads();
  u64 left = l.goal;
  const int64_t begin = (int64_t)l.at * a.chunks * kChunk;
  auto keeps = [&](uint32_t bits, int64_t i) {
    return i < a.vocab && place_of(vkey16(bits), i) <= border && bin_of(r, value_of(bits)) < kOut;
  };
#pragma unroll 1
  for (int c = 0; c < a.chunks; ++c) {
    // 8 logits a thread in a row: the thread that the goal falls to, then its token
    const int64_t from = begin + (int64_t)c * kChunk;
    const u32x4 q = logits8(x, from + tid * 8, a.vocab);
    uint32_t in = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) in |= (uint32_t)keeps(bits_at(q, e), from + tid * 8 + e) << e;
    u64 m = 0, sum;
    if (__ballot(in != 0) != 0) {
      u64 w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = mass_of(r, value_of(bits_at(q, e)), l.tab);
#pragma unroll
      for (int e = 0; e < 8; ++e) m += in >> e & 1u ? w[e] : 0;
    }
    const u64 bef = block_prefix(m, l.sh64, sum);
    if (left >= sum) {
      left -= sum;
      continue;
    }
    if (bef <= left && left < bef + m) {
      l.at = tid;
      l.goal = left - bef;
    }
    __syncthreads();
    if (tid < 64) {
      const int64_t i = from + l.at * 8 + tid;
      const uint32_t bits = tid < 8 && i < a.vocab ? reinterpret_cast<const uint16_t*>(x)[i] : 0xff80u;
      const u64 w = tid < 8 && keeps(bits, i) ? mass_of(r, value_of(bits), l.tab) : 0, inc = wave_prefix(w);
      if (w > 0 && inc - w <= l.goal && l.goal < inc) a.tok[row] = i;
    }
    return;
  }
}

struct DrawLayout {
  int64_t chunks, slices, bin_mass, bin_count, mass, list, plan, count, bytes;
};
DrawLayout draw_layout(int64_t n, int64_t vocab) {
  DrawLayout l;
  const int64_t pieces = (vocab + kChunk - 1) / kChunk;
  // about kWorkgroups slices in all
  l.chunks = std::min(pieces, std::max<int64_t>({2, (n * pieces + kWorkgroups - 1) / kWorkgroups, (pieces + kMaxSlices - 1) / kMaxSlices}));
  l.slices = (pieces + l.chunks - 1) / l.chunks;
  l.bin_mass = n * l.slices * (int64_t)sizeof(u64);
  l.mass = l.bin_mass + n * kBins * (int64_t)sizeof(u64);
  l.list = l.mass + n * l.slices * (int64_t)sizeof(u64);
  l.plan = l.list + n * kListed * (int64_t)sizeof(u64);
  l.bin_count = l.plan + n * (int64_t)sizeof(RowPlan);
  l.count = l.bin_count + n * kBins * (int64_t)sizeof(uint32_t);
  l.bytes = l.count + n * 4 * (int64_t)sizeof(uint32_t);
  return l;
}

}  // namespace

extern "C" int64_t swl_sample_tokens_workspace(int64_t n, int64_t vocab) {
  if (n <= 0 || vocab <= 0) return 0;
  return draw_layout(n, vocab).bytes;
}

extern "C" int swl_sample_tokens_bf16(const void* logits, int64_t ld, int64_t n, int64_t vocab, const float* u,
                                      const float* temperature, const int32_t* top_k, const float* top_p,
                                      const float* min_p, int64_t* out_tokens, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
  SWL_CHECK(n >= 0 && n <= 65535, SWL_ERR_INVALID, "swl_sample_tokens_bf16: at most 65535 rows");
  SWL_CHECK(vocab > 0 && vocab <= (int64_t)1 << 21, SWL_ERR_INVALID,
            "swl_sample_tokens_bf16: the vocabulary must be 1 to 2097152");
  if (n == 0) return SWL_OK;
  SWL_CHECK(logits && u && temperature && out_tokens, SWL_ERR_INVALID, "swl_sample_tokens_bf16: null argument");
  SWL_CHECK(ld >= vocab, SWL_ERR_INVALID, "swl_sample_tokens_bf16: row stride smaller than the vocabulary");
  const DrawLayout l = draw_layout(n, vocab);
  SWL_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= l.bytes, SWL_ERR_INVALID,
            "swl_sample_tokens_bf16: workspace smaller than swl_sample_tokens_workspace");
  DrawArgs a{};
  a.logits = reinterpret_cast<const bf16*>(logits);
  a.ld = ld;
  a.vocab = vocab;
  a.u = u;
  a.temp = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.tok = out_tokens;
  a.slices = (int32_t)l.slices;
  a.chunks = (int32_t)l.chunks;
  int bits = 0;  // vocab <= 2^bits
  while (((int64_t)1 << bits) < vocab) ++bits;
  a.unit = (double)((int64_t)1 << std::min(46, 63 - bits));
  char* ws = reinterpret_cast<char*>(workspace);
  a.top = reinterpret_cast<u64*>(ws);
  a.bin_mass = reinterpret_cast<u64*>(ws + l.bin_mass);
  a.mass = reinterpret_cast<u64*>(ws + l.mass);
  a.plan = reinterpret_cast<RowPlan*>(ws + l.plan);
  a.list = reinterpret_cast<u64*>(ws + l.list);
  a.bin_count = reinterpret_cast<uint32_t*>(ws + l.bin_count);
  a.count = reinterpret_cast<uint32_t*>(ws + l.count);
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)l.slices, (unsigned)n);
  hipLaunchKernelGGL(draw_max_kernel, grid, dim3(kThreads), 0, st, a);
  SWL_LAUNCH_CHECK("draw_max_kernel launch");
  if (top_k || top_p || min_p) {
    hipLaunchKernelGGL(draw_bins_kernel, grid, dim3(kThreads), 0, st, a);
    SWL_LAUNCH_CHECK("draw_bins_kernel launch");
  }
  hipLaunchKernelGGL(draw_token_kernel, grid, dim3(kThreads), 0, st, a);
  SWL_LAUNCH_CHECK("draw_token_kernel launch");
  return SWL_OK;
}
