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
// any order, whatever atomics and slices do.  Three launches:
//   1. the largest logit of every slice of a row;
//   2. counts and weights of the row's tokens by their distance from the largest,
//      in bins of a 16th of a power of two (1024 of them; weights under 2^-63.9
//      are 0 and in none);
//   3. from the bins, which of them are kept wholly, and which hold the border of
//      one of the filters; the former's weight by slice, the latter's tokens as a
//      list; by the workgroup that ends last of a row the borders among the listed
//      tokens, the slice that the random number falls in, and its token.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "dev_util.h"
#include "swl.h"
#include "swl_common.h"

namespace {

typedef unsigned long long u64;

constexpr int kSlice = 8192;    // logits of a workgroup, 32 a thread
constexpr int kBins = 1024;
constexpr int kOut = kBins - 1; // the bin of what weighs nothing
constexpr int kListed = 4096;   // tokens of a row's list (of more than that, the row itself is gone through)
constexpr int kMaxSlices = 256;
constexpr u64 kAll = ~(u64)0;

struct DrawArgs {
  const bf16* logits;   // [n, vocab], row stride ld
  int64_t ld, vocab;
  const float* u;
  const float* temp;
  const int32_t* top_k; // or null, likewise the next two
  const float* top_p;
  const float* min_p;
  int64_t* tok;
  int32_t slices;
  double unit;          // 2^46, or less for large vocabularies
  u64* top;             // [n][slices] key of the slice's largest << 32 | ~index
  u64* bin_mass;        // [n][kBins]
  uint32_t* bin_count;  // [n][kBins]
  u64* mass;            // [n][slices] weight of the slice's tokens in wholly kept bins
  u64* list;            // [n][kListed]
  uint32_t* count;      // [n][2] listed tokens, slices that are done
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
__device__ __forceinline__ u32x4 logits8(const bf16* row, int64_t i, int64_t vocab, bool vec) {
  if (vec && i + 8 <= vocab) return ldg16(row + i);
  u32x4 q;
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = i + 2 * e < vocab ? p[i + 2 * e] : 0xff80u;
    const uint32_t hi = i + 2 * e + 1 < vocab ? p[i + 2 * e + 1] : 0xff80u;
    q[e] = lo | hi << 16;
  }
  return q;
}
__device__ __forceinline__ uint32_t bits_at(const u32x4& q, int e) {
  return (e & 1) ? q[e >> 1] >> 16 : q[e >> 1] & 0xffffu;
}
__device__ __forceinline__ bool row_vec(const bf16* row) { return (reinterpret_cast<uintptr_t>(row) & 15) == 0; }

// What a row's weights and bins are taken by.
struct Row {
  float mx;      // the largest logit
  float by_bin;  // bins of a unit of logits
  double rate;   // powers of two of a unit
  double unit;
};
__device__ __forceinline__ Row row_of(float mx, float temp, double unit) {
  Row r;
  r.mx = mx;
  r.rate = 1.44269504088896340735992468100 / (double)temp;
  r.by_bin = fminf((float)(16.0 * r.rate), 1e30f);
  r.unit = unit;
  return r;
}
__device__ __forceinline__ int bin_of(const Row& r, float x) {
  return (int)fminf((r.mx - x) * r.by_bin, (float)kOut);  // (-inf, and the NaN of a rate of 0 times it: kOut)
}
// 2^y for y <= 0 in 64 bits: the series of 2^f for |f| <= 1/2 (the next term is
// under 2e-16 of it)
__device__ __forceinline__ double power(double y) {
  y = fmax(y, -2000.0);
  const double n = rint(y), f = (y - n) * 0.693147180559945309417232121458;
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
  return ldexp(p, (int)n);
}
__device__ __forceinline__ double weight(const Row& r, float x) {
  return x == -INFINITY ? 0.0 : power(((double)x - (double)r.mx) * r.rate);
}
// as a whole number of 1 / unit (at most 2^46: added to 2^52 it is the sum's low bits)
__device__ __forceinline__ u64 mass_of(const Row& r, float x) {
  return (u64)__double_as_longlong(weight(r, x) * r.unit + 0x1p52) - (u64)__double_as_longlong(0x1p52);
}

template <typename T>
__device__ __forceinline__ T wave_add(T v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <typename T>
__device__ __forceinline__ T block_add(T v, T* sh) {
  v = wave_add(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
// Exclusive prefix over the 256 threads.
template <typename T>
__device__ __forceinline__ T block_prefix(T v, T* sh) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  T inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(inc, o, 64);
    if (lane >= o) inc += y;
  }
  __syncthreads();
  if (lane == 63) sh[w] = inc;
  __syncthreads();
  T before = 0;
  for (int i = 0; i < w; ++i) before += sh[i];
  return before + inc - v;
}

__global__ __launch_bounds__(256) void draw_max_kernel(DrawArgs a) {
  __shared__ uint32_t sh[4];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, base = (int64_t)blockIdx.x * kSlice;
  const bf16* x = a.logits + row * a.ld;
  const bool vec = row_vec(x);
  u32x4 q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = logits8(x, base + (j * 256 + tid) * 8, a.vocab, vec);
  for (int b = blockIdx.x * 256 + tid; b < kBins; b += a.slices * 256) {
    a.bin_mass[row * kBins + b] = 0;
    a.bin_count[row * kBins + b] = 0;
  }
  if (blockIdx.x == 0 && tid < 2) a.count[2 * row + tid] = 0;
  uint32_t best = 0;  // key, then the index counted down
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = (j * 256 + tid) * 8 + e;
      if (base + at < a.vocab) best = max(best, vkey16(bits_at(q[j], e)) << 13 | (uint32_t)(kSlice - 1 - at));
    }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, o, 64));
  if ((tid & 63) == 0) sh[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    best = max(max(sh[0], sh[1]), max(sh[2], sh[3]));
    const uint32_t i = (uint32_t)base + kSlice - 1 - (best & (kSlice - 1));
    a.top[row * a.slices + blockIdx.x] = (u64)(best >> 13) << 32 | (uint32_t)~i;
  }
}

// The row's largest logit (key << 32 | ~index), by every wave for itself.
__device__ __forceinline__ u64 row_top(const DrawArgs& a, int64_t row) {
  const int lane = threadIdx.x & 63;
  u64 best = 0;
  for (int i = lane; i < a.slices; i += 64) best = max(best, a.top[row * a.slices + i]);
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

__global__ __launch_bounds__(256) void draw_bins_kernel(DrawArgs a) {
  __shared__ u64 mass[kBins];
  __shared__ uint32_t count[kBins];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, base = (int64_t)blockIdx.x * kSlice;
  const Asked ask = asked_of(a, row);
  if (!ask.k && !ask.p) return;
  const bf16* x = a.logits + row * a.ld;
  const bool vec = row_vec(x);
  u32x4 q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = logits8(x, base + (j * 256 + tid) * 8, a.vocab, vec);
  const float temp = a.temp[row];
  const u64 top = row_top(a, row);
  const uint32_t key = (uint32_t)(top >> 32);
  if (row_greedy(key, temp)) return;
  const Row r = row_of(vkey_value(key), temp, a.unit);
  for (int b = tid; b < kBins; b += 256) {
    mass[b] = 0;
    count[b] = 0;
  }
  __syncthreads();
#pragma unroll 1
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __uint_as_float(bits_at(q[0], e) << 16);
      const int b = bin_of(r, v);
      if (b < kOut) {
        atomicAdd(&count[b], 1u);
        if (ask.p) atomicAdd(&mass[b], mass_of(r, v));
      }
    }
    q[0] = q[1];
    q[1] = q[2];
    q[2] = q[3];
  }
  __syncthreads();
  for (int b = tid; b < kOut; b += 256)
    if (count[b]) {
      atomicAdd(&a.bin_count[row * kBins + b], count[b]);
      if (ask.p) atomicAdd(&a.bin_mass[row * kBins + b], mass[b]);
    }
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

struct DrawLds {
  u64 sh64[4];
  uint32_t sh32[4];
  int bk, p_lo, p_hi, bp;  // bins of the borders
  u64 above_k, bin_k, above_p;
  uint32_t before_k;
  int key_m;
  int last;
  // select
  u64 mass[256], most[256];
  uint32_t count[256];
  int digit;
  u64 found_mass, found_before;
  uint32_t found_count, found_n;
  // the draw
  u64 slice[kMaxSlices];
  int at;
  u64 goal;
};

// f(place) for the row's tokens whose bins are in question: the list, or where it
// is too short the row.
template <typename F>
__device__ __forceinline__ void for_listed(const DrawArgs& a, int64_t row, const Row& r, uint32_t listed, F f) {
  if (listed <= kListed) {
    for (uint32_t i = threadIdx.x; i < listed; i += 256) f(get(&a.list[row * kListed + i]));
  } else {
    const bf16* x = a.logits + row * a.ld;
    const bool vec = row_vec(x);
    for (int64_t i = threadIdx.x * 8; i < a.vocab; i += 2048) {
      const u32x4 q = logits8(x, i, a.vocab, vec);
#pragma unroll 1
      for (int e = 0; e < 8; ++e)
        if (i + e < a.vocab) f(place_of(vkey16(bits_at(q, e)), i + e));
    }
  }
}

// The place of the goal-th token of bin b (by_mass: of the first whose cumulative
// weight reaches the goal), and the weight of the bin's tokens up to it: by digits
// of the place, eight bits at a time, the logit's first; a digit that one token
// has, or whose tokens are all wanted, ends it.  Tokens of one logit weigh the
// same: then weights are counts.
__device__ u64 select_place(const DrawArgs& a, int64_t row, const Row& r, uint32_t listed, int b, bool by_mass, uint32_t goal,
                            double goal_mass, DrawLds& l, u64& up_to) {
  u64 prefix = 0;
  up_to = 0;
  const int tid = threadIdx.x;
#pragma unroll 1
  for (int shift = 40;; shift -= 8) {
    __syncthreads();
    l.mass[tid] = l.most[tid] = 0;
    l.count[tid] = 0;
    if (tid == 0) l.digit = -1;
    __syncthreads();
    for_listed(a, row, r, listed, [&](u64 p) {
      if (p >> (shift + 8) != prefix) return;
      const float v = vkey_value(place_key(p));
      if (bin_of(r, v) != b) return;
      const int d = (int)(p >> shift) & 255;
      atomicAdd(&l.count[d], 1u);
      atomicAdd(&l.mass[d], mass_of(r, v));
      atomicMax(&l.most[d], p);
    });
    __syncthreads();
    const uint32_t n = l.count[tid];
    const u64 m = l.mass[tid];
    const uint32_t nb = block_prefix(n, l.sh32);
    const u64 mb = block_prefix(m, l.sh64);
    // the digit that holds the border: of several with the same cumulative weight
    // the first (no weight: the first with a token)
    const bool here = n > 0 && (by_mass ? (double)(mb + m) >= goal_mass && (nb == 0 || (double)mb < goal_mass)
                                        : nb < goal && nb + n >= goal);
    if (here) {
      l.digit = tid;
      l.found_n = n;
      l.found_count = nb;
      l.found_before = mb;
      l.found_mass = m;
    }
    __syncthreads();
    if (l.digit < 0) {  // (not met: a goal above all by a rounding) all of it
      up_to += block_add(m, l.sh64);
      u64 most = l.most[tid];
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) most = max(most, (u64)__shfl_xor((long long)most, o, 64));
      __syncthreads();
      if ((tid & 63) == 0) l.sh64[tid >> 6] = most;
      __syncthreads();
      return max(max(l.sh64[0], l.sh64[1]), max(l.sh64[2], l.sh64[3]));
    }
    prefix = prefix << 8 | (u64)l.digit;
    up_to += l.found_before;
    if (by_mass) {
      goal_mass -= (double)l.found_before;
      if (shift == 32) {  // one logit left: so many of it
        by_mass = false;
        const u64 each = l.found_mass / l.found_n;
        const double want = each ? ceil(goal_mass / (double)each) : 1.0;
        goal = (uint32_t)fmin(fmax(want, 1.0), (double)l.found_n);
      }
    } else {
      goal -= l.found_count;
    }
    if (l.found_n == 1 || (!by_mass && goal == l.found_n)) {
      up_to += l.found_mass;
      return l.most[l.digit];
    }
    if (shift == 0) return prefix;  // (indexes are distinct: not reached)
  }
}

__global__ __launch_bounds__(256) void draw_token_kernel(DrawArgs a) {
  __shared__ DrawLds l;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.y, base = (int64_t)blockIdx.x * kSlice;
  const bf16* x = a.logits + row * a.ld;
  const bool vec = row_vec(x);
  u32x4 q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = logits8(x, base + (j * 256 + tid) * 8, a.vocab, vec);
  const Asked ask = asked_of(a, row);
  const float temp = a.temp[row];
  const u64 top = row_top(a, row);
  const uint32_t top_key = (uint32_t)(top >> 32);
  const int64_t first = (int64_t)(uint32_t)~(uint32_t)top;
  if (row_greedy(top_key, temp)) {
    if (blockIdx.x == 0 && tid == 0) a.tok[row] = first;
    return;
  }
  const Row r = row_of(vkey_value(top_key), temp, a.unit);

  // bins of the borders: 4 bins a thread, counts and weights above them
  u64 m4[4] = {0, 0, 0, 0}, m_before = 0;
  uint32_t c4[4] = {0, 0, 0, 0}, c_before = 0;
  if (tid == 0) {
    l.bk = l.p_lo = l.p_hi = kBins;
    l.key_m = -1;
  }
  bool by_k = ask.k;
  if (ask.k || ask.p) {
    u64 m = 0;
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c4[e] = a.bin_count[row * kBins + 4 * tid + e];
      m4[e] = a.bin_mass[row * kBins + 4 * tid + e];
      c += c4[e];
      m += m4[e];
    }
    c_before = block_prefix(c, l.sh32);
    m_before = block_prefix(m, l.sh64);
    const u64 all = block_add(m, l.sh64);
    if (ask.k) {
      uint32_t cb = c_before;
      u64 mb = m_before;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (cb < (uint32_t)ask.top_k && cb + c4[e] >= (uint32_t)ask.top_k) {
          l.bk = 4 * tid + e;
          l.above_k = mb;
          l.bin_k = m4[e];
          l.before_k = cb;
        }
        cb += c4[e];
        mb += m4[e];
      }
    }
    __syncthreads();
    by_k = l.bk < kBins;  // (else all that weighs anything is among the first top_k)
    if (ask.p) {
      const double lo = ask.top_p * (double)(by_k ? l.above_k : all), hi = ask.top_p * (double)(by_k ? l.above_k + l.bin_k : all);
      u64 mb = m_before;
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // the first bins whose weight and that above reaches them
        mb += m4[e];
        if (c4[e] && (double)mb >= lo) atomicMin(&l.p_lo, 4 * tid + e);
        if (c4[e] && (double)mb >= hi) atomicMin(&l.p_hi, 4 * tid + e);
      }
    }
  }
  __syncthreads();
  // the least logit of weight min_p: 256 keys apart, then each
  int bm = kBins;
  uint32_t key_m = 0;
  if (ask.m) {
    auto over = [&](int key) { return key > 0x007f && weight(r, vkey_value((uint32_t)key)) >= ask.min_p; };
    if (over((int)top_key - 256 * tid)) atomicMax(&l.key_m, tid);
    __syncthreads();
    const int far = l.key_m;
    __syncthreads();
    if (tid == 0) l.key_m = -1;
    __syncthreads();
    if (far >= 0 && over((int)top_key - 256 * far - tid)) atomicMax(&l.key_m, tid);
    __syncthreads();
    key_m = far >= 0 ? top_key - 256 * far - l.key_m : 0x10000u;  // (over 1: no token of the sort, but the first)
    bm = far >= 0 ? bin_of(r, vkey_value(key_m)) : 0;
  }
  const int bk = by_k ? l.bk : kBins, p_lo = ask.p ? l.p_lo : kBins, p_hi = ask.p ? l.p_hi : kBins;
  // bins under lo are kept, those over hi are not; those between, and top_k's
  // (its weight is what top_p is taken of), are listed
  const int lo = min(min(bk, p_lo), bm), hi = min(min(bk, p_hi), bm);

  u64 own = 0;
  uint32_t mask = 0;  // of the thread's 32 tokens, the listed ones
  auto turn = [&] {
    const u32x4 t = q[0];
    q[0] = q[1];
    q[1] = q[2];
    q[2] = q[3];
    q[3] = t;
  };
#pragma unroll 1
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __uint_as_float(bits_at(q[0], e) << 16);
      const int b = bin_of(r, v);
      const bool in = b < lo && b < kOut;
      if (__ballot(in) != 0) own += in ? mass_of(r, v) : 0;
      mask |= (uint32_t)(b >= lo && b < kOut && (b <= hi || b == bk)) << (8 * j + e);
    }
    turn();
  }
  if (__syncthreads_or(mask != 0)) {
    const uint32_t mine = __popc(mask);
    uint32_t at = block_prefix(mine, l.sh32);
    const uint32_t some = block_add(mine, l.sh32);
    if (tid == 0) l.last = (int)atomicAdd(&a.count[2 * row], some);
    __syncthreads();
    at += (uint32_t)l.last;
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      if (mask >> (8 * j) & 255u)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (mask >> (8 * j + e) & 1u) {
            if (at < kListed)
              put(&a.list[row * kListed + at], place_of(vkey16(bits_at(q[0], e)), base + (j * 256 + tid) * 8 + e));
            ++at;
          }
      turn();
    }
  }
  own = block_add(own, l.sh64);
  // In memory, for every XCD, before the slice is counted: device-scope stores,
  // waited for by every wave.
  if (tid == 0) put(&a.mass[row * a.slices + blockIdx.x], own);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) l.last = (int)__hip_atomic_fetch_add(&a.count[2 * row + 1], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (l.last != a.slices - 1) return;

  // The row's last workgroup: the borders' places
  const uint32_t listed = get(&a.count[2 * row]);
  u64 border = kAll, kept_k = 0, up_to;
  if (by_k) {
    border = select_place(a, row, r, listed, bk, false, (uint32_t)ask.top_k - l.before_k, 0.0, l, up_to);
    kept_k = l.above_k + up_to;
  } else if (ask.p) {
    u64 m = (m4[0] + m4[1]) + (m4[2] + m4[3]);
    kept_k = block_add(m, l.sh64);
  }
  if (ask.p) {
    const double goal = ask.top_p * (double)kept_k;
    if (tid == 0) l.bp = kBins;
    __syncthreads();
    u64 mb = m_before;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mb += m4[e];
      if (c4[e] && (double)mb >= goal) atomicMin(&l.bp, 4 * tid + e);
    }
    __syncthreads();
    const int bp = l.bp;
    mb = m_before;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (4 * tid + e == bp) l.above_p = mb;
      mb += m4[e];
    }
    __syncthreads();
    if (bp < kBins && bp <= hi)
      border = min(border, select_place(a, row, r, listed, bp, true, 0, goal - (double)l.above_p, l, up_to));
  }
  if (ask.m) border = min(border, key_m > 0xffffu ? 0 : place_of(key_m, 0xffffffffll));
  border = max(border, place_of(top_key, first));  // at least one

  // weights of the slices: what is kept wholly, and the listed tokens up to the border
  __syncthreads();
  for (int s = tid; s < a.slices; s += 256) l.slice[s] = get(&a.mass[row * a.slices + s]);
  __syncthreads();
  if (lo < kOut)
    for_listed(a, row, r, listed, [&](u64 p) {
      if (p > border) return;
      const float v = vkey_value(place_key(p));
      const int b = bin_of(r, v);
      if (b >= lo && b < kOut) atomicAdd(&l.slice[(uint32_t)p / kSlice], mass_of(r, v));
    });
  __syncthreads();
  const u64 mine = tid < a.slices ? l.slice[tid] : 0;
  const u64 before = block_prefix(mine, l.sh64);
  const u64 all = block_add(mine, l.sh64);
  // (a u outside [0, 1) draws the first or the last that weighs anything)
  const double want = (double)a.u[row] * (double)all;
  const u64 goal = want > 0.0 ? (want < (double)all ? min((u64)want, all - 1) : all - 1) : 0;
  // the first token with a cumulative weight above goal: of whole numbers, one with
  // more than floor(u all) has more than u all, and the other way round
  if (mine > 0 && before <= goal && goal < before + mine) {
    l.at = tid;
    l.goal = goal - before;
  }
  __syncthreads();
  const int64_t from = (int64_t)l.at * kSlice;
  u64 left = l.goal;
#pragma unroll 1
  for (int j = 0; j < 4; ++j) {
    const int64_t i = from + (j * 256 + tid) * 8;
    const u32x4 v = logits8(x, i, a.vocab, vec);
    auto mass_at = [&](int e) -> u64 {
      const uint32_t bits = bits_at(v, e);
      const float f = __uint_as_float(bits << 16);
      const bool kept = i + e < a.vocab && place_of(vkey16(bits), i + e) <= border && bin_of(r, f) < kOut;
      return kept ? mass_of(r, f) : 0;
    };
    u64 m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m += mass_at(e);
    const u64 bef = block_prefix(m, l.sh64), sum = block_add(m, l.sh64);
    if (left < sum) {
      if (bef <= left && left < bef + m) {
        u64 c = bef;
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const u64 w = mass_at(e);
          c += w;
          if (left < c) {
            a.tok[row] = i + e;
            break;
          }
        }
      }
      return;
    }
    left -= sum;
  }
}

struct DrawLayout {
  int64_t slices, bin_mass, bin_count, mass, list, count, bytes;
};
DrawLayout draw_layout(int64_t n, int64_t vocab) {
  DrawLayout l;
  l.slices = (vocab + kSlice - 1) / kSlice;
  l.bin_mass = n * l.slices * (int64_t)sizeof(u64);
  l.mass = l.bin_mass + n * kBins * (int64_t)sizeof(u64);
  l.list = l.mass + n * l.slices * (int64_t)sizeof(u64);
  l.bin_count = l.list + n * kListed * (int64_t)sizeof(u64);
  l.count = l.bin_count + n * kBins * (int64_t)sizeof(uint32_t);
  l.bytes = l.count + n * 2 * (int64_t)sizeof(uint32_t);
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
  SWL_CHECK(vocab > 0 && vocab <= (int64_t)kMaxSlices * kSlice, SWL_ERR_INVALID,
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
  int bits = 0;  // vocab <= 2^bits
  while (((int64_t)1 << bits) < vocab) ++bits;
  a.unit = (double)((int64_t)1 << std::min(46, 63 - bits));
  char* ws = reinterpret_cast<char*>(workspace);
  a.top = reinterpret_cast<u64*>(ws);
  a.bin_mass = reinterpret_cast<u64*>(ws + l.bin_mass);
  a.mass = reinterpret_cast<u64*>(ws + l.mass);
  a.list = reinterpret_cast<u64*>(ws + l.list);
  a.bin_count = reinterpret_cast<uint32_t*>(ws + l.bin_count);
  a.count = reinterpret_cast<uint32_t*>(ws + l.count);
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)l.slices, (unsigned)n);
  hipLaunchKernelGGL(draw_max_kernel, grid, dim3(256), 0, st, a);
  SWL_LAUNCH_CHECK("draw_max_kernel launch");
  if (top_k || top_p) {
    hipLaunchKernelGGL(draw_bins_kernel, grid, dim3(256), 0, st, a);
    SWL_LAUNCH_CHECK("draw_bins_kernel launch");
  }
  hipLaunchKernelGGL(draw_token_kernel, grid, dim3(256), 0, st, a);
  SWL_LAUNCH_CHECK("draw_token_kernel launch");
  return SWL_OK;
}
