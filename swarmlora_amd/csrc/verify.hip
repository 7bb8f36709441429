// Verification of drafted tokens (speculative decoding) against the target's
// probabilities, from given random numbers.
//
// With p_j, q_j the target's and the drafter's probabilities at draft j (the
// softmax of logits / temperature), draft d_j is accepted while u_j q_j(d_j) <
// p_j(d_j).  The token after the accepted ones is drawn by inverse CDF, in index
// order, from max(p - q, 0) where a draft was refused, from p of the row after
// the last draft where none was: its distribution is the target's.  A drafter
// without probabilities counts as certain of its draft (q = 1 at d_j).
//
// What decides is held in 64 bits: with 128256 tokens a cumulative sum that is
// off by 1e-7 of the total picks another token once in about forty draws.  A
// 64-bit exponential costs fifteen times an fp32 one, though (28 sequences of 1
// to 5 drafts, 128256 tokens: 77 us with 64 bits throughout, 32 now), and most
// rows only have to show that their draft is accepted: u q < p is clear in fp32
// unless the two are within 2^-14 of each other.  So, in two launches: every
// row's maximum and sum in fp32, a workgroup per slice of a row (the logits'
// bytes are its bound); then a workgroup per slice of every sequence's last row:
// acceptance (each for itself; a comparison that is not clear again in 64 bits
// over the whole row), the weights of the slice's four shares (a wave's each) in
// 64 bits, and by the workgroup that ends last the share that the random number
// falls in, and its token.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "dev_util.h"
#include "swl.h"
#include "swl_common.h"

namespace {

struct RowStat {
  float z;        // sum of e^((x - max) / temperature) over the slice
  float mx;       // its largest logit
  int32_t idx;    // the first index of that (greedy rows)
  int32_t pad;
};
// A wave's share of a sequence's last row: sums of the target's and the drafter's
// e^(..), of the residual and the drafter's part of it at a given ratio, and the
// target's part that is next to no residual.
struct ShareSum {
  double p, q, res, act, near;
};

struct VerifyArgs {
  const bf16* tgt;      // [T + nseq, vocab]
  const bf16* drf;      // [T, vocab] or null
  int64_t ld_t, ld_d, vocab, T;
  const int64_t* ids;
  const int32_t* cu;    // null: per tokens each
  const float* temp;
  const float* u;
  const float* u_last;
  int64_t* tok;         // [nseq, max_drafts + 1]
  int32_t* acc;
  int32_t nseq, per, max_drafts;
  int32_t stats, slices;  // slices of a row: of its statistics, of a sequence's last row
  int32_t share;          // logits of a wave of a slice
  RowStat* stat;        // [T + nseq rows, then T rows][stats]
  ShareSum* sum;        // [nseq][4 slices]
  uint32_t* done;       // [nseq] slices that are (set to 0 by the first launch)
  double* pow;          // [256] 2^(k / 256) (made by it)
};

// order-preserving maps of a bf16's bits to 16 bits and back, a NaN of either
// sign above all, -0 the same as +0
__device__ __forceinline__ uint32_t vkey16(uint32_t bits) {
  if ((bits & 0x7fffu) > 0x7f80u) return 0xffffu;
  if (bits == 0x8000u) return 0x8000u;
  return (bits & 0x8000u) ? (~bits & 0xffffu) : (bits | 0x8000u);
}
__device__ __forceinline__ float vkey_value(uint32_t key) {
  return __uint_as_float(((key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu)) << 16);
}

// First draft and number of drafts of sequence s.
__device__ __forceinline__ void drafts_of(const VerifyArgs& a, int s, int64_t& t0, int& n) {
  t0 = a.cu ? a.cu[s] : (int64_t)s * a.per;
  const int64_t m = a.cu ? (int64_t)a.cu[s + 1] - t0 : a.per;
  n = t0 < 0 || m < 0 || t0 + m > a.T ? 0 : (int)min<int64_t>(m, a.max_drafts);
  if (t0 < 0 || t0 > a.T) t0 = 0;  // (offsets that are none: in range all the same)
}

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

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kPow = 256;  // entries of the table of 2^(k / 256)

// e^((x - max) / temperature) in 64 bits; rate = 256 log2(e) / temperature, tab
// the 256 powers 2^(k / 256) (made by the first launch).  The series of 2^f for
// the rest |f| <= 1/512 to the fourth power (the next term is under 4e-17).
// -inf gives 0, a NaN itself.
__device__ __forceinline__ double weight(uint32_t bits, float mx, double rate, const double* tab) {
  constexpr double c = 0.693147180559945309417232121458 / kPow;  // ln 2 / 256
  constexpr double c2 = c * c;
  const double x = __uint_as_float(bits == 0xff80u ? 0xff7f0000u : bits << 16);  // (-inf: no NaN from a rate of 0)
  const double y = (x - (double)mx) * rate, n = rint(y), f = y - n;
  // (at a temperature of 1e-5 n may leave 32 bits, and a NaN is no int at all: the
  // language defines no conversion then, the instruction gives the nearest int,
  // whose power is 0 as well, and 0.  f keeps the NaN.  A clamp before a plain
  // conversion is 0.7 us of the batch of 28 below.)
  int k;
  asm("v_cvt_i32_f64 %0, %1" : "=v"(k) : "v"(n));
  double r = c2 * c2 / 24;
  r = fma(r, f, c2 * c / 6);
  r = fma(r, f, c2 / 2);
  r = fma(r, f, c);
  r = fma(r, f, 1.0);
  return bits == 0xff80u ? 0.0 : ldexp(r * tab[k & (kPow - 1)], k >> 8);
}
__device__ __forceinline__ double rate_of(float temp) {
  return kPow * 1.44269504088896340735992468100 / (double)temp;
}

// Sum over the workgroup's 256 threads, the same order always.
__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
__device__ __forceinline__ void block_sum2(double& v, double& w, double* sh) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    v += __shfl_xor(v, o, 64);
    w += __shfl_xor(w, o, 64);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    sh[threadIdx.x >> 6] = v;
    sh[4 + (threadIdx.x >> 6)] = w;
  }
  __syncthreads();
  v = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  w = (sh[4] + sh[5]) + (sh[6] + sh[7]);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Inclusive prefix over them, likewise.
__device__ __forceinline__ double block_prefix(double v, double* sh) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 63) sh[wv] = v;
  __syncthreads();
  for (int w = 0; w < wv; ++w) v += sh[w];
  return v;
}

// Slices of a row: 256 threads with 32 logits each, all requested at once.
// (Slices of 2048 for calls of few rows were level at best: one sequence of 4
// drafts and 32000 tokens 13.6 us for both launches instead of 13.7, 28 rows of
// 128256 19.3 instead of 17.4, 448 rows 70 instead of 60.)  The logits' bytes
// bound it: 196 rows of 128256 take 13 us, 3.9 TB/s.
constexpr int kStatsSlice = 8192;
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  __shared__ uint32_t shk[4];
  __shared__ float shz[4];
  constexpr int E = kStatsSlice / 256;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t R = a.T + a.nseq;
  const int64_t r = blockIdx.y, t = r - R;  // target rows, then draft rows
  const bool draft = t >= 0;
  if (blockIdx.x == 0 && r < a.nseq && tid == 0) a.done[r] = 0;
  if (blockIdx.x == 0 && r == 0) a.pow[tid] = exp2((double)tid / kPow);
  const bf16* row = draft ? a.drf + t * a.ld_d : a.tgt + r * a.ld_t;
  const bool vec = row_vec(row);
  const int64_t base = (int64_t)blockIdx.x * kStatsSlice;
  u32x4 q[E / 8];  // (requested before the sequence is looked for)
#pragma unroll
  for (int j = 0; j < E / 8; ++j) q[j] = logits8(row, base + (j * 256 + tid) * 8, a.vocab, vec);
  int s = 0;
  if (a.cu) {
    for (int i0 = 0; i0 < a.nseq; i0 += 64) {
      const int i = i0 + lane;
      s += __popcll(__ballot(i < a.nseq && (draft ? a.cu[i + 1] <= t : (int64_t)a.cu[i + 1] + i + 1 <= r)));
    }
  } else {
    s = (int)(draft ? t / max(a.per, 1) : r / (a.per + 1));
  }
  if (s >= a.nseq) return;  // (rows behind the last sequence)
  const float temp = a.temp[s];
  if (draft && temp <= 0.f) return;
  if (temp <= 0.f) {  // greedy: the largest and its first index are all there is to know
    uint32_t best = 0;  // order key, then the index counted down
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = (j * 256 + tid) * 8 + e;
        if (base + at < a.vocab) best = max(best, vkey16(bits_at(q[j], e)) << 13 | (uint32_t)(8191 - at));
      }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, o, 64));
    if (lane == 0) shk[wv] = best;
    __syncthreads();
    best = max(max(shk[0], shk[1]), max(shk[2], shk[3]));
    if (tid == 0)
      a.stat[r * a.stats + blockIdx.x] = RowStat{0.f, vkey_value(best >> 13), (int32_t)(base + 8191 - (best & 8191)), 0};
    return;
  }
  float mx = -INFINITY;  // (a NaN is passed over, and met again in the sum)
#pragma unroll
  for (int j = 0; j < E / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      mx = fmaxf(mx, fmaxf(__uint_as_float(q[j][e] << 16), __uint_as_float(q[j][e] & 0xffff0000u)));
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if (lane == 0) shk[wv] = __float_as_uint(mx);
  __syncthreads();
  mx = fmaxf(fmaxf(__uint_as_float(shk[0]), __uint_as_float(shk[1])),
             fmaxf(__uint_as_float(shk[2]), __uint_as_float(shk[3])));
  float z = 0.f;
  if (mx != -INFINITY) {  // (a slice of nothing but -inf weighs 0; so does what is past the row)
    const float c = kLog2e / temp;
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z += __builtin_amdgcn_exp2f((__uint_as_float(q[j][e] << 16) - mx) * c);
        z += __builtin_amdgcn_exp2f((__uint_as_float(q[j][e] & 0xffff0000u) - mx) * c);
      }
  } else {
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((bits_at(q[j], e) & 0x7fffu) > 0x7f80u) z = NAN;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) z += __shfl_xor(z, o, 64);
  if (lane == 0) shz[wv] = z;
  __syncthreads();
  if (tid == 0) a.stat[r * a.stats + blockIdx.x] = RowStat{(shz[0] + shz[1]) + (shz[2] + shz[3]), mx, 0, 0};
}

// A row's statistics from its slices', by sixteen lanes.
struct RowAll {
  float z, mx;
  int64_t best;  // (greedy rows)
};
__device__ __forceinline__ RowAll row_all(const VerifyArgs& a, int64_t r, float c, bool greedy, int l16) {
  const RowStat* st = a.stat + r * a.stats;
  RowAll x{0.f, -INFINITY, 0};
  RowStat own{0.f, -INFINITY, 0x7fffffff, 0};  // (sixteen slices hold 131072 logits: no round of the loops, mostly)
  if (l16 < a.stats) own = st[l16];
  if (greedy) {
    auto key = [](const RowStat& v) {
      return (uint64_t)vkey16(__float_as_uint(v.mx) >> 16) << 32 | (uint32_t)~(uint32_t)v.idx;
    };
    uint64_t best = key(own);
    for (int i = 16 + l16; i < a.stats; i += 16) best = max(best, key(st[i]));
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) best = max(best, (uint64_t)__shfl_xor((long long)best, o, 16));
    x.best = (int64_t)(uint32_t)~(uint32_t)best;
    return x;
  }
  x.mx = own.mx;
  for (int i = 16 + l16; i < a.stats; i += 16) x.mx = fmaxf(x.mx, st[i].mx);
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) x.mx = fmaxf(x.mx, __shfl_xor(x.mx, o, 16));
  // (slices of nothing but -inf weigh 0, or are a NaN)
  auto part = [&](const RowStat& v) { return v.z == 0.f ? 0.f : v.z * __builtin_amdgcn_exp2f((v.mx - x.mx) * c); };
  if (l16 < a.stats) x.z = part(own);
  for (int i = 16 + l16; i < a.stats; i += 16) x.z += part(st[i]);
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) x.z += __shfl_xor(x.z, o, 16);
  return x;
}

// What a sequence's last row is, and what is taken from it.
struct Last {
  const bf16* p;  // target row
  const bf16* q;  // draft row subtracted from it, or null
  int64_t skip;   // token whose weight is 0, -1: none
  float p_max, q_max;
  double ratio;   // the target's sum over the drafter's
};
// f(e, e^(..) of the target, of the drafter) for the eight tokens from i, in
// order; 0 at `skip` and past the row.  (Not unrolled: these kernels run once
// through their code, and its fetching would be their time.)
template <typename F>
__device__ __forceinline__ void weights8(const VerifyArgs& a, const Last& x, int64_t i, double rate,
                                         const double* tab, F f) {
  u32x4 p = logits8(x.p, i, a.vocab, row_vec(x.p)), q = p;
  if (x.q) q = logits8(x.q, i, a.vocab, row_vec(x.q));
#pragma unroll 1
  for (int e = 0; e < 8; e += 2) {
    double wp[2], wq[2] = {0, 0};
    wp[0] = weight(p[0] & 0xffffu, x.p_max, rate, tab);
    wp[1] = weight(p[0] >> 16, x.p_max, rate, tab);
    if (x.q) {
      wq[0] = weight(q[0] & 0xffffu, x.q_max, rate, tab);
      wq[1] = weight(q[0] >> 16, x.q_max, rate, tab);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const bool in = i + e + k < a.vocab;
      f(e + k, in && i + e + k != x.skip ? wp[k] : 0.0, in ? wq[k] : 0.0);
    }
    p = u32x4{p[1], p[2], p[3], p[0]};
    q = u32x4{q[1], q[2], q[3], q[0]};
  }
}

// The two rows' sums in 64 bits, by the workgroup (q 0 without a draft row).
__device__ __forceinline__ void row_sums64(const VerifyArgs& a, const Last& x, double rate, const double* tab,
                                           double* sh, double (&z)[2]) {
  z[0] = z[1] = 0;
  for (int64_t i = threadIdx.x * 8; i < a.vocab; i += 2048)
    weights8(a, x, i, rate, tab, [&](int, double p, double q) {
      z[0] += p;
      z[1] += q;
    });
  block_sum2(z[0], z[1], sh);
}

// The first largest logit of a row, a NaN above all: for rows whose weights are
// no numbers.
__device__ int64_t row_best(const bf16* row, int64_t vocab, unsigned long long* sh) {
  if (threadIdx.x == 0) *sh = 0;
  __syncthreads();
  unsigned long long best = 0;
  for (int64_t i = threadIdx.x * 8; i < vocab; i += 2048) {
    const u32x4 q = logits8(row, i, vocab, row_vec(row));
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < vocab)
        best = max(best, (unsigned long long)vkey16(bits_at(q, e)) << 32 | (uint32_t)~(uint32_t)(i + e));
  }
  atomicMax(sh, best);
  __syncthreads();
  return (int64_t)(uint32_t)~(uint32_t)*sh;
}

// Device-scope accesses, past the caches that other XCDs do not see.
__device__ __forceinline__ void put(double* p, double v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Acceptance of a sequence's drafts (sixteen lanes for a draft's target row and
// sixteen for the drafter's, eight drafts at a time), the weight of a slice of
// its last row, every wave's share of the slice for itself, and by the last
// workgroup of the sequence the token: the share that the random number falls
// in, then the thread and the token of that share: the first whose cumulative
// weight is above u * (sum of all); where rounding leaves none, the last of any
// weight.  Shares lie in index order, at most 256 of a row, one a thread.
//
// The residual max(p - q, 0) needs the two rows' sums, which are known only when
// all slices are: its weight is added up at the fp32 sums' ratio (off by a
// relative d of under 2^-14, 1e-6 as a rule) together with the drafter's part F
// of it, and put right by - d F at the end.  What that leaves out are the tokens
// between the two ratios, d of themselves each and mostly about d of all: d^2.
// Where it could be more than 2^-30 of the residual (rows that are nearly the
// same) the last workgroup adds the shares up again at the exact ratio.
//
// 10.5 us for one sequence of 4 drafts (32000 tokens, no drafter): a chain of
// loads, sums and one count in memory (5 us until the weights, 6 behind them); 22
// for 28 of up to 5 (128256 tokens, with a drafter): the same chain, met once, for
// every slice is there at once, and 64-bit arithmetic of some 6 us by its count,
// spread over the card.  (What the other 6 are has not been found.)  Sums of whole
// slices, 4096 logits instead of 1024 to look through at the end: 27 us.
constexpr double kNear = 0x1p-18;  // (the fp32 sums' ratio is nearer than half of it but for rows out of the way)
constexpr int kPiece = 1024;  // logits of a share that the last workgroup looks at together, four a thread

__global__ __launch_bounds__(256) void verify_last_kernel(VerifyArgs a) {
  constexpr int kNone = 0x7fffffff;
  __shared__ int first_bad, ended;
  __shared__ double tab[kPow], sh[8], wt[4][256], below, first;
  __shared__ int sh_hit[4], sh_any[4];
  __shared__ float sh_mx[16], sh_z[16];  // maxima and sums of the eight drafts: target, drafter
  __shared__ int64_t sh_best[8];
  __shared__ unsigned long long shb;
  const int tid = threadIdx.x, l16 = tid & 15, s = blockIdx.y;
  tab[tid] = a.pow[tid];  // (a barrier follows)
  int64_t t0;
  int n;
  drafts_of(a, s, t0, n);
  const float temp = a.temp[s];
  const bool greedy = temp <= 0.f;
  const float c = kLog2e / temp;
  const double rate = rate_of(temp);
  const float u_last = a.u_last[s];
  const int64_t R = a.T + a.nseq, row0 = t0 + s;
  Last x;
  // Drafts before `sure` are accepted; index n, behind the last draft, is where
  // it ends at the latest.
  int take, sure = 0;
  int64_t d;
  for (int j0 = 0;;) {
    __syncthreads();
    if (tid == 0) first_bad = kNone;
    __syncthreads();
    const int j = j0 + (tid >> 5);
    const bool second = tid >> 4 & 1;
    if (j <= n) {  // (the 32 lanes together)
      const bool draft = j < n;
      d = draft ? a.ids[t0 + j] : -1;
      const bool in = d >= 0 && d < a.vocab;
      const bf16* row = second && draft && a.drf ? a.drf + (t0 + j) * a.ld_d : a.tgt + (row0 + j) * a.ld_t;
      const float lg = in ? bf2f(ldg(row + d)) : 0.f;
      const float u = draft ? a.u[t0 + j] : 0.f;
      const RowAll r = row_all(a, second && draft && a.drf && !greedy ? R + t0 + j : row0 + j, c, greedy, l16);
      const float prob = __builtin_amdgcn_exp2f((lg - r.mx) * c) / r.z, other = __shfl_xor(prob, 16, 32);
      if (l16 == 0) {
        sh_mx[tid >> 4] = r.mx;
        sh_z[tid >> 4] = r.z;
        if (!second) {
          sh_best[tid >> 5] = r.best;
          bool ok = false, clear = true;
          if (j < sure) {
            ok = true;
          } else if (greedy) {
            ok = in && d == r.best;
          } else if (in) {
            const float v = a.drf ? u * other : u;
            // (fp32: the exponents' roundings, under 2^-16 of a term that counts)
            ok = v < prob * (1.f - 0x1p-14f) && prob > 0x1p-100f;
            clear = ok || (v > prob * (1.f + 0x1p-14f) && v > 0x1p-100f && v < INFINITY);
          }
          if (!ok) atomicMin(&first_bad, 2 * j + (clear ? 0 : 1));
        }
      }
    }
    __syncthreads();
    const int bad = first_bad;
    if (bad == kNone) {
      j0 += 8;
      continue;
    }
    take = bad >> 1;
    d = take < n ? a.ids[t0 + take] : -1;  // the refused draft
    const bool subtract = d >= 0 && d < a.vocab;
    x.p = a.tgt + (row0 + take) * a.ld_t;
    x.q = subtract && a.drf ? a.drf + (t0 + take) * a.ld_d : nullptr;
    x.skip = -1;
    x.p_max = sh_mx[2 * (take - j0)];
    x.q_max = sh_mx[2 * (take - j0) + 1];
    const float zp = sh_z[2 * (take - j0)], zq = sh_z[2 * (take - j0) + 1];
    x.ratio = (double)zp / (double)zq;
    // A comparison that is not clear, or sums that fp32 does not have (an
    // infinite rate, a NaN): from the whole rows, in 64 bits.
    const bool poor = !greedy && x.q && !(zp >= 0.5f && zp < INFINITY && zq >= 0.5f && zq < INFINITY);
    if (bad & 1 || poor) {
      double z[2];
      row_sums64(a, x, rate, tab, sh, z);
      x.ratio = z[0] / z[1];
      if (bad & 1) {
        const double qd =
            x.q ? weight(*reinterpret_cast<const uint16_t*>(x.q + d), x.q_max, rate, tab) / z[1] : 1.0;
        const double pd = weight(*reinterpret_cast<const uint16_t*>(x.p + d), x.p_max, rate, tab) / z[0];
        if ((double)a.u[t0 + take] * qd < pd) {
          sure = take + 1;
          continue;  // the same drafts again, this one taken
        }
      }
    }
    if (subtract && !x.q) x.skip = d;
    break;
  }
  const int64_t best = sh_best[take & 7];  // (batches begin at multiples of eight)
  int64_t* out = a.tok + (int64_t)s * (a.max_drafts + 1);
  if (blockIdx.x == 0) {
    if (tid == 0) a.acc[s] = take;
    for (int j = tid; j <= a.max_drafts; j += 256)
      if (j != take || greedy) out[j] = j < take ? a.ids[t0 + j] : j == take ? best : -1;
  }
  if (greedy) return;
  ShareSum own{0, 0, 0, 0, 0};
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t from = ((int64_t)blockIdx.x * 4 + wave) * a.share, end = min(from + a.share, a.vocab);
#pragma unroll 1
  for (int64_t i = from + (tid & 63) * 8; i < end; i += 512)
    weights8(a, x, i, rate, tab, [&](int, double p, double q) {
      own.p += p;
      own.q += q;
      const double v = p - x.ratio * q;
      if (x.q && !(v < 0)) {
        own.res += v;
        own.act += q;
      }
      if (x.q && fabs(v) < p * kNear) own.near += p;
    });
  own.p = wave_sum(own.p);
  if (x.q) {
    own.q = wave_sum(own.q);
    own.res = wave_sum(own.res);
    own.act = wave_sum(own.act);
    if (__ballot(own.near > 0) != 0) own.near = wave_sum(own.near);
  }
  // The shares' sums are in memory, for every XCD, before the slice is counted:
  // device-scope stores, waited for.  (A release fence would write back the XCD's
  // whole L2, once a workgroup, and an acquire empty it.)
  ShareSum* sums = a.sum + (int64_t)s * 4 * a.slices;
  if ((tid & 63) == 0) {
    ShareSum* mine = sums + blockIdx.x * 4 + wave;
    put(&mine->p, own.p);
    if (x.q) {
      put(&mine->q, own.q);
      put(&mine->res, own.res);
      put(&mine->act, own.act);
      put(&mine->near, own.near);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  }
  __syncthreads();
  if (tid == 0) ended = (int)__hip_atomic_fetch_add(&a.done[s], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (ended != a.slices - 1) return;
  ShareSum v{0, 0, 0, 0, 0};  // of share tid
  if (tid < 4 * a.slices) {
    v.p = get(&sums[tid].p);
    if (x.q)
      v = ShareSum{v.p, get(&sums[tid].q), get(&sums[tid].res), get(&sums[tid].act), get(&sums[tid].near)};
  }
  double m = v.p, off = 0;  // off: how far all may be off, by this share of it
  if (x.q) {  // the exact ratio, and the weights put right to it
    block_sum2(v.p, v.q, sh);
    const double ratio = v.p / v.q;
    m = v.res - (ratio - x.ratio) * v.act;
    m = m < 0 ? 0 : m;
    const double d = fabs(ratio - x.ratio) / ratio;
    off = d < kNear / 2 ? d * v.near : v.p;
    x.ratio = ratio;
  }
  // The first thread whose cumulative weight `inc` is above `goal` (where there
  // is none, the last of any weight), by the workgroup; -1: no weight at all.
  auto pick = [&](double w, double inc, double goal) {
    const uint64_t over = __ballot(w > 0 && inc > goal), some = __ballot(w > 0);
    __syncthreads();
    if ((tid & 63) == 0) {
      sh_hit[tid >> 6] = over ? tid + __builtin_ctzll(over) : kNone;
      sh_any[tid >> 6] = some ? tid + 63 - __builtin_clzll(some) : -1;
    }
    __syncthreads();
    const int hit = min(min(sh_hit[0], sh_hit[1]), min(sh_hit[2], sh_hit[3]));
    return hit != kNone ? hit : max(max(sh_any[0], sh_any[1]), max(sh_any[2], sh_any[3]));
  };
  double inc = block_prefix(m, sh);
  if (tid == 255) below = inc;  // the sum of all
  __syncthreads();
  if (__syncthreads_or(off > below * 0x1p-38)) {  // (256 shares at most: 2^-30 together)
    m = 0;
#pragma unroll 1
    for (int k = 0; k < 4 * a.slices; ++k) {
      double y = 0;
#pragma unroll 1
      for (int64_t i = (int64_t)k * a.share + tid * 8; i < min((int64_t)(k + 1) * a.share, a.vocab); i += 2048)
        weights8(a, x, i, rate, tab, [&](int, double p, double q) { y += fmax(p - x.ratio * q, 0.0); });
      y = block_sum(y, sh);
      if (tid == k) m = y;
    }
    inc = block_prefix(m, sh);
    if (tid == 255) below = inc;
    __syncthreads();
  }
  const double all = below, want = (double)u_last * all;
  if (!(all > 0)) {  // a NaN, or nothing left
    const int64_t b = row_best(x.p, a.vocab, &shb);
    if (tid == 0) out[take] = b;
    return;
  }
  const int at = pick(m, inc, want);
  if (tid == at) below = want - (inc - m);  // what is left for the share (read behind pick's barriers)
  __syncthreads();
  const double goal = below;
  // the share's pieces: the first whose weight passes that, else the last of any
  const int64_t begin = (int64_t)at * a.share, stop = min(begin + a.share, a.vocab);
  const int pieces = (a.share + kPiece - 1) / kPiece;
  double before = 0, w = 0;
  int piece = -1, who = 0, k = 0;
  auto weigh = [&](int k) {
    const int64_t i = begin + (int64_t)k * kPiece + tid * 4;
    uint32_t pb[4], qb[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pb[e] = qb[e] = 0xff80u;
      if (i + e < stop) {
        pb[e] = reinterpret_cast<const uint16_t*>(x.p)[i + e];
        if (x.q) qb[e] = reinterpret_cast<const uint16_t*>(x.q)[i + e];
      }
    }
    w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      double y = i + e < stop && i + e != x.skip ? weight(pb[e], x.p_max, rate, tab) : 0.0;
      if (x.q) y = i + e < stop ? fmax(y - x.ratio * weight(qb[e], x.q_max, rate, tab), 0.0) : 0.0;
      w += y;
      wt[e][tid] = y;
    }
  };
#pragma unroll 1
  for (;; ++k) {
    weigh(k);
    inc = before + block_prefix(w, sh);
    const int t = pick(w, inc, goal);
    if (t >= 0) {
      piece = k;
      who = t;
      if (tid == t) first = inc - w;
      if (tid == 255) below = inc;
      __syncthreads();
      before = below;
      __syncthreads();
    }
    if ((piece >= 0 && before > goal) || k == pieces - 1) break;
  }
  if (piece < 0) {  // (a weight that was the other ratio's alone: the residual is nothing)
    const int64_t b = row_best(x.p, a.vocab, &shb);
    if (tid == 0) out[take] = b;
    return;
  }
  if (piece != k) weigh(piece);  // (the last pieces had no weight)
  if (tid != who) return;
  double cum = first;  // its tokens, one after another
  int hit = 0;
  for (int e = 0; e < 4; ++e) {
    const double y = wt[e][tid];
    cum += y;
    if (y > 0) {
      hit = e;
      if (cum > goal) break;
    }
  }
  out[take] = begin + (int64_t)piece * kPiece + tid * 4 + hit;
}

struct VerifyLayout {
  int share;
  int64_t stats, slices, sum, pow, done, bytes;
};
VerifyLayout verify_layout(int64_t nseq, int64_t T, int64_t vocab, bool draft) {
  VerifyLayout l;
  const int64_t rows = T + nseq + (draft ? T : 0);
  l.stats = (vocab + kStatsSlice - 1) / kStatsSlice;
  // (slices of the last rows, multiples of 2048: about 1024 workgroups, which run
  // at once, and 64 of a row at most)
  const int64_t chunks = (vocab + 2047) / 2048;
  const int64_t each = std::min(chunks, std::max((chunks + 63) / 64, (nseq * chunks + 1023) / 1024));
  l.share = (int)(each * 512);
  l.slices = (chunks + each - 1) / each;
  l.sum = rows * l.stats * (int64_t)sizeof(RowStat);
  l.pow = l.sum + nseq * 4 * l.slices * (int64_t)sizeof(ShareSum);
  l.done = l.pow + kPow * (int64_t)sizeof(double);
  l.bytes = l.done + nseq * (int64_t)sizeof(uint32_t);
  return l;
}

int launch_verify(const VerifyArgs& a, hipStream_t st) {
  const dim3 rows((unsigned)a.stats, (unsigned)(a.T + a.nseq + (a.drf ? a.T : 0)));
  hipLaunchKernelGGL(verify_stats_kernel, rows, dim3(256), 0, st, a);
  SWL_LAUNCH_CHECK("verify_stats_kernel launch");
  const dim3 last((unsigned)a.slices, (unsigned)a.nseq);
  hipLaunchKernelGGL(verify_last_kernel, last, dim3(256), 0, st, a);
  SWL_LAUNCH_CHECK("verify_last_kernel launch");
  return SWL_OK;
}

}  // namespace

extern "C" int64_t swl_verify_drafts_workspace(int nseq, int64_t ndraft, int64_t vocab, int with_draft) {
  if (nseq <= 0 || ndraft < 0 || vocab <= 0) return 0;
  return verify_layout(nseq, ndraft, vocab, with_draft != 0 && ndraft > 0).bytes;
}

extern "C" int swl_verify_drafts_bf16(const void* target, int64_t ld_target, const void* draft, int64_t ld_draft,
                                      int64_t vocab, const int64_t* draft_ids, const int32_t* cu_drafts, int nseq,
                                      int64_t ndraft, int max_drafts, const float* temperature, const float* u_accept,
                                      const float* u_final, int64_t* out_tokens, int32_t* out_accepted,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  SWL_CHECK(nseq >= 0 && ndraft >= 0 && max_drafts >= 0 && max_drafts <= (1 << 20), SWL_ERR_INVALID,
            "swl_verify_drafts_bf16: bad sequence or draft count");
  SWL_CHECK(vocab > 0 && vocab < ((int64_t)1 << 31) - 8192, SWL_ERR_INVALID, "swl_verify_drafts_bf16: bad vocabulary");
  if (nseq == 0) return SWL_OK;
  SWL_CHECK(2 * ndraft + nseq <= 65535, SWL_ERR_INVALID, "swl_verify_drafts_bf16: at most 65535 rows");
  SWL_CHECK(cu_drafts || ndraft % nseq == 0, SWL_ERR_INVALID,
            "swl_verify_drafts_bf16: without cu_drafts every sequence has as many drafts");
  SWL_CHECK(target && temperature && u_final && out_tokens && out_accepted, SWL_ERR_INVALID,
            "swl_verify_drafts_bf16: null argument");
  SWL_CHECK(ndraft == 0 || (draft_ids && u_accept), SWL_ERR_INVALID, "swl_verify_drafts_bf16: null argument");
  SWL_CHECK(ld_target >= vocab && (!draft || ld_draft >= vocab), SWL_ERR_INVALID,
            "swl_verify_drafts_bf16: row strides smaller than the vocabulary");
  const VerifyLayout l = verify_layout(nseq, ndraft, vocab, draft && ndraft > 0);
  SWL_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= l.bytes,
            SWL_ERR_INVALID, "swl_verify_drafts_bf16: workspace smaller than swl_verify_drafts_workspace");
  VerifyArgs a{};
  a.tgt = reinterpret_cast<const bf16*>(target);
  a.drf = ndraft > 0 ? reinterpret_cast<const bf16*>(draft) : nullptr;
  a.ld_t = ld_target;
  a.ld_d = ld_draft;
  a.vocab = vocab;
  a.T = ndraft;
  a.ids = draft_ids;
  a.cu = cu_drafts;
  a.temp = temperature;
  a.u = u_accept;
  a.u_last = u_final;
  a.tok = out_tokens;
  a.acc = out_accepted;
  a.nseq = nseq;
  a.per = (int32_t)(ndraft / nseq);
  a.max_drafts = max_drafts;
  a.stats = (int32_t)l.stats;
  a.slices = (int32_t)l.slices;
  a.share = l.share;
  char* ws = reinterpret_cast<char*>(workspace);
  a.stat = reinterpret_cast<RowStat*>(ws);
  a.sum = reinterpret_cast<ShareSum*>(ws + l.sum);
  a.pow = reinterpret_cast<double*>(ws + l.pow);
  a.done = reinterpret_cast<uint32_t*>(ws + l.done);
  return launch_verify(a, (hipStream_t)stream);
}
