// Attention for a batch whose sequences share a prefix, over bf16 pages.
//
// Sequences come in groups; the sequences of a group share the group's prefix
// tokens (a page table row and a length of their own) and go on in pages of their
// own.  out_i = sum_j softmax_j(scale q_i . k_j) v_j, j over the prefix and the
// sequence's own tokens up to i.
//
// Rows are (new token, query head) pairs of one kv head, row = token * G + head.
// A prefix is walked once for the rows of all its sequences together, a
// sequence's own tokens for its rows alone, and what the two leave (a row's
// maximum, its sum of probabilities and the mean of values under them, fp32) is
// merged.  A sequence with a block of rows to itself (128: a prompt) gains nothing
// from company: it walks its prefix and its own tokens in one go and is not
// merged.
//
// One workgroup of the first launch makes the plan while the others rotate and
// store the new tokens: how many keys a part has (as many as let all parts run at
// once), and for every part (block of 128 rows, kv head, steps of 64 keys) what
// it needs to know, 64 bytes that a workgroup of the second launch reads with one
// load.  The host knows none of the lengths, so a captured call follows them.
//
// Measured on an MI355X (32 query heads over 8, replayed in a graph), with the bytes
// or operations that a pass cannot do without at the rates of a large copy (5.2
// TB/s) and a large bf16 product (1108 TFLOP/s):
//   4 tokens behind 700                  17.0 us (0.6): three launches, each a chain
//                                        of loads that wait for one another
//   32 tokens behind 4096, 0.5 K own     31.7 us (12.7): traced start 7.2, parts 18.6,
//                                        merge 6.2
//   48 tokens, 6 prefixes up to 12000    65 us (48): the pages' stream
//   28 sequences' drafts behind 8191     48.5 us (20)
//   12 prompts up to 1024 behind 8000    712-732 us (526): 796-818 TFLOP/s
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <cmath>

#include "dev_util.h"
#include "swl.h"
#include "swl_common.h"

namespace {

constexpr int kD = 128;         // head dim
constexpr int kRows = 128;      // rows of a block
constexpr int kKeys = 64;       // keys of a step
// rows of a block whose keys its waves share out, 16 each of a step (a wave's registers
// hold the results of two sets of 16 rows)
constexpr int kFew = 32;
constexpr int kMaxEntries = 1024;
constexpr int kCus = 256;       // of an MI355X
constexpr int kPerCu = 2;       // workgroups of a CU (LDS, registers)
constexpr int kSlots = kCus * kPerCu;
// Steps of a part at least (blocks of many rows: half of it).  4 tokens behind 700:
// 18.0 us at 3, 18.7 at 4, 20.1 at 6, 21.4 at 8; 32 tokens behind 4096: 34.1, 33.5,
// 33.8, 33.3; 28 sequences' drafts 52.4, 51.5, 50.9, 51.4.
constexpr int kMinSteps = 4;
// Shares of more steps than kLong are cut into kCuts: places do not end together.  12
// prompts over 1, 2, 3, 4 and 5 times the places 867, 844, 773, 782, 785 us; but 48
// tokens, whose shares are short, 67.8, 72.6, 74.2, 84, 84.
constexpr int kLong = 32;
constexpr int kCuts = 3;
constexpr int kKinds = 8;       // of parts, by their work: the ones with the most start first

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

// What a workgroup of the attention needs to know of its part.
struct Part {
  int32_t tok0;     // first token, or its place in the list of tokens
  int32_t n;        // tokens
  int32_t r0;       // first row of the block
  int32_t st0, nst; // steps: the prefix's, then the own tokens'
  int32_t pre;      // steps of the prefix
  int32_t seq, group;
  int32_t len, plen;  // own tokens before the new ones, tokens of the prefix
  int32_t flags;    // kListed, kDirect
  int32_t pad;
  int64_t rec;      // record of row 0 of the block's tokens, kv head 0
  int64_t head;     // records between kv heads
};
constexpr int kListed = 1;  // tokens are in the list
constexpr int kDirect = 2;  // the part is all there is of its rows
static_assert(sizeof(Part) == 64, "one load of 16 dwords");

// Where the records of a sequence's rows are: parts of its own tokens, and of the
// group's prefix.
struct SeqRec {
  int64_t own, own_head, pre, pre_head;
  int32_t own_rows, own_parts, pre_rows, pre_parts;
  int32_t t0, n;
  int32_t pad[2];
};
static_assert(sizeof(SeqRec) == 64, "");

struct PrefixArgs {
  const bf16* q;        // [T, hq, 128], token stride qs (rotated)
  const bf16* q_in;     // before the rotation
  const bf16* k;        // [T, hkv, 128]
  const bf16* v;
  int64_t qs, q_in_s, ks, vs;
  bf16* qrot;           // [T, hq * 128] or null
  bf16* kc;             // [num_blocks, bs, hkv, 128]
  bf16* vc;
  const int32_t* pt;    // [ngroups, max_pre]
  const int32_t* plens;
  const int32_t* cg;    // [ngroups + 1], null: one group
  const int32_t* bt;    // [nseq, max_blocks]
  const int32_t* lens;
  const int32_t* cu;    // [nseq + 1], null: L tokens each
  const int64_t* pos;
  const bf16* cs;       // [max_pos, 128]
  bf16* out;            // [T, hq * 128]
  int64_t max_pre, max_blocks, max_pos, T;
  int32_t num_blocks;
  int32_t nseq, ngroups, L, hq, hkv, G, bs;
  int32_t kmax, pmax;   // keys of the tables
  FastDiv by_g, by_hkv, by_bs, by_l;
  float scale;
  // workspace
  int32_t* n_parts;     // [1] parts of the plan (of one kv head)
  Part* part;           // [max_parts]
  SeqRec* seq;          // [nseq]
  int32_t* list;        // [T] tokens of the sequences that share their prefix, group by group
  float* rec_o;         // [max_rec][128]
  float* rec_ml;        // [max_rec][2]
  int64_t max_rec;
  int32_t max_parts;
  int32_t slots, min_steps;  // parts that run at once, steps of a part at least
  int32_t rows_wg;      // rows of a workgroup of the merge
};

// First token and number of tokens of sequence s (offsets that are none: nothing).
__device__ __forceinline__ void tokens_of(const PrefixArgs& a, int s, int& t0, int& n) {
  t0 = a.cu ? a.cu[s] : s * a.L;
  n = a.cu ? a.cu[s + 1] - t0 : a.L;
  if (t0 < 0 || n < 0 || (int64_t)t0 + n > a.T) t0 = n = 0;
}
__device__ __forceinline__ int steps_of(int keys) { return (keys + kKeys - 1) / kKeys; }

// A lane's value from a lane below it (DPP; 0 where there is none).
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T below(T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
  } else {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)v >> 32), CTRL, ROWS, 0xF, false);
    return (T)((uint64_t)hi << 32 | lo);
  }
}
// Sums over the lanes up to each: in rows of 16, then across them.
template <typename T>
__device__ __forceinline__ T wave_prefix(T v) {
  v += below<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += below<0x112, 0xF>(v);
  v += below<0x114, 0xF>(v);
  v += below<0x118, 0xF>(v);
  v += below<0x142, 0xA>(v);  // row_bcast 15, 31
  return v + below<0x143, 0xC>(v);
}
// Exclusive prefix over the 256 threads; `all` the sum.
template <typename T>
__device__ __forceinline__ T block_prefix(T v, T* sh, T& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T inc = wave_prefix(v);
  __syncthreads();
  if (lane == 63) sh[w] = inc;
  __syncthreads();
  T before = 0;
  for (int i = 0; i < w; ++i) before += sh[i];
  all = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  return before + inc - v;
}

struct PlanLds {  // of E = ngroups + nseq entries: the groups' prefixes, then the sequences
  int64_t* rec;   // [E] first record
  int32_t* rows;  // [E]
  int32_t* steps; // [E]
  int32_t* pre;   // [E] of them, the prefix's
  int32_t* first; // [E] first part
  int32_t* parts; // [E] of a block of its rows
  int32_t* len;   // [E] tokens of the prefix; own tokens before the new ones
  int32_t* few;   // [nseq + 1] tokens before it that share their prefix
  int32_t* t0;    // [nseq] first token
  int32_t* cg;    // [ngroups + 1] first sequence, in range
};
constexpr int kPlanEntry = 8 + 9 * 4;

__device__ void make_plan(const PrefixArgs& a, char* lds) {
  __shared__ int64_t sh64[4];
  __shared__ int32_t sh32[4];
  __shared__ float shf[4];
  __shared__ int32_t kind[kKinds], at_kind[kKinds];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int ng = a.ngroups, ns = a.nseq, E = ng + ns;
  PlanLds l;
  l.rec = reinterpret_cast<int64_t*>(lds);
  l.rows = reinterpret_cast<int32_t*>(l.rec + E);
  l.steps = l.rows + E;
  l.pre = l.steps + E;
  l.first = l.pre + E;
  l.parts = l.first + E;
  l.len = l.parts + E;
  l.few = l.len + E;
  l.t0 = l.few + ns + 1;
  l.cg = l.t0 + ns;

  for (int g = tid; g <= ng; g += 256) {
    l.cg[g] = a.cg ? min(max(a.cg[g], 0), ns) : g > 0 ? ns : 0;
    if (g < ng) l.len[g] = min(max(a.plens[g], 0), a.pmax);
  }
  for (int s = tid; s < ns; s += 256) {
    int t0, n;
    tokens_of(a, s, t0, n);
    l.t0[s] = t0;
    l.rows[ng + s] = n * a.G;
    l.len[ng + s] = min(a.lens[s], 1 << 30);
  }
  __syncthreads();
  auto group_of = [&](int s) {  // -1: none
    int lo = 0, hi = ng;        // the last g with cg[g] <= s
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (l.cg[mid] <= s)
        lo = mid;
      else
        hi = mid;
    }
    return ng > 0 && l.cg[lo] <= s && s < l.cg[lo + 1] ? lo : -1;
  };
  // sequences: steps, and the tokens that walk their prefix in company
  int run = 0;
  for (int s0 = 0; s0 < ns; s0 += 256) {
    const int s = s0 + tid;
    int share = 0;
    if (s < ns) {
      const int g = group_of(s), plen = g >= 0 ? l.len[g] : 0, rows = l.rows[ng + s], n = (uint32_t)rows / a.by_g;
      const bool alone = rows >= kRows;
      const int own = steps_of((int)min<int64_t>(max<int64_t>((int64_t)l.len[ng + s] + n, 0), a.kmax));
      const int pre = alone ? steps_of(plen) : 0;
      share = plen > 0 && !alone ? n : 0;
      l.pre[ng + s] = pre;
      l.steps[ng + s] = max(own + pre, 1);
    }
    int all;
    const int at = run + block_prefix(share, sh32, all);
    if (s < ns) l.few[s] = at;
    run += all;
  }
  if (tid == 0) l.few[ns] = run;
  __syncthreads();
  for (int g = tid; g < ng; g += 256) {
    const int s0 = l.cg[g], s1 = max(l.cg[g + 1], s0);
    const int n = l.few[s1] - l.few[s0], st = n > 0 ? steps_of(l.len[g]) : 0;
    l.rows[g] = st > 0 ? n * a.G : 0;
    l.steps[g] = l.pre[g] = max(st, 1);
  }
  __syncthreads();

  // Steps of a part: as many as give every place its share of all the work, at
  // least min_steps; a step of a block of many rows counts twice.  Long shares are
  // cut into kCuts, as the places do not end together and a step costs much more
  // than what a part adds.  So there are at most slots, or kCuts * slots, full
  // parts, whatever the lengths are.
  float sum = 0.f;
  for (int e = tid; e < E; e += 256) {
    const int rows = l.rows[e];
    sum += (float)((rows + kRows - 1) / kRows) * (float)l.steps[e] * (rows > kFew ? 2.f : 1.f);
  }
  sum = wave_prefix(sum);
  if (lane == 63) shf[w] = sum;
  __syncthreads();
  // (rounded up past what the sums' roundings may have lost)
  sum = ((shf[0] + shf[1]) + (shf[2] + shf[3])) * 1.0001f * (float)a.hkv;
  const int whole = (int)fminf(sum / (float)a.slots + 1.f, 1073741824.f);
  const int share = max(a.min_steps, max((whole + kCuts - 1) / kCuts, min(whole, kLong)));
  auto steps_per_part = [&](int e) { return l.rows[e] > kFew ? (share + 1) >> 1 : share; };

  // first parts and records
  int parts_run = 0;
  int64_t rec_run = 0;
  for (int e0 = 0; e0 < E; e0 += 256) {
    const int e = e0 + tid;
    int units = 0;
    int64_t recs = 0;
    if (e < E) {
      const int rows = l.rows[e], spp = steps_per_part(e), parts = (l.steps[e] + spp - 1) / spp;
      l.parts[e] = parts;
      units = (rows + kRows - 1) / kRows * parts;
      const bool joined = e < ng || l.few[e - ng + 1] > l.few[e - ng];
      recs = joined || parts > 1 ? (int64_t)rows * parts * a.hkv : 0;
    }
    int all;
    int64_t all64;
    const int at = parts_run + block_prefix(units, sh32, all);
    const int64_t rec = rec_run + block_prefix(recs, sh64, all64);
    if (e < E) {
      l.first[e] = at;
      l.rec[e] = recs ? rec : -1;
    }
    parts_run += all;
    rec_run += all64;
  }
  __syncthreads();
  const int total = min(parts_run, a.max_parts);
  if (tid == 0) a.n_parts[0] = total;
  if (tid < kKinds) kind[tid] = 0;
  for (int s = tid; s < ns; s += 256) {
    const int e = ng + s;
    SeqRec r{};
    r.t0 = l.t0[s];
    r.n = (uint32_t)l.rows[e] / a.by_g;
    if (l.rec[e] >= 0) {
      r.own = l.rec[e];
      r.own_rows = l.rows[e];
      r.own_parts = l.parts[e];
      r.own_head = (int64_t)r.own_rows * r.own_parts;
    }
    if (l.few[s + 1] > l.few[s]) {
      const int g = group_of(s);
      r.pre_rows = l.rows[g];
      r.pre_parts = l.parts[g];
      r.pre_head = (int64_t)r.pre_rows * r.pre_parts;
      r.pre = l.rec[g] + (int64_t)(l.few[s] - l.few[l.cg[g]]) * a.G;
      for (int i = 0; i < r.n && l.few[s] + i < a.T; ++i) a.list[l.few[s] + i] = r.t0 + i;
    }
    // (what lies outside the workspace, by offsets that are none, is left out)
    const int64_t own_end = r.own + r.own_head * a.hkv, pre_end = r.pre + r.pre_head * a.hkv;
    if (r.own < 0 || own_end > a.max_rec || r.pre < 0 || pre_end > a.max_rec) r.own_parts = r.pre_parts = 0;
    a.seq[s] = r;
  }
  __syncthreads();
  // The parts, the ones with the most work first: counted by kind (eighths of the
  // largest), then put where their kind begins.
  auto part_of = [&](int u, Part& o) {
    int lo_e = 0, hi_e = E;  // the last entry with parts whose first is <= u
    while (hi_e - lo_e > 1) {
      const int mid = (lo_e + hi_e) >> 1;
      if (l.first[mid] <= u)
        lo_e = mid;
      else
        hi_e = mid;
    }
    const int e = lo_e, spp = steps_per_part(e), parts = l.parts[e], rows = l.rows[e];
    const int local = u - l.first[e], b = local / parts, p = local - b * parts;
    o = Part{};
    if (local < 0 || (int64_t)b * kRows >= rows) return;  // (counts past 32 bits, by offsets that are none)
    o.r0 = b * kRows;
    o.n = (uint32_t)rows / a.by_g;
    o.st0 = p * spp;
    o.pre = l.pre[e];
    if (e < ng) {
      o.tok0 = l.few[l.cg[e]];
      o.group = e;
      o.plen = l.len[e];
      o.nst = min(spp, l.steps[e] - o.st0);
    } else {
      o.seq = e - ng;
      o.tok0 = l.t0[o.seq];
      o.len = l.len[e];
      if (o.pre > 0) {
        o.group = group_of(o.seq);
        o.plen = l.len[o.group];
      }
      // the block's own end: its last row may see fewer keys than the sequence's
      const int last = (uint32_t)(min(o.r0 + kRows, rows) - 1) / a.by_g;
      const int kend = (int)min<int64_t>(max<int64_t>((int64_t)o.len + last + 1, 0), a.kmax);
      o.nst = min(spp, o.pre + steps_of(kend) - o.st0);
    }
    o.nst = max(o.nst, 0);
    o.flags = (e < ng ? kListed : 0) | (l.rec[e] < 0 ? kDirect : 0);
    o.rec = l.rec[e] + (int64_t)p * rows;
    o.head = (int64_t)rows * parts;
  };
  auto kind_of = [&](const Part& o) {
    const int work = o.n * a.G > kFew ? 2 * o.nst : o.nst;
    return kKinds - 1 - (int)min<int64_t>((int64_t)work * kKinds / (share + 2), kKinds - 1);
  };
  Part o;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
    for (int u = tid; u < total; u += 256) {
      if (pass == 0 || total > 256) part_of(u, o);
      const int k = kind_of(o);
      if (pass == 0)
        atomicAdd(&kind[k], 1);
      else
        a.part[atomicAdd(&at_kind[k], 1)] = o;
    }
    __syncthreads();
    if (tid < kKinds) {
      int before = 0;
      for (int i = 0; i < tid; ++i) before += kind[i];
      at_kind[tid] = before;
    }
    __syncthreads();
  }
}

// The sequence of packed token t (the same for the whole wave): how many
// sequences end at or before it; nseq for a token behind the last one.
__device__ __forceinline__ int seq_of(const PrefixArgs& a, int64_t t, int lane) {
  if (!a.cu) return (int)((uint32_t)t / a.by_l);
  int s = 0;
  for (int i0 = 0; i0 < a.nseq; i0 += 64) {
    const int i = i0 + lane;
    s += __popcll(__ballot(i < a.nseq && a.cu[i + 1] <= t));
  }
  return s;
}

// Workgroup 0 makes the plan; the others rotate the new queries into the
// workspace and the new keys into the pages (NeoX, each rounded once), and store
// the values: a workgroup per (token, 32 heads), eight threads a head with
// 16-byte accesses.
__global__ __launch_bounds__(256) void prefix_start_kernel(PrefixArgs a, int heads_wg) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  if (blockIdx.x == 0) {
    make_plan(a, lds);
    return;
  }
  const int64_t t = (blockIdx.x - 1) / heads_wg;
  const int h = (int)((blockIdx.x - 1) - t * heads_wg) * 32 + (threadIdx.x >> 3);  // q, then k, then v heads
  const int nq = a.qrot ? a.hq : 0, nk = a.k ? a.hkv : 0;
  const int s = seq_of(a, t, threadIdx.x & 63);
  if (s >= a.nseq || h >= nq + 2 * nk) return;
  const int d = 8 * (threadIdx.x & 7);
  const bool is_q = h < nq, is_k = !is_q && h < nq + nk;
  const int kvh = is_k ? h - nq : h - nq - nk;
  const bf16* row = (is_q ? a.q_in + t * a.q_in_s + h * kD : is_k ? a.k + t * a.ks + kvh * kD : a.v + t * a.vs + kvh * kD) + d;
  u32x4 w1 = ldg16(row), w2 = ldg16(row + 64);
  const int64_t pos = a.pos ? a.pos[t] : -1;
  if ((is_q || is_k) && pos >= 0 && pos < a.max_pos) {
    const bf16* cs = a.cs + pos * kD + d;
    float x1[8], x2[8], co[8], sn[8];
    unpack8(ldg16(cs), co);
    unpack8(ldg16(cs + 64), sn);
    unpack8(w1, x1);
    unpack8(w2, x2);
    bf16x8 o1, o2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // (products of two bf16 are exact: one rounding before the last)
      o1[e] = f2bf(x1[e] * co[e] - x2[e] * sn[e]);
      o2[e] = f2bf(x2[e] * co[e] + x1[e] * sn[e]);
    }
    w1 = __builtin_bit_cast(u32x4, o1);
    w2 = __builtin_bit_cast(u32x4, o2);
  }
  bf16* dst;
  if (is_q) {
    dst = a.qrot + (t * a.hq + h) * kD + d;
  } else {
    int t0, n;
    tokens_of(a, s, t0, n);
    const int64_t i = t - t0, p = (int64_t)a.lens[s] + i;
    if (i < 0 || i >= n || p < 0 || p >= a.kmax) return;
    const uint32_t bi = (uint32_t)p / a.by_bs;
    const int32_t blk = a.bt[(int64_t)s * a.max_blocks + bi];
    if (blk < 0 || blk >= a.num_blocks) return;
    dst = (is_k ? a.kc : a.vc) + (((int64_t)blk * a.bs + ((uint32_t)p - bi * a.bs)) * a.hkv + kvh) * kD + d;
  }
  *reinterpret_cast<u32x4*>(dst) = w1;
  *reinterpret_cast<u32x4*>(dst + 64) = w2;
}

// ------------------------------------------------------------- attention ---
__device__ __forceinline__ float max_groups(float v) {  // over the four lane groups
  const uint32_t x = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t y = __float_as_uint(v);
  auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// e^(m - M) in powers of two; a side without a key (-inf) counts for nothing.
__device__ __forceinline__ float merge_factor(float m, float M) {
  return m == M ? (m == -INFINITY ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - M);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// 4 x 16 values turned: of the 16 lanes, lane i gives the address of 4 values of
// row i / 4 and gets column i of all four rows.
__device__ __forceinline__ u32x2 turned(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p)));
}

__device__ __forceinline__ f32x4 mfma16k16(u32x2 a, u32x2 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}

// Token i of a part.  The list holds T tokens: where offsets that overlap make the
// sequences' tokens more than that (each sequence's lie in 0 .. T - 1 all the same),
// the last one stands for those that found no place.
__device__ __forceinline__ int token_at(const PrefixArgs& a, const Part& u, int i) {
  return u.flags & kListed ? a.list[min(u.tok0 + i, (int)a.T - 1)] : u.tok0 + i;
}

// Where a block of keys is: the prefix's pages or the sequence's.
struct Keys {
  const int32_t* table;
  int first, end;  // first key of the step, keys that some row sees
};
__device__ __forceinline__ Keys keys_of(const PrefixArgs& a, const Part& u, int st, int kend) {
  const bool pre = st < u.pre;
  return Keys{pre ? a.pt + (int64_t)u.group * a.max_pre : a.bt + (int64_t)u.seq * a.max_blocks,
              (pre ? st : st - u.pre) * kKeys, pre ? u.plen : kend};
}

// One row of a part by a wave, seeing its own keys alone: sixteen lanes a key (8
// dims each), four keys at a time.  For rows that an infinity or a NaN of a key they
// do not see may have reached (0 times it is a NaN), and those whose scores are past
// what is subtracted of them.
// acc: sums of the values times `by`.  Whether it sees a key.
__device__ bool slow_sums(const PrefixArgs& a, const Part& u, int h, int kend, int r, int lane, float by, float& mx,
                          float& sm, float (&acc)[8]) {
  bool seen = false;
  const int i = (uint32_t)r / a.by_g;
  const bf16* qp = a.q + (int64_t)token_at(a, u, i) * a.qs + (int64_t)(h * a.G + r - i * a.G) * kD + 8 * (lane & 15);
  const float c2 = a.scale * 1.44269504088896340736f;
  float q[8];
  unpack8(ldg16(qp), q);
  mx = -INFINITY;
  sm = 0.f;
#pragma unroll
  for (int d = 0; d < 8; ++d) acc[d] = 0.f;
#pragma unroll 1
  for (int st = u.st0; st < u.st0 + u.nst; ++st) {
    const Keys ks = keys_of(a, u, st, kend);
    const int end = st < u.pre ? ks.end : min(ks.end, (int)max((int64_t)u.len + i + 1, (int64_t)0));
#pragma unroll 1
    for (int key = ks.first + (lane >> 4); key < min(ks.first + kKeys, end); key += 4) {
      const uint32_t bi = (uint32_t)key / a.by_bs;
      const int32_t blk = ks.table[bi];
      if (blk < 0 || blk >= a.num_blocks) continue;
      seen = true;
      const int64_t at = (((int64_t)blk * a.bs + (key - bi * a.bs)) * a.hkv + h) * kD + 8 * (lane & 15);
      float kf[8], vf[8], sc = 0.f;
      unpack8(ldg16(a.kc + at), kf);
      unpack8(ldg16(a.vc + at), vf);
#pragma unroll
      for (int d = 0; d < 8; ++d) sc += q[d] * kf[d];
#pragma unroll
      for (int o = 8; o >= 1; o >>= 1) sc += __shfl_xor(sc, o, 16);
      {  // rounded before the largest is subtracted of it, as that is (not one fma with it)
#pragma clang fp contract(off)
        sc *= c2;
      }
      const float nm = fmaxf(mx, sc), corr = merge_factor(mx, nm), p = __builtin_amdgcn_exp2f(sc - (nm == -INFINITY ? 0.f : nm));
      sm = sm * corr + p;
#pragma unroll
      for (int d = 0; d < 8; ++d) acc[d] = acc[d] * corr + p * (vf[d] * by);
      mx = nm;
    }
  }
  for (int o = 16; o <= 32; o += 16) {
    const float mo = __shfl_xor(mx, o, 64), so = __shfl_xor(sm, o, 64), nm = fmaxf(mx, mo);
    const float ca = merge_factor(mx, nm), cb = merge_factor(mo, nm);
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] = acc[d] * ca + __shfl_xor(acc[d], o, 64) * cb;
    sm = sm * ca + so * cb;
    mx = nm;
  }
  return __ballot(seen) != 0;
}

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }  // (0: no key)

// mean: the row's result.  Where sums of large values are no 32-bit numbers though
// their means are (2^31 keys at most), the sums are those of 2^-32 of them.  A row
// whose keys all have the score -inf has no weight (sm 0) and, which tells it from one
// without a key, a NaN as its maximum: what it sees elsewhere is its result, or else
// a NaN.
__device__ void slow_row(const PrefixArgs& a, const Part& u, int h, int kend, int r, int lane, float& mx, float& sm,
                         float (&mean)[8]) {
  const bool seen = slow_sums(a, u, h, kend, r, lane, 1.f, mx, sm, mean);
  const float inv = inverse(sm), max_or_nan = sm == 0.f && seen ? NAN : mx;
  bool large = false;
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    large |= not_finite(mean[d]);
    mean[d] *= inv;
  }
  mx = max_or_nan;
  if (__ballot(large) == 0) return;
  float of_part[8], mx_again;
  slow_sums(a, u, h, kend, r, lane, 0x1p-32f, mx_again, sm, of_part);
#pragma unroll
  for (int d = 0; d < 8; ++d)
    if (not_finite(mean[d])) mean[d] = of_part[d] * inv * 0x1p32f;
}

// K dims from d of a row's result, o * inv: to the output where the part is all
// there is of it, else to its record.  Records hold means: what is merged of them
// is no larger than they are.
template <int K>
__device__ __forceinline__ void put_row(const PrefixArgs& a, const Part& u, int h, int r, int d, float m, float L,
                                        const float (&o)[K], float inv) {
  if (u.flags & kDirect) {
    const int i = (uint32_t)r / a.by_g;
    bf16* dst = a.out + ((int64_t)token_at(a, u, i) * a.hq + h * a.G + r - i * a.G) * kD + d;
    bf16x2 y[K / 2];  // (m a NaN: keys, but none of any weight; a row without a key has zeros)
#pragma unroll
    for (int e = 0; e < K / 2; ++e)
      y[e] = m != m ? bf16x2{f2bf(m), f2bf(m)} : bf16x2{f2bf(o[2 * e] * inv), f2bf(o[2 * e + 1] * inv)};
#pragma unroll
    for (int e = 0; e < K / 4; ++e)
      stg(dst + 4 * e, u32x2{__builtin_bit_cast(uint32_t, y[2 * e]), __builtin_bit_cast(uint32_t, y[2 * e + 1])});
  } else {
    const int64_t at = u.rec + h * u.head + r;
    if (at < 0 || at >= a.max_rec) return;  // (only where offsets are none)
    float* dst = a.rec_o + at * kD + d;
#pragma unroll
    for (int e = 0; e < K; e += 4)
      *(__attribute__((address_space(1))) f32x4*)(dst + e) = f32x4{o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv};
    if (d == 0) {
      a.rec_ml[2 * at] = m;
      a.rec_ml[2 * at + 1] = L;
    }
  }
}

// 16 bytes a lane from global memory to LDS at `to` (the same for the wave) + 16
// lane.  The compiler puts a wait for all of these before every turned read, also
// of the other buffer (it does not for the builtin's plain reads), so they are
// issued past it: no register is written, wait_dma is the wait.  m0 is left as it was:
// the compiler does not know that it is written (it takes it for reserved, and warns of
// it as a clobber).
__device__ __forceinline__ void dma16(const char* from, char* to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr)to);
  uint32_t was;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(was)
               : "v"((gbl_ptr)from), "s"(at)
               : "memory");
}
// (the builtin, so that the compiler knows its own loads to be there as well)
__device__ __forceinline__ void wait_dma() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kWaitVm0);
  asm volatile("" ::: "memory");
}

// A part by a workgroup of four waves.  Keys and values of a step go from the
// pages to LDS (16 bytes a lane, no register between), a step ahead: wave w
// fetches keys 16 w .. + 15 of the step.  In LDS a key's 16-byte piece c is at
// place c ^ (key % 16), so that reading one piece of 16 keys, and turning 4 keys x
// 16 dims, meet every bank alike.  S^T = K Q^T leaves in a lane keys 4 g .. + 3 of
// each 16 of its row (g = lane / 16), which is the B operand of O^T = V^T P^T as
// it is; the turned read gives V^T with the same keys.
//
// MANY: a wave takes 32 of the block's 128 rows over all 64 keys.  Otherwise the
// block has at most 32 rows, which every wave takes over the 16 keys it fetched,
// without a barrier, and the waves' results meet in LDS.
//
// Two workgroups fit a CU, and a SIMD has a wave of each.  Of the busy CUs' time the
// matrix units take 42 % in a step of many rows and the vector units about as much;
// the two hardly overlap, and more waves do not make them.  Measured against this, 12
// prompts at 779 us: 256 rows a block by eight waves over a ring of four steps 847,
// the same with 32 x 32 products 803, the halves of a workgroup of eight waves
// taking turns at products and exponents, a barrier between, 873; and, at 755, eight
// waves of 16 rows each, four a SIMD, 776 (48 tokens 64 -> 85).
constexpr int kStepBytes = kKeys * kD * 2;  // keys, or values, of a step

struct AttnLds {
  char kv[2][2][kStepBytes];  // [step % 2][keys, values]
  uint32_t none[2][4];        // of a wave's 16 keys, those without a page
};

template <bool MANY, int SETS>
__device__ __forceinline__ void attend_part(const PrefixArgs& a, const Part& u, int h, AttnLds& sh) {
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = u.n * a.G, wr0 = u.r0 + (MANY ? 32 * w : 0);
  const int last = (uint32_t)(min(u.r0 + kRows, rows) - 1) / a.by_g;
  const int kend = (int)min<int64_t>(max<int64_t>((int64_t)u.len + last + 1, 0), a.kmax);  // of the own tokens
  const int all_see = max(min(u.len + (int)((uint32_t)u.r0 / a.by_g) + 1, kend), 0);       // those that every row sees
  const bool idle = wr0 >= rows;  // the wave has no row
  // Keys of the part that a row with `see` own ones sees (those without a page among
  // them), and whether the sum l of such a row's probabilities is not to be trusted:
  // the key of the largest score has a probability of about 1, unless scores are past
  // 2^31 and what is subtracted of them is rounded so far from theirs that it has none.
  auto no_sum = [&](float l, int see) {
    const int own0 = max(u.st0 - u.pre, 0) * kKeys;
    return l < 0x1p-60f && u.nst > 0 && (u.st0 < u.pre || (u.st0 + u.nst > u.pre && see > own0));
  };

  // Row of the pages that holds the lane's key of a step (key 16 w + col), and
  // the wave's keys that have none.  Keys past the last are the last one.
  auto block_of = [&](int st) {
    const Keys ks = keys_of(a, u, st, kend);
    const int key = min(ks.first + 16 * w + col, ks.end - 1);
    return ks.table[(uint32_t)key / a.by_bs];
  };
  auto row_of = [&](int st, int32_t blk, uint32_t& none) {
    const Keys ks = keys_of(a, u, st, kend);
    const int key = min(ks.first + 16 * w + col, ks.end - 1);
    const bool there = blk >= 0 && blk < a.num_blocks;
    none = (uint32_t)__ballot(!there) & 0xffffu;
    return there ? blk * a.bs + (int)((uint32_t)key - (uint32_t)key / a.by_bs * (uint32_t)a.bs) : 0;
  };
  // (16 bytes of four keys an instruction: lane i of it has place i % 16 of key i / 16)
  const uint32_t row_bytes = (uint32_t)a.hkv * (kD * 2), lane_at = (uint32_t)h * (kD * 2) + 16 * (col ^ g);
  const char *kc = reinterpret_cast<const char*>(a.kc), *vc = reinterpret_cast<const char*>(a.vc);
  auto fetch = [&](int row, int buf) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (4 * i + g), row);
      const uint64_t at = (uint64_t)r * row_bytes + (lane_at ^ (uint32_t)(64 * i));
      dma16(kc + at, sh.kv[buf][0] + (16 * w + 4 * i) * 256);
      dma16(vc + at, sh.kv[buf][1] + (16 * w + 4 * i) * 256);
    }
  };

  const int st_end = u.st0 + u.nst;
  uint32_t none = 0, none_next = 0;
  bool there = false;  // some key of the part has a page
  int32_t blk = 0;
  if (u.nst > 0) {
    blk = block_of(u.st0);
    const int row = row_of(u.st0, blk, none);
    fetch(row, 0);
    if (MANY && lane == 0) sh.none[0][w] = none;
    if (u.nst > 1) blk = block_of(u.st0 + 1);
  }

  u32x4 q[SETS][4];
  int see[SETS];  // own tokens that the lane's rows see
#pragma unroll
  for (int e = 0; e < SETS; ++e) {
    const int r = min(wr0 + e * 16 + col, rows - 1), i = (uint32_t)r / a.by_g;
    const bf16* qp = a.q + (int64_t)token_at(a, u, i) * a.qs + (int64_t)(h * a.G + r - i * a.G) * kD + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) q[e][s] = ldg16(qp + 32 * s);
    see[e] = min(max(u.len + i + 1, 0), kend);
  }
  const float c2 = a.scale * 1.44269504088896340736f;  // scores in powers of two
  float m[SETS];
  f32x4 l[SETS], acc[SETS][8];  // (l: of a product with ones, four times the same)
#pragma unroll
  for (int e = 0; e < SETS; ++e) {
    m[e] = -INFINITY;
    l[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[e][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  wait_dma();
  if (MANY) lds_barrier();

  constexpr int T = MANY ? 4 : 1;  // tiles of 16 keys of the wave
  const int t0 = MANY ? 0 : w;
  for (int st = u.st0; st < st_end; ++st) {
    const int buf = (st - u.st0) & 1;
    if (st + 1 < st_end) {
      const int row = row_of(st + 1, blk, none_next);
      if (st + 2 < st_end) blk = block_of(st + 2);
      fetch(row, buf ^ 1);
      if (MANY && lane == 0) sh.none[buf ^ 1][w] = none_next;
    }
    const char* kv = sh.kv[0][0];
    if (!idle) {
      // K: 16 bytes of key col of a tile, dims 32 k + 8 g ..
      const uint32_t k_at = buf * 32768 + t0 * 4096 + col * 256 + ((g ^ col) << 4);
      f32x4 s[SETS][T];
#pragma unroll
      for (int t = 0; t < T; ++t) {
#pragma unroll
        for (int e = 0; e < SETS; ++e) s[e][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const u32x4 kf = *reinterpret_cast<const u32x4*>(kv + (k_at ^ (64 * k)) + t * 4096);
#pragma unroll
          for (int e = 0; e < SETS; ++e) s[e][t] = mfma16(kf, q[e][k], s[e][t]);
        }
      }
      // keys that some row does not see
      uint64_t gone = none;
      if (MANY)
        gone = (uint64_t)(sh.none[buf][3] << 16 | sh.none[buf][2]) << 32 | (sh.none[buf][1] << 16 | sh.none[buf][0]);
      there |= gone != (MANY ? ~(uint64_t)0 : 0xffffu);
      const bool pre = st < u.pre;
      const int first = (pre ? st : st - u.pre) * kKeys;
      if (first + kKeys > (pre ? u.plen : all_see) || gone != 0) {
#pragma unroll
        for (int e = 0; e < SETS; ++e) {
          const int end = (pre ? u.plen : see[e]) - first;
#pragma unroll
          for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (16 * (t0 + t) + 4 * g + i >= end || (gone >> (16 * t + 4 * g + i) & 1)) s[e][t][i] = -INFINITY;
        }
      }
      u32x2 p[SETS][T];
#pragma unroll
      for (int e = 0; e < SETS; ++e) {
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < T; ++t) mx = fmaxf(mx, fmaxf(fmaxf(s[e][t][0], s[e][t][1]), fmaxf(s[e][t][2], s[e][t][3])));
        // the reference the exponents are taken from moves only when the maximum
        // has grown by 2^8 since: any reference gives the same quotient
        if (__ballot(mx * c2 > m[e] + 8.f) != 0) {
          const float mn = fmaxf(m[e], c2 * max_groups(mx)), corr = mn == m[e] ? 1.f : __builtin_amdgcn_exp2f(m[e] - mn);
          m[e] = mn;
          l[e] *= corr;
#pragma unroll
          for (int d = 0; d < 8; ++d) acc[e][d] *= corr;
        }
        const float mr = m[e] == -INFINITY ? 0.f : m[e];
#pragma unroll
        for (int t = 0; t < T; ++t) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e][t][i], c2, -mr));
          const bf16x2 lo = {f2bf(x[0]), f2bf(x[1])}, hi = {f2bf(x[2]), f2bf(x[3])};
          p[e][t] = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
        }
      }
      // The sums of the probabilities (as rounded: then the weights sum to 1) are
      // products with ones: the vector units, not the matrix ones, are what a step of
      // many rows waits for.
      const uint32_t one = 0x3f803f80u;
#pragma unroll
      for (int e = 0; e < SETS; ++e) {
        if constexpr (MANY) {
#pragma unroll
          for (int t = 0; t < 4; t += 2)
            l[e] = mfma16(u32x4{one, one, one, one}, u32x4{p[e][t][0], p[e][t][1], p[e][t + 1][0], p[e][t + 1][1]}, l[e]);
        } else {
          l[e] = mfma16k16(u32x2{one, one}, p[e][0], l[e]);
        }
      }
      // V^T: of four keys 4 g + (lane / 4) % 4 ..., dims 32 c + 4 (d ^ c % 2) .. + 3, c = lane % 4
      const int c = lane & 3, key = 4 * g + (col >> 2);
      const uint32_t v_at = buf * 32768 + 16384 + key * 256 + (((4 * c) ^ key) << 4) + 8 * (c & 1);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const char* vp = kv + (v_at ^ (8 * d));
        if constexpr (MANY) {
#pragma unroll
          for (int t = 0; t < 4; t += 2) {
            const u32x2 v0 = turned(vp + t * 4096), v1 = turned(vp + (t + 1) * 4096);
#pragma unroll
            for (int e = 0; e < SETS; ++e)
              acc[e][d] = mfma16(u32x4{v0[0], v0[1], v1[0], v1[1]}, u32x4{p[e][t][0], p[e][t][1], p[e][t + 1][0], p[e][t + 1][1]},
                                 acc[e][d]);
          }
        } else {
          const u32x2 v0 = turned(vp + t0 * 4096);
#pragma unroll
          for (int e = 0; e < SETS; ++e) acc[e][d] = mfma16k16(v0, p[e][0], acc[e][d]);
        }
      }
    }
    none = none_next;
    if (MANY) {
      wait_dma();     // the next step is there
      lds_barrier();  // for all waves, and this one read by all
    } else {
      wait_dma();
      __builtin_amdgcn_s_waitcnt(0xC07F);  // (lgkmcnt 0: this one is read)
      asm volatile("" ::: "memory");
    }
  }

  // Rows in order by way of LDS: 128 dims (the lane has 32 g + 4 (d ^ g % 2) .. + 3
  // in acc[d]), maximum, sum.
  constexpr int F = 132;
  float* mg = reinterpret_cast<float*>(sh.kv);
  static_assert(4 * 16 * F * 4 <= (int)sizeof(sh.kv), "the waves' rows");
  auto leave = [&](int e) {
    float* dst = mg + (w * 16 + col) * F;
#pragma unroll
    for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(dst + 32 * g + 4 * (d ^ (g & 1))) = acc[e][d];
    if (g == 0) {
      dst[128] = m[e];
      dst[129] = l[e][0];
      dst[130] = MANY ? inverse(l[e][0]) : there ? 1.f : 0.f;
    }
  };
  auto again = [&](int r) {
    float mx, sm, y[8];
    slow_row(a, u, h, kend, r, lane, mx, sm, y);
    if (lane < 16) put_row<8>(a, u, h, r, 8 * lane, mx, sm, y, 1.f);
  };
  if constexpr (MANY) {  // every wave its own, 32 lanes a row
    if (idle) return;
#pragma unroll
    for (int e = 0; e < SETS; ++e) {
      const int r0 = wr0 + 16 * e;
      bool bad = not_finite(l[e][0]) || (there && no_sum(l[e][0], see[e]));
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= not_finite(acc[e][d][i]);
      uint64_t redo = __ballot(bad && r0 + col < rows);
      redo = (redo | redo >> 16 | redo >> 32 | redo >> 48) & 0xffffu;
      leave(e);
      __builtin_amdgcn_s_waitcnt(0xC07F);
      asm volatile("" ::: "memory");
      const int d = 4 * (lane & 31);
#pragma unroll 4
      for (int i = lane >> 5; i < 16; i += 2) {
        const float* src = mg + (w * 16 + i) * F;
        const f32x4 v = *reinterpret_cast<const f32x4*>(src + d);
        const float o[4] = {v[0], v[1], v[2], v[3]};
        if (r0 + i < rows && !(redo >> i & 1)) put_row<4>(a, u, h, r0 + i, d, src[128], src[129], o, src[130]);
      }
      for (; redo; redo &= redo - 1) again(r0 + __builtin_ctzll(redo));
      __builtin_amdgcn_s_waitcnt(0xC07F);
      asm volatile("" ::: "memory");
    }
  } else {  // the waves' shares of a row merged
#pragma unroll
    for (int e = 0; e < SETS; ++e) {
      const int nr = min(rows - u.r0 - 16 * e, 16);
      if (nr <= 0) return;  // the same for the whole workgroup
      __syncthreads();
      leave(e);
      __syncthreads();
      const int row = threadIdx.x >> 4, x8 = 8 * (threadIdx.x & 15);
      float M = -INFINITY, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      bool bad = false;
      if (row < nr) {
#pragma unroll
        for (int v = 0; v < 4; ++v) M = fmaxf(M, mg[(v * 16 + row) * F + 128]);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float* src = mg + (v * 16 + row) * F;
          const float f = merge_factor(src[128], M);
          L += src[129] * f;
#pragma unroll
          for (int d = 0; d < 8; ++d) o[d] += src[x8 + d] * f;
        }
        bad = not_finite(L);
#pragma unroll
        for (int d = 0; d < 8; ++d) bad |= not_finite(o[d]);
        if (L < 0x1p-60f) {
          float some = 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) some += mg[(v * 16 + row) * F + 130];
          const int i = (uint32_t)(u.r0 + 16 * e + row) / a.by_g;
          bad |= some != 0.f && no_sum(L, min(max(u.len + i + 1, 0), kend));
        }
      }
      const uint64_t redo = __ballot(bad);
      if (row < nr && (redo >> (lane & 48) & 0xffffu) == 0)
        put_row<8>(a, u, h, u.r0 + 16 * e + row, x8, M, L, o, inverse(L));
      for (int i = 0; i < 4; ++i)  // the wave's four rows
        if (redo >> (16 * i) & 0xffffu) again(u.r0 + 16 * e + 4 * w + i);
    }
  }
}

__global__ __launch_bounds__(256, kPerCu) void prefix_attention_kernel(PrefixArgs a) {
  __shared__ __attribute__((aligned(16))) AttnLds sh;
  const uint32_t p = blockIdx.x / a.by_hkv;
  const int h = (int)(blockIdx.x - p * (uint32_t)a.hkv);
  if ((int)p >= a.n_parts[0]) return;
  const Part u = a.part[p];
  const int rows = u.n * a.G - u.r0;
  if (rows <= 0) return;
  if (rows <= 16)
    attend_part<false, 1>(a, u, h, sh);
  else if (rows <= kFew)
    attend_part<false, 2>(a, u, h, sh);
  else
    attend_part<true, 2>(a, u, h, sh);
}

// Merges the parts of rows that have several: 32 lanes a row with 4 dims each, its
// prefix's parts, then its own.
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixArgs a, int wgs) {
  const int t = blockIdx.x / wgs, lane = threadIdx.x & 63;
  const int s = seq_of(a, t, lane);
  if (s >= a.nseq) return;
  const SeqRec r = a.seq[s];
  if (r.own_parts + r.pre_parts == 0) return;
  const int d = 4 * (threadIdx.x & 31), i = t - r.t0;
  if (i < 0 || i >= r.n) return;
  const int j0 = (blockIdx.x - t * wgs) * a.rows_wg;
  for (int j = j0 + (threadIdx.x >> 5); j < min(j0 + a.rows_wg, a.hq); j += 8) {
    const int h = (uint32_t)j / a.by_g, row = i * a.G + j - h * a.G;
    float M = -INFINITY, L = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    bool weightless = false;
    const int64_t pre = r.pre + h * r.pre_head + row, own = r.own + h * r.own_head + row;
    const int parts = r.pre_parts + r.own_parts;
    constexpr int B = 8;  // records in flight together (4: a few % slower, 12: 40 %)
    for (int p0 = 0; p0 < parts; p0 += B) {
      float pm[B], pl[B];
      f32x4 po[B];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int p = min(p0 + b, parts - 1), q = p - r.pre_parts;
        const int64_t at = q < 0 ? pre + (int64_t)p * r.pre_rows : own + (int64_t)q * r.own_rows;
        pm[b] = a.rec_ml[2 * at];
        pl[b] = a.rec_ml[2 * at + 1];
        po[b] = *(const __attribute__((address_space(1))) f32x4*)(a.rec_o + at * kD + d);
      }
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (p0 + b >= parts) break;
        const float mn = fmaxf(M, pm[b]), fa = merge_factor(M, mn), fb = merge_factor(pm[b], mn);
        weightless |= pm[b] != pm[b];
        if (pl[b] != 0.f) {  // (a part without a key counts for nothing)
          const float la = L * fa, lb = pl[b] * fb, inv = __builtin_amdgcn_rcpf(la + lb);  // (off by 2^-23)
          L = la + lb;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = o[e] * (la * inv) + po[b][e] * (lb * inv);
          M = mn;
        }
      }
    }
    if (weightless) {  // 0 times the values of keys without weight: 0 or a NaN, all NaN where there are no others
      for (int p = 0; p < parts; ++p) {
        const int q = p - r.pre_parts;
        const int64_t at = q < 0 ? pre + (int64_t)p * r.pre_rows : own + (int64_t)q * r.own_rows;
        if (a.rec_ml[2 * at + 1] == 0.f) o += *(const __attribute__((address_space(1))) f32x4*)(a.rec_o + at * kD + d);
      }
      if (L == 0.f) o = f32x4{NAN, NAN, NAN, NAN};
    }
    bf16 y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = f2bf(o[e]);  // (without a key 0)
    stg(a.out + ((int64_t)t * a.hq + j) * kD + d, __builtin_bit_cast(u32x2, *reinterpret_cast<bf16(*)[4]>(&y)));
  }
}

// -------------------------------------------------------------- launchers ---
// Bounds of a call, from shapes alone (make_plan keeps to them whatever the
// lengths are).
struct PrefixLayout {
  int64_t parts, recs;                             // of the plan
  int64_t part, seq, list, qrot, rec_o, rec_ml, bytes;  // places in the workspace
};
PrefixLayout prefix_layout(int64_t nseq, int64_t T, int64_t ngroups, int hq, int hkv, int64_t pmax, int64_t kmax, bool rotate) {
  PrefixLayout l{};
  const int64_t G = hq / hkv;
  const int64_t blocks = nseq + ngroups + T * G / kRows;
  const int64_t steps = (pmax + kKeys - 1) / kKeys + (kmax + kKeys - 1) / kKeys;
  const int64_t most = std::max<int64_t>(1, (steps + kMinSteps / 2 - 1) / (kMinSteps / 2));
  // (full parts: kCuts * kSlots only where the work is enough for long ones)
  const int64_t full = 4 * blocks * hkv * steps > (int64_t)kLong * kSlots ? kCuts * kSlots : kSlots;
  l.parts = std::min<int64_t>(blocks * most, blocks + (full + hkv - 1) / hkv);
  // rows that share their prefix, twice, and those of blocks that are cut
  const int64_t few = std::min<int64_t>(T, nseq * ((kRows - 1) / G));
  const int64_t cut = most > 1 ? std::min<int64_t>(2 * full, blocks * most * hkv) * kRows : 0;
  l.recs = 2 * few * hq + cut;
  auto place = [&](int64_t bytes) {
    const int64_t at = l.bytes;
    l.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  place(sizeof(int32_t));
  l.part = place(l.parts * (int64_t)sizeof(Part));
  l.seq = place(nseq * (int64_t)sizeof(SeqRec));
  l.list = place(T * (int64_t)sizeof(int32_t));
  l.qrot = place(rotate ? T * hq * kD * 2 : 0);
  l.rec_ml = place(l.recs * 2 * (int64_t)sizeof(float));
  l.rec_o = place(l.recs * kD * (int64_t)sizeof(float));
  return l;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" int64_t swl_prefix_attention_workspace(int nseq, int64_t ntok, int ngroups, int hq, int hkv,
                                                  int64_t max_prefix_keys, int64_t max_keys, int rotate) {
  if (nseq <= 0 || ntok <= 0 || ngroups < 0 || hq <= 0 || hkv <= 0 || hq % hkv || max_keys <= 0 || max_prefix_keys < 0)
    return 0;
  return prefix_layout(nseq, ntok, ngroups, hq, hkv, max_prefix_keys, max_keys, rotate != 0).bytes;
}

extern "C" int swl_prefix_attention_bf16(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                         int64_t v_stride, int nseq, int64_t ntok, const int32_t* cu_seqlens, int hq,
                                         int hkv, int d, void* k_cache, void* v_cache, int64_t num_blocks,
                                         int block_size, const int32_t* prefix_table, int64_t max_prefix_blocks,
                                         const int32_t* prefix_lens, const int32_t* cu_groups, int ngroups,
                                         const int32_t* block_table, int64_t max_blocks, const int32_t* cache_seqlens,
                                         const int64_t* positions, const void* cos_sin, int64_t max_pos,
                                         float softmax_scale, void* out, void* workspace, int64_t workspace_bytes,
                                         void* stream) {
  auto bad = [](const char* m) { return swl::fail(SWL_ERR_INVALID, std::string("swl_prefix_attention_bf16: ") + m); };
  if (d != kD) return bad("head_dim must be 128");
  if (nseq < 0 || ntok < 0 || ntok >= ((int64_t)1 << 25) || ngroups < 0) return bad("bad sequence, token or group count");
  if (hkv < 1 || hkv > 4096 || hq < 1 || hq > 65536 || hq % hkv) return bad("bad head counts");
  if (block_size < 1 || block_size > (1 << 20)) return bad("bad block_size");
  if (num_blocks < 1 || num_blocks * block_size >= ((int64_t)1 << 31) || max_blocks < 1 ||
      max_blocks > ((int64_t)1 << 30) / block_size || max_prefix_blocks < 0 ||
      max_prefix_blocks > ((int64_t)1 << 30) / block_size)
    return bad("bad page geometry");
  if (!(softmax_scale > 0.f && std::isfinite(softmax_scale))) return bad("softmax_scale must be positive and finite");
  if ((positions == nullptr) != (cos_sin == nullptr) || (positions && max_pos < 1))
    return bad("positions and cos_sin go together");
  if ((k == nullptr) != (v == nullptr)) return bad("k and v go together");
  if (nseq == 0 || ntok == 0) return SWL_OK;
  if (!q || !out || !k_cache || !v_cache || !block_table || !cache_seqlens) return bad("null argument");
  if (ngroups == 0 && cu_groups) return bad("cu_groups without a group");
  if (ngroups > 0 && (!prefix_table || !prefix_lens || max_prefix_blocks < 1)) return bad("null argument");
  if (!cu_groups && ngroups > 1) return bad("more than one group needs cu_groups");
  if (nseq + ngroups > kMaxEntries) return bad("at most 1024 sequences and groups");
  if (!cu_seqlens && ntok % nseq) return bad("without cu_seqlens every sequence has as many tokens");
  if (ntok * (int64_t)(hq / hkv) >= ((int64_t)1 << 31)) return bad("too many rows");
  if (q == out) return bad("out must not be q");
  if (q_stride < (int64_t)hq * d || (k && (k_stride < (int64_t)hkv * d || v_stride < (int64_t)hkv * d)))
    return bad("token strides smaller than a token row");
  if (!aligned16(q) || !aligned16(out) || (q_stride & 7) || !aligned16(k) || !aligned16(v) ||
      (k && ((k_stride & 7) || (v_stride & 7))) || !aligned16(cos_sin) || !aligned16(k_cache) || !aligned16(v_cache))
    return bad("q, k, v, out rows, the caches and cos_sin must be 16-byte aligned");
  const int64_t pmax = ngroups > 0 ? max_prefix_blocks * block_size : 0, kmax = max_blocks * block_size;
  const PrefixLayout l = prefix_layout(nseq, ntok, ngroups, hq, hkv, pmax, kmax, positions != nullptr);
  const int heads = (positions ? hq : 0) + (k ? 2 * hkv : 0), heads_wg = (heads + 31) / 32;
  const int64_t start = 1 + ntok * heads_wg;  // workgroups of the first launch
  const int rows_wg = ntok * hq > 32768 ? hq : 8, wgs = (hq + rows_wg - 1) / rows_wg;  // of the merge
  if (!swl::grid_fits(start, 256) || !swl::grid_fits(l.parts * hkv, 256) || !swl::grid_fits(ntok * wgs, 256) ||
      l.recs >= ((int64_t)1 << 40))
    return bad("too many rows");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < l.bytes)
    return bad("workspace smaller than swl_prefix_attention_workspace");
  PrefixArgs a{};
  char* ws = reinterpret_cast<char*>(workspace);
  a.q_in = reinterpret_cast<const bf16*>(q);
  a.q_in_s = q_stride;
  a.qrot = positions ? reinterpret_cast<bf16*>(ws + l.qrot) : nullptr;
  a.q = positions ? a.qrot : a.q_in;
  a.qs = positions ? (int64_t)hq * d : q_stride;
  a.k = reinterpret_cast<const bf16*>(k);
  a.v = reinterpret_cast<const bf16*>(v);
  a.ks = k_stride;
  a.vs = v_stride;
  a.kc = reinterpret_cast<bf16*>(k_cache);
  a.vc = reinterpret_cast<bf16*>(v_cache);
  a.pt = prefix_table;
  a.plens = prefix_lens;
  a.cg = cu_groups;
  a.bt = block_table;
  a.lens = cache_seqlens;
  a.cu = cu_seqlens;
  a.pos = positions;
  a.cs = reinterpret_cast<const bf16*>(cos_sin);
  a.out = reinterpret_cast<bf16*>(out);
  a.max_pre = max_prefix_blocks;
  a.max_blocks = max_blocks;
  a.max_pos = max_pos;
  a.T = ntok;
  a.num_blocks = (int32_t)num_blocks;
  a.nseq = nseq;
  a.ngroups = ngroups;
  a.L = (int32_t)(ntok / nseq);
  a.hq = hq;
  a.hkv = hkv;
  a.G = hq / hkv;
  a.bs = block_size;
  a.kmax = (int32_t)kmax;
  a.pmax = (int32_t)pmax;
  a.by_g = fast_div((uint32_t)a.G);
  a.by_hkv = fast_div((uint32_t)hkv);
  a.by_bs = fast_div((uint32_t)block_size);
  a.by_l = fast_div((uint32_t)std::max(a.L, 1));
  a.scale = softmax_scale;
  a.n_parts = reinterpret_cast<int32_t*>(ws);
  a.part = reinterpret_cast<Part*>(ws + l.part);
  a.seq = reinterpret_cast<SeqRec*>(ws + l.seq);
  a.list = reinterpret_cast<int32_t*>(ws + l.list);
  a.rec_o = reinterpret_cast<float*>(ws + l.rec_o);
  a.rec_ml = reinterpret_cast<float*>(ws + l.rec_ml);
  a.max_rec = l.recs;
  a.max_parts = (int32_t)l.parts;
  a.slots = kSlots;
  a.min_steps = kMinSteps;
  a.rows_wg = rows_wg;
  const hipStream_t st = (hipStream_t)stream;
  const size_t lds = (size_t)(nseq + ngroups + 1) * kPlanEntry;
  hipLaunchKernelGGL(prefix_start_kernel, dim3((unsigned)start), dim3(256), lds, st, a, std::max(heads_wg, 1));
  SWL_LAUNCH_CHECK("prefix_start_kernel launch");
  hipLaunchKernelGGL(prefix_attention_kernel, dim3((unsigned)(l.parts * hkv)), dim3(256), 0, st, a);
  SWL_LAUNCH_CHECK("prefix_attention_kernel launch");
  if (l.recs == 0) return SWL_OK;
  hipLaunchKernelGGL(prefix_merge_kernel, dim3((unsigned)(ntok * wgs)), dim3(256), 0, st, a, wgs);
  SWL_LAUNCH_CHECK("prefix_merge_kernel launch");
  return SWL_OK;
}
