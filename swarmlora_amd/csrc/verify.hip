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
// Probabilities are held in 64 bits: with 128256 tokens a cumulative sum that is
// off by 1e-7 of the total picks another token once in about forty draws.
// Three launches: statistics of every row (maximum, sum; a workgroup per slice
// of a row); acceptance and the weight of every slice of the sequence's last
// row; the slice and token the random number falls in.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "dev_util.h"
#include "swl.h"
#include "swl_common.h"

namespace {

struct RowStat {
  double z;       // sum of exp((x - max) / temperature) over the slice
  uint32_t key;   // order key of the slice's largest logit
  int32_t idx;    // its first index
};
struct SeqPick {
  double p_inv, q_inv;  // 1 / sum
  float p_max, q_max;
  int64_t row;          // last row (target), -1: nothing to draw, the token is set
  int64_t q_row;        // draft row subtracted from it, -1: none
  int64_t skip;         // token whose weight is 0, -1: none
  int64_t best;         // first index of the row's largest logit
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
  int32_t nseq, per, max_drafts, slices, slice;  // slice: logits of one
  RowStat* stat;        // [T + nseq rows, then T rows][slices]
  SeqPick* pick;        // [nseq]
  double* mass;         // [nseq][slices]
};

// order-preserving maps of a bf16's bits to 16 bits and back, a NaN of either
// sign above all
__device__ __forceinline__ uint32_t vkey16(uint32_t bits) {
  if ((bits & 0x7fffu) > 0x7f80u) return 0xffffu;
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

// e^((x - max) / temperature)
__device__ __forceinline__ double weight(uint32_t bits, float mx, double invt) {
  return exp(((double)__uint_as_float(bits << 16) - (double)mx) * invt);
}

// Slices of a row, 256 threads with E logits each.
template <int E>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  __shared__ uint32_t shk[4];
  __shared__ double shz[4];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t R = a.T + a.nseq;
  const int64_t r = blockIdx.y, t = r - R;  // target rows, then draft rows
  const bool draft = t >= 0;
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
  const bf16* row = draft ? a.drf + t * a.ld_d : a.tgt + r * a.ld_t;
  const bool vec = row_vec(row);
  const int64_t base = (int64_t)blockIdx.x * a.slice;
  u32x4 q[E / 8];
#pragma unroll
  for (int j = 0; j < E / 8; ++j) q[j] = logits8(row, base + (j * 256 + tid) * 8, a.vocab, vec);
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
  const float mx = vkey_value(best >> 13);
  double z = 0;
  if (temp > 0.f || temp != temp) {
    const double invt = 1.0 / (double)temp;
    if (mx != -INFINITY) {  // (a slice of nothing but -inf weighs 0)
#pragma unroll
      for (int j = 0; j < E / 8; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (base + (j * 256 + tid) * 8 + e < a.vocab) z += weight(bits_at(q[j], e), mx, invt);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) z += __shfl_xor(z, o, 64);
    if (lane == 0) shz[wv] = z;
    __syncthreads();
    z = (shz[0] + shz[1]) + (shz[2] + shz[3]);
  }
  if (tid == 0) a.stat[r * a.slices + blockIdx.x] = RowStat{z, best >> 13, (int32_t)(base + 8191 - (best & 8191))};
}

// A row's statistics from its slices', by sixteen lanes.
struct RowAll {
  double z;
  float mx;
  int64_t best;
};
__device__ __forceinline__ RowAll row_all(const VerifyArgs& a, int64_t r, double invt, int l16) {
  const RowStat* st = a.stat + r * a.slices;
  uint64_t best = 0;
  for (int c = l16; c < a.slices; c += 16)
    best = max(best, (uint64_t)st[c].key << 32 | (uint32_t)~(uint32_t)st[c].idx);
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) best = max(best, (uint64_t)__shfl_xor((long long)best, o, 16));
  RowAll x;
  x.mx = vkey_value((uint32_t)(best >> 32));
  x.best = (int64_t)(uint32_t)~(uint32_t)best;
  x.z = 0;
  for (int c = l16; c < a.slices; c += 16)
    x.z += st[c].z * exp(((double)vkey_value(st[c].key) - (double)x.mx) * invt);
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) x.z += __shfl_xor(x.z, o, 16);
  return x;
}

// Acceptance of a sequence's drafts (sixteen lanes a draft, sixteen drafts at a
// time; every workgroup of the sequence for itself) and the weight of one slice
// of its last row.
template <int E>
__global__ __launch_bounds__(256) void verify_mass_kernel(VerifyArgs a) {
  __shared__ int first_bad;
  __shared__ double shz[4];
  __shared__ SeqPick sp;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, l16 = tid & 15;
  const int s = blockIdx.y;
  int64_t t0;
  int n;
  drafts_of(a, s, t0, n);
  const float temp = a.temp[s];
  const bool greedy = temp <= 0.f;
  const double invt = 1.0 / (double)temp;
  const int64_t R = a.T + a.nseq, row0 = t0 + s;
  if (tid == 0) first_bad = n;
  __syncthreads();
  for (int j0 = 0; j0 < n; j0 += 16) {
    const int j = j0 + (tid >> 4);
    if (j < n) {  // (the sixteen lanes together)
      const int64_t d = a.ids[t0 + j];
      bool ok = d >= 0 && d < a.vocab;
      const RowAll p = row_all(a, row0 + j, invt, l16);
      if (greedy) {
        ok = ok && d == p.best;
      } else if (ok) {
        const uint16_t pb = *reinterpret_cast<const uint16_t*>(a.tgt + (row0 + j) * a.ld_t + d);
        double qd = 1.0;
        if (a.drf) {
          const RowAll q = row_all(a, R + t0 + j, invt, l16);
          const uint16_t qb = *reinterpret_cast<const uint16_t*>(a.drf + (t0 + j) * a.ld_d + d);
          qd = weight(qb, q.mx, invt) / q.z;
        }
        ok = (double)a.u[t0 + j] * qd < weight(pb, p.mx, invt) / p.z;
      }
      if (!ok && l16 == 0) atomicMin(&first_bad, j);
    }
    __syncthreads();
    const int bad = first_bad;
    __syncthreads();  // read by all before the next drafts change it
    if (bad < n) break;
  }
  const int take = first_bad;
  if (tid < 16) {
    SeqPick x{};
    const RowAll p = row_all(a, row0 + take, invt, l16);
    x.row = greedy ? -1 : row0 + take;
    x.best = p.best;
    x.p_max = p.mx;
    x.p_inv = 1.0 / p.z;
    x.q_row = x.skip = -1;
    if (!greedy && take < n) {
      const int64_t d = a.ids[t0 + take];
      if (d >= 0 && d < a.vocab) {
        if (a.drf) {
          const RowAll q = row_all(a, R + t0 + take, invt, l16);
          x.q_row = t0 + take;
          x.q_max = q.mx;
          x.q_inv = 1.0 / q.z;
        } else {
          x.skip = d;
        }
      }
    }
    if (tid == 0) {
      sp = x;
      if (blockIdx.x == 0) {
        a.pick[s] = x;
        a.acc[s] = take;
      }
    }
  }
  if (blockIdx.x == 0)
    for (int j = tid; j <= a.max_drafts; j += 256) a.tok[(int64_t)s * (a.max_drafts + 1) + j] = j < take ? a.ids[t0 + j] : -1;
  if (greedy) return;
  __syncthreads();
  const bf16* prow = a.tgt + sp.row * a.ld_t;
  const bf16* qrow = sp.q_row >= 0 ? a.drf + sp.q_row * a.ld_d : nullptr;
  const int64_t base = (int64_t)blockIdx.x * a.slice;
  double z = 0;
  for (int j = 0; j < E / 8; ++j) {
    const int64_t i = base + (j * 256 + tid) * 8;
    if (i >= a.vocab) break;
    const u32x4 p = logits8(prow, i, a.vocab, row_vec(prow));
    u32x4 q = p;
    if (qrow) q = logits8(qrow, i, a.vocab, row_vec(qrow));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      double w = weight(bits_at(p, e), sp.p_max, invt) * sp.p_inv;
      if (qrow) {
        w -= weight(bits_at(q, e), sp.q_max, invt) * sp.q_inv;
        w = w < 0 ? 0 : w;  // (a NaN stays one)
      }
      if (i + e == sp.skip) w = 0;
      if (i + e < a.vocab) z += w;
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) z += __shfl_xor(z, o, 64);
  if (lane == 0) shz[wv] = z;
  __syncthreads();
  if (tid == 0) a.mass[(int64_t)s * a.slices + blockIdx.x] = (shz[0] + shz[1]) + (shz[2] + shz[3]);
}

// The slice that u * (sum of all) falls in, then the token of it: the first
// whose cumulative weight is above that.  1024 threads, E / 4 logits each.
template <int E>
__global__ __launch_bounds__(1024) void verify_pick_kernel(VerifyArgs a) {
  constexpr int N = E / 4;  // 8, or 2 (then 8 logits for every fourth thread)
  __shared__ double shz[16];
  __shared__ double shm[1024];
  __shared__ int slot, first, last_any;
  __shared__ double below;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int s = blockIdx.x;
  const SeqPick x = a.pick[s];
  int64_t* out = a.tok + (int64_t)s * (a.max_drafts + 1) + a.acc[s];
  if (x.row < 0) {
    if (tid == 0) *out = x.best;
    return;
  }
  const double* mass = a.mass + (int64_t)s * a.slices;
  const double invt = 1.0 / (double)a.temp[s];
  // the masses 1024 at a time through LDS: their sum, then where it passes u of it
  double total = 0, sum = 0, before = 0;
  int at = -1;
  bool found = false;
  for (int pass = 0; pass < 2; ++pass)
    for (int c0 = 0; c0 < a.slices; c0 += 1024) {
      __syncthreads();
      if (c0 + tid < a.slices) shm[tid] = mass[c0 + tid];
      __syncthreads();
      if (tid == 0) {
        const int m = min(1024, a.slices - c0);
        const double want = (double)a.u_last[s] * total;
        for (int c = 0; c < m && !found; ++c) {
          if (pass == 0) {
            total += shm[c];
          } else {
            if (shm[c] > 0) {  // the last slice of any weight where none passes it
              at = c0 + c;
              before = sum;
              found = sum + shm[c] > want;
            }
            sum += shm[c];
          }
        }
      }
    }
  if (tid == 0) {
    slot = total > 0 ? at : -1;  // a NaN, or nothing left: the largest logit
    below = (double)a.u_last[s] * total - before;
    first = 1 << 30;
    last_any = -1;
  }
  __syncthreads();
  if (slot < 0) {
    if (tid == 0) *out = x.best;
    return;
  }
  const bf16* prow = a.tgt + x.row * a.ld_t;
  const bf16* qrow = x.q_row >= 0 ? a.drf + x.q_row * a.ld_d : nullptr;
  const int64_t i = (int64_t)slot * a.slice + tid * 8;
  double w8[8];
  sum = 0;
  const bool in = tid < 128 * N && i < a.vocab;
#pragma unroll
  for (int e = 0; e < 8; ++e) w8[e] = 0;
  if (in) {
    const u32x4 p = logits8(prow, i, a.vocab, row_vec(prow));
    u32x4 q = p;
    if (qrow) q = logits8(qrow, i, a.vocab, row_vec(qrow));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      double w = weight(bits_at(p, e), x.p_max, invt) * x.p_inv;
      if (qrow) {
        w -= weight(bits_at(q, e), x.q_max, invt) * x.q_inv;
        w = w < 0 ? 0 : w;
      }
      if (i + e == x.skip || i + e >= a.vocab) w = 0;
      w8[e] = w;
      sum += w;
    }
  }
  double inc = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(inc, o, 64);
    if (lane >= o) inc += y;
  }
  if (lane == 63) shz[wv] = inc;
  __syncthreads();
  double cum = inc - sum;
  for (int w = 0; w < wv; ++w) cum += shz[w];
  // the first token above `below`, and the last of any weight (where rounding
  // puts the slice's sum under it)
  int mine = -1, last = -1;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cum += w8[e];
    if (w8[e] > 0) {
      last = tid * 8 + e;
      if (mine < 0 && cum > below) mine = tid * 8 + e;
    }
  }
  if (mine >= 0) atomicMin(&first, mine);
  if (last >= 0) atomicMax(&last_any, last);
  __syncthreads();
  if (tid == 0) *out = (int64_t)slot * a.slice + (first < (1 << 30) ? first : max(last_any, 0));
}

// Logits of a slice: 8192, or 2048 where that leaves under four workgroups a CU.
int slice_of(int64_t rows, int64_t vocab) { return rows * ((vocab + 8191) / 8192) >= 1024 ? 8192 : 2048; }

struct VerifyLayout {
  int slice;
  int64_t slices, pick, mass, bytes;
};
VerifyLayout verify_layout(int64_t nseq, int64_t T, int64_t vocab, bool draft) {
  VerifyLayout l;
  const int64_t rows = T + nseq + (draft ? T : 0);
  l.slice = slice_of(rows, vocab);
  l.slices = (vocab + l.slice - 1) / l.slice;
  l.pick = rows * l.slices * (int64_t)sizeof(RowStat);
  l.mass = l.pick + nseq * (int64_t)sizeof(SeqPick);
  l.bytes = l.mass + nseq * l.slices * (int64_t)sizeof(double);
  return l;
}

template <int E>
int launch_verify(const VerifyArgs& a, hipStream_t st) {
  const unsigned rows = (unsigned)(a.T + a.nseq + (a.drf ? a.T : 0));
  hipLaunchKernelGGL(verify_stats_kernel<E>, dim3((unsigned)a.slices, rows), dim3(256), 0, st, a);
  SWL_LAUNCH_CHECK("verify_stats_kernel launch");
  hipLaunchKernelGGL(verify_mass_kernel<E>, dim3((unsigned)a.slices, (unsigned)a.nseq), dim3(256), 0, st, a);
  SWL_LAUNCH_CHECK("verify_mass_kernel launch");
  hipLaunchKernelGGL(verify_pick_kernel<E>, dim3((unsigned)a.nseq), dim3(1024), 0, st, a);
  SWL_LAUNCH_CHECK("verify_pick_kernel launch");
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
  a.slices = (int32_t)l.slices;
  a.slice = l.slice;
  char* ws = reinterpret_cast<char*>(workspace);
  a.stat = reinterpret_cast<RowStat*>(ws);
  a.pick = reinterpret_cast<SeqPick*>(ws + l.pick);
  a.mass = reinterpret_cast<double*>(ws + l.mass);
  return l.slice == 8192 ? launch_verify<32>(a, (hipStream_t)stream) : launch_verify<8>(a, (hipStream_t)stream);
}
