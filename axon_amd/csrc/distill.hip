// Distillation from a teacher's top logits: per position, a divergence between the teacher's probabilities q of k given tokens
// and the student's p of the same tokens under the softmax over the whole vocabulary, optionally with what is left of both as
// one more outcome, and its gradient with respect to the student's logits.
//
// Every divergence is a function of the outcomes' log-probabilities lp, with G_o = dL / dlp_o:
//   forward  sum q (lq - lp)                                  G = -q
//   reverse  sum p (lp - lq)                                  G = p (lp - lq + 1)
//   jsd      m = b q + (1 - b) p:  sum b q (lq - lm) + (1 - b) p (lp - lm)   G = (1 - b) p (lp - lm)
//   dz_j = (sum_{o: id_o = j} G_o - p_j sum_o G_o + [j is not given] G_rest p_j / p_rest) / T
// so that a row is its softmax statistics, k gathered logits, and one multiple of p_j for all tokens that are not given.  What
// the student has left over is summed over these tokens themselves: 1 minus the rest has no digits where it matters.  With
// what is left as an outcome their p_j is never formed: p_j / p_rest = 2^((z_j - lse_rest) log2(e) / T) against the log-sum-exp of
// what is left, times G_rest - p_rest sum_o G_o, which stays in range however little that is.
//
// Bound by memory (a large copy takes 4.8 TB/s).  Where the losses' weights are known a row is read once and written once: 4096 x 151936
// bf16, a third of weight 0, 446 us (2.08 GB, 4.7 TB/s); 2500 x 201088 bf16 448 us (4.5 TB/s, a twentieth of a row is read twice); 1500 x
// 151936 fp32 428 us (4.3 TB/s, a third of a row twice).  Where they are not, it is read for the statistics and again for the gradient:
// 2047 x 50257 bf16 42 us (4.9 TB/s, what rows that start on 2 bytes reach) and 93 us (4.4 TB/s).
#include "logits_rows.h"
#include <type_traits>

namespace axon {

constexpr int kMaxParts = 64;
constexpr int kMaxIds = AXON_MAX_TOKEN_IDS;
constexpr int kMaxShare = 49152;  // vectors of a workgroup's share: a byte each in LDS says which of its elements are given

struct Teacher {
  const void* ids;        // [n][k]
  const float* logprobs;  // [n][k]
  const float* weights;   // [n], null: all rows count
  int ids_i64, k, divergence, tail;
  float beta, inv_t, step;
};
// What the teacher has left, 1 - sum q, is known to the rounding of its log-probabilities: a softmax in 32 bits is off by about 2^-21 (1 +
// |lq|) (up to 5.6 2^-24 (1 + |lq|) in all tokens alike, from 2 to 512 of them), and one that is stored in fewer bits by `step` |lq|: two
// half steps of its type, since errors of the same sign add up.
constexpr double kTeacherError = 0x1p-21;
__device__ __forceinline__ int teacher_id(const Teacher& t, int64_t at, int vocab) {
  const int64_t id = t.ids_i64 ? static_cast<const int64_t*>(t.ids)[at] : (int64_t) static_cast<const int32_t*>(t.ids)[at];
  return id >= 0 && id < vocab ? (int)id : -1;
}

// What a row leaves for its backward: the log-sum-exp (of z, before the temperature) in two parts, of what is not given where that is
// an outcome, else of the whole row; the multiple of 2^((z - lse) log2(e) / T) for tokens that are not given, and that for those that
// are (0 where what is left is an outcome: the p_j sum G of a given token is in its own gradient then).
enum Coef { kLse, kRest, kOut, kIn, kCoefs };
struct RowOut {
  float *losses, *covered;
  float* grads;  // [n][k]: G of every given token, less p_j sum G of its id where what is left is an outcome
  float* coef;   // [kCoefs][n]
  int n;
};

// Sum of 2^((z - M) log2(e) / T) over a set of logits and their largest.  A thread's sum is in 64 bits: beside a likely token's
// term every other addition to it would round at that term's size.
struct Sum { float M; double s; };
constexpr float kLowest = -3.402823466e38f;
template <int N>
__device__ __forceinline__ void fold(Sum& a, const float (&z)[8], float k) {
  float m = z[0];
#pragma unroll
  for (int j = 1; j < N; ++j) m = fmaxf(m, z[j]);
  if (m > a.M) {
    a.s *= (double)__builtin_amdgcn_exp2f((a.M - m) * k);
    a.M = m;
  }
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) s += __builtin_amdgcn_exp2f((z[j] - a.M) * k);
  a.s += (double)s;
}

// The bytes that say which elements of a share's vectors are given, and the same for the few elements outside vectors.
struct GivenBytes {
  uint32_t* bytes;   // LDS, a byte per vector of [q_lo, q_hi)
  uint32_t* single;  // LDS, a bit per element outside the vectors
};
template <typename T>
__device__ __forceinline__ void mark_given(const GivenBytes& g, const Teacher& t, int64_t row, int vocab, const RowSpan& sp, int threads) {
  constexpr int kPer = Row<T>::kPer;
  const int words = (sp.q_hi - sp.q_lo + 3) / 4;
  for (int i = threadIdx.x; i < words; i += threads) g.bytes[i] = 0;
  if (threadIdx.x == 0) *g.single = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < t.k; i += threads) {
    const int id = teacher_id(t, row * t.k + i, vocab);
    if (id < 0) continue;
    const int in = id - sp.head, q = in >= 0 ? in / kPer : -1;
    if (q >= 0 && q < sp.n_vec) {
      const int at = q - sp.q_lo;
      if (at >= 0 && q < sp.q_hi) atomicOr(g.bytes + (at >> 2), 1u << ((at & 3) * 8 + in % kPer));
    } else {
      atomicOr(g.single, 1u << (in < 0 ? id : id - sp.n_vec * kPer));
    }
  }
  __syncthreads();
}

// What one lane has written to LDS, for the others of its wavefront: LDS serves a wavefront in order, the compiler is told to.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// In 64 bits, as functions that are called: inlined a dozen times their registers and their code would be those of the kernel.
__device__ __attribute__((noinline)) double exp64(double x) { return exp(x); }
__device__ __attribute__((noinline)) double log64(double x) { return log(x); }

// One outcome of which the teacher has q = exp(lq) and the student p = exp(lp): its share of the loss and G.
struct Term { double loss, g; };
__device__ __forceinline__ Term outcome(const Teacher& t, double q, double lq, double p, double lp) {
  if (t.divergence == AXON_DISTILL_FORWARD) return {q > 0.0 ? q * (lq - lp) : q - q, -q};
  if (t.divergence == AXON_DISTILL_REVERSE) {
    if (p == 0.0) return {0.0, 0.0};
    const double d = p * (lp - lq);
    return {d, d + p};
  }
  const double b = (double)t.beta, lm = log64(b * q + (1.0 - b) * p);
  const double mine = p == 0.0 ? 0.0 : (1.0 - b) * p * (lp - lm);
  return {(q == 0.0 ? 0.0 : b * q * (lq - lm)) + mine, mine};
}

// The outcome of what is left.  Where the teacher has no more than its error e of it, the list may well be complete:
//   forward  what the student has no more of either counts 0: q log(q / p) of a rounding q is infinite where p is 0 (lists of all legal
//            tokens).  Where it has none at all 8 e are let pass, which is what a softmax written as z - logsumexp(z) leaves with z up to 60.
//   reverse  the teacher has e: against 0, p log(p / q) is infinite wherever a sure teacher's log-probability is rounded to 0.
// The third is bounded either way.
__device__ __forceinline__ Term what_is_left(const Teacher& t, double q, double e, double p, double lp) {
  if (t.divergence == AXON_DISTILL_FORWARD && p <= e && q <= (p == 0.0 ? 8.0 * e : e)) return {0.0, 0.0};
  q = fmax(q, t.divergence == AXON_DISTILL_REVERSE ? e : 0.0);
  return outcome(t, q, log64(q), p, lp);
}

// The given tokens of a row, in LDS.
constexpr int kAgain = -2;
struct Given {
  int id[kMaxIds];               // -1: a filler
  int16_t next[kMaxIds];         // kAgain: an id that has come before, or none; else -1, or the next of its chain
  float a[kMaxIds], b[kMaxIds];  // the teacher's log-probabilities, then G; the logits, then p, then what is written in their place
  float best, best_q;            // the largest of either
  double sum, sum_q;             // REST: of exp((z - best) / T), every token once, and of q; else of exp(lq - best_q)
  double error_q;                // REST: of 1 - sum q
};
// By one wavefront; everything that can be known before the row's statistics.  firsts: whether ids that come again are looked for.
template <typename T, bool REST>
__device__ __forceinline__ void fetch_given(Given& s, const Teacher& t, int row_i, const T* row, int vocab, int lane, bool firsts = REST) {
  for (int i = lane; i < t.k; i += kWave) {
    const int id = teacher_id(t, (int64_t)row_i * t.k + i, vocab);
    const float lq = t.logprobs[(int64_t)row_i * t.k + i], z = Row<T>::one(row + max(id, 0));
    s.id[i] = id;
    s.a[i] = id < 0 ? -INFINITY : lq;
    s.b[i] = id < 0 ? -INFINITY : z;
  }
  wave_sync();
  for (int i = lane; i < t.k; i += kWave) {
    const int id = s.id[i];
    bool first = id >= 0;
    if (firsts) {
#pragma unroll 8
      for (int j = 0; j < t.k; ++j) first = first && !(j < i && s.id[j] == id);
    }
    s.next[i] = first ? -1 : kAgain;
  }
  float best = -INFINITY, best_q = -INFINITY;
  for (int i = lane; i < t.k; i += kWave) {
    best = fmaxf(best, s.b[i]);
    best_q = fmaxf(best_q, s.a[i]);
  }
  best = wave_max(best);
  best_q = wave_max(best_q);
  double sum = 0.0, sum_q = 0.0, error_q = 0.0;
  if (REST || t.tail == AXON_DISTILL_RENORMALIZE) {
#pragma unroll 1
    for (int i = lane; i < t.k; i += kWave) {
      if (s.id[i] < 0) continue;
      if (REST && s.next[i] != kAgain) sum += exp64(((double)s.b[i] - (double)best) * (double)t.inv_t);
      const double lq = (double)s.a[i], q = exp64(lq - (REST ? 0.0 : (double)best_q));
      sum_q += q;
      if (REST && q > 0.0) error_q += q * (kTeacherError + fabs(lq) * (kTeacherError + (double)t.step));
    }
    if (REST) {
      sum = wave_sum_d(sum);
      error_q = wave_sum_d(error_q);
    }
    sum_q = wave_sum_d(sum_q);
  }
  if (lane == 0) {
    s.best = best;
    s.best_q = best_q;
    s.sum = sum;
    s.sum_q = sum_q;
    s.error_q = error_q;
  }
  wave_sync();
}

// The outcomes of a row in 64 bits, by one wavefront, from the statistics that its lanes have of parts of the row (REST: of what is not
// given): losses, G (also in s.a), p (in s.b), and the row's coefficients.
struct RowCoefs { float lse, rest, c_out; double sum_g; };
template <bool REST>
__device__ __forceinline__ RowCoefs finish_row(Given& s, const Teacher& t, const RowOut& out, int row_i, float part_m, double part_s, int lane) {
  const float k = t.inv_t * kLog2e;
  const double inv_t = (double)t.inv_t;
  // The parts against the largest of themselves: what is left over may be next to nothing beside what is given.
  const float best = s.best, M_parts = wave_max(part_m), M = fmaxf(M_parts, best);
  const float d = fmaxf((part_m - M_parts) * k, -2000.f), n = rintf(d);
  const double s_parts = wave_sum_d(ldexp(part_s * (double)__builtin_amdgcn_exp2f(d - n), (int)n));
  const double below = ((double)M_parts - (double)M) * inv_t, s_in_all = s_parts > 0.0 ? s_parts * exp64(below) : s_parts;
  const double s_all = REST && best > -INFINITY ? s_in_all + s.sum * exp64(((double)best - (double)M) * inv_t) : s_in_all;
  const double ln_s = s_all > 0.0 ? log64(s_all) : (double)NAN;  // a row of -inf alone has no softmax
  // given tokens that the teacher rules out all together have no sum to be divided by: they stay at 0
  const double norm_q = !REST && t.tail == AXON_DISTILL_RENORMALIZE && s.best_q > -INFINITY ? (double)s.best_q + log64(s.sum_q) : 0.0;
  double loss = 0.0, sum_g = 0.0, covered = 0.0;
#pragma unroll 1
  for (int i = lane; i < t.k; i += kWave) {
    Term o{0.0, 0.0};
    double p = 0.0;
    if (s.id[i] >= 0) {
      const double lp = ((double)s.b[i] - (double)M) * inv_t - ln_s;
      const double lq = (double)s.a[i] - norm_q;
      p = exp64(lp);
      o = outcome(t, exp64(lq), lq, p, lp);
      covered += p;
    }
    loss += o.loss;
    sum_g += o.g;
    s.a[i] = (float)o.g;
    s.b[i] = (float)p;
    if (!REST) out.grads[(int64_t)row_i * t.k + i] = (float)o.g;
  }
  loss = wave_sum_d(loss);
  sum_g = wave_sum_d(sum_g);
  covered = wave_sum_d(covered);
  // of the parts, against which the gradient of what is not given is formed; of what a row of no such logits has, the whole row's
  const bool some = REST && s_parts > 0.0;
  const double ln_ref = some ? log64(s_parts) : ln_s;
  const float M_ref = some ? M_parts : M;
  RowCoefs r;
  // a number of 32 bits (at a temperature of 1e38 the sum's logarithm is none): `rest` is what it lacks.  (NaN stays.)
  const auto within = [](double x, double most) { return x > most ? most : x < -most ? -most : x; };
  r.lse = (float)within((double)M_ref + within(ln_ref / inv_t, 0x1p126), 3.402823466e38);
  r.rest = (float)((((double)M_ref - (double)r.lse) * inv_t + ln_ref) * 1.4426950408889634);
  if (REST) {
    const double lp_rest = some ? below + ln_ref - ln_s : log64(s_parts) - ln_s;
    const double p_rest = exp64(lp_rest);
    const Term o = what_is_left(t, 1.0 - s.sum_q, s.error_q, p_rest, lp_rest);
    loss += o.loss;
    sum_g += o.g;
    r.c_out = some ? (float)(o.g - p_rest * sum_g) : (float)(0.0 * s_all);
    for (int i = lane; i < t.k; i += kWave)
      out.grads[(int64_t)row_i * t.k + i] = s.next[i] == kAgain ? s.a[i] : (float)((double)s.a[i] - (double)s.b[i] * sum_g);
  } else {
    r.c_out = (float)-sum_g;
  }
  r.sum_g = sum_g;
  if (lane == 0) {
    out.losses[row_i] = (float)loss;
    out.covered[row_i] = (float)covered;
    float* const c = out.coef + row_i;
    c[(int64_t)kLse * out.n] = r.lse;
    c[(int64_t)kRest * out.n] = r.rest;
    c[(int64_t)kOut * out.n] = r.c_out;
    c[(int64_t)kIn * out.n] = REST ? 0.f : r.c_out;
  }
  wave_sync();
  return r;
}

// Workgroup (row, part): the statistics of its share of the row, of what is not given where that is an outcome (REST), in
// parts[row][part].  A row of one part is finished here, by a wavefront, while the compute unit's other workgroups read theirs.
template <typename T, bool REST>
__global__ __launch_bounds__(kBlock) void distill_stats_kernel(const T* __restrict__ logits, int64_t ld, int vocab, int n_parts, Teacher t,
                                                               float4* __restrict__ parts, RowOut out, int cached_from) {
  extern __shared__ __align__(16) uint32_t s_given[];
  __shared__ uint32_t s_single;
  __shared__ float red_m[kBlock / kWave];
  __shared__ double red_s[kBlock / kWave];
  __shared__ Given s_row;
  const int row_i = blockIdx.x / n_parts, part = blockIdx.x % n_parts, tid = threadIdx.x;
  if (t.weights != nullptr && t.weights[row_i] == 0.f) {
    if (n_parts == 1 && tid == 0) out.losses[row_i] = out.covered[row_i] = 0.f;
    return;
  }
  const T* row = logits + (int64_t)row_i * ld;
  constexpr int kPer = Row<T>::kPer;
  const RowSpan sp(row, vocab, true, part, n_parts);
  if (REST) mark_given<T>(GivenBytes{s_given, &s_single}, t, row_i, vocab, sp, kBlock);
  const uint8_t* const given = reinterpret_cast<const uint8_t*>(s_given);
  const T* body = row + sp.head;
  const float k = t.inv_t * kLog2e;
  Sum st{kLowest, 0.0};
  auto one = [&](int q, float (&v)[8]) {
    if (REST) {
      const uint32_t out = given[q - sp.q_lo];
      if (out != 0) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] = (out >> j & 1) ? -INFINITY : v[j];
      }
    }
    fold<kPer>(st, v, k);
  };
  // rows from cached_from on are left in the cache in front of the memory, for a backward that follows
  auto walk = [&](auto cached) {
    constexpr bool kCached = decltype(cached)::value;
    int q = sp.q_lo + tid;
    for (; q + kBlock < sp.q_hi; q += 2 * kBlock) {
      float v0[8], v1[8];
      Row<T>::template load<kCached>(body + (uint32_t)q * kPer, v0);
      Row<T>::template load<kCached>(body + (uint32_t)(q + kBlock) * kPer, v1);
      one(q, v0);
      one(q + kBlock, v1);
    }
    for (; q < sp.q_hi; q += kBlock) {
      float v[8];
      Row<T>::template load<kCached>(body + (uint32_t)q * kPer, v);
      one(q, v);
    }
  };
  if (row_i >= cached_from) walk(std::true_type{}); else walk(std::false_type{});
  if (part == 0 && tid < sp.n_scalar && !(REST && (s_single >> tid & 1))) {
    const float v[8] = {Row<T>::one(row + sp.scalar<T>(tid))};
    fold<1>(st, v, k);
  }
  const float m = wave_max(st.M);
  const double s = wave_sum_d(st.s * (double)__builtin_amdgcn_exp2f((st.M - m) * k));
  if ((tid & (kWave - 1)) == 0) { red_m[tid / kWave] = m; red_s[tid / kWave] = s; }
  __syncthreads();
  if (n_parts == 1) {
    if (tid >= kWave) return;
    fetch_given<T, REST>(s_row, t, row_i, row, vocab, tid);
    const bool mine = tid < kBlock / kWave;
    finish_row<REST>(s_row, t, out, row_i, mine ? red_m[tid] : kLowest, mine ? red_s[tid] : 0.0, tid);
    return;
  }
  if (tid != 0) return;
  float M = red_m[0];
  for (int w = 1; w < kBlock / kWave; ++w) M = fmaxf(M, red_m[w]);
  double total = 0.0;
  for (int w = 0; w < kBlock / kWave; ++w) total += red_s[w] * (double)__builtin_amdgcn_exp2f((red_m[w] - M) * k);
  parts[blockIdx.x] = make_float4(M, (float)total, (float)(total - (float)total), 0.f);
}

// The end of rows that several workgroups have read, by a wavefront per row.
template <typename T, bool REST>
__global__ __launch_bounds__(kWave) void distill_finish_kernel(const T* __restrict__ logits, int64_t ld, int vocab, int n_parts, Teacher t,
                                                               const float4* __restrict__ parts, RowOut out) {
  __shared__ Given s;
  const int row_i = blockIdx.x, lane = threadIdx.x;
  if (t.weights != nullptr && t.weights[row_i] == 0.f) {
    if (lane == 0) out.losses[row_i] = out.covered[row_i] = 0.f;
    return;
  }
  const float4 p = lane < n_parts ? parts[(int64_t)row_i * n_parts + lane] : make_float4(kLowest, 0.f, 0.f, 0.f);
  fetch_given<T, REST>(s, t, row_i, logits + (int64_t)row_i * ld, vocab, lane);
  finish_row<REST>(s, t, out, row_i, p.x, (double)p.y + (double)p.z, lane);
}

// Workgroup (row, part): dlogits of its share.  The row is streamed without a look at the given tokens; their few elements are
// written again afterwards, from logits that were read before (dlogits may be the logits' own storage).  Equal ids of a row add
// up in their order, in the thread of the first of them.  upstream: of every row's loss, or (weights) one for all, and where that
// is 1 the gradient is there already (`ready`).  Where it is 0 the row is not read.
template <typename T>
__global__ __launch_bounds__(kBlock) void distill_grad_kernel(const T* logits, int64_t ld, int vocab, Teacher t, RowOut saved,
                                                              const float* __restrict__ upstream, int ready, T* dlogits, int64_t ld_d,
                                                              int vec_ok, int n_parts) {
  constexpr int kPer = Row<T>::kPer, kSlots = kMaxIds / kBlock;
  __shared__ int ids[kMaxIds];
  const int b = gridDim.x - 1 - blockIdx.x, row_i = b / n_parts, part = b - row_i * n_parts, tid = threadIdx.x;
  const float up = upstream != nullptr ? upstream[t.weights != nullptr ? 0 : row_i] : 1.f;
  if (ready && up == 1.f) return;
  const float w = t.weights != nullptr ? t.weights[row_i] : 1.f;
  const float g = up * w * t.inv_t;
  const bool skip = w == 0.f || g == 0.f;  // nothing comes of the row, whatever it holds
  const T* row = logits + (int64_t)row_i * ld;
  T* out = dlogits + (int64_t)row_i * ld_d;
  const float* const c = saved.coef + row_i;
  const float lse = skip ? 0.f : c[(int64_t)kLse * saved.n], rest = skip ? 0.f : c[(int64_t)kRest * saved.n];
  const float c_out = skip ? 0.f : g * c[(int64_t)kOut * saved.n], c_in = skip ? 0.f : g * c[(int64_t)kIn * saved.n];
  const float k = t.inv_t * kLog2e;
  auto prob = [&](float z) { return __builtin_amdgcn_exp2f(fmaf(z - lse, k, -rest)); };
  const RowSpan sp(row, vocab, vec_ok != 0, part, n_parts);
  float again[kSlots];
  int where[kSlots];
  for (int i = tid; i < t.k; i += kBlock) ids[i] = skip ? -1 : teacher_id(t, (int64_t)row_i * t.k + i, vocab);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSlots; ++u) {
    const int i = tid + u * kBlock;
    where[u] = -1;
    const int id = i < t.k ? ids[i] : -1;
    if (id < 0) continue;
    const int in = id - sp.head, q = in / kPer;
    const bool vec = in >= 0 && q < sp.n_vec;
    if (vec) {
      if (q < sp.q_lo || q >= sp.q_hi) continue;
    } else if ((in < 0 ? id : id - sp.n_vec * kPer) / kBlock % n_parts != part) {
      continue;
    }
    float total = 0.f;
    bool first = true;
    for (int j = 0; j < t.k && first; ++j) {
      if (ids[j] != id) continue;
      first = j >= i;
      total += saved.grads[(int64_t)row_i * t.k + j];
    }
    if (!first) continue;
    where[u] = id;
    const float p = prob(Row<T>::one(row + id));  // against what is left it may be any number, of which c_in takes nothing
    again[u] = fmaf(p > 1.f ? 1.f : p, c_in, g * total);
  }
  __syncthreads();  // nothing of the row is written before these are read
  const T* body = row + sp.head;
  T* body_out = out + sp.head;
  auto finish = [&](int q, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = prob(v[j]) * c_out;
    Row<T>::store(body_out + (uint32_t)q * kPer, v);
  };
  if (skip) {
    for (int q = sp.q_lo + tid; q < sp.q_hi; q += kBlock) {
      const float v[8] = {};
      Row<T>::store(body_out + (uint32_t)q * kPer, v);
    }
    for (int i = part * kBlock + tid; i < sp.n_scalar; i += n_parts * kBlock) Row<T>::store_one(out + sp.scalar<T>(i), 0.f);
    return;
  }
  int q = sp.q_hi - 1 - tid;
  for (; q - kBlock >= sp.q_lo; q -= 2 * kBlock) {  // two loads in flight per thread
    float v0[8], v1[8];
    Row<T>::load(body + (uint32_t)q * kPer, v0);
    Row<T>::load(body + (uint32_t)(q - kBlock) * kPer, v1);
    finish(q, v0);
    finish(q - kBlock, v1);
  }
  for (; q >= sp.q_lo; q -= kBlock) {
    float v[8];
    Row<T>::load(body + (uint32_t)q * kPer, v);
    finish(q, v);
  }
  for (int i = part * kBlock + tid; i < sp.n_scalar; i += n_parts * kBlock) {
    const int j = sp.scalar<T>(i);
    Row<T>::store_one(out + j, prob(Row<T>::one(row + j)) * c_out);
  }
  // the stores above are acknowledged before another thread of the workgroup writes the same element
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0)
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSlots; ++u)
    if (where[u] >= 0) Row<T>::store_one(out + where[u], again[u]);
}

// The loss and its gradient from ONE read of a row.  A workgroup walks rows; it holds a row, NREG 16-byte vectors of every thread in
// registers and NLDS in LDS, from its statistics to its gradient (what is longer is read again).  As the vectors of a row leave, those
// of the next are asked for in their place, and looked at as they come: between the two there are only the sums over the workgroup and
// the outcomes.  ROW threads do that; the wavefront behind them looks after the given tokens: where they lie, two rows ahead, and the
// outcomes when a row's statistics are there.
// A thread's vectors that hold a given token are marked by a bit; statistics leave them out and take them one by one, with the tokens
// found through a hash of the vector's number, and the tokens' gradients are written over the vector's by the thread that has written it.
constexpr int kBuckets = 256, kMaxTiles = 64, kAhead = 3;
template <int ROW>
struct RowLds {
  Given given[kAhead];
  int heads[kAhead][kBuckets];  // chains of the ids that come for the first time
  uint32_t marks[kAhead][2][ROW];  // bit i % 32 of word i / 32: this thread's vector of tile i holds a given token
  uint32_t single[kAhead];         // a bit per element outside the vectors
  double red_s[ROW / kWave];
  float red_m[ROW / kWave];
  float lse, c_out;
  int is_far;
};

template <typename T> struct Packed;
template <> struct Packed<float> {
  typedef float Loose __attribute__((ext_vector_type(4), aligned(4)));
  __device__ static float get(const uint4& r, int j) { return __uint_as_float(j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w); }
  __device__ static void store(float* p, const float (&v)[8]) {
    const Loose x = {v[0], v[1], v[2], v[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<Loose*>(p));
  }
};
template <> struct Packed<unsigned short> {
  typedef uint32_t Loose __attribute__((ext_vector_type(4), aligned(2)));
  __device__ static float get(const uint4& r, int j) {
    const uint32_t w = j < 2 ? r.x : j < 4 ? r.y : j < 6 ? r.z : r.w;
    return __uint_as_float((j & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  __device__ static void store(unsigned short* p, const float (&v)[8]) {
    const Loose x = {f32x2_to_bf16(v[0], v[1]), f32x2_to_bf16(v[2], v[3]), f32x2_to_bf16(v[4], v[5]), f32x2_to_bf16(v[6], v[7])};
    __builtin_nontemporal_store(x, reinterpret_cast<Loose*>(p));
  }
};
constexpr float kFar = 1e9f;  // a reference in log2 units whose rounding (64) leaves the exponentials in range

// A barrier for what the threads have written to LDS themselves: loads on their way, to registers or to LDS, stay on their way.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A row as its threads see it.
template <typename T>
struct RowView {
  const T* row;
  RowSpan sp;
  __amdgpu_buffer_rsrc_t rsrc;  // of the vectors: behind the last a load gives zeros
  __device__ __forceinline__ RowView(const T* logits, int64_t ld, int i, int vocab, bool wanted = true)
      : row(logits + (int64_t)i * ld), sp(row, vocab, true, 0, 1),
        rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(row + sp.head), 0, wanted ? sp.n_vec * 16 : 0, 0x00020000)) {}
};

// Where the given tokens of a row lie, by one wavefront.
template <typename T, bool REST, int ROW>
__device__ __forceinline__ void mark_row(RowLds<ROW>& s, int buf, const Teacher& t, int row_i, const RowView<T>& v, int vocab, int lane) {
  constexpr int kPer = Row<T>::kPer;
  Given& g = s.given[buf];
  for (int i = lane; i < ROW; i += kWave) s.marks[buf][0][i] = s.marks[buf][1][i] = 0;
  for (int i = lane; i < kBuckets; i += kWave) s.heads[buf][i] = -1;
  if (lane == 0) s.single[buf] = 0;
  fetch_given<T, REST>(g, t, row_i, v.row, vocab, lane, true);
  for (int i = lane; i < t.k; i += kWave) {
    if (g.next[i] == kAgain) continue;
    const int id = g.id[i], in = id - v.sp.head, q = in >= 0 ? in / kPer : -1;
    if (q >= 0 && q < v.sp.n_vec) {
      atomicOr(&s.marks[buf][q / ROW / 32][q % ROW], 1u << (q / ROW % 32));
      g.next[i] = (int16_t)atomicExch(&s.heads[buf][q & (kBuckets - 1)], i);
    } else {
      atomicOr(&s.single[buf], 1u << (in < 0 ? id : id - v.sp.n_vec * kPer));
    }
  }
  wave_sync();
}

// The constants of a row for its threads, and what is written in the given tokens' places (in given.b), by one wavefront.
template <bool REST, int ROW>
__device__ __forceinline__ void settle_row(RowLds<ROW>& s, int buf, const Teacher& t, const RowOut& out, int row_i, float weight, int lane) {
  constexpr int kRowWaves = ROW / kWave;
  Given& gv = s.given[buf];
  const float k = t.inv_t * kLog2e, g = weight * t.inv_t;
  const float part_m = lane < kRowWaves ? s.red_m[lane] : kLowest;
  const double part_s = lane < kRowWaves ? s.red_s[lane] : 0.0;
  const RowCoefs r = finish_row<REST>(gv, t, out, row_i, part_m, part_s, lane);
  // p = 2^(z k - off) f with off = lse k rounded; far from 0 by the difference from lse
  const float off = r.lse * k;
  const bool is_far = !(fabsf(off) < kFar);
  const float f = __builtin_amdgcn_exp2f((is_far ? 0.f : (float)((double)off - (double)r.lse * (double)k)) - r.rest);
  const float c_in = -g * (float)r.sum_g;
  if (lane == 0) {
    s.lse = is_far ? r.lse : off;
    s.is_far = is_far;
    s.c_out = g * r.c_out * f;
  }
  for (int i = lane; i < t.k; i += kWave) {
    if (gv.next[i] == kAgain) continue;
    float total = gv.a[i];
#pragma unroll 8
    for (int j = i + 1; j < t.k; ++j) total += gv.id[j] == gv.id[i] ? gv.a[j] : 0.f;
    gv.b[i] = fmaf(gv.b[i], c_in, g * total);
  }
}

// RESIDENT: workgroups on a compute unit.
template <typename T, bool REST, int ROW, int NREG, int NLDS, int RESIDENT>
__global__ __launch_bounds__(ROW + kWave, RESIDENT * (ROW + kWave) / 256) void distill_row_kernel(
    const T* __restrict__ logits, int64_t ld, int vocab, Teacher t, RowOut out, T* __restrict__ dlogits, int64_t ld_d) {
  __shared__ RowLds<ROW> s;
  __shared__ int s_count[256 * RESIDENT], s_list[2][kWave];
  __shared__ uint4 s_tiles[NLDS * ROW];  // an array of its own: reads of the rest do not wait for what is on its way here
  constexpr int kPer = Row<T>::kPer;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const float k = t.inv_t * kLog2e;
  // Rows that are looked at and rows of weight 0 go round the workgroups by their number among their kind, 64 rows of each kind a
  // workgroup at a time: list[0] and list[1].
  const int grid = (int)gridDim.x, me = (int)blockIdx.x, n = out.n;
  for (int64_t batch = 0; batch < n; batch += (int64_t)kWave * grid) {
    const int rows = (int)min((int64_t)kWave * grid, n - batch), chunks = (rows + kWave - 1) / kWave;
    lds_barrier();  // the lists of the batch before have been read
    for (int c = wave; c < chunks; c += ROW / kWave + 1) {
      const int at = c * kWave + lane;
      const uint64_t on = __ballot(at < rows && t.weights[batch + min(at, rows - 1)] != 0.f);
      if (lane == 0) s_count[c] = __popcll(on);
    }
    lds_barrier();
    for (int c = wave; c < chunks; c += ROW / kWave + 1) {
      int before = 0;
      for (int i = lane; i < c; i += kWave) before += s_count[i];
      before = (int)wave_sum((float)before);  // at most 2^16
      const int at = c * kWave + lane;
      const bool there = at < rows, on = there && t.weights[batch + min(at, rows - 1)] != 0.f;
      const uint64_t kind = __ballot(there && on), other = __ballot(there && !on), below = (1ull << lane) - 1;
      const int rank = on ? before + __popcll(kind & below) : c * kWave - before + __popcll(other & below);
      if (there && rank % grid == me) s_list[on ? 0 : 1][rank / grid] = at;
    }
    int total = 0;
    lds_barrier();
    for (int i = lane; i < chunks; i += kWave) total += s_count[i];
    total = (int)wave_sum((float)total);
    const int n_on = (total - me + grid - 1) / grid, n_off = (rows - total - me + grid - 1) / grid;  // (0 where me is beyond)
    const int on_l = s_list[0][lane], off_l = s_list[1][lane];
    const auto row_of = [&](int j) { return (int)batch + __builtin_amdgcn_readlane(on_l, j); };

    if (wave == ROW / kWave) {
      if (lane < n_off) out.losses[batch + off_l] = out.covered[batch + off_l] = 0.f;
      const auto mark = [&](int j) {
        if (j < n_on) mark_row<T, REST, ROW>(s, j % kAhead, t, row_of(j), RowView<T>(logits, ld, row_of(j), vocab), vocab, lane);
      };
      mark(0);
      lds_barrier();  // the marks of row 0
      mark(1);
      for (int j = 0; j < n_on; ++j) {
        const int row_i = row_of(j);
        const float weight = t.weights[row_i];
        lds_barrier();  // the statistics of row j, the marks of row j + 1
        settle_row<REST, ROW>(s, j % kAhead, t, out, row_i, weight, lane);
        lds_barrier();  // its constants
        mark(j + 2);
      }
      continue;
    }

    // A tile: ROW vectors.  Buffer loads leave no branch between them, so that every tile is waited for by itself; those to LDS
    // write there themselves, 64 vectors of a wavefront side by side.
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) void* LdsPtr;
    int first = tid * 16;  // all of an offset in the lane's part: the bounds are of that
    asm volatile("" : "+v"(first));  // offsets are made where they are used: held over the rows they are registers
    const auto load = [&](__amdgpu_buffer_rsrc_t rsrc, int i) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rsrc, first + i * ROW * 16, 0, 2);  // non-temporal
      return make_uint4(x.x, x.y, x.z, x.w);
    };
    const auto load_cached = [&](__amdgpu_buffer_rsrc_t rsrc, int i) {  // what is read twice
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rsrc, first + i * ROW * 16, 0, 0);
      return make_uint4(x.x, x.y, x.z, x.w);
    };
    const auto load_lds = [&](__amdgpu_buffer_rsrc_t rsrc, int i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LdsPtr)(s_tiles + i * ROW + wave * kWave), 16, first + (NREG + i) * ROW * 16, 0, 0, 2);
    };
    uint4 reg[NREG];
    float single_z;

    // Statistics of a row.  Against a reference c = ref k rounded (ref: the largest of its given tokens' logits) an element is one
    // instruction beside its exponential, and what c is off by is taken back at the end.
    double terms = 0.0;  // of a vector's sums, in 64 bits: beside a likely token's term others would be rounded at its size
    float cc = 0.f, ref = 0.f;
    uint32_t mark_lo = 0, mark_hi = 0;
    const auto marked = [&](int i) { return REST && ((i < 32 ? mark_lo >> i : mark_hi >> (i - 32)) & 1) != 0; };
    const auto begin_stats = [&](int j) {
      const int buf = j % kAhead;
      ref = s.given[buf].best > -INFINITY ? s.given[buf].best : 0.f;
      cc = ref * k;
      mark_lo = s.marks[buf][0][tid];
      mark_hi = s.marks[buf][1][tid];
      terms = 0.0;
    };
    const auto add = [&](const uint4& r) {
      float s2[2] = {};
#pragma unroll
      for (int j = 0; j < kPer; ++j) s2[j & 1] += __builtin_amdgcn_exp2f(fmaf(Packed<T>::get(r, j), k, -cc));
      terms += (double)(s2[0] + s2[1]);
    };
    const auto each_given = [&](int buf, int id0, int q, auto&& f) {  // f(element, number among the given) of vector q
      for (int h = s.heads[buf][q & (kBuckets - 1)]; h >= 0; h = s.given[buf].next[h]) {
        const int e = s.given[buf].id[h] - id0;
        if (e >= 0 && e < kPer) f(e, h);
      }
    };
    const auto read_left = [&](int buf, const RowView<T>& v, int q, float (&x)[8]) {  // vector q without what is given
      Row<T>::template load<true>(v.row + v.sp.head + (uint32_t)q * kPer, x);
      uint32_t off = 0;
      if (REST) each_given(buf, v.sp.head + q * kPer, q, [&](int e, int) { off |= 1u << e; });
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[e] = (off >> e & 1) ? -INFINITY : x[e];
    };
    const auto add_marked = [&](int j, const RowView<T>& v) {
      if (!REST) return;
      for (uint64_t m = ((uint64_t)mark_hi << 32) | mark_lo; m != 0; m &= m - 1) {
        float x[8];
        read_left(j % kAhead, v, __builtin_ctzll(m) * ROW + tid, x);
#pragma unroll
        for (int e = 0; e < kPer; ++e) terms += (double)__builtin_amdgcn_exp2f(fmaf(x[e], k, -cc));
      }
    };
    const auto add_beyond = [&](const RowView<T>& v) {  // tiles that are not held
      const int last_q = v.sp.n_vec - 1, tiles = last_q / ROW + 1;
#pragma unroll 1
      for (int i = NREG + NLDS; i < tiles; i += 2) {
        const uint4 r0 = load_cached(v.rsrc, i), r1 = load_cached(v.rsrc, i + 1);
        if (i * ROW + tid <= last_q && !marked(i)) add(r0);
        if ((i + 1) * ROW + tid <= last_q && !marked(i + 1)) add(r1);
      }
    };
    const auto end_stats = [&](int j, const RowView<T>& v) {
      const bool single_in = tid < v.sp.n_scalar && !(REST && (s.single[j % kAhead] >> tid & 1));
      if (single_in) terms += (double)__builtin_amdgcn_exp2f(fmaf(single_z, k, -cc));
      double sum = wave_sum_d(terms) * (double)__builtin_amdgcn_exp2f(fmaf(-ref, k, cc));
      float m = ref;
      if (!(fabsf(cc) < kFar && sum > 0x1p-60 && sum < 0x1p80)) {
        // another scale, logits far from 0, infinite, or not numbers: by differences from the largest, read again
        Sum st{kLowest, 0.0};
#pragma unroll 1
        for (int q = tid; q < v.sp.n_vec; q += ROW) {
          float x[8];
          read_left(j % kAhead, v, q, x);
          fold<kPer>(st, x, k);
        }
        if (single_in) {
          const float x[8] = {single_z};
          fold<1>(st, x, k);
        }
        m = wave_max(st.M);
        sum = wave_sum_d(st.s * (double)__builtin_amdgcn_exp2f((st.M - m) * k));
      }
      if (lane == 0) { s.red_m[wave] = m; s.red_s[wave] = sum; }
    };

    {
      const RowView<T> v(logits, ld, n_on > 0 ? row_of(0) : 0, vocab, n_on > 0);
      single_z = tid < v.sp.n_scalar ? Row<T>::one(v.row + v.sp.template scalar<T>(tid)) : -INFINITY;
#pragma unroll
      for (int i = 0; i < NREG; ++i) reg[i] = load(v.rsrc, i);
#pragma unroll
      for (int i = 0; i < NLDS; ++i) load_lds(v.rsrc, i);
      // rows of weight 0, while the first row comes
      for (int j = 0; j < n_off; ++j) {
        const int row_i = (int)batch + __builtin_amdgcn_readlane(off_l, j);
        const RowSpan sp(logits + (int64_t)row_i * ld, vocab, true, 0, 1);
        T* const drow = dlogits + (int64_t)row_i * ld_d;
        const float none[8] = {};
        for (int q = tid; q < sp.n_vec; q += ROW) Packed<T>::store(drow + sp.head + (uint32_t)q * kPer, none);
        if (tid < sp.n_scalar) Row<T>::store_one(drow + sp.scalar<T>(tid), 0.f);
      }
      lds_barrier();  // the marks of row 0
      if (n_on > 0) {
        begin_stats(0);
        const int last_q = v.sp.n_vec - 1;
#pragma unroll
        for (int i = 0; i < NREG; ++i)
          if (i * ROW + tid <= last_q && !marked(i)) add(reg[i]);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the tiles in LDS are there
        asm volatile("" ::: "memory");
#pragma unroll 1
        for (int i = 0; i < NLDS; ++i)
          if ((NREG + i) * ROW + tid <= last_q && !marked(NREG + i)) add(s_tiles[i * ROW + tid]);
        add_beyond(v);
        add_marked(0, v);
        end_stats(0, v);
      }
    }
    for (int j = 0; j < n_on; ++j) {
      const int buf = j % kAhead, row_i = row_of(j);
      asm volatile("" : "+v"(first));
      lds_barrier();  // the statistics of row j, the marks of row j + 1
      const bool more = j + 1 < n_on;
      const RowView<T> v(logits, ld, row_i, vocab), next(logits, ld, more ? row_of(j + 1) : row_i, vocab, more);
      T* const drow = dlogits + (int64_t)row_i * ld_d;
      T* const dbody = drow + v.sp.head;
      const int last_q = v.sp.n_vec - 1, tiles = last_q / ROW + 1, next_q = more ? next.sp.n_vec - 1 : -1;
      uint64_t mine = ((uint64_t)s.marks[buf][1][tid] << 32) | s.marks[buf][0][tid];
      const float z_now = single_z;
      if (more && tid < next.sp.n_scalar) single_z = Row<T>::one(next.row + next.sp.template scalar<T>(tid));
      if (more) begin_stats(j + 1);
      lds_barrier();  // its constants
      const float lse = s.lse, c_out = s.c_out;
      const bool is_far = s.is_far != 0;
      const auto power = [&](float x) { return __builtin_amdgcn_exp2f(is_far ? (x - lse) * k : fmaf(x, k, -lse)); };
      const auto write = [&](const uint4& r, int i) {
        if (i * ROW + tid > last_q) return;
        float x[8];
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(Packed<T>::get(r, e), k, -lse)) * c_out;
        Packed<T>::store(dbody + (int64_t)i * ROW * kPer + (uint32_t)tid * kPer, x);
      };
      const auto look = [&](const uint4& r, int i) {
        if (i * ROW + tid <= next_q && !marked(i)) add(r);
      };
#pragma unroll
      for (int i = 0; i < NLDS; ++i) {
        write(s_tiles[i * ROW + tid], NREG + i);
        asm volatile("" ::: "memory");  // the tile has been read
        load_lds(next.rsrc, i);
      }
      asm volatile("" ::: "memory");  // the loads that follow are behind these
      constexpr int kLag = 3;  // tiles between a load and its use
#pragma unroll
      for (int i = 0; i < NREG + kLag; ++i) {
        if (i < NREG) {
          write(reg[i], i);
          reg[i] = load(next.rsrc, i);
        }
        if (i == kLag) {  // as many loads behind those to LDS: these are there
          __builtin_amdgcn_s_waitcnt(0x0F70 | kLag);
          asm volatile("" ::: "memory");
        }
        if (i >= kLag) look(reg[i - kLag], i - kLag);
        if (i > kLag && i - kLag - 1 < NLDS) look(s_tiles[(i - kLag - 1) * ROW + tid], NREG + i - kLag - 1);
      }
#pragma unroll 1
      for (int i = NREG + NLDS; i < tiles; i += 2) {
        const uint4 r0 = load_cached(v.rsrc, i), r1 = load_cached(v.rsrc, i + 1);
        write(r0, i);
        write(r1, i + 1);
      }
      if (is_far) {
#pragma unroll 1
        for (int q = tid; q <= last_q; q += ROW) {
          float x[8];
          Row<T>::template load<true>(v.row + v.sp.head + (uint32_t)q * kPer, x);
#pragma unroll
          for (int e = 0; e < kPer; ++e) x[e] = power(x[e]) * c_out;
          Packed<T>::store(dbody + (uint32_t)q * kPer, x);
        }
      }
      // the given tokens, each by the thread that has written its vector
      for (; mine != 0; mine &= mine - 1) {
        const int q = __builtin_ctzll(mine) * ROW + tid, id0 = v.sp.head + q * kPer;
        each_given(buf, id0, q, [&](int e, int h) { Row<T>::store_one(drow + id0 + e, s.given[buf].b[h]); });
      }
      if (tid < v.sp.n_scalar) {
        const int at = v.sp.template scalar<T>(tid);
        float x = power(z_now) * c_out;
        if (s.single[buf] >> tid & 1)
          for (int i = 0; i < t.k; ++i)
            if (s.given[buf].id[i] == at) {
              x = s.given[buf].b[i];  // the first of them has it all
              break;
            }
        Row<T>::store_one(drow + at, x);
      }
      if (more) {
        add_beyond(next);
        add_marked(j + 1, next);
        end_stats(j + 1, next);
      }
    }
    // the loads that the last row has asked for come back before the tiles are asked for again
    __builtin_amdgcn_s_waitcnt(0x0F70);
    asm volatile("" ::: "memory");
  }
}

// sum_t w_t loss_t in 64 bits, in a fixed order.
constexpr int kSumBlock = 1024;
__global__ __launch_bounds__(kSumBlock) void distill_sum_kernel(const float* __restrict__ losses, const float* __restrict__ weights, int n,
                                                                float* __restrict__ loss) {
  __shared__ double red[kSumBlock / kWave];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kSumBlock) {
    const float w = weights[i];
    if (w != 0.f) s += (double)w * (double)losses[i];
  }
  s = wave_sum_d(s);
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kSumBlock / kWave; ++w) s += red[w];
  *loss = (float)s;
}

}  // namespace axon

using namespace axon;

namespace {

constexpr int64_t kCacheBytes = int64_t(256) << 20;

int elem_bytes(int dtype) { return dtype == AXON_LOGITS_F32 ? 4 : 2; }

int check_rows(const void* p, int dtype, int64_t ld, int64_t n, int64_t v) {
  if (n < 0 || v <= 0 || ld < v || (dtype != AXON_LOGITS_F32 && dtype != AXON_LOGITS_BF16)) return AXON_ERR_ARG;
  if (n >= (int64_t)1 << 24 || v > (int64_t)kMaxShare * kMaxParts) return AXON_ERR_SHAPE;
  if (n > 0 && (!p || reinterpret_cast<uintptr_t>(p) % elem_bytes(dtype) != 0)) return AXON_ERR_ARG;
  return AXON_OK;
}

// The tail's flags: the type that the teacher's log-probabilities were stored in.
constexpr int kTailBits = 3, kTailFlags = AXON_DISTILL_FROM_BF16 | AXON_DISTILL_FROM_F16;
float step_of(int tail) { return tail & AXON_DISTILL_FROM_BF16 ? 0x1p-7f : tail & AXON_DISTILL_FROM_F16 ? 0x1p-10f : 0.f; }

bool usable(float temperature) { return temperature >= 0x1p-126f && temperature <= 3.402823466e38f; }  // smaller ones have no reciprocal

int check_teacher(const void* ids, const float* logprobs, int64_t k, int divergence, int flagged_tail, float beta, float temperature) {
  if (k < 1 || k > kMaxIds) return AXON_ERR_SHAPE;
  const int tail = flagged_tail & ~kTailFlags;
  if (!ids || !logprobs || divergence < AXON_DISTILL_FORWARD || divergence > AXON_DISTILL_JSD || tail < AXON_DISTILL_DROP ||
      tail > AXON_DISTILL_RENORMALIZE)
    return AXON_ERR_ARG;
  if (!usable(temperature)) return AXON_ERR_ARG;
  if (divergence == AXON_DISTILL_JSD && !(beta > 0.f && beta < 1.f)) return AXON_ERR_ARG;
  return AXON_OK;
}

// Workgroups per row of the backward: as in logits.hip, whose backward moves the same bytes.
int grad_parts(int64_t n, int64_t vocab, int eb) {
  if (n >= 1536) return 1;
  const int64_t fill = 8192 / (n > 0 ? n : 1), work = vocab * eb / (8 * 16 * kBlock);
  const int64_t p = fill < work ? fill : work;
  return (int)(p < 1 ? 1 : (p < kMaxParts ? p : kMaxParts));
}
// ... and of the forward: about 2048 pieces, what the part holds at once, none of them beyond what LDS describes.  One part where there
// are as many rows finishes them without a second launch (2047 x 50257 bf16 with gradient 144 us, 158 with it).
int stats_parts(int64_t n, int64_t vocab, int eb) {
  const int64_t fill = 2048 / (n > 0 ? n : 1), work = vocab * eb / (4 * 16 * kBlock), least = (vocab * eb / 16 + kMaxShare - 1) / kMaxShare;
  int64_t p = fill < work ? fill : work;
  p = p < least ? least : p;
  return (int)(p < 1 ? 1 : (p < kMaxParts ? p : kMaxParts));
}

}  // namespace

#define AXON_ROWS(dtype, CALL)                  \
  do {                                          \
    if ((dtype) == AXON_LOGITS_F32) CALL(float); \
    else CALL(unsigned short);                  \
  } while (0)

extern "C" int64_t axon_distill_workspace_bytes(int dtype, int64_t n, int64_t vocab) {
  if (n < 0 || vocab <= 0 || (dtype != AXON_LOGITS_F32 && dtype != AXON_LOGITS_BF16)) return AXON_ERR_ARG;
  return n * stats_parts(n, vocab, elem_bytes(dtype)) * (int64_t)sizeof(float4);
}

extern "C" int axon_distill_fwd(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab, const void* ids, int ids_i64,
                                const float* teacher_logprobs, int64_t k, const float* weights, int divergence, int tail, float beta,
                                float temperature, float* losses, float* covered, float* grads, float* coef, void* workspace,
                                int64_t workspace_bytes, int bwd_follows, void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc == AXON_OK && n > 0) rc = check_teacher(ids, teacher_logprobs, k, divergence, tail, beta, temperature);
  if (rc != AXON_OK || n == 0) return rc;
  if (!losses || !covered || !grads || !coef) return AXON_ERR_ARG;
  if (!workspace || workspace_bytes < axon_distill_workspace_bytes(dtype, n, vocab) || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return AXON_ERR_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  const int eb = elem_bytes(dtype), parts = stats_parts(n, vocab, eb);
  const Teacher t{ids, teacher_logprobs, weights, ids_i64, (int)k, divergence, tail & kTailBits, beta, 1.f / temperature, step_of(tail)};
  const RowOut out{losses, covered, grads, coef, (int)n};
  float4* const ws = static_cast<float4*>(workspace);
  const int64_t cached = bwd_follows ? kCacheBytes / (vocab * eb) : 0;
  const int cached_from = (int)(cached < n ? n - cached : 0);
  const unsigned lds = (unsigned)(((vocab * eb / 16 + parts - 1) / parts + 1 + 3) / 4 * 4);
#define AXON_FWD(T, REST)                                                                                                          \
  do {                                                                                                                             \
    hipLaunchKernelGGL((distill_stats_kernel<T, REST>), dim3((unsigned)(n * parts)), dim3(kBlock), REST ? lds : 0, st,             \
                       static_cast<const T*>(logits), ld, (int)vocab, parts, t, ws, out, cached_from);                             \
    AXON_CHECK_LAUNCH();                                                                                                           \
    if (parts > 1)                                                                                                                 \
      hipLaunchKernelGGL((distill_finish_kernel<T, REST>), dim3((unsigned)n), dim3(kWave), 0, st, static_cast<const T*>(logits), ld, \
                       (int)vocab, parts, t, ws, out);                                                                             \
  } while (0)
#define AXON_FWD_OF(T) \
  do {                 \
    if (t.tail == AXON_DISTILL_REST) AXON_FWD(T, true); else AXON_FWD(T, false); \
  } while (0)
  AXON_ROWS(dtype, AXON_FWD_OF);
#undef AXON_FWD_OF
#undef AXON_FWD
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

extern "C" int axon_distill_bwd(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab, const void* ids, int ids_i64,
                                int64_t k, const float* weights, float temperature, const float* grads, const float* coef,
                                const float* upstream, int ready, void* dlogits, int64_t ld_d, void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc == AXON_OK) rc = check_rows(dlogits, dtype, ld_d, n, vocab);
  if (rc != AXON_OK || n == 0) return rc;
  if (k < 1 || k > kMaxIds) return AXON_ERR_SHAPE;
  if (!ids || !grads || !coef || !usable(temperature) || (!upstream && !weights) || (ready && (!weights || !upstream))) return AXON_ERR_ARG;
  const hipStream_t st = (hipStream_t)stream;
  const int eb = elem_bytes(dtype), parts = grad_parts(n, vocab, eb);
  // every row of dlogits sits on the same offset from a 16-byte boundary as the row of logits
  const int vec_ok = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15) == 0 &&
                     (n <= 1 || ((ld - ld_d) * eb) % 16 == 0);
  const Teacher t{ids, nullptr, weights, ids_i64, (int)k, 0, 0, 0.f, 1.f / temperature, 0.f};
  const RowOut saved{nullptr, nullptr, const_cast<float*>(grads), const_cast<float*>(coef), (int)n};
#define AXON_GRAD(T)                                                                                                              \
  hipLaunchKernelGGL((distill_grad_kernel<T>), dim3((unsigned)(n * parts)), dim3(kBlock), 0, st, static_cast<const T*>(logits), ld, \
                     (int)vocab, t, saved, upstream, ready, static_cast<T*>(dlogits), ld_d, vec_ok, parts)
  AXON_ROWS(dtype, AXON_GRAD);
#undef AXON_GRAD
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

namespace {

// Rows of up to 66 KB: 192 threads that hold the row, three workgroups on a compute unit; up to 133 KB: 448, two; longer: 960, one, of
// which 375 KB are held and the rest is read twice.  More workgroups hide each other's outcomes, as many as hold their rows: 8192 x 33792
// bf16 take 250, 269 and 428 us with 192, 448 and 960 threads, 4096 x 65536 217 with 448 and 268 with 960.  Beyond kMaxTiles the marks
// of the given tokens have no room: such rows take the statistics and the gradient one after the other.
constexpr int64_t kMaxRowVecs = kMaxTiles * 960;
template <typename T, bool REST>
int launch_rows(const void* logits, int64_t ld, int64_t n, int64_t vocab, const Teacher& t, const RowOut& out, void* dlogits, int64_t ld_d,
                hipStream_t st) {
  const int64_t vecs = vocab / Row<T>::kPer;
#define AXON_ROW(ROW, NREG, NLDS, RESIDENT)                                                                                          \
  hipLaunchKernelGGL((distill_row_kernel<T, REST, ROW, NREG, NLDS, RESIDENT>), dim3((unsigned)(n < 256 * RESIDENT ? n : 256 * RESIDENT)),       \
                     dim3(ROW + kWave), 0, st, static_cast<const T*>(logits), ld, (int)vocab, t, out, static_cast<T*>(dlogits), ld_d)
  if (vecs <= 192 * 22) AXON_ROW(192, 18, 4, 3);
  else if (vecs <= 448 * 19) AXON_ROW(448, 14, 5, 2);
  else AXON_ROW(960, 18, 7, 1);
#undef AXON_ROW
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

}  // namespace

extern "C" int axon_distill_loss(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab, const void* ids, int ids_i64,
                                 const float* teacher_logprobs, int64_t k, const float* weights, int divergence, int tail, float beta,
                                 float temperature, float* loss, float* losses, float* covered, float* grads, float* coef, void* dlogits,
                                 int64_t ld_d, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!loss || (n > 0 && !weights)) return AXON_ERR_ARG;
  int rc = dlogits ? check_rows(dlogits, dtype, ld_d, n, vocab) : AXON_OK;
  const bool rows = rc == AXON_OK && dlogits && n >= 1 && vocab * elem_bytes(dtype) / 16 <= kMaxRowVecs;
  if (rows) {
    rc = check_rows(logits, dtype, ld, n, vocab);
    if (rc == AXON_OK) rc = check_teacher(ids, teacher_logprobs, k, divergence, tail, beta, temperature);
    if (rc != AXON_OK) return rc;
    if (!losses || !covered || !grads || !coef) return AXON_ERR_ARG;
    const Teacher t{ids, teacher_logprobs, weights, ids_i64, (int)k, divergence, tail & kTailBits, beta, 1.f / temperature, step_of(tail)};
    const RowOut out{losses, covered, grads, coef, (int)n};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == AXON_LOGITS_F32)
      rc = t.tail == AXON_DISTILL_REST ? launch_rows<float, true>(logits, ld, n, vocab, t, out, dlogits, ld_d, st)
                                     : launch_rows<float, false>(logits, ld, n, vocab, t, out, dlogits, ld_d, st);
    else
      rc = t.tail == AXON_DISTILL_REST ? launch_rows<unsigned short, true>(logits, ld, n, vocab, t, out, dlogits, ld_d, st)
                                     : launch_rows<unsigned short, false>(logits, ld, n, vocab, t, out, dlogits, ld_d, st);
  } else if (rc == AXON_OK) {
    rc = axon_distill_fwd(logits, dtype, ld, n, vocab, ids, ids_i64, teacher_logprobs, k, weights, divergence, tail, beta, temperature, losses,
                          covered, grads, coef, workspace, workspace_bytes, dlogits != nullptr, stream);
  }
  if (rc == AXON_OK && dlogits && !rows)
    rc = axon_distill_bwd(logits, dtype, ld, n, vocab, ids, ids_i64, k, weights, temperature, grads, coef, nullptr, 0, dlogits, ld_d, stream);
  if (rc != AXON_OK) return rc;
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(kSumBlock), 0, (hipStream_t)stream, losses, weights, (int)n, loss);
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}
