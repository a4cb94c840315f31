// Alternatives of materialised logits: the k largest of every row with their log-probabilities, or the log-probabilities
// of k given tokens per row, beside the entropy (and the label's log-probability); and the backward of both, which is
// one: dz_j = sum_i g_i [j = id_i] - p_j (sum_i g_i + g_H (log p_j + H)).
//
// Forward: ONE read of the row gives the softmax statistics and, for the k largest, the maxima of the row's segments of
// 256 bytes, from which select.h finds the few segments that are read again.  Bound by memory: 4096 x 151936 bf16 with 20
// alternatives and a label 214 us, 5.8 TB/s (a large device copy 4.8 to 5.0, read and write); 1500 x 151936 fp32 with 32 given
// tokens 149 us, 6.1 TB/s.  Short batches are bound by the two launches' latency: one row of 151936 5.4 + 7.0 us, of which the
// selection's trips to memory are most.
#include "logits_rows.h"
#include "select.h"
#include <type_traits>

namespace axon {

constexpr int kMaxParts = 64;
constexpr int kPartFloats = 4;      // what a part of a row leaves: M, e, s in two
constexpr int kSegVecs = 16;        // 16-byte vectors per segment: what sixteen neighbouring lanes load together
constexpr int kMaxTokenIds = AXON_MAX_TOKEN_IDS;  // given tokens per row

__device__ __forceinline__ int64_t load_id(const void* ids, int i64, int64_t at) {
  return i64 ? static_cast<const int64_t*>(ids)[at] : (int64_t) static_cast<const int32_t*>(ids)[at];
}

// A row as it is walked: the 16-byte vectors of its aligned middle in tiles of 256 (4 KB), one wavefront each at a time; the
// share of workgroup `part` of `parts` is whole tiles, and some of the elements outside the vectors.
constexpr int kTileVecs = 256;
struct SegSpan {
  int head, n_vec, n_scalar, n_seg, tile_lo, tile_hi;
  template <typename T>
  __device__ __forceinline__ SegSpan(const T* row, int vocab, int part, int parts) {
    const RowSpan sp(row, vocab, true, 0, 1);
    head = sp.head; n_vec = sp.n_vec; n_scalar = sp.n_scalar;
    n_seg = (n_vec + kSegVecs - 1) / kSegVecs;
    const int tiles = (n_vec + kTileVecs - 1) / kTileVecs;
    tile_lo = (int)((int64_t)tiles * part / parts);
    tile_hi = (int)((int64_t)tiles * (part + 1) / parts);
  }
  template <typename T>
  __device__ __forceinline__ int scalar(int i) const { return i < head ? i : i + n_vec * Row<T>::kPer; }
};

// Statistics of a set of logits: M >= every one of them (the largest, once there is one), s = sum 2^d, e = sum d 2^d over
// d = (z - M) log2(e).  The difference comes first: scaled by themselves, the type's lowest value overflows, -1e9 is off by 64,
// and every logit by what log2(e) has been rounded by (with the scaled maximum subtracted in one fused operation: 209 us for 215,
// log-probabilities near 0 off by 3e-6 of themselves for 4e-7).
constexpr float kLowest = -3.402823466e38f;

// Folds U times N logits into a thread's statistics, given the maxima of the U sets: one rescale at most.  A NaN or +inf among
// the logits makes the sums NaN, as it does those of a softmax; -inf adds nothing.
template <int N, int U, int M>
__device__ __forceinline__ void fold_all(Stats& a, const float (&z)[U][M], const float (&set_max)[U]) {
  float m = set_max[0];
#pragma unroll
  for (int u = 1; u < U; ++u) m = fmaxf(m, set_max[u]);
  if (m > a.M) {
    const float d = fmaxf((a.M - m) * kLog2e, kTiny), f = __builtin_amdgcn_exp2f(d);
    a.e = f * fmaf(a.s, d, a.e);
    a.s = a.s * f;
    a.M = m;
  }
  float s4[4] = {}, e4[4] = {};  // what is there joins at the end: one rounding of its size, not one per logit
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = (z[u][j] - a.M) * kLog2e, f = __builtin_amdgcn_exp2f(d);
      s4[j & 3] += f;
      e4[j & 3] = fmaf(f, fmaxf(d, kTiny), e4[j & 3]);
    }
  a.s += (s4[0] + s4[1]) + (s4[2] + s4[3]);
  a.e += (e4[0] + e4[1]) + (e4[2] + e4[3]);
}
template <int N, int M>
__device__ __forceinline__ float max_of(const float (&z)[M]) {
  float m = z[0];
#pragma unroll
  for (int j = 1; j < N; ++j) m = fmaxf(m, z[j]);
  return m;
}

// The threads' statistics together: the sum in 64 bits, since its roundings at each of the dozen merges are what the logarithm of a
// sum near 1 would consist of (a row with one likely token).
struct RowStats {
  float M, e;
  double s;
};
__device__ __forceinline__ RowStats merge(const RowStats& a, const RowStats& b) {
  const float M = fmaxf(a.M, b.M);
  const float d1 = fmaxf((a.M - M) * kLog2e, kTiny), d2 = fmaxf((b.M - M) * kLog2e, kTiny);
  const float f1 = __builtin_amdgcn_exp2f(d1), f2 = __builtin_amdgcn_exp2f(d2);
  return {M, f1 * fmaf((float)a.s, d1, a.e) + f2 * fmaf((float)b.s, d2, b.e), a.s * f1 + b.s * f2};
}
__device__ __forceinline__ RowStats wave_merge(RowStats st) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    st = merge(st, RowStats{__shfl_down(st.M, off, kWave), __shfl_down(st.e, off, kWave), __shfl_down(st.s, off, kWave)});
  return st;
}

// The lanes of a wavefront as rows of sixteen: row 1 of a changes place with row 0 of b and row 3 of a with row 2 of b, or
// rows 2 and 3 of a with rows 0 and 1 of b.  Written as instructions: through the builtins the compiler takes the two
// results for one value.  The s_nop covers the wait states that the swaps need after a vector instruction.
__device__ __forceinline__ void swap_rows16(float& a, float& b) {
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void swap_rows32(float& a, float& b) {
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}

// A tile's 256 vectors in the lanes: lane 16 r + c loads, of every 64 consecutive ones, number 16 (c / 4) + 4 r + c % 4, so
// that a segment's sixteen vectors of load u lie in the four lanes of the same c / 4 in each row.
__device__ __forceinline__ int tile_vec(int lane) { return ((lane & 12) << 2) + ((lane >> 4) << 2) + (lane & 3); }
// The maxima of the tile's sixteen segments from those of a lane's four vectors: segment 4 u + c / 4 in the lanes 16 u + c.
// Three swaps carry the four values over the rows at once, two steps the rest: 13 instructions for 4 KB, where a reduction
// of each value by itself took 32 and its store as many again.
__device__ __forceinline__ float tile_maxima(const float (&v)[4]) {
  float a = v[0], b = v[1], c = v[2], d = v[3];
  swap_rows16(a, b);
  swap_rows16(c, d);
  float x = fmaxf(a, b), y = fmaxf(c, d);
  swap_rows32(x, y);
  x = fmaxf(x, y);
  x = fmaxf(x, dpp_or_own<0xb1, 0xf>(x));  // lane ^ 1
  return fmaxf(x, dpp_or_own<0x4e, 0xf>(x));  // lane ^ 2
}

struct RowOut {
  float *logprob, *entropy, *lse;  // logprob, entropy may be null; lse [2][n]
  const void* labels;              // may be null
  int labels_i64, n;
};
// A log-sum-exp and what its rounding to 32 bits has left of it: the log-probability of logit z is (z - lse) - rest.
struct RowLse {
  float lse, rest;
  __device__ __forceinline__ float logprob(float z) const { return (z - lse) - rest; }
};
// ln s of s >= 1 from its exponent and its mantissa in [0.7, 1.4), by the series of 2 artanh: to 2^-23 of itself also near s = 1.
__device__ __forceinline__ double log_of_sum(double s) {
  int ex = __builtin_amdgcn_frexp_exp(s);
  double m = __builtin_amdgcn_frexp_mant(s);
  if (m < 0.70710678) { m *= 2.0; ex -= 1; }
  const float f = (float)(m - 1.0) / (float)(m + 1.0), f2 = f * f;
  const float series = fmaf(f2, fmaf(f2, fmaf(f2, fmaf(f2, 1.f / 9, 1.f / 7), 1.f / 5), 1.f / 3), 1.f);
  return (double)ex * 0.6931471805599453 + (double)(2.f * f * series);
}
__device__ __forceinline__ RowLse row_lse(const RowStats& st, double ln_s) {
  const float lse = st.s > 0.0 ? (float)((double)st.M + ln_s) : NAN;  // NaN: a row of -inf alone
  return RowLse{lse, (float)(((double)st.M - lse) + ln_s)};
}

struct Picks {
  const void* ids;  // [n][k]
  int ids_i64, k;
  float* out;       // [n][k]
};
template <typename T>
__device__ __forceinline__ void write_picks(const Picks& p, int t, const T* row, int vocab, RowLse lse) {
  for (int i = threadIdx.x; i < p.k; i += kBlock) {
    const int64_t id = load_id(p.ids, p.ids_i64, (int64_t)t * p.k + i);
    p.out[(int64_t)t * p.k + i] = (id >= 0 && id < vocab) ? lse.logprob(Row<T>::one(row + id)) : 0.f;
  }
}

// A row of logits as select_top reads it.
template <typename T, int HELD>
struct LogitsSource {
  static constexpr int kPer = Row<T>::kPer, kItems = kSegVecs, kHeld = HELD;
  const T* row;
  const float* seg_max;  // LDS or global
  SegSpan sp;
  int vocab;
  __device__ int n_segs() const { return sp.n_seg; }
  __device__ uint32_t max_key(int i) const { return order_key(seg_max[i]); }
  __device__ int limit() const { return vocab; }
  __device__ int load(const int* segs, int j, float (&v)[kPer]) const {
    const int q = segs[j / kSegVecs] * kSegVecs + (j & (kSegVecs - 1));
    if (q >= sp.n_vec) return -1;
    float x[8];
    const int at = sp.head + q * kPer;
    Row<T>::template load<true>(row + at, x);
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = x[e];
    return at;
  }
  __device__ int n_single() const { return sp.n_scalar; }
  __device__ float single(int i, int& index) const {
    index = sp.scalar<T>(i);
    return Row<T>::one(row + index);
  }
};

struct TopOut {
  float* logprobs;  // [n][k]
  int64_t* ids;     // [n][k]
  int k;
};
// What is wanted of a row beside its statistics.
enum Want { kTokens, kTop };

// The end of a row: log-sum-exp and entropy from its statistics (in thread 0), then what is wanted of it.  HELD: how many
// maxima a thread holds, 0 where they are in LDS.
template <typename T, Want WANT, int HELD>
__device__ __forceinline__ void finish_row(RowStats st, int t, const T* row, int vocab, const float* seg_max, const RowOut& out,
                                           const Picks& picks, const TopOut& top, SelectLds* sel) {
  __shared__ RowLse s_lse;
  const int tid = threadIdx.x;
  if (tid == 0) {
    const double ln_s = log_of_sum(st.s);
    s_lse = row_lse(st, ln_s);
    out.lse[t] = s_lse.lse;
    out.lse[(int64_t)out.n + t] = s_lse.rest;
    if (out.entropy != nullptr) out.entropy[t] = (float)ln_s - st.e / (float)st.s * kLn2;
  }
  if (WANT == kTokens) {
    __syncthreads();
    write_picks<T>(picks, t, row, vocab, s_lse);
    return;
  }
  // the last thread asks for the label's logit here and uses it at the end: the label is a trip to memory, its logit another
  const bool with_label = tid == kBlock - 1 && out.logprob != nullptr;
  const int64_t lab = with_label ? load_id(out.labels, out.labels_i64, t) : -1;
  const bool inside = lab >= 0 && lab < vocab;
  const float label_z = inside ? Row<T>::one(row + lab) : 0.f;
  // (the selection's own barriers come before the first use of s_lse)
  const LogitsSource<T, HELD> src{row, seg_max, SegSpan(row, vocab, 0, 1), vocab};
  select_top(src, top.k, *sel, tid, [&](int rank, float z, int index) {
    top.logprobs[(int64_t)t * top.k + rank] = s_lse.logprob(z);
    top.ids[(int64_t)t * top.k + rank] = index;
  });
  if (with_label) out.logprob[t] = inside ? s_lse.logprob(label_z) : 0.f;
}

// Workgroup (row, part): blockIdx.x = row * parts + part.  Where a row has one part it is finished here: a row's selection
// runs beside the reading of the rows that the compute unit's other workgroups have (the maxima of its segments are in
// LDS).  Else the statistics go to ws[row][part][kPartFloats] and the maxima to seg_max[row][seg], for the kernels below.
// Rows from `cached_from` on are left in the cache in front of the memory, for what reads them next.
template <typename T, Want WANT>
__global__ __launch_bounds__(kBlock) void alternatives_kernel(const T* __restrict__ logits, int64_t ld, int vocab, int parts,
                                                              float* __restrict__ ws, float* __restrict__ seg_max, int seg_stride,
                                                              RowOut out, Picks picks, TopOut top, int cached_from) {
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[2][kBlock / kWave];
  __shared__ double red_s[kBlock / kWave];
  const int t = blockIdx.x / parts, part = blockIdx.x - t * parts;
  const T* row = logits + (int64_t)t * ld;
  constexpr int kPer = Row<T>::kPer;
  const SegSpan sp(row, vocab, part, parts);
  const T* body = row + sp.head;
  const bool whole = parts == 1 && seg_max == nullptr;
  float* const segs = reinterpret_cast<float*>(smem + sizeof(SelectLds));  // where the row is finished here
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  Stats mine_st{kLowest, 0.f, 0.f};
  auto walk = [&](auto cached) {
    constexpr bool kCached = decltype(cached)::value;
    const int mine = tile_vec(lane);
    for (int tile = sp.tile_lo + wave; tile < sp.tile_hi; tile += kBlock / kWave) {
      float v[4][8], m[4];
      const int q0 = tile * kTileVecs + mine;
      if ((tile + 1) * kTileVecs <= sp.n_vec) {
#pragma unroll
        for (int u = 0; u < 4; ++u) Row<T>::template load<kCached>(body + (uint32_t)(q0 + u * kWave) * kPer, v[u]);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
          for (int j = 0; j < kPer; ++j) v[u][j] = -INFINITY;
          if (q0 + u * kWave < sp.n_vec) Row<T>::template load<kCached>(body + (uint32_t)(q0 + u * kWave) * kPer, v[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) m[u] = max_of<kPer>(v[u]);
      fold_all<kPer>(mine_st, v, m);
      if (WANT == kTop) {
        const float best = tile_maxima(m);
        const int seg = tile * (kTileVecs / kSegVecs) + (lane >> 2);
        if ((lane & 3) == 0 && seg < sp.n_seg) {
          if (whole) segs[seg] = best;
          else seg_max[(int64_t)t * seg_stride + seg] = best;
        }
      }
    }
  };
  if (t >= cached_from) walk(std::true_type{}); else walk(std::false_type{});
  for (int i = part * kBlock + tid; i < sp.n_scalar; i += parts * kBlock) {
    const float v[1][1] = {{Row<T>::one(row + sp.scalar<T>(i))}};
    fold_all<1>(mine_st, v, v[0]);
  }
  RowStats st = wave_merge(RowStats{mine_st.M, mine_st.e, mine_st.s});
  if (lane == 0) { red[0][wave] = st.M; red[1][wave] = st.e; red_s[wave] = st.s; }
  __syncthreads();
  if (tid == 0)
    for (int w = 1; w < kBlock / kWave; ++w) st = merge(st, RowStats{red[0][w], red[1][w], red_s[w]});
  if (whole) {
    finish_row<T, WANT, 0>(st, t, row, vocab, segs, out, picks, top, reinterpret_cast<SelectLds*>(smem));
  } else if (tid == 0) {
    float* o = ws + (int64_t)blockIdx.x * kPartFloats;
    o[0] = st.M; o[1] = st.e; o[2] = (float)st.s; o[3] = (float)(st.s - (float)st.s);
  }
}

// The statistics of a row's parts (at most kMaxParts), in a fixed tree; the total in thread 0.
__device__ __forceinline__ RowStats merge_parts(const float* ws, int t, int parts) {
  RowStats st{kLowest, 0.f, 0.0};
  if ((int)threadIdx.x < parts) {
    const float* o = ws + ((int64_t)t * parts + threadIdx.x) * kPartFloats;
    st = RowStats{o[0], o[1], (double)o[2] + (double)o[3]};
  }
  return threadIdx.x < kWave ? wave_merge(st) : st;
}

// The end of rows that several workgroups have read, by a workgroup per row.  (In the launch before, by the workgroup that draws
// a row's last ticket: one row of 151936 11.6 us for 12.5, but 61 x 201088 fp32 34 for 21 and 187 x 151936 51 for 23, for the
// maxima that have to be written through to the level that the XCDs share.)
template <typename T, Want WANT>
__global__ __launch_bounds__(kBlock) void alternatives_finish_kernel(const T* __restrict__ logits, int64_t ld, int vocab, int parts,
                                                                     const float* __restrict__ ws,
                                                                     const float* __restrict__ seg_max, int seg_stride, RowOut out,
                                                                     Picks picks, TopOut top) {
  __shared__ SelectLds s;
  const int t = blockIdx.x;
  const T* row = logits + (int64_t)t * ld;
  // 13 maxima per thread: 3328, 201088 fp32 logits have 3142
  finish_row<T, WANT, 13>(merge_parts(ws, t, parts), t, row, vocab, WANT == kTop ? seg_max + (int64_t)t * seg_stride : nullptr,
                          out, picks, top, &s);
}

// Upstream gradients of a row's chosen tokens: k of them, and a label's.  Either may be absent (g null).
struct TokenGrads {
  const void* ids;  // [n][k]
  const float* g;   // [n][k]
  const void* labels;
  const float* g_label;
  int ids_i64, k, labels_i64;
};

// dz_j = sum_i g_i [j = id_i] - p_j (G + g_H (log p_j + H)), G the sum of the g of the ids in the vocabulary.
// The row is streamed without a look at the ids; the few elements that have one are written again afterwards, from
// logits that were read before (dlogits may be the logits' own storage).  Equal ids of a row add up in their order, in the
// thread of the first of them, so that the result repeats bit for bit.  Rows are walked from the last to the first, as
// the forward leaves them in the cache.  Bound by memory: 1500 x 151936 fp32 360 us, 5.1 TB/s read and written; 2047 x 50257
// bf16, rows on every boundary, 83 us, 5.0 TB/s.
template <typename T>
__global__ __launch_bounds__(kBlock) void tokens_grad_kernel(const T* logits, int64_t ld, int vocab, TokenGrads tg,
                                                             int n, const float* __restrict__ lse,
                                                             const float* __restrict__ entropy,
                                                             const float* __restrict__ g_entropy, T* dlogits, int64_t ld_d,
                                                             int vec_ok, int parts) {
  constexpr int kMost = kMaxTokenIds + 1, kSlots = (kMost + kBlock - 1) / kBlock;
  __shared__ int ids[kMost];
  __shared__ float gs[kMost];
  __shared__ float red[kBlock / kWave];
  const int b = gridDim.x - 1 - blockIdx.x, t = b / parts, part = b - t * parts, tid = threadIdx.x;
  const T* row = logits + (int64_t)t * ld;
  T* out = dlogits + (int64_t)t * ld_d;
  constexpr int kPer = Row<T>::kPer;
  const int with_label = tg.g_label != nullptr, n_ids = (tg.g != nullptr ? tg.k : 0) + with_label;
  float sum = 0.f;
  for (int i = tid; i < n_ids; i += kBlock) {
    const bool lab = with_label && i == 0;
    const int64_t at = (int64_t)t * tg.k + i - with_label;
    const int64_t id = lab ? load_id(tg.labels, tg.labels_i64, t) : load_id(tg.ids, tg.ids_i64, at);
    const bool ok = id >= 0 && id < vocab;
    const float g = !ok ? 0.f : lab ? tg.g_label[t] : tg.g[at];
    ids[i] = ok ? (int)id : -1;
    gs[i] = g;
    sum += g;
  }
  sum = wave_sum(sum);
  if ((tid & (kWave - 1)) == 0) red[tid / kWave] = sum;
  __syncthreads();
  const float G = (red[0] + red[1]) + (red[2] + red[3]);
  const float lse_v = lse[t], rest = lse[n + t], g_en = g_entropy ? g_entropy[t] : 0.f;
  const float H = (g_entropy ? entropy[t] : 0.f) - rest, rest2 = rest * kLog2e;
  auto grad = [&](float z) {  // log p = z - lse - rest
    const float d = z - lse_v, p = __builtin_amdgcn_exp2f(fmaf(d, kLog2e, -rest2));
    return p * ((p > 0.f) ? fmaf(-g_en, d + H, -G) : -G);  // a probability of 0 takes nothing from the entropy
  };
  const RowSpan sp(row, vocab, vec_ok != 0, part, parts);
  // the ids that are this part's, each in the thread of its first occurrence
  float again[kSlots];
  int where[kSlots];
#pragma unroll
  for (int u = 0; u < kSlots; ++u) {
    const int i = tid + u * kBlock;
    where[u] = -1;
    if (i >= n_ids) continue;
    const int id = ids[i];
    if (id < 0) continue;
    const int in = id - sp.head, q = in / kPer;
    const int single = in < 0 ? id : id - sp.n_vec * kPer;  // its number among the elements outside the vectors
    const bool vec = in >= 0 && q < sp.n_vec;
    if (vec ? (q < sp.q_lo || q >= sp.q_hi) : (single / kBlock % parts != part)) continue;
    float total = 0.f;
    bool first = true;
    for (int j = 0; j < n_ids; ++j) {
      if (ids[j] != id) continue;
      if (j < i) { first = false; break; }
      total += gs[j];
    }
    if (!first) continue;
    where[u] = id;
    again[u] = grad(Row<T>::one(row + id)) + total;
  }
  __syncthreads();  // nothing of the row is written before these are read
  const T* body = row + sp.head;
  T* body_out = out + sp.head;
  auto finish = [&](int q, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = grad(v[j]);
    Row<T>::store(body_out + (uint32_t)q * kPer, v);
  };
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
  for (int i = part * kBlock + tid; i < sp.n_scalar; i += parts * kBlock) {
    const int j = sp.scalar<T>(i);
    Row<T>::store_one(out + j, grad(Row<T>::one(row + j)));
  }
  // the stores above are acknowledged before another thread of the workgroup writes the same element
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0)
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSlots; ++u)
    if (where[u] >= 0) Row<T>::store_one(out + where[u], again[u]);
}

}  // namespace axon

using namespace axon;

namespace {

// Workgroups per row of the backward: as in logits.hip, whose backward moves the same bytes.
int row_parts(int64_t n, int64_t vocab, int elem_bytes) {
  if (n >= 1536) return 1;
  const int64_t fill = 8192 / (n > 0 ? n : 1), work = vocab * elem_bytes / (8 * 16 * kBlock);
  const int64_t p = fill < work ? fill : work;
  return (int)(p < 1 ? 1 : (p < kMaxParts ? p : kMaxParts));
}
// ... and of the forward.  From 512 rows on a row is left to one workgroup, which finishes it (20 alternatives, split / whole, us:
// 512 x 201088 fp32 82 / 72, 1300 x 201088 194 / 184, 1500 x 151936 bf16 92 / 83, 512 x 151936 bf16 42 / 45; 320 x 201088
// 55 / 65).  Fewer rows are split into about 2048 pieces, what the part holds at once, of at least a tile per wavefront (250 x
// 151936 bf16 25.9 us for 27.0 with 8192 pieces, 400 32.5 for 35.4; one row 11.8 for 12.4 with pieces twice as long).
int fwd_parts(int64_t n, int64_t vocab, int elem_bytes) {
  if (n >= 512) return 1;
  const int64_t fill = 2048 / (n > 0 ? n : 1), work = vocab * elem_bytes / (kTileVecs * 16 * (kBlock / kWave));
  const int64_t p = fill < work ? fill : work;
  return (int)(p < 1 ? 1 : (p < kMaxParts ? p : kMaxParts));
}

constexpr int64_t kCacheBytes = int64_t(256) << 20;

int elem_bytes(int dtype) { return dtype == AXON_LOGITS_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == AXON_LOGITS_F32 || dtype == AXON_LOGITS_BF16; }
int64_t seg_stride(int dtype, int64_t vocab) {
  const int64_t per = 16 / elem_bytes(dtype) * kSegVecs;
  return (vocab + per - 1) / per;
}

// What a workgroup that finishes its row holds in LDS; more than this and the rows are finished by a kernel of their own.
constexpr int64_t kMaxTopLds = 48 * 1024;
int64_t top_lds(int dtype, int64_t vocab) { return (int64_t)sizeof(SelectLds) + seg_stride(dtype, vocab) * 4; }

int check_rows(const void* logits, int dtype, int64_t ld, int64_t n, int64_t v) {
  if (n < 0 || v <= 0 || ld < v || !dtype_ok(dtype)) return AXON_ERR_ARG;
  if (n >= (int64_t)1 << 24 || v >= (int64_t)1 << 30) return AXON_ERR_SHAPE;  // rows times parts are a grid
  if (n > 0 && (!logits || reinterpret_cast<uintptr_t>(logits) % elem_bytes(dtype) != 0)) return AXON_ERR_ARG;
  return AXON_OK;
}

int cached_from(int64_t n, int64_t vocab, int eb, int bwd_follows) {
  const int64_t cached = bwd_follows ? kCacheBytes / (vocab * eb) : 0;
  return (int)(cached < n ? n - cached : 0);
}

}  // namespace

#define AXON_ROWS(dtype, CALL)                     \
  do {                                             \
    if ((dtype) == AXON_LOGITS_F32) CALL(float);   \
    else CALL(unsigned short);                     \
  } while (0)

extern "C" int64_t axon_logits_top_workspace_bytes(int dtype, int64_t n, int64_t vocab) {
  if (n < 0 || vocab <= 0 || !dtype_ok(dtype)) return AXON_ERR_ARG;
  const int parts = fwd_parts(n, vocab, elem_bytes(dtype));
  if (parts == 1 && top_lds(dtype, vocab) <= kMaxTopLds) return 0;
  return n * (parts * kPartFloats + seg_stride(dtype, vocab)) * (int64_t)sizeof(float);
}

extern "C" int axon_logits_top_fwd(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab, int64_t k,
                                   const void* labels, int labels_i64, float* logprob, float* entropy, float* lse,
                                   float* top_logprobs, int64_t* top_ids, float* workspace, int64_t workspace_bytes,
                                   int bwd_follows, void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc != AXON_OK) return rc;
  if (k < 1 || k > kMaxTop || k > vocab) return AXON_ERR_SHAPE;
  if (n == 0) return AXON_OK;
  if (!lse || !top_logprobs || !top_ids || (logprob && !labels)) return AXON_ERR_ARG;
  const int64_t need = axon_logits_top_workspace_bytes(dtype, n, vocab);
  if (need > 0 && !workspace) return AXON_ERR_ARG;
  if (need > workspace_bytes) return AXON_ERR_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  const int eb = elem_bytes(dtype), parts = fwd_parts(n, vocab, eb);
  const bool whole = need == 0;
  float* const seg_max = whole ? nullptr : workspace + n * parts * kPartFloats;
  const int stride = (int)seg_stride(dtype, vocab), from = cached_from(n, vocab, eb, bwd_follows);
  const unsigned lds = whole ? (unsigned)top_lds(dtype, vocab) : 0;
  const RowOut out{logprob, entropy, lse, labels, labels_i64, (int)n};
  const TopOut top{top_logprobs, top_ids, (int)k};
#define AXON_TOP(T)                                                                                                        \
  do {                                                                                                                     \
    hipLaunchKernelGGL((alternatives_kernel<T, kTop>), dim3((unsigned)(n * parts)), dim3(kBlock), lds, st,                 \
                       static_cast<const T*>(logits), ld, (int)vocab, parts, workspace, seg_max, stride, out, Picks{}, top, \
                       from);                                                                                              \
    AXON_CHECK_LAUNCH();                                                                                                   \
    if (!whole)                                                                                                            \
      hipLaunchKernelGGL((alternatives_finish_kernel<T, kTop>), dim3((unsigned)n), dim3(kBlock), 0, st, static_cast<const T*>(logits),    \
                         ld, (int)vocab, parts, workspace, seg_max, stride, out, Picks{}, top);                                     \
  } while (0)
  AXON_ROWS(dtype, AXON_TOP);
#undef AXON_TOP
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

extern "C" int64_t axon_logits_tokens_workspace_bytes(int dtype, int64_t n, int64_t vocab) {
  if (n < 0 || vocab <= 0 || !dtype_ok(dtype)) return AXON_ERR_ARG;
  const int parts = fwd_parts(n, vocab, elem_bytes(dtype));
  return parts > 1 ? n * parts * kPartFloats * (int64_t)sizeof(float) : 0;
}

extern "C" int axon_logits_tokens_fwd(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab, const void* ids,
                                      int ids_i64, int64_t k, float* logprobs, float* entropy, float* lse, float* workspace,
                                      int64_t workspace_bytes, int bwd_follows, void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc != AXON_OK) return rc;
  if (k < 1 || k > kMaxTokenIds) return AXON_ERR_SHAPE;
  if (n == 0) return AXON_OK;
  if (!lse || !ids || !logprobs) return AXON_ERR_ARG;
  const int eb = elem_bytes(dtype), parts = fwd_parts(n, vocab, eb);
  const int64_t need = axon_logits_tokens_workspace_bytes(dtype, n, vocab);
  if (need > 0 && (!workspace || need > workspace_bytes)) return AXON_ERR_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  const RowOut out{nullptr, entropy, lse, nullptr, 0, (int)n};
  const Picks picks{ids, ids_i64, (int)k, logprobs};
  const int from = cached_from(n, vocab, eb, bwd_follows);
#define AXON_TOKENS(T)                                                                                                      \
  do {                                                                                                                      \
    hipLaunchKernelGGL((alternatives_kernel<T, kTokens>), dim3((unsigned)(n * parts)), dim3(kBlock), 0, st,                 \
                       static_cast<const T*>(logits), ld, (int)vocab, parts, workspace, nullptr, 0, out, picks, TopOut{},   \
                       from);                                                                                               \
    AXON_CHECK_LAUNCH();                                                                                                    \
    if (parts > 1)                                                                                                          \
      hipLaunchKernelGGL((alternatives_finish_kernel<T, kTokens>), dim3((unsigned)n), dim3(kBlock), 0, st, static_cast<const T*>(logits),  \
                         ld, (int)vocab, parts, workspace, nullptr, 0, out, picks, TopOut{});                                                     \
  } while (0)
  AXON_ROWS(dtype, AXON_TOKENS);
#undef AXON_TOKENS
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

extern "C" int axon_logits_tokens_bwd(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab, const void* ids,
                                      int ids_i64, int64_t k, const void* labels, int labels_i64, const float* lse,
                                      const float* entropy, const float* g_ids, const float* g_label, const float* g_entropy,
                                      void* dlogits, int64_t ld_d, void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc != AXON_OK) return rc;
  if (k < 0 || k > kMaxTokenIds) return AXON_ERR_SHAPE;
  if (n == 0) return AXON_OK;
  if (!lse || !dlogits || ld_d < vocab || reinterpret_cast<uintptr_t>(dlogits) % elem_bytes(dtype) != 0) return AXON_ERR_ARG;
  if ((g_ids && !ids) || (g_label && !labels) || (g_entropy && !entropy)) return AXON_ERR_ARG;
  const hipStream_t st = (hipStream_t)stream;
  const int eb = elem_bytes(dtype), parts = row_parts(n, vocab, eb);
  // every row of dlogits sits on the same offset from a 16-byte boundary as the row of logits
  const int vec_ok = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15) == 0 &&
                     (n <= 1 || ((ld - ld_d) * eb) % 16 == 0);
  const TokenGrads tg{ids, g_ids, labels, g_label, ids_i64, (int)k, labels_i64};
#define AXON_GRAD(T)                                                                                                       \
  hipLaunchKernelGGL((tokens_grad_kernel<T>), dim3((unsigned)(n * parts)), dim3(kBlock), 0, st,                             \
                     static_cast<const T*>(logits), ld, (int)vocab, tg, (int)n, lse, entropy, g_entropy, static_cast<T*>(dlogits), \
                     ld_d, vec_ok, parts)
  AXON_ROWS(dtype, AXON_GRAD);
#undef AXON_GRAD
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}
