// The balance loss of a mixture of experts and the experts' loads.  For every layer and every sequence (or the batch as one)
// with T unmasked tokens
//   loss = sum_e E / (k T^2) c_e P_e,   P_e = sum_t m_t p_te,   c_e = choices of expert e among the unmasked tokens,
// averaged over the sequences that have tokens and over the layers; p: softmax of a token's logits, or their sigmoids divided
// by their sum.  c is a count and constant for the gradient:
//   d loss / d x_te = m_t E / (k T^2) slope_te (c_e - sum_j p_tj c_j),   slope = p (softmax), p (1 - sigmoid(x)).
//
// A row of E logits lies in G neighbouring lanes, 8 or 16 consecutive ones per lane.  Tokens go in chunks, one workgroup per
// chunk and layer; a chunk leaves one partial (P and c of every expert, T) per sequence that it meets, at index chunk +
// sequence, which is different for every such pair and below chunks + sequences.  A second kernel adds the partials of a
// sequence in a fixed order, so that results repeat bit for bit.
#include "common.h"
#include "select.h"
#include <algorithm>

namespace axon {

constexpr int kMaxLayers = 64;     // per launch: their pointers travel as kernel arguments
constexpr int kMaxExperts = AXON_MAX_EXPERTS;

enum Score { kSoftmax = 0, kSigmoid = 1 };

struct LayerPtrs { const void* p[kMaxLayers]; };

struct BalanceParams {
  int64_t ld;              // elements between rows of logits
  int n_tokens, experts, k, chunk, n_chunks, layers, first_layer;  // layers: of the whole call
  const void* mask;        // may be null
  const int32_t* cu;       // null: one sequence of all tokens
  int n_seqs, ids_i64, quads;  // quads: rows can be read four elements at a time (1), or sixteen bytes (2)
  float* part_p;           // [slots][layers][experts]
  int* part_c;             // the same
  int* part_t;             // [slots]
  int* ticket;                 // zeroed by the first kernel
  unsigned long long* counts;  // [layers][experts]
  const float* coef;       // [n_seqs][layers][experts]
  const float* scale;      // what the mean over sequences and layers multiplies by
  const float* g_loss;
};

template <typename T> struct RouterRow;
template <> struct RouterRow<float> {
  static __device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  }
  static __device__ __forceinline__ float load1(const float* p) { return *p; }
  static __device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
    const f32x4 x = {v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p) = x;
  }
  static __device__ __forceinline__ void store1(float* p, float v) { *p = v; }
};
template <> struct RouterRow<__bf16> {
  static __device__ __forceinline__ void load4(const __bf16* p, float (&v)[4]) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
    v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
  }
  static __device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
  static __device__ __forceinline__ void store4(__bf16* p, const float (&v)[4]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = {v[0], v[1]}, b = {v[2], v[3]};
    uint2 x;
    x.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(a, bf16x2));
    x.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(b, bf16x2));
    *reinterpret_cast<uint2*>(p) = x;
  }
  static __device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }
};

// Reductions over the G lanes of a row, the result in each of them: DPP steps inside sixteen lanes, register swaps beyond (a
// shuffle would take a trip through the LDS crossbar with a wait behind it).  All 64 lanes have to be active.
template <int CTRL, class T>
__device__ __forceinline__ T dpp(T v) {
  const int i = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, i, CTRL, 0xf, 0xf, true));  // every lane has a source
}
// The compiler takes the two results of a swap for one value where the builtin is used; the s_nop covers the wait states
// behind the instruction that has written the operands.
template <class T, class Op>
__device__ __forceinline__ T over_rows16(T v, Op op) {
  T w = v;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(w));
  return op(v, w);
}
template <class T, class Op>
__device__ __forceinline__ T over_rows32(T v, Op op) {
  T w = v;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(v), "+v"(w));
  return op(v, w);
}
template <int G, class T, class Op>
__device__ __forceinline__ T row_reduce(T v, Op op) {
  if (G > 1) v = op(v, dpp<0xb1>(v));    // lane ^ 1
  if (G > 2) v = op(v, dpp<0x4e>(v));    // lane ^ 2
  if (G > 4) v = op(v, dpp<0x141>(v));   // the mirror lane of eight: any of the other four
  if (G > 8) v = op(v, dpp<0x140>(v));   // the mirror lane of sixteen
  if (G > 16) v = over_rows16(v, op);
  if (G > 32) v = over_rows32(v, op);
  return v;
}
// The other way: over the lanes of a wavefront that hold the same experts of different rows (the same lane modulo G).
template <int G, class T, class Op>
__device__ __forceinline__ T column_reduce(T v, Op op) {
  if (G <= 1) v = op(v, dpp<0xb1>(v));
  if (G <= 2) v = op(v, dpp<0x4e>(v));
  if (G <= 4) v = op(v, dpp<0x124>(v));  // turned by four inside sixteen lanes
  if (G <= 8) v = op(v, dpp<0x128>(v));  // by eight
  if (G <= 16) v = over_rows16(v, op);
  if (G <= 32) v = over_rows32(v, op);
  return v;
}

struct Add { template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; } };
struct MaxF { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct MaxU { __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); } };

template <typename T, int V>
__device__ __forceinline__ void load_row(const T* row, int e0, int experts, int quads, float (&x)[V]) {
  if (sizeof(T) == 2 && quads == 2) {
#pragma unroll
    for (int j = 0; j < V; j += 8) {
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      u32x4 w = {0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};  // -inf
      if (e0 + j < experts) w = *reinterpret_cast<const u32x4*>(row + e0 + j);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        x[j + 2 * q] = __uint_as_float(w[q] << 16);
        x[j + 2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; j += 4) {
    float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (quads) {
      if (e0 + j < experts) RouterRow<T>::load4(row + e0 + j, v);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e0 + j + q < experts) v[q] = RouterRow<T>::load1(row + e0 + j + q);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) x[j + q] = v[q];
  }
}

// A row's scores are w * inv; for sigmoids also 1 - sigmoid (from the exponential where the sigmoid is close to 1, and would
// cancel).  What lies beyond the experts (-inf) gets w = 0.
template <int G, int V, int SCORE>
__device__ __forceinline__ float scores(const float (&x)[V], float (&w)[V], float (&rest)[V]) {
  constexpr float kLog2e = 1.4426950408889634f;
  float sum = 0.f;
  if constexpr (SCORE == kSoftmax) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < V; ++j) m = fmaxf(m, x[j]);
    m = row_reduce<G>(m, MaxF());
#pragma unroll
    for (int j = 0; j < V; ++j) sum += w[j] = __builtin_amdgcn_exp2f((x[j] - m) * kLog2e);  // m * log2(e) may overflow
    return __builtin_amdgcn_rcpf(row_reduce<G>(sum, Add()));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float ex = __builtin_amdgcn_exp2f(x[j] * -kLog2e);
      sum += w[j] = __builtin_amdgcn_rcpf(1.f + ex);
      rest[j] = x[j] > 0.f ? ex * w[j] : 1.f - w[j];
    }
    sum = row_reduce<G>(sum, Add());
    // rows whose sigmoids are all next to nothing: there they are exponentials, to a relative 2^-90, and their ratios a softmax
    const bool tiny = sum < 0x1p-90f;
    if (__builtin_amdgcn_ballot_w64(tiny) != 0) {
      float s[V], unused[V];
      const float inv = scores<G, V, kSoftmax>(x, s, unused);
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = tiny ? s[j] : w[j];
      return tiny ? inv : __builtin_amdgcn_rcpf(sum);
    }
    return __builtin_amdgcn_rcpf(sum);
  }
}

// Keys in descending order (Batcher's odd-even merge sort: 19 exchanges for eight).
template <int V>
__device__ __forceinline__ void sort_keys(uint32_t (&s)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint32_t a = s[i + j], b = s[i + j + k];
            s[i + j] = max(a, b);
            s[i + j + k] = min(a, b);
          }
}

// Ordered keys of a lane's elements; 0 where there is no expert (no expert's key is 0).  fp32: the value's 32 bits.  bf16: the
// value's 16 bits above the index, so that no two keys of a row are equal (two values at a time: sign and magnitude to an
// integer in the order of the values, -0 to that of 0).  A NaN has the value of -inf in both.
template <typename T, int V>
__device__ __forceinline__ void make_keys(const float (&x)[V], int e0, int experts, uint32_t (&key)[V]) {
  if (sizeof(T) == 2) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const uint32_t low = 0xffff - e0;
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const uint32_t w = __builtin_amdgcn_perm(__float_as_uint(x[j + 1]), __float_as_uint(x[j]), 0x07060302u);
      const s16x2 sign = __builtin_bit_cast(s16x2, w) >> 15, mag = __builtin_bit_cast(s16x2, w & 0x7fff7fffu);
      // +inf moves to the largest integer, a positive NaN wraps to where the negative ones are: below -inf, which takes them up
      const s16x2 value = __builtin_bit_cast(s16x2, __builtin_bit_cast(u16x2, (s16x2)((mag ^ sign) - sign)) + (unsigned short)0x7f);
      const s16x2 ordered = __builtin_elementwise_max(value, (s16x2)(short)(0x7f - 0x7f80));
      const uint32_t u = __builtin_bit_cast(uint32_t, ordered) ^ 0x80008000u;
      key[j] = e0 + j < experts ? (u << 16) | (low - j) : 0u;
      key[j + 1] = e0 + j + 1 < experts ? (u & 0xffff0000u) | (low - j - 1) : 0u;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) key[j] = e0 + j < experts ? order_key(x[j]) : 0u;
}

// Adds 1 to cnt of the lane's elements that are among the row's k first by (value descending, index ascending), where `in`.
// Every lane sorts its keys; k times the lane with the largest head gives it up.  bf16: the last head given up is the bound.
// fp32: equal heads go to the first lane, and of a lane's equal keys the first ones count.
template <typename T, int G, int V>
__device__ __forceinline__ void count_choices(const float (&x)[V], int e0, int experts, int k, bool in, int lane, int (&cnt)[V]) {
  constexpr bool kUnique = sizeof(T) == 2;
  uint32_t key[V], s[V];
  make_keys<T>(x, e0, experts, key);
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = key[j];
  sort_keys(s);
  uint32_t bound = 0;
  int given = 0;
  for (int i = 0; i < k; ++i) {
    const uint32_t best = row_reduce<G>(s[0], MaxU());
    bool mine = s[0] == best;
    if (kUnique) {
      bound = best;
    } else {
      const uint64_t have = __builtin_amdgcn_ballot_w64(mine) >> (lane & ~(G - 1));
      mine = mine && (have & ((uint64_t(1) << (lane & (G - 1))) - 1)) == 0;
      bound = mine ? best : bound;
      given += mine;
    }
    const uint32_t m = mine ? ~0u : 0u;  // as bits: selects between neighbours become selects by index
#pragma unroll
    for (int j = 0; j + 1 < V; ++j) s[j] = (s[j + 1] & m) | (s[j] & ~m);
    s[V - 1] &= ~m;
  }
  if (!in) return;  // whatever its row holds
  if (kUnique) {
#pragma unroll
    for (int j = 0; j < V; ++j) cnt[j] += key[j] >= bound;
    return;
  }
  if (given == 0) return;
#pragma unroll
  for (int j = 0; j < V; ++j) given -= key[j] > bound;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const bool equal = key[j] == bound && given > 0;
    given -= equal;
    cnt[j] += equal || key[j] > bound;
  }
}

template <int KIND>
__device__ __forceinline__ bool counts_in(const void* mask, int64_t t) {
  if (mask == nullptr) return true;
  return KIND == AXON_MASK_F32 ? static_cast<const float*>(mask)[t] != 0.f : static_cast<const int64_t*>(mask)[t] != 0;
}

// f(sequence, first token, end) for what every sequence has of tokens [c0, c1), in ascending order; the same for all threads.
template <class F>
__device__ __forceinline__ void each_run(const BalanceParams& p, int c0, int c1, F&& f) {
  if (p.cu == nullptr) { f(0, c0, c1); return; }
  int pos = max(c0, p.cu[0]);
  while (pos < c1) {
    const int s = RowFinder::upper(p.cu, 0, p.n_seqs, pos);
    if (s >= p.n_seqs) return;
    const int end = min(p.cu[s + 1], c1);
    f(s, pos, end);
    pos = end;
  }
}

// Workgroup (chunk, layer).  48 layers x 8192 x 128 bf16, 8 choices: 65 us, where one read of the logits is 21: bound by
// instructions, those of the choices (a sort of a lane's eight keys, then eight times the largest head of sixteen lanes): with
// given choices it is 27 us.
template <typename T, int G, int V, int SCORE, int MASK>
__global__ __launch_bounds__(kBlock) void balance_fwd_kernel(BalanceParams p, LayerPtrs logits, LayerPtrs ids) {
  constexpr int kRows = kBlock / G, kE = G * V;
  __shared__ float red[kBlock / kWave][kE];
  __shared__ int hist[kE];
  __shared__ int s_tokens;
  const int chunk = blockIdx.x % p.n_chunks, layer = blockIdx.x / p.n_chunks, tid = threadIdx.x;
  const int lane_g = tid & (G - 1), e0 = lane_g * V, wave = tid / kWave, lane = tid & (kWave - 1);
  const T* const x0 = static_cast<const T*>(logits.p[layer]);
  const void* const chosen = ids.p[layer];
  const int64_t out_layer = p.first_layer + layer;
  if (out_layer == 0 && chunk == 0 && tid == 0) *p.ticket = 0;
  if (chunk == 0)
    for (int e = tid; e < p.experts; e += kBlock) p.counts[out_layer * p.experts + e] = 0;
  const int c0 = chunk * p.chunk, c1 = min(c0 + p.chunk, p.n_tokens);
  each_run(p, c0, c1, [&](int seq, int t0, int t1) {
    for (int e = tid; e < kE; e += kBlock) hist[e] = 0;
    if (tid == 0) s_tokens = 0;
    __syncthreads();
    float acc[V] = {};
    int cnt[V] = {}, tokens = 0;
    for (int b = t0; b < t1; b += kRows) {  // the same number of times for all threads
      const int t = b + tid / G;
      const bool in = t < t1 && counts_in<MASK>(p.mask, t);
      float x[V], w[V], rest[V];
      load_row<T, V>(x0 + (int64_t)(t < t1 ? t : t0) * p.ld, e0, p.experts, p.quads, x);
      const float inv = scores<G, V, SCORE>(x, w, rest);
      if (in) {
        ++tokens;
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = fmaf(w[j], inv, acc[j]);
      }
      if (chosen == nullptr) count_choices<T, G>(x, e0, p.experts, p.k, in, lane, cnt);
    }
    if (lane_g == 0 && tokens > 0) atomicAdd(&s_tokens, tokens);
    if (chosen != nullptr) {
      for (int i = tid; i < (t1 - t0) * p.k; i += kBlock) {
        const int t = t0 + i / p.k;
        if (!counts_in<MASK>(p.mask, t)) continue;
        const int64_t at = (int64_t)t0 * p.k + i;
        const int64_t e = p.ids_i64 ? static_cast<const int64_t*>(chosen)[at] : (int64_t) static_cast<const int32_t*>(chosen)[at];
        if (e >= 0 && e < p.experts) atomicAdd(&hist[e], 1);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      acc[j] = column_reduce<G>(acc[j], Add());
      if (lane < G) red[wave][e0 + j] = acc[j];
      if (chosen == nullptr) {
        cnt[j] = column_reduce<G>(cnt[j], Add());
        if (lane < G && cnt[j]) atomicAdd(&hist[e0 + j], cnt[j]);
      }
    }
    __syncthreads();
    const int64_t slot = chunk + seq;
    for (int e = tid; e < p.experts; e += kBlock) {
      const int64_t at = (slot * p.layers + out_layer) * p.experts + e;
      p.part_p[at] = (red[0][e] + red[1][e]) + (red[2][e] + red[3][e]);
      p.part_c[at] = hist[e];
    }
    if (tid == 0 && out_layer == 0) p.part_t[slot] = s_tokens;
    __syncthreads();
  });
}

// Workgroup (sequence, layer): adds its partials, leaves E / (k T^2) c per expert for the backward, the loads and the
// sequence's loss.  The workgroup that draws the last ticket adds the losses, in a fixed order, to the mean over the sequences
// that have tokens and the layers.  Up to 256 experts the chunks are shared by groups of threads: 48 x
// 8192 x 128 7 us (one load at a time and thread, and a launch for the mean: 18).
__global__ __launch_bounds__(kBlock) void balance_sum_kernel(BalanceParams p, float* __restrict__ coef, double* __restrict__ losses,
                                                             int* __restrict__ tokens, float* __restrict__ loss,
                                                             float* __restrict__ scale) {
  __shared__ double prob[kBlock];
  __shared__ int cnt[kBlock];
  __shared__ double red[2][kBlock / kWave];
  __shared__ int s_last;
  const int seq = blockIdx.x % p.n_seqs, layer = blockIdx.x / p.n_seqs, tid = threadIdx.x, lane = tid & (kWave - 1);
  const int a = p.cu ? max(p.cu[seq], 0) : 0, b = min(p.cu ? p.cu[seq + 1] : p.n_tokens, p.n_tokens);
  const int first = a / p.chunk, last = b > a ? (b - 1) / p.chunk : first - 1;
  int n = 0;
  for (int c = first + lane; c <= last; c += kWave) n += p.part_t[c + seq];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, kWave);
  const double w = n > 0 ? (double)p.experts / ((double)p.k * n * n) : 0.0;
  const int width = p.experts >= kBlock ? kBlock : 1 << (32 - __builtin_clz(p.experts - 1 | 1));  // at least the experts
  const int groups = kBlock / width, group = tid / width;
  double sum = 0.0;
  for (int e0 = 0; e0 < p.experts; e0 += width) {
    const int e = e0 + (tid & (width - 1));
    double pr = 0.0;
    int ct = 0;
    if (e < p.experts) {
#pragma unroll 4
      for (int c = first + group; c <= last; c += groups) {
        const int64_t at = ((int64_t)(c + seq) * p.layers + layer) * p.experts + e;
        pr += p.part_p[at];
        ct += p.part_c[at];
      }
    }
    prob[tid] = pr;
    cnt[tid] = ct;
    __syncthreads();
    if (group == 0 && e < p.experts) {
      for (int g = 1; g < groups; ++g) { pr += prob[g * width + tid]; ct += cnt[g * width + tid]; }
      const double wc = w * ct;
      coef[((int64_t)seq * p.layers + layer) * p.experts + e] = (float)wc;
      if (ct) atomicAdd(&p.counts[(int64_t)layer * p.experts + e], (unsigned long long)ct);
      sum += n > 0 ? wc * pr : 0.0;
    }
    __syncthreads();
  }
  sum = wave_sum_d(sum);
  if (lane == 0) red[0][tid / kWave] = sum;
  __syncthreads();
  if (tid == 0) {
    losses[(int64_t)seq * p.layers + layer] = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    if (layer == 0) tokens[seq] = n;
    __threadfence();
    s_last = __hip_atomic_fetch_add(p.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  sum = 0.0;
  double with = 0.0;
  for (int i = tid; i < p.n_seqs * p.layers; i += kBlock) sum += losses[i];
  for (int i = tid; i < p.n_seqs; i += kBlock) with += tokens[i] > 0 ? 1.0 : 0.0;
  sum = wave_sum_d(sum);
  with = wave_sum_d(with);
  if (lane == 0) { red[0][tid / kWave] = sum; red[1][tid / kWave] = with; }
  __syncthreads();
  if (tid != 0) return;
  for (int v = 1; v < kBlock / kWave; ++v) { sum += red[0][v]; with += red[1][v]; }
  const double s = with > 0.0 ? 1.0 / (with * p.layers) : 0.0;
  *loss = (float)(sum * s);
  *scale = (float)s;
}

// The gradient, a row in the lanes that had it in the forward; nothing but the coefficients is kept from there.  48 x 8192 x 128
// bf16 38 us, 5.3 TB/s read and written: memory.
template <typename T, int G, int V, int SCORE, int MASK>
__global__ __launch_bounds__(kBlock) void balance_bwd_kernel(BalanceParams p, LayerPtrs logits, LayerPtrs grads) {
  constexpr int kRows = kBlock / G;
  const int chunk = blockIdx.x % p.n_chunks, layer = blockIdx.x / p.n_chunks, tid = threadIdx.x;
  const int e0 = (tid & (G - 1)) * V;
  const T* const x0 = static_cast<const T*>(logits.p[layer]);
  T* const d0 = static_cast<T*>(const_cast<void*>(grads.p[layer]));
  if (d0 == nullptr) return;  // a layer that needs no gradient
  const float factor = *p.scale * *p.g_loss;
  auto store = [&](int t, const float (&v)[V]) {
    T* const out = d0 + (int64_t)t * p.experts + e0;
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float q[4] = {v[j], v[j + 1], v[j + 2], v[j + 3]};
      if (p.quads) {
        if (e0 + j < p.experts) RouterRow<T>::store4(out + j, q);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (e0 + j + r < p.experts) RouterRow<T>::store1(out + j + r, q[r]);
      }
    }
  };
  const int c0 = chunk * p.chunk, c1 = min(c0 + p.chunk, p.n_tokens);
  const float zero[V] = {};
  int done = c0;  // tokens before it have their gradient: those of no sequence are filled up with zeros
  auto fill = [&](int to) {
    for (int t = done + tid / G; t < to; t += kRows) store(t, zero);
  };
  each_run(p, c0, c1, [&](int seq, int t0, int t1) {
    fill(t0);
    done = t1;
    float wc[V];
    const float* const coef = p.coef + ((int64_t)seq * p.layers + p.first_layer + layer) * p.experts;
#pragma unroll
    for (int j = 0; j < V; ++j) wc[j] = e0 + j < p.experts ? coef[e0 + j] : 0.f;
    for (int b = t0; b < t1; b += kRows) {
      const int t = b + tid / G;
      const bool in = t < t1 && counts_in<MASK>(p.mask, t);
      float x[V], w[V], rest[V], d[V], dot = 0.f;
      load_row<T, V>(x0 + (int64_t)(t < t1 ? t : t0) * p.ld, e0, p.experts, p.quads, x);
      const float inv = scores<G, V, SCORE>(x, w, rest);
#pragma unroll
      for (int j = 0; j < V; ++j) dot = fmaf(w[j], wc[j], dot);
      dot = row_reduce<G>(dot, Add()) * inv;
      const float by = factor * inv;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float slope = w[j] * by;
        if (SCORE == kSigmoid) slope *= rest[j];
        d[j] = in ? slope * (wc[j] - dot) : 0.f;
      }
      if (t < t1) store(t, d);
    }
  });
  fill(c1);
}

}  // namespace axon

using namespace axon;

namespace {

// Tokens per chunk: 256, fewer where that leaves less than four workgroups per compute unit, at least 32.
int chunk_of(int64_t n, int64_t layers) {
  int c = 256;
  while (c > 32 && (n + c - 1) / c * layers < 1024) c /= 2;
  return c;
}

struct BalanceWs {
  float* part_p;
  int *part_c, *part_t, *tokens, *ticket;
  double* losses;
  int64_t bytes;
};
BalanceWs balance_ws(int64_t n, int64_t n_seqs, int64_t layers, int64_t experts, void* base) {
  const int64_t c = chunk_of(n, layers), slots = (n + c - 1) / c + n_seqs, cells = slots * layers * experts;
  char* p = static_cast<char*>(base);
  BalanceWs w;
  w.losses = reinterpret_cast<double*>(p);  p += n_seqs * layers * 8;
  w.part_p = reinterpret_cast<float*>(p);   p += cells * 4;
  w.part_c = reinterpret_cast<int*>(p);     p += cells * 4;
  w.part_t = reinterpret_cast<int*>(p);     p += slots * 4;
  w.tokens = reinterpret_cast<int*>(p);     p += n_seqs * 4;
  w.ticket = reinterpret_cast<int*>(p);     p += 4;
  w.bytes = p - static_cast<char*>(base);
  return w;
}

int check_balance(const void* const* logits, int dtype, int64_t ld, int64_t layers, int64_t n, int64_t experts,
                  const void* mask, int mask_kind, const int32_t* cu, int64_t n_seqs, int score) {
  if (dtype != AXON_LOGITS_F32 && dtype != AXON_LOGITS_BF16) return AXON_ERR_ARG;
  if (score != kSoftmax && score != kSigmoid) return AXON_ERR_ARG;
  if (mask && mask_kind != AXON_MASK_F32 && mask_kind != AXON_MASK_I64) return AXON_ERR_ARG;
  if (layers < 1 || n < 0 || experts < 1 || ld < experts || n_seqs < 0 || (!cu && n_seqs != 1)) return AXON_ERR_ARG;
  if (experts > kMaxExperts || layers > (1 << 16) || n >= (int64_t)1 << 30 || n_seqs >= (int64_t)1 << 24 ||
      (n / 32 + 1) * kMaxLayers >= INT32_MAX || n_seqs * layers >= INT32_MAX)
    return AXON_ERR_SHAPE;
  if (!logits) return AXON_ERR_ARG;
  const int eb = dtype == AXON_LOGITS_F32 ? 4 : 2;
  for (int64_t l = 0; n > 0 && l < layers; ++l)
    if (!logits[l] || reinterpret_cast<uintptr_t>(logits[l]) % eb != 0) return AXON_ERR_ARG;
  return AXON_OK;
}

// how rows of every layer can be read: sixteen bytes at a time (2), four elements (1), one (0)
int quads_ok(const void* const* ptrs, int64_t layers, int64_t ld, int64_t experts, int eb) {
  uintptr_t bits = (uintptr_t)(ld * eb) | (uintptr_t)(experts * eb);
  for (int64_t l = 0; l < layers; ++l) bits |= reinterpret_cast<uintptr_t>(ptrs[l]);  // a null is on every boundary
  return bits % 16 == 0 ? 2 : bits % (4 * eb) == 0 ? 1 : 0;
}

template <typename T, int SCORE, int MASK, bool BWD>
int launch_balance(const BalanceParams& p, const LayerPtrs& a, const LayerPtrs& b, int layers, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.n_chunks * layers)), blk(kBlock);
#define AXON_BALANCE(G, V)                                                                                          \
  do {                                                                                                              \
    if constexpr (BWD) hipLaunchKernelGGL((balance_bwd_kernel<T, G, V, SCORE, MASK>), grid, blk, 0, st, p, a, b);   \
    else hipLaunchKernelGGL((balance_fwd_kernel<T, G, V, SCORE, MASK>), grid, blk, 0, st, p, a, b);                 \
  } while (0)
  const int e = p.experts;
  if (e <= 8) AXON_BALANCE(1, 8);
  else if (e <= 16) AXON_BALANCE(2, 8);
  else if (e <= 32) AXON_BALANCE(4, 8);
  else if (e <= 64) AXON_BALANCE(8, 8);
  else if (e <= 128) AXON_BALANCE(16, 8);
  else if (e <= 256) AXON_BALANCE(32, 8);
  else if (e <= 512) AXON_BALANCE(64, 8);
  else AXON_BALANCE(64, 16);
#undef AXON_BALANCE
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

template <bool BWD>
int launch_typed(int dtype, int score, int mask_kind, const BalanceParams& p, const LayerPtrs& a, const LayerPtrs& b, int layers,
                 hipStream_t st) {
  const bool i64 = p.mask && mask_kind == AXON_MASK_I64;
#define AXON_SCORE(T)                                                                                  \
  (score == kSoftmax ? (i64 ? launch_balance<T, kSoftmax, AXON_MASK_I64, BWD>(p, a, b, layers, st)     \
                            : launch_balance<T, kSoftmax, AXON_MASK_F32, BWD>(p, a, b, layers, st))    \
                     : (i64 ? launch_balance<T, kSigmoid, AXON_MASK_I64, BWD>(p, a, b, layers, st)     \
                            : launch_balance<T, kSigmoid, AXON_MASK_F32, BWD>(p, a, b, layers, st)))
  return dtype == AXON_LOGITS_F32 ? AXON_SCORE(float) : AXON_SCORE(__bf16);
#undef AXON_SCORE
}

}  // namespace

extern "C" int64_t axon_router_balance_workspace_bytes(int64_t n, int64_t n_seqs, int64_t layers, int64_t experts) {
  if (n < 0 || n_seqs < 0 || layers < 1 || experts < 1) return AXON_ERR_ARG;
  return balance_ws(n, n_seqs, layers, experts, nullptr).bytes;
}

extern "C" int axon_router_balance_fwd(const void* const* logits, int dtype, int64_t ld, int64_t layers, int64_t n,
                                       int64_t experts, int64_t k, const void* const* ids, int ids_i64, const void* mask,
                                       int mask_kind, const int32_t* cu, int64_t n_seqs, int score, float* loss, float* coef,
                                       float* scale, int64_t* counts, void* workspace, int64_t ws_bytes, void* stream) {
  int rc = check_balance(logits, dtype, ld, layers, n, experts, mask, mask_kind, cu, n_seqs, score);
  if (rc != AXON_OK) return rc;
  if (k < 1 || k > experts) return AXON_ERR_SHAPE;
  if (!loss || !scale || !counts || (n_seqs > 0 && !coef)) return AXON_ERR_ARG;
  if (n == 0 || n_seqs == 0) {
    rc = axon_fill_zero(loss, 4, stream);
    if (rc == AXON_OK) rc = axon_fill_zero(scale, 4, stream);
    if (rc == AXON_OK) rc = axon_fill_zero(counts, layers * experts * 8, stream);
    if (rc == AXON_OK && n_seqs > 0) rc = axon_fill_zero(coef, n_seqs * layers * experts * 4, stream);
    return rc;
  }
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7)) return AXON_ERR_ARG;
  for (int64_t l = 0; ids && l < layers; ++l)
    if (!ids[l]) return AXON_ERR_ARG;
  const BalanceWs w = balance_ws(n, n_seqs, layers, experts, workspace);
  if (w.bytes > ws_bytes) return AXON_ERR_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  BalanceParams p{};
  p.ld = ld;
  p.n_tokens = (int)n;  p.experts = (int)experts;  p.k = (int)k;  p.layers = (int)layers;
  p.chunk = chunk_of(n, layers);
  p.n_chunks = (int)((n + p.chunk - 1) / p.chunk);
  p.mask = mask;  p.cu = cu;  p.n_seqs = (int)n_seqs;  p.ids_i64 = ids_i64;
  p.part_p = w.part_p;  p.part_c = w.part_c;  p.part_t = w.part_t;  p.ticket = w.ticket;
  p.counts = reinterpret_cast<unsigned long long*>(counts);
  const int eb = dtype == AXON_LOGITS_F32 ? 4 : 2;
  for (int64_t l0 = 0; l0 < layers; l0 += kMaxLayers) {
    const int nl = (int)(layers - l0 < kMaxLayers ? layers - l0 : kMaxLayers);
    LayerPtrs x{}, c{};
    for (int l = 0; l < nl; ++l) { x.p[l] = logits[l0 + l]; c.p[l] = ids ? ids[l0 + l] : nullptr; }
    p.first_layer = (int)l0;
    p.quads = quads_ok(x.p, nl, ld, experts, eb);
    rc = launch_typed<false>(dtype, score, mask_kind, p, x, c, nl, st);
    if (rc != AXON_OK) return rc;
  }
  hipLaunchKernelGGL(balance_sum_kernel, dim3((unsigned)(n_seqs * layers)), dim3(kBlock), 0, st, p, coef, w.losses, w.tokens, loss,
                     scale);
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

extern "C" int axon_router_balance_bwd(const void* const* logits, int dtype, int64_t ld, int64_t layers, int64_t n,
                                       int64_t experts, const void* mask, int mask_kind, const int32_t* cu, int64_t n_seqs,
                                       int score, const float* coef, const float* scale, const float* g_loss,
                                       void* const* dlogits, void* stream) {
  int rc = check_balance(logits, dtype, ld, layers, n, experts, mask, mask_kind, cu, n_seqs, score);
  if (rc != AXON_OK) return rc;
  if (n == 0) return AXON_OK;
  if (!scale || !g_loss || !dlogits || (n_seqs > 0 && !coef)) return AXON_ERR_ARG;
  const int eb = dtype == AXON_LOGITS_F32 ? 4 : 2;
  for (int64_t l = 0; l < layers; ++l)
    if (reinterpret_cast<uintptr_t>(dlogits[l]) % eb != 0) return AXON_ERR_ARG;
  BalanceParams p{};
  p.ld = ld;
  p.n_tokens = (int)n;  p.experts = (int)experts;  p.layers = (int)layers;
  p.chunk = chunk_of(n, layers);
  p.n_chunks = (int)((n + p.chunk - 1) / p.chunk);
  p.mask = mask;  p.cu = cu;  p.n_seqs = (int)n_seqs;
  p.coef = coef;  p.scale = scale;  p.g_loss = g_loss;
  for (int64_t l0 = 0; l0 < layers; l0 += kMaxLayers) {
    const int nl = (int)(layers - l0 < kMaxLayers ? layers - l0 : kMaxLayers);
    LayerPtrs x{}, d{};
    for (int l = 0; l < nl; ++l) { x.p[l] = logits[l0 + l]; d.p[l] = dlogits[l0 + l]; }
    p.first_layer = (int)l0;
    p.quads = std::min(quads_ok(x.p, nl, ld, experts, eb), quads_ok(d.p, nl, experts, experts, eb));
    rc = launch_typed<true>(dtype, score, mask_kind, p, x, d, nl, (hipStream_t)stream);
    if (rc != AXON_OK) return rc;
  }
  return AXON_OK;
}
