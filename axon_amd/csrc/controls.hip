// What a sampler does to a position's logits before it draws: penalties for tokens that the sequence holds already, biases,
// a grammar's mask, the temperature.  Written out (for a decoder), or as the log-probability of a label and the entropy of
// what is left (for a trainer, which has to score a rollout under the distribution that it was drawn from), forward and
// backward.
//
//   y_j = (z_j > 0 ? z_j / rep : z_j rep  where j is in the row's history)  - freq count_j - pres [count_j > 0] + bias_j,
//   -inf where the row's mask has a 0 bit;  out = y / T;  log p = out - logsumexp(out).
//
// A wavefront owns 4 KB of consecutive ids of the vocabulary and walks a run of rows: the ids stay the same from row to row,
// so what the histories do to them is kept where it is used (the sum of the additive terms in LDS, whether an id was
// seen in a bit of the owning lane), and a row of a packed batch differs from the row before by ONE token.  Vectors are
// loaded at whatever boundary a row of an odd vocabulary starts on, so that lanes keep their ids.
//
// Memory takes 6.4 TB/s read and 4.8 copied in rows of whole vectors, 4.9 and 4.7 at a boundary of 2 bytes.  It bounds fp32 rows and the
// gradients; bf16 rows of log-probabilities are bound by instructions and by the loads that wait for them, since a row of few ids
// takes as long as its loads do (masks that leave out half of all vectors save nothing).
//   log-probability and entropy   1500 x 151936 fp32 174 us (5.2 TB/s); 4096 x 151936 bf16 under masks, penalties and 40 biases 300 to
//     315 us, under the penalties alone 285, under the masks alone and without controls 244 (5.1 TB/s): what the penalties take of every
//     element, four waves to a SIMD (five spill, 666 us); 2047 x 50257 bf16 75 us, without controls 50: short runs
//   their gradient                1500 x 151936 fp32 329 us (5.5 TB/s, in part from the cache in front of the memory), 2047 x 50257 bf16 89 us
//   written out                   61 x 201088 fp32, histories of 4000 tokens, 32 us (17 without controls); 1024 x 32768 bf16, 1500
//     tokens, 42 us (24 without controls): a workgroup's history and its terms are trips to memory and through
//     LDS before the row's arithmetic, which the four other workgroups of a compute unit hide in part
//   their gradient                1024 x 151936 fp32, 1500 tokens, 325 us (5.8 TB/s of the two reads and the write), bf16 170 us (5.5)
#include "logits_rows.h"
#include <type_traits>

namespace axon {

constexpr int kVecs = 4;                  // 16-byte vectors of a lane: a wavefront's chunk of a row is 4 KB
constexpr int kChunkBytes = kVecs * kWave * 16;
constexpr int kWaves = kBlock / kWave;
constexpr int kMaxRun = kWave;            // rows of a run: a lane holds what belongs to a row

enum Mode { kStats, kGrad, kApply, kApplyGrad };

// 16-byte vectors on any boundary of their elements.
template <typename T> struct Unaligned;
template <> struct Unaligned<float> {
  static constexpr int kPer = 4;
  typedef f32x4 Raw;
  typedef Raw Loose __attribute__((aligned(4)));
  template <bool CACHED>
  __device__ static Raw load(const float* p) {
    const Loose* const q = reinterpret_cast<const Loose*>(p);
    return CACHED ? *q : __builtin_nontemporal_load(q);
  }
  __device__ static float get(const Raw& r, int j) { return r[j]; }
  __device__ static void set(Raw& r, int j, const float* p) { r[j] = *p; }
  __device__ static void store(float* p, const float* v) {
    const Raw x = {v[0], v[1], v[2], v[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<Loose*>(p));
  }
};
template <> struct Unaligned<unsigned short> {
  static constexpr int kPer = 8;
  typedef uint32_t Raw __attribute__((ext_vector_type(4)));
  typedef Raw Loose __attribute__((aligned(2)));
  template <bool CACHED>
  __device__ static Raw load(const unsigned short* p) {
    const Loose* const q = reinterpret_cast<const Loose*>(p);
    return CACHED ? *q : __builtin_nontemporal_load(q);
  }
  __device__ static float get(const Raw& r, int j) {
    return __uint_as_float((j & 1) ? (r[j >> 1] & 0xffff0000u) : (r[j >> 1] << 16));
  }
  __device__ static void set(Raw& r, int j, const unsigned short* p) { r[j >> 1] |= (uint32_t)*p << ((j & 1) * 16); }  // of a 0
  __device__ static void store(unsigned short* p, const float* v) {
    const Raw x = {f32x2_to_bf16(v[0], v[1]), f32x2_to_bf16(v[2], v[3]), f32x2_to_bf16(v[4], v[5]), f32x2_to_bf16(v[6], v[7])};
    __builtin_nontemporal_store(x, reinterpret_cast<Loose*>(p));
  }
};

__device__ __forceinline__ int64_t index_at(const void* p, int i64, int64_t at) {
  return i64 ? static_cast<const int64_t*>(p)[at] : (int64_t) static_cast<const int32_t*>(p)[at];
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
// What one lane has written to LDS, for the others of its wavefront: LDS serves a wavefront in order, the compiler is told to.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
constexpr float kBanned = -1e30f;  // stands for -inf where a product with it has to stay finite
constexpr float kFar = 1e9f;       // a reference in log2 units whose rounding (64) leaves the exponentials in range
constexpr float kNear = 8.f;       // ... and of which a term is off by at most 2^-22 ln 2
constexpr float kNoLogit = -3.402823466e38f;  // the reference of a set without a logit: any there is is at least as large

// A token of a history: its id, or -1 where it counts for nothing; bit 30 where the model has generated it.  (Both loads at once.)
constexpr int kOwn = 1 << 30;
__device__ __forceinline__ int history_token(const axon_controls& c, int64_t at, int vocab) {
  const int64_t id = index_at(c.token_ids, c.token_ids_i64, at);
  bool own = true;
  if (c.own_mask != nullptr)
    own = c.mask_kind == AXON_MASK_I64 ? static_cast<const int64_t*>(c.own_mask)[at] != 0 : static_cast<const float*>(c.own_mask)[at] != 0.f;
  return id < 0 || id >= vocab ? -1 : (int)id | (own ? kOwn : 0);
}

// The additive part of what controls do to one id.
__device__ __forceinline__ float penalty(int count, float frequency, float presence) {
  return count > 0 ? fmaf(frequency, (float)count, presence) : 0.f;
}

struct RowIo {
  const void* labels;  // [rows]
  int labels_i64;
  float* label_y;             // [rows], kStats
  float4* parts;              // [rows][chunks] (M, s, e), kStats
  const float* stats;         // [3][rows]: what controls_finish_kernel has left, kGrad
  const float *g_logprob, *g_entropy;
  int cached_from;  // rows from here on are left in the cache in front of the memory, for a backward that follows (256 MB of them:
                    // 2047 x 50257 bf16 with gradient 155 us, 166 where nothing is; 1500 x 151936 fp32 505 and 512)
};

// The additive terms of a wavefront's ids in LDS, in the order in which the lanes read them: 16 bytes of neighbouring
// lanes lie side by side.
template <int PER>
__device__ __forceinline__ constexpr int slot(int off) {
  return PER == 4 ? off : (off & ~511) | ((off & 4) << 6) | ((off & 0x1f8) >> 1) | (off & 3);
}

// Bits of one lane's ids as masks of 32 bits, and a choice by such a mask: two instructions per element and no branch.
__device__ __forceinline__ uint32_t bit_mask(uint32_t bits, int i) { return (uint32_t)((int32_t)(bits << (31 - i)) >> 31); }
__device__ __forceinline__ float pick(uint32_t mask, float yes, float no) {
  return __uint_as_float((mask & __float_as_uint(yes)) | (~mask & __float_as_uint(no)));
}

template <typename T, Mode MODE, bool ADJ, bool MASK, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 4) void controls_kernel(const T* logits, int64_t ld, int n_rows, int vocab, int chunks, int run,
                                                          axon_controls c, RowIo io, const T* other, int64_t ld_other, T* out,
                                                          int64_t ld_out) {
  constexpr int kPer = Unaligned<T>::kPer, kLaneIds = kVecs * kPer, kIds = kLaneIds * kWave, kGroupIds = kIds * WAVES, kThreads = WAVES * kWave;
  constexpr uint32_t kVecBits = (1u << kPer) - 1, kAll = kLaneIds == 32 ? ~0u : (1u << (kLaneIds & 31)) - 1;
  __shared__ __align__(16) uint32_t s_adj[ADJ ? kGroupIds : 4];  // counts (bit 31: seen) while they are collected, then floats
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);  // bases in scalar registers
  const int groups = (chunks + WAVES - 1) / WAVES;
  // kGrad from the last row to the first: the end of what the forward read last is still in the cache in front of the memory
  const unsigned block = MODE == kGrad ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const int first = (int)(block / groups) * run, group = (int)(block % groups);
  const bool cached = MODE == kStats && first >= io.cached_from;
  const int rows = min(run, n_rows - first);
  const int chunk = group * WAVES + wave, base = chunk * kIds;

  // what belongs to row first + lane
  const int mine = min(first + lane, n_rows - 1);
  int seq = 0, start = 0, state = -1, label = -1, token = -1;
  const int n_seqs = (int)c.n_seqs;
  int64_t begin = 0, end = 0;  // the row's history
  const bool history = ADJ && c.token_ids != nullptr, offsets = c.uniform_len == 0 && c.cu_seqlens != nullptr;
  if (n_seqs > 0 && c.every_position && offsets && n_seqs <= kWave) {
    // few sequences: all of their ends in one load, a lane each, instead of a search with its loads one after the other
    // (2047 x 50257 bf16 with gradient 160 us, with the search 167)
    const int ends = c.cu_seqlens[min(lane + 1, n_seqs)], base0 = c.cu_seqlens[0];
    for (int i = 0; i < n_seqs - 1; ++i) seq += lane_value(ends, i) <= mine;
    end = __shfl(ends, seq, kWave);
    begin = __shfl(ends, max(seq - 1, 0), kWave);
    if (seq == 0) begin = base0;
  } else if (n_seqs > 0) {
    if (!c.every_position) seq = mine;
    else if (c.uniform_len > 0) seq = (int)(mine / c.uniform_len);
    else seq = RowFinder::upper4(c.cu_seqlens, 0, n_seqs, mine);
    seq = min(max(seq, 0), n_seqs - 1);
    if (history) {
      begin = c.uniform_len > 0 ? (int64_t)seq * c.uniform_len : (int64_t)c.cu_seqlens[seq];
      end = c.uniform_len > 0 ? begin + c.uniform_len : (int64_t)c.cu_seqlens[seq + 1];
    }
  }
  if (history) {
    if (c.every_position) {
      if (mine < begin || mine >= end) begin = mine + 1;  // a position of no sequence
      end = (int64_t)mine + 1;
    }
    begin = max(begin, (int64_t)0);
    end = min(end, c.n_tokens);
    start = (int)begin;
    if (c.every_position && begin < end) token = history_token(c, end - 1, vocab);
  } else {
    start = c.bias_per_seq ? seq : 0;  // no history: rows differ where their biases do
  }
  const float rep_l = c.repetition ? c.repetition[seq] : c.repetition_all;
  const float freq_l = c.frequency ? c.frequency[seq] : c.frequency_all;
  const float pres_l = c.presence ? c.presence[seq] : c.presence_all;
  const float inv_t_l = 1.f / (c.temperature ? c.temperature[seq] : c.temperature_all);
  if (MASK) {
    const int64_t s = c.allowed_index ? index_at(c.allowed_index, c.allowed_index_i64, mine) : (c.allowed_rows == 1 ? 0 : mine);
    state = s >= 0 && s < c.allowed_rows ? (int)s : -1;
  }
  if (MODE == kStats || MODE == kGrad) {
    const int64_t l = index_at(io.labels, io.labels_i64, mine);
    label = l >= 0 && l < vocab ? (int)l : -1;
  }
  // kGrad: dz = 2^t (A + B t) slope with t = (y - M) log2(e) / T, the row's constants in A and B
  float top_l = 0.f, a_l = 0.f, b_l = 0.f, glp_l = 0.f;
  uint64_t live = ~0ull >> (kMaxRun - rows);  // rows that are looked at: of the others nothing is asked
  if (MODE == kGrad) {
    top_l = io.stats[mine];
    const float sum = io.stats[(int64_t)n_rows + mine], ls = __log2f(sum), H = io.stats[2 * (int64_t)n_rows + mine];
    const float g_en = io.g_entropy ? io.g_entropy[mine] : 0.f;
    const float q = inv_t_l / sum, g_lp = io.g_logprob && label >= 0 ? io.g_logprob[mine] : 0.f;
    glp_l = g_lp * inv_t_l;
    a_l = q * -fmaf(g_en, fmaf(-kLn2, ls, H), g_lp);
    b_l = q * -g_en * kLn2;
    live &= __ballot(g_lp != 0.f || g_en != 0.f);
  }

  uint32_t* const adj = s_adj + (ADJ ? wave * kIds : 0);
  uint32_t seen = 0;     // bit u * kPer + j: this lane's id of vector u, element j
  uint32_t touched = 0;  // bit i / 4: some lane's ids of these four bits are not left as they are; the same in all lanes
  // A row's own token is counted with the run's first rows, for all rows at once: by a sum of additions as the rows go by, the
  // term would drift.  count: how often the row's token is among the own tokens up to the row; bias: of that id.
  const int mine_off = token < 0 ? -1 : (token & (kOwn - 1)) - base;
  const bool in_chunk = ADJ && mine_off >= 0 && mine_off < kIds;
  int count_l = 0;
  float bias_l = 0.f;
  // counts and seen bits in LDS to additive terms, biases with them
  auto settle = [&](int row) {
    const float f = lane_value(freq_l, row), a = lane_value(pres_l, row);
    const int sq = lane_value(seq, row);
    const bool of_it = in_chunk && start == lane_value(start, row);
    const int before = of_it ? (int)(adj[slot<kPer>(mine_off)] & 0x7fffffffu) : 0;
    uint32_t any = 0;
    seen = 0;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      uint32_t w[kPer], some = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        w[j] = adj[slot<kPer>((u * kWave + lane) * kPer + j)];
        some |= w[j];
      }
      if (!__any(some != 0)) continue;  // 0 is 0.f
#pragma unroll
      for (int j = 0; j < kPer; j += 4)
        if (__any((w[j] | w[j + 1] | w[j + 2] | w[j + 3]) != 0)) any |= 1u << ((u * kPer + j) / 4);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        seen |= (w[j] >> 31) << (u * kPer + j);
        adj[slot<kPer>((u * kWave + lane) * kPer + j)] = __float_as_uint(penalty((int)(w[j] & 0x7fffffffu), f, a));
      }
    }
    wave_sync();
    for (int64_t i0 = 0; i0 < c.n_bias; i0 += kWave) {
      const int64_t i = i0 + lane, at = (c.bias_per_seq ? (int64_t)sq * c.n_bias : 0) + i;
      const int64_t off = i < c.n_bias ? index_at(c.bias_ids, c.bias_ids_i64, at) - base : -1;
      const bool in = off >= 0 && off < kIds && off + base < vocab;
      if (in) atomicAdd(reinterpret_cast<float*>(adj) + slot<kPer>((int)off), -c.bias[at]);
      const int quad = in ? ((int)off / (kWave * kPer) * kPer + (int)off % kPer) / 4 : -1;
#pragma unroll
      for (int v = 0; v < kLaneIds / 4; ++v)
        if (__any(quad == v)) any |= 1u << v;
    }
    touched = __builtin_amdgcn_readfirstlane(any);
    wave_sync();
    if (of_it) {
      count_l += before;
      if (c.n_bias > 0) bias_l = penalty(before, f, a) - __uint_as_float(adj[slot<kPer>(mine_off)]);
    }
  };

  // the ids of this lane that there are
  const bool whole = base + kIds <= vocab;
  uint32_t there = kAll;
  if (!whole) {
    there = 0;
#pragma unroll
    for (int i = 0; i < kLaneIds; ++i) there |= (uint32_t)(base + ((i / kPer) * kWave + lane) * kPer + i % kPer < vocab) << i;
  }
  // What of them row r may keep, in two halves: the bytes are asked for a row before they are put together.
  uint32_t bytes[MASK ? kVecs : 1];
  auto ask_mask = [&](int r) {
    const int st = lane_value(state, r);
    const uint8_t* const from = reinterpret_cast<const uint8_t*>(c.allowed + (int64_t)max(st, 0) * c.allowed_stride) + base / 8;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int id0 = (u * kWave + lane) * kPer;
      bytes[MASK ? u : 0] = whole || base + id0 < vocab ? from[(uint32_t)id0 >> 3] : 0;
    }
  };
  auto mask_of = [&](int r) {
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) m |= (bytes[MASK ? u : 0] >> (kPer == 4 ? (lane & 1) * 4 : 0) & kVecBits) << (u * kPer);
    return lane_value(state, r) < 0 ? there : m & there;
  };

  // A row's vectors are asked for while the row before is worked on, as soon as the registers are free; its mask a row
  // earlier, since what is not kept is not read either.  Where a mask leaves no lane more than kFew ids (a grammar's
  // state that allows a handful of tokens), only these are looked at: 4096 x 151936 bf16 under such and other masks take
  // 288 us, 307 with all elements of all rows.  kFew is what the row's registers hold one element to a vector.
  constexpr int kFew = 4;
  static_assert(kFew <= kVecs, "");
  // The lane's id number `bit` as an offset from the wavefront's first, and the next one of those that are left: behind the last
  // it is an id of the lane still, so that what is addressed by it lies in the wavefront's own terms.
  auto offset_of = [&](int bit) { return (uint32_t)((bit / kPer * kWave + lane) * kPer + bit % kPer); };
  constexpr uint32_t kLastId = 1u << (kLaneIds - 1);
  static_assert((kLaneIds - 1) / kPer < kVecs && slot<kPer>(((kLaneIds - 1) / kPer * kWave + kWave - 1) * kPer + kPer - 1) < kIds, "");
  auto first_of = [&](uint32_t left) { return __builtin_ctz(left | kLastId); };
  typename Unaligned<T>::Raw raw[kVecs], raw_g[MODE == kApplyGrad ? kVecs : 1];
  auto is_few = [&](uint32_t keep) {
    if (MODE != kStats || !MASK) return false;
    uint32_t x = keep;
#pragma unroll
    for (int i = 0; i < kFew; ++i) x &= x - 1;
    return !__any(x != 0);
  };
  auto read = [&](const T* from, uint32_t keep, int u, typename Unaligned<T>::Raw& into) {
    const int id0 = (u * kWave + lane) * kPer;
    if (MASK || !whole) {
      into = typename Unaligned<T>::Raw{};
      if ((keep >> (u * kPer) & kVecBits) == 0) return;
      if (!whole && base + id0 + kPer > vocab) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (base + id0 + j < vocab) Unaligned<T>::set(into, j, from + id0 + j);
        return;
      }
    }
    into = cached ? Unaligned<T>::template load<true>(from + (uint32_t)id0) : Unaligned<T>::template load<false>(from + (uint32_t)id0);
  };
  const T* const from = logits + (int64_t)first * ld + base;
  const T* const from_g = MODE == kApplyGrad ? other + (int64_t)first * ld_other + base : nullptr;
  auto read_row = [&](int r, uint32_t keep, bool few) {
    if (few) {
      uint32_t x = keep;
#pragma unroll
      for (int i = 0; i < kFew; ++i, x &= x - 1) {
        raw[i] = typename Unaligned<T>::Raw{};
        if (x != 0) Unaligned<T>::set(raw[i], 0, from + r * ld + offset_of(first_of(x)));
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      read(from + r * ld, keep, u, raw[u]);
      if constexpr (MODE == kApplyGrad) read(from_g + r * ld_other, keep, u, raw_g[u]);
    }
  };

  const bool works = chunk < chunks;
  uint32_t keep_next = there;
  bool few_next = false;
  const auto after = [&](int r) {  // the next row that is looked at, or rows
    if (MODE != kGrad || r >= rows) return r;
    const uint64_t left = live & ~0ull << r;
    return left != 0 ? __builtin_ctzll(left) : rows;
  };
  int next = after(0), later = next;
  if (works && next < rows) {  // on their way while the history is counted
    if (MASK) ask_mask(next);
    else read_row(next, keep_next, false);
  }
  if (ADJ) {  // the history before the run's first row, by the whole workgroup (of the row itself, where a row is a sequence)
    const uint4 none = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < kGroupIds / 4; i += kThreads) reinterpret_cast<uint4*>(s_adj)[i] = none;
    __syncthreads();
    const int from = lane_value(start, 0);
    const int n_history = (c.every_position ? first : max(lane_value((int)end, 0), 0)) - from;  // offsets are 32-bit integers
    if (c.token_ids != nullptr) {
      const auto count = [&](auto id_of, auto own_of) {
        constexpr int kBatch = 8;  // loads in flight per thread
        // counted from the first token, and no step is added behind the last batch: positions may reach 2^31
        for (int i0 = tid; i0 < n_history;) {
          int off[kBatch];
          bool own[kBatch];
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const unsigned i = (unsigned)i0 + b * kThreads;
            const int at = from + (int)min(i, (unsigned)(n_history - 1));
            const int64_t id = id_of(at);
            own[b] = own_of(at);
            off[b] = i < (unsigned)n_history && id >= 0 && id < vocab ? (int)id - group * kGroupIds : -1;
          }
#pragma unroll
          for (int b = 0; b < kBatch; ++b)
            if (off[b] >= 0 && off[b] < kGroupIds) {
              uint32_t* const w = s_adj + (off[b] & ~(kIds - 1)) + slot<kPer>(off[b] & (kIds - 1));
              atomicOr(w, 0x80000000u);
              if (own[b]) atomicAdd(w, 1u);
            }
          if (n_history - i0 <= kThreads * kBatch) break;
          i0 += kThreads * kBatch;
        }
      };
      const auto with_ids = [&](auto id_of) {
        const void* const m = c.own_mask;
        if (m == nullptr) count(id_of, [](int) { return true; });
        else if (c.mask_kind == AXON_MASK_I64) count(id_of, [m](int i) { return static_cast<const int64_t*>(m)[i] != 0; });
        else count(id_of, [m](int i) { return static_cast<const float*>(m)[i] != 0.f; });
      };
      const void* const ids = c.token_ids;
      if (c.token_ids_i64) with_ids([ids](int i) { return static_cast<const int64_t*>(ids)[i]; });
      else with_ids([ids](int i) { return (int64_t)static_cast<const int32_t*>(ids)[i]; });
    }
    __syncthreads();
  }
  if (!works) return;
  if (ADJ && c.every_position && __any(in_chunk))
    for (int r = 0; r < rows; ++r)
      count_l += lane >= r && token == lane_value(token, r) && start == lane_value(start, r);
  if (MASK && next < rows) {
    keep_next = mask_of(next);
    later = after(next + 1);
    if (later < rows) ask_mask(later);
    few_next = is_few(keep_next);
    read_row(next, keep_next, few_next);
  }
  if (MODE == kGrad) {
    for (int r = 0; r < rows; ++r) {
      if (live >> r & 1) continue;
      T* const o = out + (first + r) * ld_out + base;
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const int id0 = (u * kWave + lane) * kPer;
        const float none[kPer] = {};
        if (whole || base + id0 + kPer <= vocab) {
          Unaligned<T>::store(o + (uint32_t)id0, none);
        } else {
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (base + id0 + j < vocab) Row<T>::store_one(o + id0 + j, 0.f);
        }
      }
    }
  }
  float refs[2] = {kNoLogit, kNoLogit};  // of whole rows, and of rows of few ids
  bool above_before = false;
  for (int r = 0; r < rows; ++r) {
    // another sequence (a row in front of the first one starts where that does)
    if (ADJ && (r == 0 || lane_value(start, r) != lane_value(start, r - 1) || lane_value(seq, r) != lane_value(seq, r - 1))) {
      if (r > 0) {
#pragma unroll
        for (int i = 0; i < kLaneIds; ++i) adj[i * kWave + lane] = 0;
        wave_sync();
      }
      settle(r);
    }
    if (ADJ && c.every_position) {
      const int t = lane_value(token, r);
      const int id = t & (kOwn - 1), off = id - base;
      if (t >= 0 && off >= 0 && off < kIds) {  // the row's own token
        const int u = off / (kWave * kPer), at = off / kPer % kWave, j = off % kPer;
        if (lane == at) seen |= 1u << (u * kPer + j);
        touched |= 1u << ((u * kPer + j) / 4);
        if (t & kOwn) {
          const float p = penalty(lane_value(count_l, r), lane_value(freq_l, r), lane_value(pres_l, r)) - lane_value(bias_l, r);
          if (lane == at) adj[slot<kPer>(off)] = __float_as_uint(p);
          wave_sync();
        }
      }
    }
    if (MODE == kGrad && r != next) continue;
    const int64_t row = first + r;
    const float inv_t = lane_value(inv_t_l, r), k = inv_t * kLog2e, rep = lane_value(rep_l, r), inv_rep = 1.f / rep;
    uint32_t keep = keep_next;
    const bool few = few_next;
    if (MASK) {
      next = later;
      keep_next = next < rows ? mask_of(next) : 0;
      later = after(next + 1);
      if (later < rows) ask_mask(later);
    } else {
      next = after(r + 1);
    }
    // masks of single bits are made where they are used: 32 of them held over the rows are 32 registers
    asm volatile("" : "+v"(keep), "+v"(seen));
    const int l = MODE == kStats || MODE == kGrad ? lane_value(label, r) - base : -1;
    const bool has_label = l >= 0 && l < kIds;
    const int label_lane = l / kPer % kWave, label_at = l / (kWave * kPer) * kPer + l % kPer;
    const bool masked = (MASK || !whole) && __any(keep != kAll);
    const bool repeats = ADJ && rep != 1.f;
    const bool more = next < rows;

    // vector u under the controls, before the temperature; banned: what stands for -inf.  slope: dy / dz of every element.
    auto controlled = [&](int u, float banned, float (&y)[kPer], float (&slope)[kPer]) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) { y[j] = Unaligned<T>::get(raw[u], j); slope[j] = 1.f; }
#pragma unroll
      for (int q = 0; q < kPer; q += 4) {
        if (!ADJ || !(touched >> ((u * kPer + q) / 4) & 1)) continue;
        float sub[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) sub[j] = __uint_as_float(adj[slot<kPer>((u * kWave + lane) * kPer + q + j)]);
        if (repeats) {
#pragma unroll
          for (int j = 0; j < 4; ++j) slope[q + j] = pick(bit_mask(seen, u * kPer + q + j), y[q + j] > 0.f ? inv_rep : rep, 1.f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) y[q + j] = fmaf(y[q + j], slope[q + j], -sub[j]);
      }
      if (masked) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) y[j] = pick(bit_mask(keep, u * kPer + j), y[j], banned);
      }
    };

    if constexpr (MODE == kStats) {
      float4* const part = io.parts + row * chunks + chunk;
      // The sum of N logits of each lane, and weighted by their exponents, against the reference m: the largest logit of an
      // earlier row of this chunk will do as long as the sum stays in range and the terms that count are near it.  Against
      // c = m k rounded it is one instruction per element, and what c is off by is the same for all of them and taken back.
      auto statistics = [&](auto n, auto& y, uint32_t bits) {
        constexpr int N = decltype(n)::value;
        auto largest = [&] {
          float m = y[0];
#pragma unroll
          for (int i = 1; i < N; ++i) m = fmaxf(m, y[i]);
          return wave_max(m);
        };
        float& ref = refs[N == kFew];
        float m = ref > kBanned ? ref : largest();
        const float cc = m * k;
        float s4[4] = {}, e4[4] = {}, s = 0.f, e = 0.f;
        // what is banned has to be out of reach of the reference (at a temperature of 1e28 it is not)
        bool plain = fabsf(cc) < kFar && (m - kBanned) * k > 2 * -kTiny, above = false;
        if (plain) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float d = fmaf(y[i], k, -cc), f = __builtin_amdgcn_exp2f(d);
            s4[i & 3] += f;
            e4[i & 3] = fmaf(f, d, e4[i & 3]);
          }
          s = wave_sum((s4[0] + s4[1]) + (s4[2] + s4[3]));
          e = wave_sum((e4[0] + e4[1]) + (e4[2] + e4[3]));
          const float off = fmaf(m, k, -cc), back = __builtin_amdgcn_exp2f(-off);  // 2^(y k - c) = 2^((y - m) k + off)
          e = fmaf(-off, s, e) * back;
          s *= back;
          // e / s: how far the terms that count are from the reference, of which their exponents carry the rounding
          plain = s > 0x1p-80f && s < 0x1p100f && fabsf(e) <= kNear * s;
          above = e > kNear * s;
        }
        if (!plain) {  // another scale (a likely token), logits far from 0, infinite, or not numbers: by differences, what is banned at -inf
          asm volatile("" : "+v"(bits));
#pragma unroll
          for (int i = 0; i < N; ++i) y[i] = pick(bit_mask(bits, i), y[i], -INFINITY);
          m = largest();
          if (!(m > -INFINITY)) m = kNoLogit;
#pragma unroll
          for (int i = 0; i < 4; ++i) s4[i] = e4[i] = 0.f;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float d = (y[i] - m) * k, f = __builtin_amdgcn_exp2f(d);
            s4[i & 3] += f;
            e4[i & 3] = fmaf(f, fmaxf(d, kTiny), e4[i & 3]);
          }
          s = wave_sum((s4[0] + s4[1]) + (s4[2] + s4[3]));
          e = wave_sum((e4[0] + e4[1]) + (e4[2] + e4[3]));
        }
        const bool once = above && !above_before;  // a likely token: what is like the rows before it stays the reference
        if (!once) ref = m;
        above_before = once;
        if (lane == 0) *part = make_float4(m, s, e, 0.f);
      };
      if (MASK && few) {
        float y[kFew];
        uint32_t x = keep, there_are = 0;
        float label_y = -INFINITY;
#pragma unroll
        for (int i = 0; i < kFew; ++i, x &= x - 1) {
          const int bit = first_of(x);
          y[i] = Unaligned<T>::get(raw[i], 0);
          if (ADJ && touched != 0) {
            const float slope = repeats && (seen >> bit & 1) ? (y[i] > 0.f ? inv_rep : rep) : 1.f;
            y[i] = fmaf(y[i], slope, -__uint_as_float(adj[slot<kPer>((int)offset_of(bit))]));
          }
          if (x != 0 && bit == label_at) label_y = y[i];
          y[i] = x != 0 ? y[i] : kBanned;
          there_are |= (uint32_t)(x != 0) << i;
        }
        few_next = is_few(keep_next);
        if (more) read_row(next, keep_next, few_next);
        if (__any(keep != 0)) statistics(std::integral_constant<int, kFew>{}, y, there_are);
        else if (lane == 0) *part = make_float4(kNoLogit, 0.f, 0.f, 0.f);
        if (has_label && lane == label_lane) io.label_y[row] = label_y;
        continue;
      }
      float y[kLaneIds];
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        float v[kPer], slope[kPer];
        controlled(u, kBanned, v, slope);
#pragma unroll
        for (int j = 0; j < kPer; ++j) y[u * kPer + j] = v[j];
      }
      few_next = is_few(keep_next);
      if (more) read_row(next, keep_next, few_next);
      statistics(std::integral_constant<int, kLaneIds>{}, y, keep);
      if (has_label) {
        const int at = lane == label_lane ? label_at : -1;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < kLaneIds; ++i) v = i == at ? y[i] : v;
        if (at >= 0) io.label_y[row] = keep >> label_at & 1 ? v : -INFINITY;
      }
    } else {
      T* const o = out + row * ld_out + base;
      const float top = lane_value(top_l, r), A = lane_value(a_l, r), B = lane_value(b_l, r), g_lp = lane_value(glp_l, r);
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const int id0 = (u * kWave + lane) * kPer;
        float y[kPer], slope[kPer], d[kPer];
        controlled(u, -INFINITY, y, slope);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (MODE == kApply) {
            d[j] = y[j] * inv_t;
          } else if (MODE == kApplyGrad) {
            d[j] = y[j] == -INFINITY ? 0.f : Unaligned<T>::get(raw_g[MODE == kApplyGrad ? u : 0], j) * (slope[j] * inv_t);
          } else {
            // a probability of 0 takes nothing from the entropy
            const float t = (y[j] - top) * k;
            d[j] = __builtin_amdgcn_exp2f(t) * fmaf(B, fmaxf(t, kTiny), A);
          }
        }
        if (more) {
          read(from + next * ld, keep_next, u, raw[u]);
          if constexpr (MODE == kApplyGrad) read(from_g + next * ld_other, keep_next, u, raw_g[u]);
        }
        if (MODE == kGrad && has_label && label_at / kPer == u) {
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (lane == label_lane && label_at % kPer == j && y[j] != -INFINITY) d[j] += g_lp;
        }
        if (MODE == kGrad && ADJ && repeats) {
#pragma unroll
          for (int q = 0; q < kPer; q += 4) {
            if (!(touched >> ((u * kPer + q) / 4) & 1)) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) d[q + j] *= slope[q + j];
          }
        }
        if (whole || base + id0 + kPer <= vocab) {
          Unaligned<T>::store(o + (uint32_t)id0, d);
        } else {
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (base + id0 + j < vocab) Row<T>::store_one(o + id0 + j, d[j]);
        }
      }
    }
  }
}

// A row's chunks together, by a wavefront, in 64 bits: log-probability of the label, entropy, and what the backward reads: the
// logarithm M of the sum of exponentials (before the temperature, rounded), the sum of 2^((y - M) log2(e) / T), the entropy.  A row that nothing is left of has
// M = 0, of which its -inf are far enough.  4 us for 187 rows of 75 chunks, 7 for 4096: latency.
__global__ __launch_bounds__(kBlock) void controls_finish_kernel(int n_rows, int vocab, int chunks, axon_controls c, RowIo io,
                                                                 float* logprob, float* entropy, float* stats) {
  const int row = (int)(blockIdx.x * kWaves + threadIdx.x / kWave), lane = threadIdx.x & (kWave - 1);
  if (row >= n_rows) return;
  float M = kNoLogit;
  for (int i = lane; i < chunks; i += kWave) M = fmaxf(M, io.parts[(int64_t)row * chunks + i].x);
  M = wave_max(M);
  float inv_t = 1.f / c.temperature_all;
  if (c.temperature != nullptr) {
    int64_t seq = !c.every_position ? row : c.uniform_len > 0 ? row / c.uniform_len : RowFinder::upper4(c.cu_seqlens, 0, (int)c.n_seqs, row);
    inv_t = 1.f / c.temperature[min(max(seq, (int64_t)0), c.n_seqs - 1)];
  }
  const float k = inv_t * kLog2e;
  double s = 0.0, e = 0.0;
  for (int i = lane; i < chunks; i += kWave) {
    const float4 p = io.parts[(int64_t)row * chunks + i];
    // the references are no maxima: a sum may be anything from 2^-80 to 2^100
    const double d = ((double)p.x - (double)M) * (double)k, f = exp2(d);
    if (f > 0.0 || p.y != p.y) {
      s += (double)p.y * f;
      e += f * ((double)p.y * d + (double)p.z);
    }
  }
  s = wave_sum_d(s);
  e = wave_sum_d(e);
  if (lane != 0) return;
  float sum = 1.f, H = 0.f, lp = 0.f;
  const int64_t l = index_at(io.labels, io.labels_i64, row);
  const bool inside = l >= 0 && l < vocab;
  if (s == 0.0) {  // nothing is left
    lp = inside ? -INFINITY : 0.f;
    M = 0.f;
  } else {
    const double ls = log2(s);
    H = (float)((ls - e / s) * 0.6931471805599453);
    if (inside) lp = (float)((((double)io.label_y[row] - (double)M) * (double)k - ls) * 0.6931471805599453);
    // for the backward against the logarithm of the sum: what is likely has an exponent near 0
    const float near = (float)((double)M + ls / (double)k);
    if (fabsf(near) <= 3.402823466e38f) {
      sum = (float)exp2(ls - ((double)near - (double)M) * (double)k);
      M = near;
    } else {
      sum = (float)s;
    }
  }
  logprob[row] = lp;
  if (entropy != nullptr) entropy[row] = H;
  stats[row] = M;
  stats[(int64_t)n_rows + row] = sum;
  stats[2 * (int64_t)n_rows + row] = H;
}

}  // namespace axon

using namespace axon;

namespace {

constexpr int64_t kCacheBytes = int64_t(256) << 20;

int elem_bytes(int dtype) { return dtype == AXON_LOGITS_F32 ? 4 : 2; }

int check_rows(const void* p, int dtype, int64_t ld, int64_t n, int64_t v) {
  if (n < 0 || v <= 0 || ld < v || (dtype != AXON_LOGITS_F32 && dtype != AXON_LOGITS_BF16)) return AXON_ERR_ARG;
  if (n >= (int64_t)1 << 24 || v >= kOwn) return AXON_ERR_SHAPE;
  if (n > 0 && (!p || reinterpret_cast<uintptr_t>(p) % elem_bytes(dtype) != 0)) return AXON_ERR_ARG;
  return AXON_OK;
}

// Whether the operands of the controls are there and belong to n rows.
int check_controls(const axon_controls* c, int64_t n, int64_t v) {
  if (!c || c->n_seqs < 0 || c->n_tokens < 0 || c->uniform_len < 0 || c->n_bias < 0 || c->allowed_rows < 0) return AXON_ERR_ARG;
  if (n == 0) return AXON_OK;
  if (c->n_seqs >= INT32_MAX || c->n_tokens >= INT32_MAX || c->n_bias >= INT32_MAX || c->allowed_rows >= INT32_MAX) return AXON_ERR_SHAPE;
  const bool per_seq = c->repetition || c->frequency || c->presence || c->temperature || (c->n_bias && c->bias_per_seq) || c->token_ids;
  if (per_seq) {
    if (c->n_seqs == 0) return AXON_ERR_ARG;
    if (c->uniform_len > 0) {
      if (c->n_seqs > INT32_MAX / c->uniform_len) return AXON_ERR_SHAPE;
      if (c->token_ids && c->n_seqs * c->uniform_len != c->n_tokens) return AXON_ERR_SHAPE;
      if (c->every_position && n != c->n_seqs * c->uniform_len) return AXON_ERR_SHAPE;
    } else if (!c->cu_seqlens && (c->every_position || c->token_ids)) {
      return AXON_ERR_ARG;
    }
    if (!c->every_position && n != c->n_seqs) return AXON_ERR_SHAPE;
    if (c->every_position && c->token_ids && n != c->n_tokens) return AXON_ERR_SHAPE;
  }
  if (c->mask_kind != AXON_MASK_F32 && c->mask_kind != AXON_MASK_I64) return AXON_ERR_ARG;
  if (c->n_bias > 0 && (!c->bias_ids || !c->bias)) return AXON_ERR_ARG;
  if (c->allowed) {
    if (c->allowed_rows < 1 || c->allowed_stride < (v + 31) / 32) return AXON_ERR_SHAPE;
    if (!c->allowed_index && c->allowed_rows != 1 && c->allowed_rows != n) return AXON_ERR_SHAPE;
  }
  const auto positive = [](float x) { return x >= 0x1p-126f && x <= 3.402823466e38f; };  // smaller ones have no reciprocal
  const auto finite = [](float x) { return x - x == 0.f; };
  if (!c->repetition && !positive(c->repetition_all)) return AXON_ERR_ARG;
  if (!c->temperature && !positive(c->temperature_all)) return AXON_ERR_ARG;
  if ((!c->frequency && !finite(c->frequency_all)) || (!c->presence && !finite(c->presence_all))) return AXON_ERR_ARG;
  return AXON_OK;
}

int chunks_of(int64_t vocab, int dtype) { return (int)((vocab * elem_bytes(dtype) + kChunkBytes - 1) / kChunkBytes); }

// Workgroups of a kernel that the device holds at once (it is the same for all devices that this is built for).
template <typename K>
int resident_of(K kernel, int threads) {
  int dev = 0, cus = 0, per_cu = 0;
  const bool known = hipGetDevice(&dev) == hipSuccess && hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess &&
                     hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, reinterpret_cast<const void*>(kernel), threads, 0) == hipSuccess;
  return known && cus * per_cu > 0 ? cus * per_cu : 1024;
}

// Rows of a run: three times as many workgroups as there is room for, so that the last ones to start are a small part, and what a
// run costs by itself (the history before it, its terms) is shared by as many rows as that leaves.  Log-probabilities with gradients
// of 2047 x 50257 bf16 take 154 us so, 151 to 154 with two, 159 with four; 4096 x 151936 under masks 284, 307 and 293 us.
int run_of(int64_t n, int groups, int resident) {
  const int64_t most = 3 * (int64_t)resident, r = (n * groups + most - 1) / most;
  return (int)(r < 1 ? 1 : (r < kMaxRun ? r : kMaxRun));
}

// Wavefronts of a workgroup that holds additive terms: those of 8192 ids, 32 KB of LDS and five workgroups on a compute unit.  Each
// reads the whole history, so fewer ids a workgroup cost reads (61 x 201088 fp32 with 4000 tokens each: 4 wavefronts 33 us, 8 30 us),
// more cost workgroups that work while another waits (16: 39 us; 1024 x 32768 bf16 with 1500 tokens each: 4 38.7, 8 39.5, 16 43 us).
template <typename T> constexpr int kAdjWaves = sizeof(T) == 4 ? 8 : 4;

template <Mode MODE>
int launch(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab, const axon_controls& given, const RowIo& io,
           const void* other, int64_t ld_other, void* out, int64_t ld_out, hipStream_t st) {
  axon_controls c = given;
  const bool penalties = c.repetition || c.frequency || c.presence || c.repetition_all != 1.f || c.frequency_all != 0.f || c.presence_all != 0.f;
  if (!penalties) c.token_ids = nullptr;  // nobody asks for the history
  const bool adj = (penalties && c.token_ids) || c.n_bias > 0, mask = c.allowed != nullptr;
  const int chunks = chunks_of(vocab, dtype);
  const bool of_rows = !c.every_position;
#define AXON_CONTROLS(T, A, M, WAVES)                                                                                                           \
  do {                                                                                                                                          \
    const auto kernel = controls_kernel<T, MODE, A, M, WAVES>;                                                                                  \
    static const int resident = resident_of(kernel, WAVES * kWave);                                                                             \
    const int groups = (chunks + WAVES - 1) / WAVES, run = A && of_rows ? 1 : run_of(n, groups, resident);                                      \
    const int64_t grid = (n + run - 1) / run * groups;                                                                                          \
    if (grid * (WAVES * kWave) > UINT32_MAX) return AXON_ERR_SHAPE;                                                                             \
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(WAVES * kWave), 0, st, static_cast<const T*>(logits), ld, (int)n, (int)vocab,         \
                       chunks, run, c, io, static_cast<const T*>(other), ld_other, static_cast<T*>(out), ld_out);                               \
  } while (0)
#define AXON_CONTROLS_OF(T)                                  \
  do {                                                       \
    if (adj && mask) AXON_CONTROLS(T, true, true, kAdjWaves<T>);             \
    else if (adj) AXON_CONTROLS(T, true, false, kAdjWaves<T>);               \
    else if (mask) AXON_CONTROLS(T, false, true, 4);         \
    else AXON_CONTROLS(T, false, false, 4);                  \
  } while (0)
  if (dtype == AXON_LOGITS_F32) AXON_CONTROLS_OF(float);
  else AXON_CONTROLS_OF(unsigned short);
#undef AXON_CONTROLS_OF
#undef AXON_CONTROLS
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

}  // namespace

extern "C" int axon_controls_apply(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab, const axon_controls* controls,
                                   void* out, int64_t ld_out, void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc == AXON_OK) rc = check_rows(out, dtype, ld_out, n, vocab);
  if (rc == AXON_OK) rc = check_controls(controls, n, vocab);
  if (rc != AXON_OK || n == 0) return rc;
  return launch<kApply>(logits, dtype, ld, n, vocab, *controls, RowIo{}, nullptr, 0, out, ld_out, (hipStream_t)stream);
}

extern "C" int axon_controls_apply_bwd(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab,
                                       const axon_controls* controls, const void* g_out, int64_t ld_g, void* dlogits, int64_t ld_d,
                                       void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc == AXON_OK) rc = check_rows(g_out, dtype, ld_g, n, vocab);
  if (rc == AXON_OK) rc = check_rows(dlogits, dtype, ld_d, n, vocab);
  if (rc == AXON_OK) rc = check_controls(controls, n, vocab);
  if (rc != AXON_OK || n == 0) return rc;
  return launch<kApplyGrad>(logits, dtype, ld, n, vocab, *controls, RowIo{}, g_out, ld_g, dlogits, ld_d, (hipStream_t)stream);
}

extern "C" int64_t axon_controls_logprob_workspace_bytes(int64_t n, int64_t vocab) {
  if (n < 0 || vocab <= 0 || vocab >= kOwn) return AXON_ERR_ARG;
  return n * (chunks_of(vocab, AXON_LOGITS_F32) * (int64_t)sizeof(float4) + (int64_t)sizeof(float));
}

extern "C" int axon_controls_logprob_fwd(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab,
                                         const axon_controls* controls, const void* labels, int labels_i64, float* logprob,
                                         float* entropy, float* stats, void* workspace, int64_t workspace_bytes, int bwd_follows,
                                         void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc == AXON_OK) rc = check_controls(controls, n, vocab);
  if (rc != AXON_OK || n == 0) return rc;
  if (!labels || !logprob || !stats) return AXON_ERR_ARG;
  if (!workspace || workspace_bytes < axon_controls_logprob_workspace_bytes(n, vocab) || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return AXON_ERR_WORKSPACE;
  const int chunks = chunks_of(vocab, dtype);
  RowIo io{};
  io.labels = labels;
  io.labels_i64 = labels_i64;
  io.parts = static_cast<float4*>(workspace);
  io.label_y = reinterpret_cast<float*>(io.parts + n * chunks);
  const int64_t cached = bwd_follows ? kCacheBytes / (vocab * elem_bytes(dtype)) : 0;
  io.cached_from = (int)(cached < n ? n - cached : 0);
  const hipStream_t st = (hipStream_t)stream;
  rc = launch<kStats>(logits, dtype, ld, n, vocab, *controls, io, nullptr, 0, nullptr, 0, st);
  if (rc != AXON_OK) return rc;
  hipLaunchKernelGGL(controls_finish_kernel, dim3((unsigned)((n + kWaves - 1) / kWaves)), dim3(kBlock), 0, st, (int)n, (int)vocab, chunks,
                     *controls, io, logprob, entropy, stats);
  AXON_CHECK_LAUNCH();
  return AXON_OK;
}

extern "C" int axon_controls_logprob_bwd(const void* logits, int dtype, int64_t ld, int64_t n, int64_t vocab,
                                         const axon_controls* controls, const void* labels, int labels_i64, const float* stats,
                                         const float* g_logprob, const float* g_entropy, void* dlogits, int64_t ld_d, void* stream) {
  int rc = check_rows(logits, dtype, ld, n, vocab);
  if (rc == AXON_OK) rc = check_rows(dlogits, dtype, ld_d, n, vocab);
  if (rc == AXON_OK) rc = check_controls(controls, n, vocab);
  if (rc != AXON_OK || n == 0) return rc;
  if (!labels || !stats) return AXON_ERR_ARG;
  RowIo io{};
  io.labels = labels;
  io.labels_i64 = labels_i64;
  io.stats = stats;
  io.g_logprob = g_logprob;
  io.g_entropy = g_entropy;
  return launch<kGrad>(logits, dtype, ld, n, vocab, *controls, io, nullptr, 0, dlogits, ld_d, (hipStream_t)stream);
}
