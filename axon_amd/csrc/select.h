// The k largest of a row, exactly, equal values by ascending index, without looking at the whole row again.
//
// A row is cut into segments of consecutive elements, whose maxima the pass that reads the row anyway has left.  Ordered
// by (maximum descending, index ascending), the first k segments hold the k first elements by (value descending, index
// ascending): an element of any other segment has k segments before its own, and the maximum of each of them comes
// before it.  So the maxima are selected from first, then the elements of k segments, those only that reach the smallest
// of the k maxima: about as many as are wanted.
#pragma once
#include "common.h"

namespace axon {

constexpr int kMaxTop = AXON_MAX_TOP;  // alternatives per row
constexpr int kCandidates = 512;  // elements that reach the smallest maximum taken and are ranked against each other
constexpr int kMaxSegs = 2 * kMaxTop;  // segments taken: the first k and a few more where that saves a look

// Unsigned integers in the order of the floats; -0 equals 0, and NaN equals -inf, as a maximum that passes it by has it (so
// that a segment's key is never above those of all its elements).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0x007fffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
// ... and of (value descending, index ascending)
__device__ __forceinline__ uint64_t order_key(float x, int index) {
  return ((uint64_t)order_key(x) << 32) | (0xffffffffu - (uint32_t)index);
}

constexpr int kHits = 96;  // items that hold a candidate and are gone through an element per thread
struct SelectLds {
  alignas(16) uint64_t cand[kCandidates];
  float hits[kHits][8];
  int hit_at[kHits], n_hits;
  int hist[256];
  int segs[kMaxSegs];
  uint32_t range[2][4];
  int n_segs, n_cand, bin, before, upto;
};

constexpr int NT = kBlock;  // threads that work on a row: a workgroup

// Permutations by DPP in which every lane has a source, and the sums up to a lane, whose missing sources are 0.
template <int CTRL>
__device__ __forceinline__ uint32_t lane_of(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, lane_of<0xb1>(v));
  v = max(v, lane_of<0x4e>(v));
  v = max(v, lane_of<0x141>(v));
  v = max(v, lane_of<0x140>(v));
  const uint32_t a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = __builtin_amdgcn_readlane((int)v, 32), d = __builtin_amdgcn_readlane((int)v, 48);
  return max(max(a, b), max(c, d));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add_i(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_upto(int v) {
  v = dpp_add_i<0x111, 0xf>(v);  // row_shr:1
  v = dpp_add_i<0x112, 0xf>(v);
  v = dpp_add_i<0x114, 0xf>(v);
  v = dpp_add_i<0x118, 0xf>(v);
  v = dpp_add_i<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  return dpp_add_i<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
}

// Smallest and largest over the threads.
__device__ __forceinline__ void group_range(SelectLds& s, int tid, uint32_t& lo, uint32_t& hi) {
  lo = ~wave_max_u32(~lo);
  hi = wave_max_u32(hi);
  if ((tid & (kWave - 1)) == 0) { s.range[0][tid / kWave] = lo; s.range[1][tid / kWave] = hi; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / kWave; ++w) { lo = min(lo, s.range[0][w]); hi = max(hi, s.range[1][w]); }
}
// The k-th largest of n keys (1 <= k <= n), eight bits at a time; `ties`: how many of the keys equal to it are among
// the k.  key_at(i) is asked for every i once per eight bits.
template <class Key, class KeyAt>
__device__ __forceinline__ Key kth_largest(KeyAt key_at, int n, int k, SelectLds& s, int tid, int& ties) {
  Key prefix = 0, mask = 0;
  int rest = k;
  for (int shift = 8 * (int)sizeof(Key) - 8; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += NT) s.hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const Key key = key_at(i);
      if ((key & mask) == prefix) atomicAdd(&s.hist[(int)(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid < kWave) {  // lane l: bins 255 - 4 l and the three below
      int c[4], sum = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) sum += c[q] = s.hist[255 - 4 * tid - q];
      int before = wave_upto(sum) - sum;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (before < rest && before + c[q] >= rest) { s.bin = 255 - 4 * tid - q; s.before = before; }
        before += c[q];
      }
    }
    __syncthreads();
    prefix |= (Key)s.bin << shift;
    mask |= (Key)255 << shift;
    rest -= s.before;
  }
  ties = rest;
  return prefix;
}

// A row's keys in the threads' registers, up to NT * Src::kHeld of them, requested together: where they are in memory, a loop
// that asks for one at a time is a trip there each, and there are three such loops.  More are asked for again wherever they are
// needed, as are those in LDS, which a loop reads faster than code for every number of them runs.
template <class Src>
struct HeldKeys {
  static constexpr int kHeld = Src::kHeld;
  const Src& src;
  const int n, tid;
  uint32_t key[kHeld > 0 ? kHeld : 1];
  __device__ __forceinline__ HeldKeys(const Src& s, int n_, int tid_) : src(s), n(n_), tid(tid_) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      if (u * NT >= n) break;
      key[u] = tid + u * NT < n ? src.max_key(tid + u * NT) : 0u;
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      if (u * NT >= n) break;
      if (tid + u * NT < n) f(tid + u * NT, key[u]);
    }
    for (int i = tid + kHeld * NT; i < n; i += NT) f(i, src.max_key(i));
  }
};

// The segments that are looked at, to s.segs: those whose maximum reaches a bound (returned) that at least k maxima reach.
// The keys' range is cut into 256 bins and the bin of the k-th taken whole if that makes at most a quarter more; else
// the bin is cut again, down to one key, of whose segments the first are taken then.  A row of a model's logits takes one cut.
template <class Src>
__device__ __forceinline__ uint32_t choose_segments(const Src& src, int n, int k, SelectLds& s, int tid) {
  const int most = k + k / 4 + 8;
  const HeldKeys<Src> keys(src, n, tid);
  uint32_t lo = 0xffffffffu, hi = 0;
  keys.each([&](int, uint32_t key) {
    lo = min(lo, key);
    hi = max(hi, key);
  });
  group_range(s, tid, lo, hi);
  int rest = k, above = 0;  // of the segments in the range, `rest` are wanted; `above`: segments above the range
  uint32_t least;
  for (uint32_t width = hi - lo;;) {  // the range: lo .. lo + width
    const int shift = width < 256 ? 0 : 24 - __builtin_clz(width);
    for (int i = tid; i < 256; i += NT) s.hist[i] = 0;
    __syncthreads();
    keys.each([&](int, uint32_t key) {
      const uint32_t at = key - lo;
      if (at <= width) atomicAdd(&s.hist[at >> shift], 1);
    });
    __syncthreads();
    if (tid < kWave) {  // lane l: bins 255 - 4 l and the three below
      int c[4], sum = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) sum += c[q] = s.hist[255 - 4 * tid - q];
      int before = wave_upto(sum) - sum;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (before < rest && before + c[q] >= rest) { s.bin = 255 - 4 * tid - q; s.before = before; s.upto = before + c[q]; }
        before += c[q];
      }
    }
    __syncthreads();
    least = lo + ((uint32_t)s.bin << shift);
    if (above + s.upto <= most || shift == 0) break;
    above += s.before;
    rest -= s.before;
    const uint32_t last = lo + width;
    lo = least;
    width = min((1u << shift) - 1, last - lo);
  }
  if (above + s.upto <= most) {
    keys.each([&](int i, uint32_t key) {
      if (key >= least) s.segs[atomicAdd(&s.n_segs, 1)] = i;
    });
    return least;
  }
  const int ties = rest - s.before;  // at a bin of one key: how many of its segments are wanted
  int one;
  auto first = [&](int i) { return src.max_key(i) == least ? 0xffffffffu - (uint32_t)i : 0u; };
  const uint32_t last = kth_largest<uint32_t>(first, n, ties, s, tid, one);
  keys.each([&](int i, uint32_t key) {
    if (key > least || (key == least && 0xffffffffu - (uint32_t)i >= last)) s.segs[atomicAdd(&s.n_segs, 1)] = i;
  });
  return least;
}

// `src`: maxima of its segments, max_key(i) for i < n_segs() (kHeld: see HeldKeys); the elements of the segments in `segs`, kPer consecutive ones
// per item: load(segs, j, v) returns the index of the first, or -1 where there is none (elements from limit() on do not
// count); and n_single() elements outside all segments, single(i, index).  out(rank, value, index) for rank < k.
template <class Src, class Out>
__device__ __forceinline__ void select_top(const Src& src, int k, SelectLds& s, int tid, Out out) {
  const int n = src.n_segs();
  uint32_t least = 0;  // what an element has to reach
  if (tid == 0) s.n_segs = s.n_cand = s.n_hits = 0;
  if (n > k) {
    least = choose_segments(src, n, k, s, tid);
  } else {
    for (int i = tid; i < n; i += NT) s.segs[i] = i;
  }
  __syncthreads();
  const int n_items = (n > k ? s.n_segs : n) * Src::kItems, limit = src.limit();
  auto offer = [&](float x, int index) {
    if (order_key(x) < least) return;
    const int at = atomicAdd(&s.n_cand, 1);
    if (at < kCandidates) s.cand[at] = order_key(x, index);
  };
  // an item of which no element reaches the bound, as most, costs a comparison (NaN passes it)
  const float bound = least == 0 ? -INFINITY : key_value(least);
  auto any = [&](const float (&v)[Src::kPer]) {
    float m = v[0];
#pragma unroll
    for (int e = 1; e < Src::kPer; ++e) m = fmaxf(m, v[e]);
    return !(m < bound);
  };
  // four loads under way together: one at a time is a trip to memory each
  constexpr int kDeep = 4;
  for (int j0 = tid; j0 < n_items; j0 += kDeep * NT) {
    float v[kDeep][Src::kPer];
    int i0[kDeep];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      i0[u] = -1;
      if (j0 + u * NT < n_items) i0[u] = src.load(s.segs, j0 + u * NT, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      if (i0[u] < 0 || !any(v[u])) continue;
      const int hit = atomicAdd(&s.n_hits, 1);
      if (hit < kHits) {
        s.hit_at[hit] = i0[u];
#pragma unroll
        for (int e = 0; e < Src::kPer; ++e) s.hits[hit][e] = v[u][e];
      } else {
#pragma unroll
        for (int e = 0; e < Src::kPer; ++e)
          if (i0[u] + e < limit) offer(v[u][e], i0[u] + e);
      }
    }
  }
  __syncthreads();
  // few items hold a candidate: their elements one per thread (all elements of every item: eight times the instructions in each
  // wavefront that has one)
  for (int i = tid, n_el = min(s.n_hits, kHits) * Src::kPer; i < n_el; i += NT) {
    const int index = s.hit_at[i / Src::kPer] + i % Src::kPer;
    if (index < limit) offer(s.hits[i / Src::kPer][i % Src::kPer], index);
  }
  for (int i = tid; i < src.n_single(); i += NT) {
    int index;
    const float x = src.single(i, index);
    offer(x, index);
  }
  __syncthreads();
  int c = s.n_cand;
  if (c > kCandidates) {  // a run of equal values, as a rule: the k-th key itself, from the elements of the segments
    const int n_el = n_items * Src::kPer + src.n_single();
    auto element = [&](int i) -> uint64_t {
      if (i >= n_items * Src::kPer) {
        int index;
        const float x = src.single(i - n_items * Src::kPer, index);
        return order_key(x, index);
      }
      float v[Src::kPer];
      const int i0 = src.load(s.segs, i / Src::kPer, v), e = i % Src::kPer;
      if (i0 < 0 || i0 + e >= limit) return 0;
      float x = v[0];
#pragma unroll
      for (int q = 1; q < Src::kPer; ++q) x = e == q ? v[q] : x;
      return order_key(x, i0 + e);
    };
    int one;
    const uint64_t last = kth_largest<uint64_t>(element, n_el, k, s, tid, one);
    if (tid == 0) s.n_cand = 0;
    __syncthreads();
    for (int i = tid; i < n_el; i += NT) {
      const uint64_t key = element(i);
      if (key >= last) s.cand[atomicAdd(&s.n_cand, 1)] = key;
    }
    __syncthreads();
    c = k;
  }
  // Ranks.  Few candidates are each compared with all; more are first put in order of 256 bins of their range, and compared
  // inside their bin.
  auto put = [&](int rank, uint64_t key) {
    if (rank < k) out(rank, key_value((uint32_t)(key >> 32)), (int)(0xffffffffu - (uint32_t)key));
  };
  if (c <= kWave) {
    if (tid == 0) s.cand[c] = 0;  // to a whole number of pairs
    __syncthreads();
    if (tid < c) {
      const uint64_t mine = s.cand[tid];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < c; j += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(s.cand + j);
        rank += (two.x > mine) + (two.y > mine);
      }
      put(rank, mine);
    }
    return;
  }
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int i = tid; i < c; i += NT) {
    const uint32_t key = (uint32_t)(s.cand[i] >> 32);
    lo = min(lo, key);
    hi = max(hi, key);
  }
  group_range(s, tid, lo, hi);
  const int shift = hi - lo < 256 ? 0 : 24 - __builtin_clz(hi - lo);
  for (int i = tid; i < 256; i += NT) s.hist[i] = 0;
  __syncthreads();
  // a candidate's bin, and its number among those of the bin that came before it
  constexpr int kSlots = kCandidates / NT;
  uint64_t mine[kSlots];
  int bin[kSlots], nth[kSlots];
#pragma unroll
  for (int u = 0; u < kSlots; ++u) {
    if (u * NT >= c) break;
    if (tid + u * NT >= c) continue;
    mine[u] = s.cand[tid + u * NT];
    bin[u] = ((uint32_t)(mine[u] >> 32) - lo) >> shift;
    nth[u] = atomicAdd(&s.hist[bin[u]], 1);
  }
  __syncthreads();
  if (tid < kWave) {  // hist[b]: how many lie in higher bins; lane l has bins 255 - 4 l and the three below
    int n4[4], sum = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) sum += n4[q] = s.hist[255 - 4 * tid - q];
    int before = wave_upto(sum) - sum;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s.hist[255 - 4 * tid - q] = before;
      before += n4[q];
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSlots; ++u) {
    if (u * NT >= c) break;
    if (tid + u * NT < c) s.cand[s.hist[bin[u]] + nth[u]] = mine[u];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSlots; ++u) {
    if (u * NT >= c) break;
    if (tid + u * NT >= c) continue;
    int rank = s.hist[bin[u]];
    if (rank >= k) continue;
    const int end = bin[u] > 0 ? s.hist[bin[u] - 1] : c;
    for (int j = rank; j < end; ++j) rank += s.cand[j] > mine[u];
    put(rank, mine[u]);
  }
}

}  // namespace axon
