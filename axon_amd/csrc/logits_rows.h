// A row of materialised logits as the streaming kernels walk it: vector loads of both types, running softmax
// statistics, and the share of a row that a workgroup has.
#pragma once
#include "common.h"

namespace axon {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float bf16_to_f32(unsigned short h) { return __uint_as_float((uint32_t)h << 16); }
// two floats to bf16, round to nearest even, NaN kept (one v_cvt_pk_bf16_f32; in integer arithmetic eight
// instructions per value, which is what held the gradient kernel back)
__device__ __forceinline__ uint32_t f32x2_to_bf16(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

template <typename T> struct Row;
template <> struct Row<float> {
  static constexpr int kPer = 4;
  // CACHED: the vector stays in the caches behind (plain load) instead of passing them by
  template <bool CACHED = false>
  __device__ static void load(const float* p, float (&v)[8]) {
    const f32x4* const q = reinterpret_cast<const f32x4*>(p);
    const f32x4 x = CACHED ? *q : __builtin_nontemporal_load(q);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  }
  __device__ static float one(const float* p) { return *p; }
  __device__ static void store(float* p, const float (&v)[8]) {
    const f32x4 x = {v[0], v[1], v[2], v[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(p));
  }
  __device__ static void store_one(float* p, float v) { *p = v; }
};
template <> struct Row<unsigned short> {
  static constexpr int kPer = 8;
  template <bool CACHED = false>
  __device__ static void load(const unsigned short* p, float (&v)[8]) {
    const u16x8* const q = reinterpret_cast<const u16x8*>(p);
    const u16x8 x = CACHED ? *q : __builtin_nontemporal_load(q);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = bf16_to_f32(x[j]);
  }
  __device__ static float one(const unsigned short* p) { return bf16_to_f32(*p); }
  __device__ static void store(unsigned short* p, const float (&v)[8]) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 x = {f32x2_to_bf16(v[0], v[1]), f32x2_to_bf16(v[2], v[3]), f32x2_to_bf16(v[4], v[5]),
                     f32x2_to_bf16(v[6], v[7])};
    __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p));
  }
  __device__ static void store_one(unsigned short* p, float v) { *p = (unsigned short)f32x2_to_bf16(v, 0.f); }
};

// Running statistics of a set of logits y (log2 units): M >= every y, s = sum 2^(y-M), e = sum 2^(y-M)(y-M).
struct Stats { float M, s, e; };

constexpr float kTiny = -150.f;  // 2^-150 flushes to zero: a logit that far below the maximum (or -inf) adds nothing

// Folds N logits (natural units) at once: one rescale at most, then four arithmetic instructions and one
// exponential per logit.
template <int N>
__device__ __forceinline__ void fold(Stats& a, const float (&z)[8]) {
  float m = z[0];
#pragma unroll
  for (int j = 1; j < N; ++j) m = fmaxf(m, z[j]);
  m *= kLog2e;
  if (m > a.M) {  // rescale what is there to the new reference
    const float d = fmaxf(a.M - m, kTiny), f = __builtin_amdgcn_exp2f(d);
    a.e = f * fmaf(a.s, d, a.e);
    a.s = a.s * f;
    a.M = m;
  }
  // four independent partial sums: the additions of consecutive logits do not wait for one another
  float s4[4] = {a.s, 0.f, 0.f, 0.f}, e4[4] = {a.e, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float d = fmaxf(fmaf(z[j], kLog2e, -a.M), kTiny), f = __builtin_amdgcn_exp2f(d);
    s4[j & 3] += f;
    e4[j & 3] = fmaf(f, d, e4[j & 3]);
  }
  a.s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
  a.e = (e4[0] + e4[1]) + (e4[2] + e4[3]);
}
__device__ __forceinline__ Stats merge(Stats a, Stats b) {
  const float Mn = fmaxf(a.M, b.M);
  const float d1 = fmaxf(a.M - Mn, kTiny), d2 = fmaxf(b.M - Mn, kTiny);
  const float f1 = __builtin_amdgcn_exp2f(d1), f2 = __builtin_amdgcn_exp2f(d2);
  Stats r;
  r.M = Mn;
  r.e = f1 * fmaf(a.s, d1, a.e) + f2 * fmaf(b.s, d2, b.e);
  r.s = a.s * f1 + b.s * f2;
  return r;
}
constexpr float kFloor = -1e30f;  // below any logit; finite, so that differences stay finite

// What one workgroup does of a row: the 16-byte vectors [q_lo, q_hi) of the row's aligned middle, counted from
// element `head` on, and its share of the n_scalar elements outside it (before `head`, then behind the last vector).
// An odd vocabulary puts every row on another boundary, so a row's first vector starts at its first 16-byte boundary
// and not at its first element.
struct RowSpan {
  int head, n_vec, n_scalar, q_lo, q_hi;
  template <typename T>
  __device__ __forceinline__ RowSpan(const T* row, int vocab, bool vec_ok, int part, int parts) {
    constexpr int kPer = Row<T>::kPer;
    const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = min((kPer - off) & (kPer - 1), vocab);
    n_vec = vec_ok ? (vocab - head) / kPer : 0;
    n_scalar = vocab - n_vec * kPer;
    q_lo = (int)((int64_t)n_vec * part / parts);
    q_hi = (int)((int64_t)n_vec * (part + 1) / parts);
  }
  template <typename T>
  __device__ __forceinline__ int scalar(int i) const { return i < head ? i : i + n_vec * Row<T>::kPer; }
};

}  // namespace axon
