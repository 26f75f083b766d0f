// nif_target.h -- the sparse target distribution of a row (a label, or a teacher's top logits) and the pieces of a
// softmax that the head losses share (nif_head.hip, nif_distill.hip).
#ifndef NIF_TARGET_H_
#define NIF_TARGET_H_

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "nif_common.h"

namespace nif {

constexpr float NO_TARGET = -1.f;  // P of a row that is left out

struct Targets {
  float* p;   // [n][k] probabilities; 0 where there is no entry
  int* at;    // [n][k] classes; -1 where there is no entry
  float* P;   // [n] sum of p, or NO_TARGET
  int k;
  float tau, inv_tau;
  double tau2;
};

typedef __attribute__((ext_vector_type(4))) float vec4f;
typedef __attribute__((ext_vector_type(8))) short vec8s;

template <int DT>
struct Elem;
template <>
struct Elem<0> {  // NIF_F32
  typedef float t;
  static constexpr int PER16 = 4;
  static __device__ __forceinline__ float load(const void* p, int64_t i) { return ((const float*)p)[i]; }
  static __device__ __forceinline__ float up(float x) { return x; }
};
template <>
struct Elem<2> {  // NIF_BF16
  typedef __bf16 t;
  static constexpr int PER16 = 8;
  static __device__ __forceinline__ float load(const void* p, int64_t i) { return (float)((const __bf16*)p)[i]; }
};
template <>
struct Elem<3> {  // NIF_F16
  typedef _Float16 t;
  static constexpr int PER16 = 8;
  static __device__ __forceinline__ float load(const void* p, int64_t i) { return (float)((const _Float16*)p)[i]; }
};

// 16 bytes -> floats
template <int DT>
__device__ __forceinline__ void unpack16(vec4f raw, float (&x)[Elem<DT>::PER16]) {
  typedef typename Elem<DT>::t t;
  t v[Elem<DT>::PER16];
  __builtin_memcpy(v, &raw, 16);
#pragma unroll
  for (int e = 0; e < Elem<DT>::PER16; ++e) x[e] = (float)v[e];
}

// (max, sum of exp(. - max)) pairs: the empty one is (-inf, 0); NaN stays in the sum
__device__ __forceinline__ void join(float& top, float& sum, float t2, float s2) {
  const float m = fmaxf(top, t2), ref = m == -INFINITY ? 0.f : m;
  sum = sum * expf(top - ref) + s2 * expf(t2 - ref);
  top = m;
}

__device__ __forceinline__ float wave_max_f32(float x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  return x;
}
__device__ __forceinline__ float wave_sum_f32(float x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// a . b over d elements by one wave, in 32 bits
template <int DT>
__device__ __forceinline__ float wave_dot(const void* a, int64_t ao, const void* b, int64_t bo, int d, int lane) {
  constexpr int V = Elem<DT>::PER16;
  typedef typename Elem<DT>::t t;
  const t* pa = (const t*)a + ao;
  const t* pb = (const t*)b + bo;
  float s = 0.f;
  if ((((uintptr_t)pa | (uintptr_t)pb) & 15) == 0) {
    int c = lane * V;
    for (; c + V <= d; c += 64 * V) {
      float x[V], y[V];
      unpack16<DT>(*(const vec4f*)(pa + c), x);
      unpack16<DT>(*(const vec4f*)(pb + c), y);
#pragma unroll
      for (int e = 0; e < V; ++e) s = fmaf(x[e], y[e], s);
    }
    for (int e = 0; e < V && c + e < d; ++e) s = fmaf((float)pa[c + e], (float)pb[c + e], s);
  } else {
    for (int c = lane; c < d; c += 64) s = fmaf((float)pa[c], (float)pb[c], s);
  }
  return wave_sum_f32(s);
}

// one target's term of a row's loss / tau^2; an entry of no weight adds nothing, whatever its logit is
__device__ __forceinline__ double target_term(const Targets& t, int64_t row, int k, float u, float lse) {
  const float p = t.p[row * t.k + k];
  if (t.at[row * t.k + k] < 0 || p == 0.f) return 0.0;
  return (double)p * ((double)logf(p) - (double)u + (double)lse);
}

// Fills p, at and P of n rows from labels or from top logits (nif_distill.hip).
void launch_targets(const int64_t* labels, int64_t ignore, const int32_t* indices, const float* values, const float* lse, int64_t n, int k,
                    int classes, const Targets& t, hipStream_t st);

}  // namespace nif

#endif  // NIF_TARGET_H_
