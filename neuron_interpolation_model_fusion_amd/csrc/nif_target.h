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

// Blocks of rows: along x up to 2^21 of them (a dimension takes fewer than 2^32 threads, of which blocks have up to 1024), the
// rest along z.  The last ones may lie behind the rows.
inline dim3 row_grid(int64_t blocks, unsigned y = 1) {
  const int64_t x = blocks < (1 << 21) ? blocks : 1 << 21;
  return dim3((unsigned)x, y, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ int64_t row_block() { return (int64_t)blockIdx.z * gridDim.x + blockIdx.x; }

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

// What is subtracted before an exponential where `top` is the largest: nothing where it is infinite.
__device__ __forceinline__ float reference_of(float top) { return fabsf(top) == INFINITY ? 0.f : top; }

// (max, sum of exp((. - reference) / tau)) pairs: the empty one is (-inf, 0), one that holds +inf (+inf, +inf); NaN stays in
// the sum
__device__ __forceinline__ void join(float& top, float& sum, float t2, float s2, float inv_tau) {
  const float m = fmaxf(top, t2), ref = reference_of(m);
  sum = sum * expf((top - ref) * inv_tau) + s2 * expf((t2 - ref) * inv_tau);
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

// One target's term of a row's loss / tau^2; an entry of no weight adds nothing, whatever its logit is.  `u` is its logit's
// distance from the row's largest, over tau, `log_sum` the logarithm of the row's exponentials from there: the log-sum-exp of
// large logits in 32 bits would be off by half a step of theirs.
__device__ __forceinline__ double target_term(const Targets& t, int64_t row, int k, double u, float log_sum) {
  const float p = t.p[row * t.k + k];
  if (t.at[row * t.k + k] < 0 || p == 0.f) return 0.0;
  return (double)p * ((double)logf(p) - u + (double)log_sum);
}

// p_k = exp(t_k / tau - L), L = lse of the teacher's row where given, else over the row's entries, whose largest is subtracted
// before anything is scaled.  Entries of a
// negative class or of value -inf carry nothing; a class that does not exist makes the row NaN.  One wave per row.
__device__ __forceinline__ float top_targets(const int32_t* __restrict__ indices, const float* __restrict__ values,
                                            const float* __restrict__ lse, int64_t row, int classes, const Targets& t, int lane) {
  const int32_t* at = indices + row * t.k;
  const float* val = values + row * t.k;
  float top = -INFINITY;
  bool any = false;
  for (int k = lane; k < t.k; k += 64) {
    const bool have = at[k] >= 0 && val[k] != -INFINITY;
    any |= have;
    if (have) top = fmaxf(top, val[k]);
  }
  const bool live = __any(any);
  top = wave_max_f32(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int k = lane; k < t.k; k += 64)
    if (at[k] >= 0 && val[k] != -INFINITY) sum += expf((val[k] - ref) * t.inv_tau);
  sum = wave_sum_f32(sum);
  float P = 0.f;
  for (int k = lane; k < t.k; k += 64) {
    const bool have = at[k] >= 0 && val[k] != -INFINITY;
    const bool good = at[k] < classes;
    // without lse: exp((. - ref) / tau) / sum, which adds up to one to rounding
    const float e = lse ? expf(fmaf(val[k], t.inv_tau, -lse[row])) : expf((val[k] - ref) * t.inv_tau) / sum;
    const float p = !have ? 0.f : good ? e : NAN;
    t.at[row * t.k + k] = !have ? -1 : good ? at[k] : 0;
    t.p[row * t.k + k] = p;
    P += p;
  }
  P = wave_sum_f32(P);
  P = live ? P : NO_TARGET;
  if (lane == 0) t.P[row] = P;
  return P;
}

// a label outside the classes that is not the ignored one has p = NaN: its row's loss and gradients are NaN
__device__ __forceinline__ void label_target(int64_t y, int64_t ignore, int classes, float& p, int& at, float& P) {
  const bool live = y != ignore, good = y >= 0 && y < classes;
  at = !live ? -1 : good ? (int)y : 0;
  p = !live ? 0.f : good ? 1.f : NAN;
  P = !live ? NO_TARGET : p;
}

// Fills p, at and P of n rows from top logits (nif_distill.hip).
void launch_targets(const int32_t* indices, const float* values, const float* lse, int64_t n, int classes, const Targets& t, hipStream_t st);

// loss = sum or mean of the rows' losses over the rows that count; count = their number, at least 1 (nif_distill.hip).
void launch_reduce(const float* row_loss, const float* P, int64_t n, bool mean, float* count, float* loss, hipStream_t st);

}  // namespace nif

#endif  // NIF_TARGET_H_
