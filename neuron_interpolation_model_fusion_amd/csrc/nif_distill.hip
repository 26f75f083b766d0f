// nif_distill.hip -- distillation of given logits from a teacher's top logits, with its gradient, and the selection of
// the top logits themselves.  The loss is the one of nif_head.hip with the logits in memory:
//
//   u = z / tau, s[v] = exp(u[v] - lse), loss = tau^2 ( sum_k p_k (log p_k - u[at_k]) + P lse ),
//   dloss / dz[v] = tau ( P s[v] - sum_{k : at_k = v} p_k ).
//
// All of it is bound by memory: the loss reads the logits once, the gradient reads them again and writes as much.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/nif.h"
#include "nif_common.h"
#include "nif_target.h"

namespace nif {

// ---- targets ------------------------------------------------------------------------------------------------

// a label outside the classes that is not the ignored one has p = NaN: its row's loss and gradients are NaN
__global__ __launch_bounds__(256) void label_targets_kernel(const int64_t* __restrict__ labels, int64_t ignore, int64_t n, int classes,
                                                            Targets t) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t y = labels[i];
  const bool live = y != ignore, good = y >= 0 && y < classes;
  t.at[i] = !live ? -1 : good ? (int)y : 0;
  t.p[i] = !live ? 0.f : good ? 1.f : NAN;
  t.P[i] = !live ? NO_TARGET : good ? 1.f : NAN;
}

// p_k = exp(t_k / tau - L), L = lse of the teacher's row where given, else over the row's entries.  Entries of a
// negative class or of value -inf carry nothing; a class that does not exist makes the row NaN.  One wave per row.
__device__ __forceinline__ void top_targets(const int32_t* __restrict__ indices, const float* __restrict__ values,
                                            const float* __restrict__ lse, int64_t row, int classes, const Targets& t, int lane) {
  const int32_t* at = indices + row * t.k;
  const float* val = values + row * t.k;
  float top = -INFINITY;
  bool any = false;
  for (int k = lane; k < t.k; k += 64) {
    const bool have = at[k] >= 0 && val[k] != -INFINITY;
    any |= have;
    if (have) top = fmaxf(top, val[k] * t.inv_tau);
  }
  const bool live = __any(any);
  top = wave_max_f32(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int k = lane; k < t.k; k += 64)
    if (at[k] >= 0 && val[k] != -INFINITY) sum += expf(val[k] * t.inv_tau - ref);
  sum = wave_sum_f32(sum);
  const float L = lse ? lse[row] : ref + logf(sum);
  float P = 0.f;
  for (int k = lane; k < t.k; k += 64) {
    const bool have = at[k] >= 0 && val[k] != -INFINITY;
    const bool good = at[k] < classes;
    // without lse: exp(. - ref) / sum, which adds up to one to rounding
    const float e = lse ? expf(val[k] * t.inv_tau - L) : expf(val[k] * t.inv_tau - ref) / sum;
    const float p = !have ? 0.f : good ? e : NAN;
    t.at[row * t.k + k] = !have ? -1 : good ? at[k] : 0;
    t.p[row * t.k + k] = p;
    P += p;
  }
  P = wave_sum_f32(P);
  if (lane == 0) t.P[row] = live ? P : NO_TARGET;
}

__global__ __launch_bounds__(256) void top_targets_kernel(const int32_t* __restrict__ indices, const float* __restrict__ values,
                                                          const float* __restrict__ lse, int64_t n, int classes, Targets t) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row < n) top_targets(indices, values, lse, row, classes, t, threadIdx.x & 63);
}

void launch_targets(const int64_t* labels, int64_t ignore, const int32_t* indices, const float* values, const float* lse, int64_t n, int k,
                    int classes, const Targets& t, hipStream_t st) {
  (void)k;
  if (labels)
    hipLaunchKernelGGL(label_targets_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, labels, ignore, n, classes, t);
  else
    hipLaunchKernelGGL(top_targets_kernel, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, indices, values, lse, n, classes, t);
}

// ---- distillation of given logits ---------------------------------------------------------------------------

// One block per row: (max, sum of exponentials) in one pass, the targets' terms, the row's loss.
template <int DT>
__global__ __launch_bounds__(256) void distill_rows_kernel(const void* __restrict__ logits, int64_t ld, int classes, Targets t,
                                                           float* __restrict__ lse_out, float* __restrict__ loss) {
  __shared__ float sh_top[4], sh_sum[4];
  __shared__ double sh_loss[4];
  const int64_t row = blockIdx.x;
  const float P = t.P[row];
  if (P == NO_TARGET) {
    if (threadIdx.x == 0) loss[row] = 0.f, lse_out[row] = 0.f;
    return;
  }
  const typename Elem<DT>::t* z = (const typename Elem<DT>::t*)logits + row * ld;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float top = -INFINITY, sum = 0.f;
  for (int c = threadIdx.x; c < classes; c += 256) {
    const float u = (float)z[c] * t.inv_tau;
    const float m = fmaxf(top, u), ref = m == -INFINITY ? 0.f : m;
    sum = sum * expf(top - ref) + expf(u - ref);
    top = m;
  }
  const float wtop = wave_max_f32(top), ref = wtop == -INFINITY ? 0.f : wtop;
  sum = wave_sum_f32(sum * expf(top - ref));
  if (lane == 0) sh_top[wave] = wtop, sh_sum[wave] = sum;
  __syncthreads();
  top = sh_top[0], sum = sh_sum[0];
  for (int w = 1; w < 4; ++w) join(top, sum, sh_top[w], sh_sum[w]);
  const float lse = top + logf(sum);
  double s = 0.0;
  for (int k = threadIdx.x; k < t.k; k += 256) {
    const int at = t.at[row * t.k + k];
    if (at >= 0) s += target_term(t, row, k, (float)z[at] * t.inv_tau, lse);
  }
  s = wave_sum_f64(s);
  if (lane == 0) sh_loss[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    lse_out[row] = lse;
    loss[row] = (float)(((sh_loss[0] + sh_loss[1]) + (sh_loss[2] + sh_loss[3])) * t.tau2);
  }
}

__global__ __launch_bounds__(1024) void distill_reduce_kernel(const float* __restrict__ rows, const float* __restrict__ P, int64_t n,
                                                              int mean, float* __restrict__ count, float* __restrict__ loss) {
  __shared__ double sh[16];
  __shared__ int sc[16];
  double s = 0.0;
  int c = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    s += (double)rows[i];
    c += P[i] != NO_TARGET;
  }
  s = wave_sum_f64(s);
  for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s, sc[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0, c = 0;
    for (int w = 0; w < 16; ++w) s += sh[w], c += sc[w];
    *count = (float)(c > 0 ? c : 1);
    if (loss) loss[0] = (float)(mean ? s / (c > 0 ? c : 1) : s);
  }
}

// One block per row and stretch of classes.  The targets' entries are stored again after the block's other stores.
template <int DT>
__global__ __launch_bounds__(256) void distill_grad_kernel(const void* __restrict__ logits, int64_t ld, int classes, Targets t,
                                                           const float* __restrict__ lse, const float* __restrict__ grad, int per_row,
                                                           const float* __restrict__ count, void* __restrict__ out, int64_t ldo,
                                                           int stretch) {
  typedef typename Elem<DT>::t E;
  const int64_t row = blockIdx.x;
  const int c0 = blockIdx.y * stretch, c1 = min(classes, c0 + stretch);
  const E* z = (const E*)logits + row * ld;
  E* o = (E*)out + row * ldo;
  const float P = t.P[row];
  if (P == NO_TARGET) {
    for (int c = c0 + threadIdx.x; c < c1; c += 256) o[c] = (E)0.f;
    return;
  }
  const float coef = (per_row ? grad[row] : count ? grad[0] / *count : grad[0]) * t.tau, cp = coef * P, l = lse[row];
  for (int c = c0 + threadIdx.x; c < c1; c += 256) o[c] = (E)(cp * expf((float)z[c] * t.inv_tau - l));
  __syncthreads();  // the block's stores are done
  for (int k = threadIdx.x; k < t.k; k += 256) {
    const int v = t.at[row * t.k + k];
    if (v < c0 || v >= c1) continue;
    float sum = 0.f;
    bool first = true;
    for (int q = 0; q < t.k; ++q)
      if (t.at[row * t.k + q] == v) {
        first &= q >= k;
        sum += t.p[row * t.k + q];
      }
    if (first) o[v] = (E)(cp * expf((float)z[v] * t.inv_tau - l) - coef * sum);
  }
}

// ---- top logits -----------------------------------------------------------------------------------------------

// Order of logits: larger first, NaN before everything, equal values (and the two zeros) by the lower class.  Larger
// keys come first; the key of an absent entry is 0, which no class has.
__device__ __forceinline__ unsigned order_of(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned b = __float_as_uint(x + 0.f);  // -0 -> +0
  return b >> 31 ? ~b : b | 0x80000000u;
}

// One block per row, one pass per entry: the largest key below the last one.  With the log-sum-exp of the row.
template <int DT>
__global__ __launch_bounds__(256) void top_logits_kernel(const void* __restrict__ logits, int64_t ld, int classes, int k, float inv_tau,
                                                         void* __restrict__ values, int* __restrict__ indices, float* __restrict__ lse) {
  typedef typename Elem<DT>::t E;
  __shared__ unsigned long long sh_key[4];
  __shared__ float sh_top[4], sh_sum[4];
  const int64_t row = blockIdx.x;
  const E* z = (const E*)logits + row * ld;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float top = -INFINITY, sum = 0.f;
  for (int c = threadIdx.x; c < classes; c += 256) {
    const float u = (float)z[c] * inv_tau;
    const float m = fmaxf(top, u), ref = m == -INFINITY ? 0.f : m;
    sum = sum * expf(top - ref) + expf(u - ref);
    top = m;
  }
  const float wtop = wave_max_f32(top), ref = wtop == -INFINITY ? 0.f : wtop;
  sum = wave_sum_f32(sum * expf(top - ref));
  if (lane == 0) sh_top[wave] = wtop, sh_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    top = sh_top[0], sum = sh_sum[0];
    for (int w = 1; w < 4; ++w) join(top, sum, sh_top[w], sh_sum[w]);
    lse[row] = top + logf(sum);
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long best = 0;
    for (int c = threadIdx.x; c < classes; c += 256) {
      const unsigned long long key = ((unsigned long long)order_of((float)z[c]) << 32) | (0xfffffffeu - (unsigned)c);
      if (key < last && key > best) best = key;
    }
    for (int o = 32; o; o >>= 1) {
      const unsigned long long x = __shfl_xor(best, o, 64);
      best = x > best ? x : best;
    }
    __syncthreads();
    if (lane == 0) sh_key[wave] = best;
    __syncthreads();
    for (int w = 0; w < 4; ++w) best = sh_key[w] > best ? sh_key[w] : best;
    last = best;
    if (threadIdx.x == 0) {
      const int c = (int)(0xfffffffeu - (unsigned)best);
      indices[row * k + j] = c;
      ((E*)values)[row * k + j] = z[c];
    }
  }
}

static bool good_type(int dt) { return dt == NIF_F32 || dt == NIF_BF16 || dt == NIF_F16; }

struct DistillState {
  size_t p, at, P, lse, count, bytes;
};
static DistillState distill_state(int64_t n, int k) {
  DistillState s;
  size_t at = 0;
  const auto take = [&](size_t b) {
    const size_t r = at;
    at += (b + 255) / 256 * 256;
    return r;
  };
  s.p = take((size_t)n * k * 4);
  s.at = take((size_t)n * k * 4);
  s.P = take((size_t)n * 4);
  s.lse = take((size_t)n * 4);
  s.count = take(4);
  s.bytes = at;
  return s;
}

static Targets distill_targets(char* state, const DistillState& s, int k, float tau) {
  Targets t;
  t.p = (float*)(state + s.p);
  t.at = (int*)(state + s.at);
  t.P = (float*)(state + s.P);
  t.k = k;
  t.tau = tau;
  t.inv_tau = 1.f / tau;
  t.tau2 = (double)tau * tau;
  return t;
}

static bool good_distill(int64_t n, int classes, int dt, int k, float tau, int reduction) {
  return n >= 0 && n <= (1 << 30) && classes > 0 && classes <= (1 << 28) && good_type(dt) && k >= 1 && k <= NIF_TOP_MAX_K && tau > 0.f &&
         tau < INFINITY && reduction >= NIF_REDUCE_NONE && reduction <= NIF_REDUCE_SUM;
}

}  // namespace nif

extern "C" size_t nif_distill_state_bytes(int64_t rows, int top) {
  if (rows < 0 || rows > (1 << 30) || top < 1 || top > NIF_TOP_MAX_K) return 0;
  return nif::distill_state(rows, top).bytes;
}

extern "C" size_t nif_distill_workspace_bytes(int64_t rows) { return rows < 0 ? 0 : (size_t)(rows + 1) * 4; }

#define NIF_BY_TYPE(DT, CALL)                     \
  do {                                            \
    if ((DT) == NIF_F32) {                        \
      constexpr int D = NIF_F32;                  \
      CALL;                                       \
    } else if ((DT) == NIF_BF16) {                \
      constexpr int D = NIF_BF16;                 \
      CALL;                                       \
    } else {                                      \
      constexpr int D = NIF_F16;                  \
      CALL;                                       \
    }                                             \
  } while (0)

extern "C" int nif_distill_forward(const void* logits, int64_t ld, int64_t rows, int classes, int dtype, const int32_t* top_indices,
                                   const float* top_values, const float* top_lse, int top, float temperature, int reduction, float* loss,
                                   void* state, size_t state_bytes, void* ws, size_t ws_bytes, void* stream) {
  nif::Range nif_range_("nif_distill_forward");
  using namespace nif;
  if (!good_distill(rows, classes, dtype, top, temperature, reduction) || ld < classes) return NIF_ERR_INVALID_ARG;
  if (rows > 0 && (!logits || !top_indices || !top_values)) return NIF_ERR_INVALID_ARG;
  if (!loss && (rows > 0 || reduction != NIF_REDUCE_NONE)) return NIF_ERR_INVALID_ARG;
  if (!state || state_bytes < nif_distill_state_bytes(rows, top) || !ws || ws_bytes < nif_distill_workspace_bytes(rows))
    return NIF_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const DistillState s = distill_state(rows, top);
  const Targets t = distill_targets((char*)state, s, top, temperature);
  float* row_loss = reduction == NIF_REDUCE_NONE ? loss : (float*)ws;
  clear_err();
  if (rows > 0) {
    launch_targets(nullptr, 0, top_indices, top_values, top_lse, rows, top, classes, t, st);
    NIF_BY_TYPE(dtype, hipLaunchKernelGGL(distill_rows_kernel<D>, dim3((unsigned)rows), dim3(256), 0, st, logits, ld, classes, t,
                                          (float*)((char*)state + s.lse), row_loss));
  }
  hipLaunchKernelGGL(distill_reduce_kernel, dim3(1), dim3(1024), 0, st, row_loss, t.P, rows, reduction == NIF_REDUCE_MEAN,
                     (float*)((char*)state + s.count), reduction == NIF_REDUCE_NONE ? nullptr : loss);
  return launch_ok() ? NIF_OK : NIF_ERR_LAUNCH;
}

extern "C" int nif_distill_backward(const void* logits, int64_t ld, int64_t rows, int classes, int dtype, int top, float temperature,
                                    int reduction, const float* grad_loss, const void* state, size_t state_bytes, void* dlogits,
                                    int64_t ldd, void* stream) {
  nif::Range nif_range_("nif_distill_backward");
  using namespace nif;
  if (!good_distill(rows, classes, dtype, top, temperature, reduction) || ld < classes || ldd < classes) return NIF_ERR_INVALID_ARG;
  if (rows > 0 && (!logits || !grad_loss || !dlogits)) return NIF_ERR_INVALID_ARG;
  if (!state || state_bytes < nif_distill_state_bytes(rows, top)) return NIF_ERR_WORKSPACE;
  if (rows == 0) return NIF_OK;
  hipStream_t st = (hipStream_t)stream;
  const DistillState s = distill_state(rows, top);
  const Targets t = distill_targets((char*)state, s, top, temperature);
  const int stretch = 16384;
  const dim3 grid((unsigned)rows, (unsigned)((classes + stretch - 1) / stretch));
  clear_err();
  NIF_BY_TYPE(dtype, hipLaunchKernelGGL(distill_grad_kernel<D>, grid, dim3(256), 0, st, logits, ld, classes, t,
                                        (const float*)((const char*)state + s.lse), grad_loss, reduction == NIF_REDUCE_NONE,
                                        reduction == NIF_REDUCE_MEAN ? (const float*)((const char*)state + s.count) : nullptr, dlogits,
                                        ldd, stretch));
  return launch_ok() ? NIF_OK : NIF_ERR_LAUNCH;
}

extern "C" int nif_top_logits(const void* logits, int64_t ld, int64_t rows, int classes, int dtype, int top, float temperature,
                              void* values, int32_t* indices, float* lse, void* stream) {
  nif::Range nif_range_("nif_top_logits");
  using namespace nif;
  if (!good_distill(rows, classes, dtype, top, temperature, NIF_REDUCE_NONE) || top > classes || ld < classes) return NIF_ERR_INVALID_ARG;
  if (rows > 0 && (!logits || !values || !indices || !lse)) return NIF_ERR_INVALID_ARG;
  if (rows == 0) return NIF_OK;
  hipStream_t st = (hipStream_t)stream;
  clear_err();
  NIF_BY_TYPE(dtype, hipLaunchKernelGGL(top_logits_kernel<D>, dim3((unsigned)rows), dim3(256), 0, st, logits, ld, classes, top,
                                        1.f / temperature, values, indices, lse));
  return launch_ok() ? NIF_OK : NIF_ERR_LAUNCH;
}
