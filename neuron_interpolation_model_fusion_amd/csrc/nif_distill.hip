// nif_distill.hip -- distillation of given logits from a teacher's top logits, with its gradient, and the selection of
// the top logits themselves.  The loss is the one of nif_head.hip with the logits in memory:
//
//   u = z / tau, s[v] = exp(u[v] - lse), loss = tau^2 ( sum_k p_k (log p_k - u[at_k]) + P lse ),
//   dloss / dz[v] = tau ( P s[v] - sum_{k : at_k = v} p_k ).
//
// A row's log-sum-exp stays in two parts, its largest logit and the sum of the exponentials from there: s[v] is exp((z[v] -
// top) / tau) / sum, as exact for logits of a thousand as for small ones.
// All of it is bound by memory: the loss reads the logits once, the gradient reads them again and writes as much.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/nif.h"
#include "nif_common.h"
#include "nif_target.h"

namespace nif {

// ---- targets ------------------------------------------------------------------------------------------------

__global__ __launch_bounds__(256) void top_targets_kernel(const int32_t* __restrict__ indices, const float* __restrict__ values,
                                                          const float* __restrict__ lse, int64_t n, int classes, Targets t) {
  const int64_t row = row_block() * 4 + (threadIdx.x >> 6);
  if (row < n) top_targets(indices, values, lse, row, classes, t, threadIdx.x & 63);
}

void launch_targets(const int32_t* indices, const float* values, const float* lse, int64_t n, int classes, const Targets& t, hipStream_t st) {
  hipLaunchKernelGGL(top_targets_kernel, row_grid((n + 3) / 4), dim3(256), 0, st, indices, values, lse, n, classes, t);
}

// ---- distillation of given logits ---------------------------------------------------------------------------

// A row as 16-byte vectors: [0, head) and [tail, n) are the elements before the first and behind the last whole one.
template <int DT>
struct RowView {
  const typename Elem<DT>::t* z;
  int n, head, vecs;
  __device__ __forceinline__ RowView(const void* base, int64_t at, int classes) {
    constexpr int V = Elem<DT>::PER16;
    z = (const typename Elem<DT>::t*)base + at;
    n = classes;
    head = min(n, (int)((16 - ((uintptr_t)z & 15)) & 15) / (16 / V));
    vecs = (n - head) / V;
  }
  __device__ __forceinline__ int tail() const { return head + vecs * Elem<DT>::PER16; }
  __device__ __forceinline__ vec4f vec(int i) const { return ((const vec4f*)(z + head))[i]; }
  // loose element j = 0 .. loose() - 1: the head's, then the tail's
  __device__ __forceinline__ int loose() const { return head + (n - tail()); }
  __device__ __forceinline__ int loose_at(int j) const { return j < head ? j : tail() + (j - head); }
};

// 2^x. 16-bit inputs: the hardware's (2^-22 relative); f32: the library's exponential of the natural argument.
template <int DT>
__device__ __forceinline__ float exp_of(float x) {
  return DT == NIF_F32 ? expf(x) : __builtin_amdgcn_exp2f(x);
}
// what differences of logits are multiplied with before exp_of: 1 / tau, and log2(e) where the hardware's exponential is used
template <int DT>
__device__ __forceinline__ float exp_scale(float inv_tau) {
  return DT == NIF_F32 ? inv_tau : inv_tau * 1.4426950408889634f;
}

// Running (maximum, sum of exponentials): one rescaling per batch of elements.  The maximum is subtracted before anything is
// scaled: a type's lowest value, the mask of a class, is finite, its product with log2(e) or 1 / tau need not be.
template <int DT>
struct Running {
  float top, sum;  // top in the logits' own units
  __device__ __forceinline__ void init() { top = -INFINITY, sum = 0.f; }
  template <int N>
  __device__ __forceinline__ float add(const float (&x)[N], float scale) {  // returns the batch's maximum
    float m = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) m = fmaxf(m, x[e]);
    const float now = fmaxf(top, m), ref = reference_of(now);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) s += exp_of<DT>((x[e] - ref) * scale);
    sum = sum * exp_of<DT>((top - ref) * scale) + s;
    top = now;
    return m;
  }
  // the block's; every thread gets them.  sh: 2 * waves floats
  template <int NT>
  __device__ __forceinline__ void join_block(float scale, float inv_tau, float* sh) {
    const float wtop = wave_max_f32(top), ref = reference_of(wtop);
    const float wsum = wave_sum_f32(sum * exp_of<DT>((top - ref) * scale));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) sh[2 * wave] = wtop, sh[2 * wave + 1] = wsum;
    __syncthreads();
    top = sh[0], sum = sh[1];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) join(top, sum, sh[2 * w], sh[2 * w + 1], inv_tau);
  }
};

// Streams a row through `f(x[batch], first element's column or -1 for the row's loose ends, vector of elements e ->
// column + e)` in batches of U vectors a thread; the next batch's loads are in flight while one is worked on.
template <int DT, int NT, int U, class F>
__device__ __forceinline__ void stream_row(const RowView<DT>& r, F&& f) {
  constexpr int V = Elem<DT>::PER16;
  vec4f next[U];
  const auto fetch = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + u * NT + (int)threadIdx.x;
      if (i < r.vecs) next[u] = r.vec(i);
    }
  };
  fetch(0);
  for (int base = 0; base < r.vecs; base += U * NT) {
    vec4f raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    fetch(base + U * NT);
    float x[U * V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float y[V];
      unpack16<DT>(raw[u], y);
      const bool have = base + u * NT + (int)threadIdx.x < r.vecs;
#pragma unroll
      for (int e = 0; e < V; ++e) x[u * V + e] = have ? y[e] : -INFINITY;
    }
    f(x, base);
  }
}

// One block per row: the targets' probabilities, (max, sum of exponentials) in one pass over the logits, the targets'
// terms and the row's loss.  Bound by the read of the logits: 4096 x 131072 bf16 in 206 us, 5.2 TB/s.
template <int DT, int NT>
__global__ __launch_bounds__(NT) void distill_rows_kernel(const void* __restrict__ logits, int64_t ld, int64_t n, int classes, Targets t,
                                                          const int32_t* __restrict__ indices, const float* __restrict__ values,
                                                          const float* __restrict__ top_lse, float* __restrict__ top_out,
                                                          float* __restrict__ sum_out, float* __restrict__ loss) {
  __shared__ float sh[2 * NT / 64], sh_P;
  __shared__ double sh_loss[NT / 64];
  const int64_t row = row_block();
  if (row >= n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave == 0) {
    const float P = top_targets(indices, values, top_lse, row, classes, t, lane);
    if (lane == 0) sh_P = P;
  }
  __syncthreads();
  if (sh_P == NO_TARGET) {
    if (threadIdx.x == 0) loss[row] = 0.f, top_out[row] = 0.f, sum_out[row] = 1.f;
    return;
  }
  const RowView<DT> r(logits, row * ld, classes);
  const float scale = exp_scale<DT>(t.inv_tau);
  Running<DT> run;
  run.init();
  if ((int)threadIdx.x < r.loose()) {
    const float x[1] = {(float)r.z[r.loose_at(threadIdx.x)]};
    run.add(x, scale);
  }
  constexpr int U = DT == NIF_F32 ? 4 : 2;
  stream_row<DT, NT, U>(r, [&](const float (&x)[U * Elem<DT>::PER16], int) { run.add(x, scale); });
  run.template join_block<NT>(scale, t.inv_tau, sh);
  const float top = run.top, sum = top == INFINITY ? NAN : run.sum, log_sum = logf(sum);  // no softmax of infinite logits
  double s = 0.0;
  for (int k = threadIdx.x; k < t.k; k += NT) {
    const int at = t.at[row * t.k + k];
    if (at >= 0) s += target_term(t, row, k, ((double)(float)r.z[at] - (double)top) * (double)t.inv_tau, log_sum);
  }
  s = wave_sum_f64(s);
  if (lane == 0) sh_loss[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < NT / 64; ++w) s += sh_loss[w];
    top_out[row] = top;
    sum_out[row] = sum;
    loss[row] = (float)(s * t.tau2);
  }
}

// sum or mean over the rows that count, in a fixed order and 64 bits; rows without a target hold 0
__global__ __launch_bounds__(1024) void reduce_rows_kernel(const float* __restrict__ rows, const float* __restrict__ P, int64_t n,
                                                              int mean, float* __restrict__ count, float* __restrict__ loss) {
  __shared__ double sh[16];
  __shared__ int sc[16];
  double s = 0.0;
  int c = 0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    s += (double)rows[i];
    c += P[i] != NO_TARGET;
  }
  s = wave_sum_f64(s);
  for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s, sc[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0, c = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) s += sh[w], c += sc[w];
    if (count) *count = (float)(c > 0 ? c : 1);
    loss[0] = (float)(mean ? s / (c > 0 ? c : 1) : s);
  }
}

void launch_reduce(const float* row_loss, const float* P, int64_t n, bool mean, float* count, float* loss, hipStream_t st) {
  hipLaunchKernelGGL(reduce_rows_kernel, dim3(1), dim3(n <= 4096 ? 256 : 1024), 0, st, row_loss, P, n, mean, count, loss);
}

// One block per row and stretch of classes, the rows in reverse: the last ones read by the loss are the likeliest to be
// in the cache still.  The targets' entries are stored again after the block's other stores.  Bound by memory: 16-byte
// loads and stores, also where the row starts off a 16-byte border (the output's rows then start alike, or go by element);
// 4096 x 131072 bf16 in 418 us, 5.1 TB/s of both; 777 x 50001 f16 in 29 us.
template <int DT>
__global__ __launch_bounds__(256) void distill_grad_kernel(const void* __restrict__ logits, int64_t ld, int64_t n, int classes, Targets t,
                                                           const float* __restrict__ tops, const float* __restrict__ sums,
                                                           const float* __restrict__ grad, int per_row,
                                                           const float* __restrict__ count, void* __restrict__ out, int64_t ldo,
                                                           int stretch) {
  typedef typename Elem<DT>::t E;
  constexpr int V = Elem<DT>::PER16, U = 4;
  const int64_t row = n - 1 - row_block();
  if (row < 0) return;
  const RowView<DT> r(logits, row * ld, classes);
  E* o = (E*)out + row * ldo;
  const float P = t.P[row];
  const bool live = P != NO_TARGET;
  const float coef = live ? (per_row ? grad[row] : count ? grad[0] / *count : grad[0]) * t.tau : 0.f;
  const float cp = live ? coef * P / sums[row] : 0.f, top = tops[row], scale = exp_scale<DT>(t.inv_tau);
  const auto dz = [&](float x) { return live ? cp * exp_of<DT>((x - top) * scale) : 0.f; };
  int c0, c1;  // this block's columns
  if (((uintptr_t)r.z & 15) == ((uintptr_t)o & 15)) {
    const int v0 = min(r.vecs, (int)blockIdx.y * (stretch / V)), v1 = min(r.vecs, v0 + stretch / V);
    vec4f* ov = (vec4f*)(o + r.head);
    const auto one = [&](vec4f raw) {
      float x[V];
      unpack16<DT>(raw, x);
      E y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = (E)dz(x[e]);
      vec4f w;
      __builtin_memcpy(&w, y, 16);
      return w;
    };
    int i = v0 + threadIdx.x;
    for (; i + (U - 1) * 256 < v1; i += U * 256) {
      vec4f raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = r.vec(i + u * 256);
#pragma unroll
      for (int u = 0; u < U; ++u) __builtin_nontemporal_store(one(raw[u]), ov + i + u * 256);
    }
    for (; i < v1; i += 256) ov[i] = one(r.vec(i));
    c0 = r.head + v0 * V, c1 = r.head + v1 * V;
    if (blockIdx.y == 0) {
      c0 = 0;
      if ((int)threadIdx.x < r.head) o[threadIdx.x] = (E)dz((float)r.z[threadIdx.x]);
    }
    if (blockIdx.y == gridDim.y - 1) {
      c1 = classes;
      if (r.tail() + (int)threadIdx.x < classes) o[r.tail() + threadIdx.x] = (E)dz((float)r.z[r.tail() + threadIdx.x]);
    }
  } else {
    c0 = blockIdx.y * stretch, c1 = blockIdx.y == gridDim.y - 1 ? classes : min(classes, c0 + stretch);
    for (int c = c0 + threadIdx.x; c < c1; c += 256) o[c] = (E)dz((float)r.z[c]);
  }
  if (!live) return;
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
    if (first) o[v] = (E)(dz((float)r.z[v]) - coef * sum);
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

__device__ __forceinline__ unsigned long long key_of(float x, int c) {
  return ((unsigned long long)order_of(x) << 32) | (0xfffffffeu - (unsigned)c);
}

// n keys (a power of two) in descending order
template <int NT>
__device__ __forceinline__ void sort_keys(unsigned long long* key, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += NT) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const unsigned long long a = key[lo], b = key[hi];
        if ((a < b) == ((lo & size) == 0)) key[lo] = b, key[hi] = a;
      }
    }
  __syncthreads();
}

// The k-th largest of the block's NT values (1 <= k <= NT), one a thread: sorted with wave shuffles, the three or more
// steps wider than a wave through LDS.
template <int NT>
__device__ __forceinline__ float kth_largest(float x, int k, float* sh) {
  for (int size = 2; size <= NT; size <<= 1)
    for (int step = size >> 1; step; step >>= 1) {
      float y;
      if (step >= 64) {
        __syncthreads();
        sh[threadIdx.x] = x;
        __syncthreads();
        y = sh[threadIdx.x ^ step];
      } else {
        y = __shfl_xor(x, step, 64);
      }
      const bool want_max = ((threadIdx.x & step) == 0) == ((threadIdx.x & size) == 0);
      x = want_max ? fmaxf(x, y) : fminf(x, y);
    }
  __syncthreads();
  sh[threadIdx.x] = x;
  __syncthreads();
  x = sh[k - 1];
  __syncthreads();
  return x;
}

constexpr int TOP_LIST = 8;  // keys a thread in the list

// Any row: the k-th largest order by four passes of eight bits each, then everything above it and the first of its
// equals by class.  `key` ends with the k entries, unordered beyond that.
template <int DT, int NT>
__device__ __forceinline__ void select_by_digits(const typename Elem<DT>::t* z, int classes, int k, unsigned long long* key, unsigned* hist,
                                                 int* sh_n) {
  unsigned prefix = 0, mask = 0;
  int need = k;  // entries still wanted among those that match the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += NT) hist[i] = 0;
    __syncthreads();
    for (int c = threadIdx.x; c < classes; c += NT) {
      const unsigned o = order_of((float)z[c]);
      if ((o & mask) == prefix) atomicAdd(&hist[o >> shift & 255], 1u);
    }
    __syncthreads();
    int d = 255, left = need;
    while (d > 0 && (int)hist[d] < left) left -= (int)hist[d--];
    need = left;
    prefix |= (unsigned)d << shift;
    mask |= 255u << shift;
    __syncthreads();
  }
  if (threadIdx.x == 0) *sh_n = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int taken = 0;  // equals before this stretch
  for (int c0 = 0; c0 < classes; c0 += NT) {
    const int c = c0 + threadIdx.x;
    const unsigned o = c < classes ? order_of((float)z[c]) : 0u;
    const bool equal = c < classes && o == prefix;
    const unsigned long long m = __ballot(equal);
    if (lane == 0) hist[wave] = __popcll(m);
    __syncthreads();
    int before = taken + __popcll(m & ((1ull << lane) - 1)), all = 0;
    for (int w = 0; w < NT / 64; ++w) {
      if (w < wave) before += hist[w];
      all += hist[w];
    }
    if ((c < classes && o > prefix) || (equal && before < need)) key[atomicAdd(sh_n, 1)] = ((unsigned long long)o << 32) | (0xfffffffeu - (unsigned)c);
    taken += all;
    __syncthreads();
  }
}

// One block per row, one pass over it.  The k-th largest of the threads' maxima so far is a bar that k elements reach, so
// whatever comes later must exceed it; it is taken anew after 1, 2, 4, 8, .. stretches, which leaves about 6 k elements
// of a row of 131072 (k log2 of the stretches) in a list in LDS.  The last bar cuts the list to little more than k, which are sorted.  Rows that
// this does not fit (more than the list holds: ties at the bar, rising rows; NaN) are selected by digits instead.  The
// log-sum-exp goes along.  Bound by the read of the logits and the exponentials: 4096 x 131072 bf16, k = 64, in 237 us,
// 4.5 TB/s; 400 x 1000 f32 in 12 us, a launch's latency.
template <int DT, int NT>
__global__ __launch_bounds__(NT, 8) void top_logits_kernel(const void* __restrict__ logits, int64_t ld, int64_t rows, int classes, int k, float inv_tau,
                                                        void* __restrict__ values, int* __restrict__ indices, float* __restrict__ lse) {
  typedef typename Elem<DT>::t E;
  constexpr int V = Elem<DT>::PER16, U = DT == NIF_F32 ? 4 : 2;
  constexpr int LIST = TOP_LIST * NT;
  __shared__ unsigned long long key[LIST];
  __shared__ float sh[NT];
  __shared__ int sh_n;
  const int64_t row = row_block();
  if (row >= rows) return;
  const RowView<DT> r(logits, row * ld, classes);
  const float scale = exp_scale<DT>(inv_tau);
  if (threadIdx.x == 0) sh_n = 0;
  __syncthreads();
  Running<DT> run;
  run.init();
  const auto put = [&](float x, int c) {
    const int at = atomicAdd(&sh_n, 1);
    if (at < LIST) key[at] = key_of(x, c);
  };
  if ((int)threadIdx.x < r.loose()) {
    const float x[1] = {(float)r.z[r.loose_at(threadIdx.x)]};
    run.add(x, scale);
  }
  // more entries than threads: no bar, such rows are selected by digits and this pass makes the log-sum-exp only
  float bar = k <= NT ? -INFINITY : INFINITY, mine = -INFINITY;
  int stretch = 0;
  stream_row<DT, NT, U>(r, [&](const float (&x)[U * V], int base) {
    const float m = run.add(x, scale);
    mine = fmaxf(mine, m);
    const bool anew = k <= NT && (stretch & (stretch + 1)) == 0;
    if (anew) bar = kth_largest<NT>(mine, k, sh);
    // elements of this stretch may be among the k that reach a new bar; those behind it must exceed it
    if (anew ? m >= bar : m > bar) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        int i = base + u * NT + (int)threadIdx.x;
        asm volatile("" : "+v"(i));  // of this rare path alone: shared with the loads it costs registers that they spill
#pragma unroll
        for (int e = 0; e < V; ++e)
          if ((anew ? x[u * V + e] >= bar : x[u * V + e] > bar) && i < r.vecs) put(x[u * V + e], r.head + i * V + e);
      }
    }
    ++stretch;
  });
  run.template join_block<NT>(scale, inv_tau, sh);
  const float l = run.top * inv_tau + logf(run.sum);
  __syncthreads();
  if (threadIdx.x == 0) lse[row] = l;
  // the row's loose ends (fewer than 16), whatever they are
  if ((int)threadIdx.x < r.loose()) put((float)r.z[r.loose_at(threadIdx.x)], r.loose_at(threadIdx.x));
  if (k <= NT && stretch > 0) bar = kth_largest<NT>(mine, k, sh);
  __syncthreads();
  int n = sh_n;
  if (k > NT || n > LIST || !(l < INFINITY) || n < k) {  // l is NaN where the row holds NaN, which floats do not order
    __syncthreads();
    select_by_digits<DT, NT>(r.z, classes, k, key, (unsigned*)sh, &sh_n);
    n = k;
  } else if (n > 2 * k) {
    unsigned long long mykeys[TOP_LIST];
    const unsigned long long least = (unsigned long long)order_of(bar) << 32;
#pragma unroll
    for (int q = 0; q < TOP_LIST; ++q) {
      const int at = q * NT + threadIdx.x;
      mykeys[q] = at < n ? key[at] : 0;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh_n = 0;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < TOP_LIST; ++q)
      if (q * NT < n && mykeys[q] > least) key[atomicAdd(&sh_n, 1)] = mykeys[q];  // no key is `least` itself: classes end below
    __syncthreads();
    n = sh_n;
  }
  int p = 64;
  while (p < n) p <<= 1;
  for (int i = n + threadIdx.x; i < p; i += NT) key[i] = 0;
  sort_keys<NT>(key, p);
  for (int j = threadIdx.x; j < k; j += NT) {
    const int c = (int)(0xfffffffeu - (unsigned)key[j]);
    indices[row * k + j] = c;
    ((E*)values)[row * k + j] = r.z[c];
  }
}

static bool good_type(int dt) { return dt == NIF_F32 || dt == NIF_BF16 || dt == NIF_F16; }

struct DistillState {
  size_t p, at, P, top, sum, count, bytes;
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
  s.top = take((size_t)n * 4);
  s.sum = take((size_t)n * 4);
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
    // blocks of 512 where rows are few and long (256 x 131072 f32: 28 us to 34; 777 x 50001 f16: 26 to 21, with 1024 threads 38)
    if (rows <= 256 && (int64_t)classes * (dtype == NIF_F32 ? 4 : 2) >= 96 << 10)
      NIF_BY_TYPE(dtype, hipLaunchKernelGGL((distill_rows_kernel<D, 512>), row_grid(rows), dim3(512), 0, st, logits, ld, rows, classes,
                                            t, top_indices, top_values, top_lse, (float*)((char*)state + s.top), (float*)((char*)state + s.sum), row_loss));
    else
      NIF_BY_TYPE(dtype, hipLaunchKernelGGL((distill_rows_kernel<D, 256>), row_grid(rows), dim3(256), 0, st, logits, ld, rows, classes, t,
                                            top_indices, top_values, top_lse, (float*)((char*)state + s.top), (float*)((char*)state + s.sum), row_loss));
  }
  if (reduction != NIF_REDUCE_NONE)
    launch_reduce(row_loss, t.P, rows, reduction == NIF_REDUCE_MEAN, (float*)((char*)state + s.count), loss, st);
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
  const dim3 grid = row_grid(rows, (unsigned)((classes + stretch - 1) / stretch));
  clear_err();
  NIF_BY_TYPE(dtype, hipLaunchKernelGGL(distill_grad_kernel<D>, grid, dim3(256), 0, st, logits, ld, rows, classes, t,
                                        (const float*)((const char*)state + s.top), (const float*)((const char*)state + s.sum), grad_loss, reduction == NIF_REDUCE_NONE,
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
  // Threads a row.  The bar is of use for k up to three quarters of them (2048 x 50001 bf16, k = 500: 328 us with 1024 threads,
  // 685 with 512; k = 300: 152 with 512, 565 by digits with 256), and the list of 512 holds enough for more entries of long rows
  // (2048 x 131072, k = 200: 233 us, 837 with 256; but 4096 rows, k = 160: 406, 315).  Wider blocks also where rows are few and entries are not
  // (64 x 131072 bf16, k = 128: 67 us with 512, 78 with 256; k = 10: 52, 47), else not (2048 x 131072 f32, k = 20: 284 us with
  // 512, 233 with 256; 2048 x 50001 bf16: 117, 72); rows over 1 MiB are as wide as the longest measured ones need.  Many of
  // short rows are selected by digits at once (2048 x 3000, k = 700: 108 us with 256 threads, 309 with 1024), and so are over
  // three quarters of 1024 (2048 x 50001, k = 1024: 584 us with 256 threads, 951 with 1024; 400 rows: 437 and 257).
  const int64_t bytes = (int64_t)classes * (dtype == NIF_F32 ? 4 : 2);
  const bool few = bytes >= 192 << 10 && (rows <= 256 ? top >= 64 : rows <= 512 && top > 128);
  const bool wide = top > 192 || (top > 160 && bytes >= 512 << 10) || few || bytes > 1 << 20;
  if (top > 384 && classes >= 8192 && (top <= 768 || rows < 1024))
    NIF_BY_TYPE(dtype, hipLaunchKernelGGL((top_logits_kernel<D, 1024>), row_grid(rows), dim3(1024), 0, st, logits, ld, rows, classes, top,
                                          1.f / temperature, values, indices, lse));
  else if (wide && top <= 384)
    NIF_BY_TYPE(dtype, hipLaunchKernelGGL((top_logits_kernel<D, 512>), row_grid(rows), dim3(512), 0, st, logits, ld, rows, classes, top,
                                          1.f / temperature, values, indices, lse));
  else
    NIF_BY_TYPE(dtype, hipLaunchKernelGGL((top_logits_kernel<D, 256>), row_grid(rows), dim3(256), 0, st, logits, ld, rows, classes, top,
                                          1.f / temperature, values, indices, lse));
  return launch_ok() ? NIF_OK : NIF_ERR_LAUNCH;
}
