// nif_head.hip -- losses of a linear head over many classes, computed without keeping its logits: softmax cross
// entropy against labels, and distillation from a teacher's top logits, each with its gradients.
//
//   z[n][v] = hidden[n] . weight[v] + bias[v],   u = z / tau,   s[n][v] = exp(u[n][v] - lse[n]),
//   loss[n] = tau^2 ( sum_k p[n][k] (log p[n][k] - u[n][at(n,k)]) + P[n] lse[n] ),   P[n] = sum_k p[n][k],
//   dloss[n] / dz[n][v] = tau ( P[n] s[n][v] - sum_{k : at(n,k) = v} p[n][k] ).
//
// Cross entropy is the case of one target k with p = 1 and tau = 1, so both share every kernel.  A row without a
// target (ignored label, padding) is left out: the rows that count are packed to the front (`rows`, `count` on the
// device), and tiles behind them end at once -- such rows cost nothing and nothing in them reaches a result.
//
// A row's log-sum-exp stays in two parts, its largest logit and the sum of the exponentials from there: s is
// exp((z - top) / tau) / sum, with differences of logits only.
//
// Forward: one matrix product whose epilogue reduces each tile of u to (maximum, sum of exponentials) per row; the
// logits never leave registers.  Backward, in pieces of the classes: the product again, its epilogue writing
// dz = coef * (P s) in 16 bits; the targets' entries are then rewritten with their -p; dW of the piece = dz^T hidden,
// and dhidden += dz W.  Recomputing costs 8 n d v operations in place of 6 and saves n * v logits.
//
// Up to 64 rows of 16 bits dz is written in two 16-bit parts, the second behind the first's rows (`Plan::two`): what the
// rounding of a few rows takes off does not average out.
//
// For few rows, where the product is bound by the weight's bytes or has too few tiles, up to 64 MiB of logits are kept in
// 32 bits instead (head_kept_kernel).
//
// 16-bit inputs run on v_mfma_f32_16x16x32 with 32-bit accumulation (head_gemm_kernel).  f32 inputs are split exactly into
// three bf16 planes (x = h + m + l, 24 bits) on their way into LDS and a product runs as the six plane pairs above 2^-24:
// f32-level accuracy (head_gemm_any_kernel, which also takes 16-bit weights whose rows are off 16-byte borders).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/nif.h"
#include "nif_common.h"
#include "nif_target.h"

namespace nif {

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// The matrix instructions are written out so that the accumulators stay where they are, in accumulation registers: left
// to itself the compiler moves them through spare vector registers, of which a 256 x 256 tile leaves none.  Volatile, so
// that they keep their order against the loads between them; mfma_done() before the results are read.
struct Bf16 {
  typedef __bf16 t;
  static constexpr bool WIDE = false;
  static __device__ __forceinline__ void mfma(f32x4& c, s16x8 a, s16x8 b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
};
struct F32 {  // products as three bf16 planes; accumulators among the other registers, of which the tiles leave enough
  typedef float t;
  static constexpr bool WIDE = true;
  static __device__ __forceinline__ void mfma(f32x4& c, s16x8 a, s16x8 b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  }
};
struct F16 {
  typedef _Float16 t;
  static constexpr bool WIDE = false;
  static __device__ __forceinline__ void mfma(f32x4& c, s16x8 a, s16x8 b) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
};
// the compiler does not know that the results take a few cycles more
template <class T, int FI, int FJ>
__device__ __forceinline__ void mfma_done(f32x4 (&acc)[FI][FJ]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      if constexpr (T::WIDE)
        asm volatile("" : "+v"(acc[i][j]));
      else
        asm volatile("" : "+a"(acc[i][j]));
    }
}

template <class T>
__device__ __forceinline__ short to16(float x) {
  return __builtin_bit_cast(short, (typename T::t)x);  // round to nearest even
}

// 16-bit types: 2^x by the hardware (2^-22 relative); f32: the library's e^x.  x: a difference of logits times 1 / tau in that
// unit -- the difference first, since a type's lowest value times log2(e) or 1 / tau is infinite.
template <class T>
__device__ __forceinline__ float head_exp(float x) {
  return T::WIDE ? expf(x) : __builtin_amdgcn_exp2f(x);
}

constexpr int K_PAD = 64;      // packed operands hold zeros up to a multiple of this along the contraction
constexpr int DZ_PAD = 128;    // rows of dz
constexpr int HEAD_PAD = 256;  // packed rows are padded to a multiple of the largest tile

// One side of a product.  Plain side: element (r, k) at base[r * ld + k]; transposed side: base[k * ld + r].  Rows behind
// rlim are read as the last one (their results are not stored).  16 bits: so are k behind klim, where the other side,
// which is always a packed one, holds zeros up to the next multiple of K_PAD.
struct Side {
  const void* base;  // 16 bits or f32
  int64_t ld;
  int rlim;          // 16 bits, transposed: a multiple of 8
  int klim;          // 16 bits, plain: a multiple of 8
};

enum { EPI_STATS = 0, EPI_DZ = 1, EPI_OUT = 2 };
enum { OUT_F32 = 0, OUT_ADD = 1, OUT_FINAL = 2 };

struct GemmArgs {
  Side A, B;
  int M, N;             // extents that are computed (N: at most *n_dev when given)
  const int* n_dev;
  int K;                // contraction length (at most *k_dev when given)
  const int* k_dev;
  int two;              // not 0: the second part of dz lies so many rows behind the first, and K (if *k_dev is not 0) covers both
  int mt, nt, splits;
  int first, tiles;     // of this launch's, and all of them (tiles x splits)
  // EPI_STATS / EPI_DZ: the logit's last steps
  const void* bias;     // of the first class of the piece; f32 or the 16-bit type
  float inv_tau;
  float2* stats;        // [m tile * waves in m][stat_ld]
  int64_t stat_ld;
  const float* top;     // the largest logit of each packed row
  const float* cp;      // coef * P / (the row's sum of exponentials from there)
  void* dz;             // [rows][ldz], 16 bits or f32
  int64_t ldz;
  // EPI_OUT
  int out_kind;
  float* acc;           // OUT_F32 / OUT_ADD target, [split][n][acc_ld]; OUT_FINAL: added when not null
  int64_t acc_ld, acc_split;
  void* out;
  int64_t out_ld;
  const int* rowmap;    // packed row -> row of out
  const float* inv_scale;
};

// blockIdx -> split and tile: blocks b and b + 8 share an XCD (and its L2), so each XCD takes a contiguous range of ids --
// with eight splits, a stretch of the contraction of its own.  Inside, tiles go in groups of 8 along n for each step along
// m, so that the blocks in flight on an XCD share their panels.
__device__ __forceinline__ void tile_of(int id, int total, int mt, int nt, int& split, int& tm, int& tn) {
  const int q = total >> 3, rr = total & 7, xcd = id & 7;
  int wg = (xcd < rr ? xcd * (q + 1) : rr * (q + 1) + (xcd - rr) * q) + (id >> 3);
  split = wg / (mt * nt);
  wg -= split * mt * nt;
  const int G = 8;
  const int group = wg / (G * mt), first = group * G;
  const int width = min(G, nt - first);
  const int in = wg - group * G * mt;
  tm = in / width;
  tn = first + in % width;
}

// Copies a 32-deep tile of one side into LDS with direct 16-byte loads.  Plain: [BT rows][4 units of 16 bytes], unit u of
// row r at u ^ row_swizzle(r / 4) (r / 8: EIGHT): 16-byte reads go 16 lanes at a time, lanes 0-3, 12-15, 20-23, 24-27 together, then 4-11,
// 16-19, 28-31, and so on (u ^ (r >> 2 & 3) measured two cycles for one).  Transposed: [32 k][BT / 8 units], pairs of units xor-ed with (k & 3) | (k >> 3 & 1) << 2.
// Both keep the fragment reads free of bank conflicts.
constexpr int BK = 32;
constexpr int64_t HEAD_MAX_LD = 1 << 20;

__device__ __forceinline__ int row_swizzle(int row) { return 0x78 >> (row & 3) * 2 & 3; }  // 0, 2, 3, 1

__device__ __forceinline__ unsigned lds_offset(const void* p) {
  return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}

// Direct loads into LDS, 16 bytes a lane, lane i to dst + 16 i.  In assembly because the compiler, which cannot tell the
// stages apart, would have every LDS read wait for all of them; step_barrier waits instead.  They write no register.
__device__ __forceinline__ void load_lds16(const void* base, unsigned off, unsigned dst, unsigned more) {
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3" ::"s"(dst), "i"(more), "v"(off), "s"(base)
               : "memory", "scc");
}
// EIGHT: the fragments of a plain side take their 16 rows as 4 of each 8, two fragments sharing 32 rows, so that a lane's
// results of such a pair are eight neighbours.
template <int BT, int NW, bool TR, bool EIGHT>
struct Stager {
  static constexpr int PIECES = BT / 16;                          // of 1 KiB
  static constexpr int CW = PIECES > NW ? PIECES / NW : 1;        // pieces per wave (some twice where waves outnumber them)
  static constexpr int U = BT / 8;
  const char* base;    // of the tile at k = 0 (the same for every lane)
  unsigned piece[CW];  // where this wave's pieces go in the first stage (LDS bytes)
  unsigned off[CW];    // bytes from there to this lane's 16, 32 bits (leading dimensions are at most HEAD_MAX_LD)
  int k_of[CW];        // the (first) k of those
  __device__ __forceinline__ void init(const Side& s, int r0, const void* lds, int wave, int lane) {
    base = (const char*)s.base + (TR ? 0 : (int64_t)r0 * s.ld * 2);
#pragma unroll
    for (int q = 0; q < CW; ++q) {
      const int c = (wave * CW + q) % PIECES;
      piece[q] = lds_offset(lds) + c * 1024;
      if (!TR) {
        const int row = 16 * c + (lane >> 2);
        k_of[q] = ((lane & 3) ^ row_swizzle(row >> (EIGHT ? 3 : 2))) * 8;
        off[q] = (unsigned)min(row, s.rlim - 1 - r0) * (unsigned)s.ld * 2 + k_of[q] * 2;
      } else {
        const int k = c * (64 / U) + lane / U, d = lane % U;
        const int f = ((k & 3) | ((k >> 3 & 1) << 2)) & (U / 2 - 1);
        k_of[q] = k;
        off[q] = (unsigned)k * (unsigned)s.ld * 2 + (unsigned)min(r0 / 8 + (d ^ (f << 1)), s.rlim / 8 - 1) * 16;
      }
    }
  }
  // piece q of the tile at `at` = base + its k (and plane), into stage STAGE
  template <int STAGE>
  __device__ __forceinline__ void issue(const char* at, int q) const {
    load_lds16(at, off[q], piece[q], STAGE * BT * 64);
  }
  // of a tile of which only `have` k exist (0 or fewer: none): the last ones again in the place of the others.  The base
  // goes back to where the tile holds one, so that the lanes' offsets, which only shrink, never fall below zero.
  template <int STAGE>
  __device__ __forceinline__ void issue_ragged(const Side& s, const char* at, int have, int q) const {
    constexpr int LEAST = TR ? 1 : 8;
    const int64_t ld = TR ? s.ld : 1;
    if (have < LEAST) at -= (LEAST - have) * ld * 2, have = LEAST;
    const int behind = k_of[q] + LEAST - have;
    load_lds16(at, off[q] - (unsigned)max(0, behind) * (unsigned)ld * 2, piece[q], STAGE * BT * 64);
  }
};

typedef __attribute__((address_space(3))) const s16x8 lds_s16x8;

template <int BT, bool TR, bool EIGHT>
struct Reader {
  unsigned at;  // LDS bytes of this lane's share of fragment 0 in the first stage
  __device__ __forceinline__ void init(const void* lds, int w0, int lane) {
    if (!TR) {
      const int r = lane & 15;
      at = (w0 + (EIGHT ? (r >> 2) * 8 + (r & 3) : r)) * 64 + ((lane >> 4) ^ row_swizzle(r >> 2)) * 16;
    } else {
      const int g = lane >> 4, q = (lane & 15) >> 2, f = (q | ((g & 1) << 2)) & (BT / 16 - 1);
      at = (8 * g + q) * (BT * 2) + (((w0 / 16) ^ f) << 5) + (lane & 3) * 8;
    }
    at += lds_offset(lds);
    asm("" : "+v"(at));  // one register: the reads' own offsets reach all stages
  }
  // fragment i: 16 rows from w0 + 16 i (EIGHT: of the 32 from w0 + 32 (i / 2)), 32 k
  __device__ __forceinline__ s16x8 get(int stage, int i) const {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"
    if (!TR) {
      return *(lds_s16x8*)(at + stage * BT * 64 + (EIGHT ? (i >> 1) * 2048 + (i & 1) * 256 : i * 1024));
    } else {
      const unsigned a = (at ^ (i << 5)) + stage * BT * 64;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 4 * BT * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma clang diagnostic pop
  }
};

// The last step of a product, a wave at a time.  acc[i][j][r]: n = n0 + 16 j + lane % 16, m = m0 + 16 i + 4 (lane / 16) + r
// (EIGHT: m0 + 32 (i / 2) + 8 (lane / 16) + 4 (i % 2) + r) -- a lane holds four or eight neighbours along m.
template <class T, int EPI, bool EIGHT, int FI, int FJ>
__device__ __forceinline__ void head_epilogue(const GemmArgs& g, f32x4 (&acc)[FI][FJ], int m0, int n0, int lane, int N, int split,
                                              int64_t stat_row) {
  const int mw = m0 + (EIGHT ? 8 : 4) * (lane >> 4), nw = n0 + (lane & 15);
  const auto m_of = [&](int i) { return mw + (EIGHT ? 32 * (i >> 1) + 4 * (i & 1) : 16 * i); };
  static_assert(DZ_PAD % (16 * FI) == 0);
  constexpr bool TWO_PARTS = EPI == EPI_DZ && !T::WIDE && FI == 2;  // tiles of 128 x 64, which such few rows take
  if constexpr (EPI == EPI_STATS || EPI == EPI_DZ) {
    const float scale = g.inv_tau * (T::WIDE ? 1.f : 1.4426950408889634f);
    float bias[FI][4];  // -inf behind the last class
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) bias[i][r] = m_of(i) + r < g.M ? 0.f : -INFINITY;
    if (g.bias) {
#pragma unroll
      for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int m = min(m_of(i) + r, g.M - 1);
          bias[i][r] += T::WIDE ? ((const float*)g.bias)[m] : (float)((const typename T::t*)g.bias)[m];
        }
    }
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int n = nw + 16 * j;
      if constexpr (EPI == EPI_STATS) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            acc[i][j][r] += bias[i][r];
            top = fmaxf(top, acc[i][j][r]);
          }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        float sum = 0.f;
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) sum += head_exp<T>((acc[i][j][r] - ref) * scale);  // a NaN stays in the sum
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lane < 16 && n < N) g.stats[stat_row * g.stat_ld + n] = make_float2(top, sum);
      } else if (m0 < g.ldz) {  // all or nothing of a wave's columns, of which DZ_PAD is a multiple
        const bool live = n < N;
        const float top = live ? g.top[n] : 0.f, cp = live ? g.cp[n] : 0.f;
        typedef typename std::conditional<T::WIDE, float, short>::type W;
        W* out = (W*)g.dz + (int64_t)n * g.ldz;
        constexpr int GROUP = EIGHT ? 2 : 1;
        if constexpr (TWO_PARTS) {
          if (g.two) {
            if (n >= g.two) continue;
#pragma unroll
            for (int i = 0; i < FI; ++i) {
              W hi[4], lo[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float x = live ? cp * head_exp<T>((acc[i][j][r] + bias[i][r] - top) * scale) : 0.f;
                hi[r] = to16<T>(x);
                lo[r] = to16<T>(x - (float)__builtin_bit_cast(typename T::t, hi[r]));
              }
              __builtin_memcpy(__builtin_assume_aligned(out + m_of(i), sizeof(hi)), hi, sizeof(hi));
              __builtin_memcpy(__builtin_assume_aligned(out + (int64_t)g.two * g.ldz + m_of(i), sizeof(lo)), lo, sizeof(lo));
            }
            continue;
          }
        }
#pragma unroll
        for (int i0 = 0; i0 < FI; i0 += GROUP) {
          W w[4 * GROUP];
#pragma unroll
          for (int e = 0; e < 4 * GROUP; ++e) {
            const int i = i0 + e / 4, r = e % 4;
            // Rounded to the 16-bit type (half a step, 2^-8 bf16 / 2^-11 f16, of each element; f16 after scaling by a
            // power of two): the size of the rounding that the gradients themselves get.  Their error grows by it -- not
            // seen for labels (1537 x 776 x 50001 bf16: 1.66e-3 -> 1.67e-3 relative), 1.4 times for distillation (2048 x 1000
            // x 32000 f16: 2.1e-4 -> 2.9e-4); two 16-bit parts would double the products of the backward pass.
            float x = cp * head_exp<T>((acc[i][j][r] + bias[i][r] - top) * scale);
            x = live ? x : 0.f;
            if constexpr (T::WIDE)
              w[e] = x;
            else
              w[e] = to16<T>(x);
          }
          __builtin_memcpy(__builtin_assume_aligned(out + m_of(i0), sizeof(w)), w, sizeof(w));
        }
      }
    }
  } else {
    const float inv = g.inv_scale ? *g.inv_scale : 1.f;
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int n = nw + 16 * j;
      if (n >= N) continue;
      float* arow = g.acc ? g.acc + split * g.acc_split + (int64_t)n * g.acc_ld : nullptr;
      const int64_t orow = (int64_t)(g.rowmap ? g.rowmap[n] : n) * g.out_ld;
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const int m = m_of(i);
        f32x4 x = acc[i][j];
        if (m >= g.M) continue;
        if (g.out_kind != OUT_FINAL) {  // acc rows are padded to a multiple of 4
          f32x4* dst = (f32x4*)(arow + m);
          *dst = g.out_kind == OUT_ADD ? *dst + x : x;
          continue;
        }
        if (arow) x += *(const f32x4*)(arow + m);
        x *= inv;
        if constexpr (T::WIDE) {
          float* o = (float*)g.out + orow + m;
          if (m + 4 <= g.M && !(((uintptr_t)o) & 15)) {
            *(f32x4*)o = x;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (m + r < g.M) o[r] = x[r];
          }
        }
      }
    }
  }
}

// Results in 16 bits, out[rowmap[n]][m] = (acc + what the pieces before left) * inv_scale, a wave at a time through its own
// part of LDS: a lane's four neighbours are 8 bytes of a row, whole rows of 2 * 16 FI bytes leave in 16-byte stores.  Units
// of 16 bytes are xor-ed with the row, which keeps both sides free of bank conflicts.
// (dweight of 1 x 2048 x 131072, 537 MB: 208 us with 8-byte stores from the registers, 165 us so.)
typedef __attribute__((ext_vector_type(8), aligned(2))) short s16x8_any;
template <class T, int FI, int FJ>
__device__ __forceinline__ void head_store(const GemmArgs& g, f32x4 (&acc)[FI][FJ], int m0, int n0, int lane, int N, char* lds) {
  constexpr int U = 2 * FI;  // units of a row
  const float inv = g.inv_scale ? *g.inv_scale : 1.f;
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    const int r = 16 * j + (lane & 15);
    const float* before = g.acc && n0 + r < N ? g.acc + (int64_t)(n0 + r) * g.acc_ld : nullptr;
#pragma unroll
    for (int i = 0; i < FI; ++i) {
      const int m = m0 + 16 * i + 4 * (lane >> 4);
      f32x4 x = acc[i][j];
      if (before && m < g.M) x += *(const f32x4*)(before + m);  // rows are padded to a multiple of 4
      s16x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = to16<T>(x[e] * inv);
      *(s16x4*)(lds + r * U * 16 + ((2 * i + (lane >> 5)) ^ (r & (U - 1))) * 16 + (lane >> 4 & 1) * 8) = w;
    }
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll 4
  for (int e = lane; e < 16 * FJ * U; e += 64) {
    const int r = e / U, u = e % U, n = n0 + r, m = m0 + 8 * u;
    if (n >= N || m >= g.M) continue;
    const s16x8 w = *(const s16x8*)(lds + r * U * 16 + (u ^ (r & (U - 1))) * 16);
    short* o = (short*)g.out + (int64_t)(g.rowmap ? g.rowmap[n] : n) * g.out_ld + m;
    if (m + 8 <= g.M) {
      *(s16x8_any*)o = w;
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (m + q < g.M) o[q] = w[q];
    }
  }
}

// A product of 16-bit operands with its epilogue.  8192 x 4096 x 131072 bf16: logits reduced 6.6 ms (1330 TFLOP/s; the
// library's product alone, writing the logits: 1494), dz 7.1 ms, dhidden and dweight 6.5 ms each (1350; the library 1157 and
// 1031).  The matrix units are busy 0.70 of the cycles at 1.7 GHz (0.62-0.67 at 1.9 GHz where results are written): power
// holds the clock there.  Few steps: 0.81 us a step of 256 x 256 x 32 and 11 us a tile around them.  Tiles of 128 x 256,
// two workgroups a CU, have one's epilogue under the other's steps but half as many loads again: 8.3 ms; workgroups that
// stay and load their next tile under the epilogue: 6.9 ms; four waves of 128 x 128: 6.9 ms.
template <class T, int BM, int BN, int WM, int WN, bool TRA, bool TRB, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void head_gemm_kernel(GemmArgs g) {
  constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, FI = WTM / 16, FJ = WTN / 16;
  __shared__ __attribute__((aligned(1024))) char lds[4 * (BM + BN) * 64];
  char *const lds_a = lds, *const lds_b = lds + 4 * BM * 64;
  int split, tm, tn;
  tile_of(g.first + blockIdx.x, g.tiles, g.mt, g.nt, split, tm, tn);
  const int N = g.n_dev ? min(g.N, *g.n_dev) : g.N;
  const int m0 = tm * BM, n0 = tn * BN;
  // dz is an operand of the next products: rows up to a multiple of K_PAD are written, as zeros
  if (n0 >= (EPI == EPI_DZ ? (N + K_PAD - 1) / K_PAD * K_PAD : N)) return;
  const int K = !g.k_dev ? g.K : g.two && *g.k_dev > 0 ? g.K : min(g.K, *g.k_dev);
  const int ktiles = (K + BK - 1) / BK;
  const int per = (ktiles + g.splits - 1) / g.splits;
  const int t0 = min(split * per, ktiles), t1 = min(t0 + per, ktiles);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  constexpr bool EIGHT = !TRA && FI % 2 == 0;
  Stager<BM, NW, TRA, EIGHT> sa;
  Stager<BN, NW, TRB, false> sb;
  sa.init(g.A, m0, lds_a, wave, lane);
  sb.init(g.B, n0, lds_b, wave, lane);
  Reader<BM, TRA, EIGHT> ra;
  Reader<BN, TRB, false> rb;
  ra.init(lds_a, wm * WTM, lane);
  rb.init(lds_b, wn * WTN, lane);

  f32x4 acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  mfma_done<T>(acc);  // written, before the first matrix instruction reads them

  // The tiles are issued in order: `at_a`, `at_b` walk along k.
  const int64_t step_a = BK * 2 * (TRA ? g.A.ld : 1), step_b = BK * 2 * (TRB ? g.B.ld : 1);
  int kt = t0;
  const char *at_a = sa.base + kt * step_a, *at_b = sb.base + kt * step_b;
  int left = t1 - t0;  // tiles that are still to be issued; behind the last one it is issued again, for the count of loads
  const auto issue = [&](auto stage, int q) {
    if (q >= sa.CW)
      sb.template issue<stage>(at_b, q - sa.CW);
    else if (kt * BK + BK <= g.A.klim)
      sa.template issue<stage>(at_a, q);
    else
      sa.template issue_ragged<stage>(g.A, at_a, g.A.klim - kt * BK, q);
    if (q == sa.CW + sb.CW - 1 && --left > 0) {
      at_a += step_a;
      at_b += step_b;
      ++kt;
    }
  };
  const auto issue_all = [&](auto stage) {
#pragma unroll
    for (int q = 0; q < sa.CW + sb.CW; ++q) issue(stage, q);
  };
  // Four stages of 32 k: while a step's matrix instructions run on fragments that are in registers, the next step's
  // fragments are read from LDS, two more tiles are in flight and the loads of the fourth go into the stage that the
  // step's own fragments came from.  One barrier a step: behind it the tile after next has landed for every wave, and
  // nobody still reads the stage that the next loads overwrite.
  constexpr int LOADS = sa.CW + sb.CW;
  s16x8 a0[FI], b0[FJ], a1[FI], b1[FJ];
  // Fragments of the next tile are read in the order b, the last two rows of a, the other rows of a: those go into the
  // registers of rows that are done with.
  constexpr int FRAGS = FI + FJ, PER_ROW = FI > 1 ? (FRAGS + FI - 2) / (FI - 1) : FRAGS;
  const auto fetch = [&](int f, int stage, s16x8(&a)[FI], s16x8(&b)[FJ]) {
    if (f < FJ) {
      b[f] = rb.get(stage, f);
    } else {
      const int i = FI < 3 ? f - FJ : f - FJ < 2 ? FI - 1 - (f - FJ) : f - FJ - 2;
      a[i] = ra.get(stage, i);
    }
  };
  // all loads but the newest two tiles' have landed, all LDS reads are done, in every wave; nothing moves across
  const auto step_barrier = [&] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // Each row of matrix instructions takes its share of the next tile's reads and of the loads along, and nothing moves
  // across rows: all waves' loads in one place would queue up (16 cycles each) with the matrix units idle behind them.
  const auto step = [&](auto stage, const s16x8(&a)[FI], const s16x8(&b)[FJ], s16x8(&an)[FI], s16x8(&bn)[FJ]) {
#pragma unroll
    for (int i = 0; i < FI; ++i) {
#pragma unroll
      for (int f = 0; f < FRAGS; ++f)
        if (f / PER_ROW == i) fetch(f, (stage + 1) & 3, an, bn);
#pragma unroll
      for (int j = 0; j < FJ; ++j) T::mfma(acc[i][j], a[i], b[j]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < LOADS; ++q)
        if (q * FI / LOADS == i) issue(stage, q);
    }
    step_barrier();
  };
  if (t0 < t1) {
    issue_all(std::integral_constant<int, 0>());
    issue_all(std::integral_constant<int, 1>());
    issue_all(std::integral_constant<int, 2>());
    issue_all(std::integral_constant<int, 3>());
    step_barrier();
#pragma unroll
    for (int f = 0; f < FRAGS; ++f) fetch(f, 0, a0, b0);
    step_barrier();  // every wave has read the first stage, which the first step overwrites
    for (int t = t0;; t += 4) {
      step(std::integral_constant<int, 0>(), a0, b0, a1, b1);
      if (t + 1 >= t1) break;
      step(std::integral_constant<int, 1>(), a1, b1, a0, b0);
      if (t + 2 >= t1) break;
      step(std::integral_constant<int, 2>(), a0, b0, a1, b1);
      if (t + 3 >= t1) break;
      step(std::integral_constant<int, 3>(), a1, b1, a0, b0);
      if (t + 4 >= t1) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the tiles issued again
  }
  mfma_done<T>(acc);

  if constexpr (EPI == EPI_OUT && TRA)
    if (g.out_kind == OUT_FINAL) {
      __syncthreads();  // no wave's loads still write the stages
      static_assert(2 * BM * BN <= sizeof(lds));
      head_store<T>(g, acc, m0 + wm * WTM, n0 + wn * WTN, lane, N, lds + wave * 2 * WTM * WTN);
      return;
    }
  head_epilogue<T, EPI, EIGHT>(g, acc, m0 + wm * WTM, n0 + wn * WTN, lane, N, split, tm * WM + wm);
}

// ---- products through registers -----------------------------------------------------------------------------
// x = h + m + l: three bf16 values, exact for 24 bits; an infinity becomes NaN.  Two at a time.
__device__ __forceinline__ void split3(float x, float y, unsigned (&w)[3]) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
#pragma unroll
  for (int pl = 0; pl < 3; ++pl) {
    w[pl] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{x, y}), bf16x2));
    x -= __uint_as_float(w[pl] << 16);
    y -= __uint_as_float(w[pl] & 0xffff0000u);
  }
}

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// A thread's share of a 32-deep tile of one side: a block of four rows and eight k, fetched into registers and stored as
// three planes of bf16.  A unit u of 16 bytes in LDS holds the k 4 u .. 4 u + 3 and 16 + 4 u .. (both sides alike, so that
// the order does not matter): four lanes fetch 64 neighbouring bytes of a row.  Row r has the slot r ^ (r / 16 & 3), which
// spreads the stores of a transposed side (four neighbouring rows a lane) over all banks.
template <class T, int BT, bool TR>
struct Splitter {
  typedef f32x4 Regs[8];
  const float* base;
  unsigned off[4];  // of the thread's rows
  unsigned first;   // transposed: of the four at the first of its k
  int u, row;       // transposed: the first of the four; plain: the rows are row + BT / 4 * j
  bool whole;       // transposed: all four exist
  __device__ __forceinline__ void init(const Side& s, int r0, int block) {
    u = TR ? block / (BT / 4) : block & 3;
    row = TR ? block % (BT / 4) * 4 : block >> 2;
    base = (const float*)s.base + (TR ? (int64_t)r0 : (int64_t)r0 * s.ld);
    whole = r0 + row + 4 <= s.rlim;
    first = TR ? 4 * u * (unsigned)s.ld + row : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      off[j] = TR ? (unsigned)min(row + j, s.rlim - 1 - r0) : (unsigned)min(row + BT / 4 * j, s.rlim - 1 - r0) * (unsigned)s.ld;
  }
  // keeps the rare path's addresses out of the loop's registers
  static __device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
  }
  // plain: x[2 j], x[2 j + 1] are row j; transposed: x[i] are the four rows at its i-th k; zeros from klim on
  __device__ __forceinline__ void load(const Side& s, int k0, int klim, f32x4 (&x)[8]) const {
    if constexpr (!TR) {
      const float* p = base + k0;
      if (k0 + BK <= klim) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q) x[2 * j + q] = *(const f32x4_any*)(p + off[j] + 16 * q + 4 * u);
      } else {
        const int have = klim - k0, k4 = opaque(4 * u);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = 16 * q + k4 + e;
              const float y = p[off[j] + (unsigned)min(k, have - 1)];
              x[2 * j + q][e] = k < have ? y : 0.f;
            }
      }
    } else {
      const float* p = base + (int64_t)k0 * s.ld;
      const unsigned ld = (unsigned)s.ld;
      if (k0 + BK <= klim && whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = *(const f32x4_any*)(p + (16 * (i >> 2) + (i & 3)) * s.ld + first);
      } else {
        const int have = klim - k0, k4 = opaque(4 * u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int k = 16 * (i >> 2) + k4 + (i & 3);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float y = p[(unsigned)min(k, have - 1) * ld + off[j]];
            x[i][j] = k < have ? y : 0.f;
          }
        }
      }
    }
  }
  __device__ __forceinline__ void store(char* lds, const f32x4 (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = TR ? row + j : row + BT / 4 * j;
      u32x4 w[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        unsigned t[3];
        split3(TR ? x[2 * e][j] : x[2 * j + e / 2][2 * e & 3], TR ? x[2 * e + 1][j] : x[2 * j + e / 2][2 * e + 1 & 3], t);
        w[0][e] = t[0], w[1][e] = t[1], w[2][e] = t[2];
      }
      char* at = lds + (r ^ (r >> 4 & 3)) * 64 + (u ^ row_swizzle(r >> 2)) * 16;
#pragma unroll
      for (int pl = 0; pl < 3; ++pl) *(u32x4*)(at + pl * BT * 64) = w[pl];
      __builtin_amdgcn_sched_barrier(0);  // a row at a time: registers
    }
  }
};

// The same for 16-bit operands of any alignment, one plane: a unit u holds the k 8 u .. 8 u + 7.
template <class T, int BT, bool TR>
struct Mover {
  typedef s16x8 Regs[4];  // plain: a row each; transposed: halves are the four rows at one k
  typedef __attribute__((ext_vector_type(4), aligned(2))) short s16x4_any;
  const short* base;
  unsigned off[4], first;
  int u, row;
  bool whole;
  __device__ __forceinline__ void init(const Side& s, int r0, int block) {
    u = TR ? block / (BT / 4) : block & 3;
    row = TR ? block % (BT / 4) * 4 : block >> 2;
    base = (const short*)s.base + (TR ? (int64_t)r0 : (int64_t)r0 * s.ld);
    whole = r0 + row + 4 <= s.rlim;
    first = TR ? 8 * u * (unsigned)s.ld + row : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      off[j] = TR ? (unsigned)min(row + j, s.rlim - 1 - r0) : (unsigned)min(row + BT / 4 * j, s.rlim - 1 - r0) * (unsigned)s.ld;
  }
  static __device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
  }
  __device__ __forceinline__ void load(const Side& s, int k0, int klim, Regs& x) const {
    const int have = klim - k0;
    if constexpr (!TR) {
      const short* p = base + k0;
      if (have >= BK) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *(const s16x8_any*)(p + off[j] + 8 * u);
      } else {
        const int k8 = opaque(8 * u);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const short y = p[off[j] + (unsigned)min(k8 + e, have - 1)];
            x[j][e] = k8 + e < have ? y : (short)0;
          }
      }
    } else {
      const short* p = base + (int64_t)k0 * s.ld;
      if (have >= BK && whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const s16x4 y = *(const s16x4_any*)(p + i * s.ld + first);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i >> 1][4 * (i & 1) + j] = y[j];
        }
      } else {
        const int k8 = opaque(8 * u);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const short y = p[(unsigned)min(k8 + i, have - 1) * (unsigned)s.ld + off[j]];
            x[i >> 1][4 * (i & 1) + j] = k8 + i < have ? y : (short)0;
          }
      }
    }
  }
  __device__ __forceinline__ void store(char* lds, const Regs& x) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = TR ? row + j : row + BT / 4 * j;
      s16x8 w;
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = TR ? x[e >> 1][4 * (e & 1) + j] : x[j][e];
      *(s16x8*)(lds + (r ^ (r >> 4 & 3)) * 64 + (u ^ row_swizzle(r >> 2)) * 16) = w;
    }
  }
};

// The same products for f32 and for 16-bit operands of any alignment, through registers.  f32: each workgroup splits the tiles that it reads (four bytes an element from memory, whatever the
// planes), and the fragments of three planes serve six products.  One LDS stage of 32 k; the loads of the next two tiles are
// in flight under the products, and the CU's other workgroup fills the waits.  4000 x 2048 x 50000: 196 TFLOP/s of the
// operands' products (planes split beforehand, copied by the 16-bit kernel: 155; the library's f32: 153); 1 x 2048 x
// 131072, forward and backward: 0.81 ms (planes split beforehand: 3.64, 10 bytes an element a pass).
template <class T, int BM, int BN, int WM, int WN, bool TRA, bool TRB, int EPI>
__global__ __launch_bounds__(256, 2) void head_gemm_any_kernel(GemmArgs g) {
  static_assert(WM * WN == 4 && BM + BN <= 256 && BM % 64 == 0 && BN % 64 == 0);
  constexpr int PLANES = T::WIDE ? 3 : 1, PAIRS = T::WIDE ? 6 : 1;
  constexpr int WTM = BM / WM, WTN = BN / WN, FI = WTM / 16, FJ = WTN / 16;
  static_assert(WTM % 64 == 0 || (WTM == 32 && FI <= 2));
  __shared__ __attribute__((aligned(1024))) char lds_a[PLANES * BM * 64];
  __shared__ __attribute__((aligned(1024))) char lds_b[PLANES * BN * 64];
  __shared__ __attribute__((aligned(1024))) char lds_out[EPI == EPI_OUT && !T::WIDE ? 2 * BM * BN : 16];
  int split, tm, tn;
  tile_of(g.first + blockIdx.x, g.tiles, g.mt, g.nt, split, tm, tn);
  const int N = g.n_dev ? min(g.N, *g.n_dev) : g.N;
  const int m0 = tm * BM, n0 = tn * BN;
  if (n0 >= N) return;
  const int K = !g.k_dev ? g.K : g.two && *g.k_dev > 0 ? g.K : min(g.K, *g.k_dev);
  const int ktiles = (K + BK - 1) / BK;
  const int per = (ktiles + g.splits - 1) / g.splits;
  const int t0 = min(split * per, ktiles), t1 = min(t0 + per, ktiles);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // the first waves fetch A, the others B
  typename std::conditional<T::WIDE, Splitter<T, BM, TRA>, Mover<T, BM, TRA>>::type sa;
  typename std::conditional<T::WIDE, Splitter<T, BN, TRB>, Mover<T, BN, TRB>>::type sb;
  typedef typename decltype(sa)::Regs Regs;
  const bool for_a = wave < BM / 64, for_b = !for_a && wave < (BM + BN) / 64;
  sa.init(g.A, m0, for_a ? threadIdx.x : 0);
  sb.init(g.B, n0, for_b ? threadIdx.x - BM : 0);
  Regs x0, x1;
  const auto load = [&](int t, Regs& x) {
    if (for_a)
      sa.load(g.A, t * BK, K, x);
    else if (for_b)
      sb.load(g.B, t * BK, K, x);
  };
  const auto fragment = [&](const char* lds, int rows, int w0, int pl, int i) {
    const int r = lane & 15, at = w0 / 16 + i;
    return *(const s16x8*)(lds + pl * rows * 64 + (w0 + 16 * i + (r ^ (at & 3))) * 64 + ((lane >> 4) ^ row_swizzle(r >> 2)) * 16);
  };
  f32x4 acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  mfma_done<T>(acc);  // written, before the first matrix instruction reads them
  const auto step = [&](int t, Regs& x) {
    if (for_a)
      sa.store(lds_a, x);
    else if (for_b)
      sb.store(lds_b, x);
    __syncthreads();
    if (t + 2 < t1) load(t + 2, x);
    s16x8 a[FI][PLANES];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int pl = 0; pl < PLANES; ++pl) a[i][pl] = fragment(lds_a, BM, wm * WTM, pl, i);
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      s16x8 b[PLANES];
#pragma unroll
      for (int pl = 0; pl < PLANES; ++pl) b[pl] = fragment(lds_b, BN, wn * WTN, pl, j);
      // smallest products first: (l, h) (h, l) (m, m) (m, h) (h, m) (h, h)
#pragma unroll
      for (int q = 6 - PAIRS; q < 6; ++q)
#pragma unroll
        for (int i = 0; i < FI; ++i) T::mfma(acc[i][j], a[i][(0x001102 >> (4 * q)) & 3], b[(0x010120 >> (4 * q)) & 3]);
    }
    __syncthreads();
  };
  if (t0 < t1) load(t0, x0);
  if (t0 + 1 < t1) load(t0 + 1, x1);
  for (int t = t0; t < t1; t += 2) {
    step(t, x0);
    if (t + 1 < t1) step(t + 1, x1);
  }
  mfma_done<T>(acc);
  if constexpr (EPI == EPI_OUT && !T::WIDE)
    if (g.out_kind == OUT_FINAL) {
      static_assert(2 * BM * BN <= sizeof(lds_out));
      head_store<T>(g, acc, m0 + wm * WTM, n0 + wn * WTN, lane, N, lds_out + wave * 2 * WTM * WTN);
      return;
    }
  head_epilogue<T, EPI, false>(g, acc, m0 + wm * WTM, n0 + wn * WTN, lane, N, split, tm * WM + wm);
}

// ---- the rows that count ------------------------------------------------------------------------------
// One workgroup: rows[i] = i-th row with a target, inv[r] = its place or -1, count; the targets themselves where they are
// labels; loss 0 for rows without.
__global__ __launch_bounds__(1024) void head_rows_kernel(Targets tg, const int64_t* __restrict__ labels, int64_t ignore, int classes,
                                                         int64_t n, int* __restrict__ rows, int* __restrict__ inv,
                                                         int* __restrict__ count, float* __restrict__ loss) {
  // each thread a run of rows: counted, the counts scanned, then written
  __shared__ int sh[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t per = (n + 1023) / 1024, r0 = min(n, threadIdx.x * per), r1 = min(n, r0 + per);
  int mine = 0;
  for (int64_t r = r0; r < r1; ++r) {
    float P;
    if (labels) {
      label_target(labels[r], ignore, classes, tg.p[r], tg.at[r], P);
      tg.P[r] = P;
    } else {
      P = tg.P[r];
    }
    mine += P != NO_TARGET;
    inv[r] = P != NO_TARGET ? 0 : -1;
    if (P == NO_TARGET) loss[r] = 0.f;
  }
  int upto = mine;
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(upto, o, 64);
    if (lane >= o) upto += x;
  }
  if (lane == 63) sh[wave] = upto;
  __syncthreads();
  int at = upto - mine;
  for (int w = 0; w < wave; ++w) at += sh[w];
  if (threadIdx.x == 1023) count[0] = at + mine, count[1] = 0;
  for (int64_t r = r0; r < r1; ++r)
    if (inv[r] == 0) {  // written by this thread above
      rows[at] = (int)r;
      inv[r] = at++;
    }
}

// dst[0 .. ldd) = src[0 .. d) by one block of 256, zeros behind d (everywhere: have = false)
template <typename W>
__device__ __forceinline__ void pack_row(const W* src, bool have, int d, W* dst, int ldd) {
  constexpr int V = 16 / sizeof(W);
  for (int c = threadIdx.x * V; c < ldd; c += 256 * V) {
    vec4f w = {0.f, 0.f, 0.f, 0.f};
    if (have && c < d) {
      if (c + V <= d && !((uintptr_t)(src + c) & 15)) {
        w = *(const vec4f*)(src + c);
      } else {
        W x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = c + e < d ? src[c + e] : (W)0;
        __builtin_memcpy(&w, x, 16);
      }
    }
    *(vec4f*)(dst + c) = w;
  }
}

// the weight rows of a piece, a block each
template <typename W>
__global__ __launch_bounds__(256) void head_pack_kernel(const W* __restrict__ src, int64_t lds, int d, W* __restrict__ dst, int ldd) {
  const int64_t i = blockIdx.x;
  pack_row<W>(src + i * lds, true, d, dst + i * ldd, ldd);
}

// The targets' logits z = hidden . weight[at] + bias as dot products of the inputs, in 32 bits: a wave for eight
// targets of a row, two for each 16 lanes (one or two targets: the whole wave), their weight rows in flight together.  Bound
// by the gathered rows' bytes (3686 rows of 64 targets, 2048 features, bf16, 0.93 GB: 150 us, 6.2 TB/s, caches included).
constexpr int DOTS = 8;
template <int DT>
__device__ __forceinline__ void target_dots(const typename Elem<DT>::t* h, const void* weight, int64_t ldw, const void* bias, int d,
                                            const Targets& tg, int64_t src, int k0, float* zk, int lane) {
  typedef typename Elem<DT>::t E;
  constexpr int V = Elem<DT>::PER16;
  const int lanes = tg.k > 2 ? 16 : 64, l = lane & (lanes - 1), k = k0 + lane / lanes * 2;
  const bool vec = (((uintptr_t)h | (uintptr_t)weight) & 15) == 0 && ldw % V == 0;
  int at[2];
  const E* w[2];
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    at[q] = k + q < tg.k ? tg.at[src * tg.k + k + q] : -1;
    w[q] = (const E*)weight + (int64_t)max(at[q], 0) * ldw;
  }
  int c = vec ? l * V : d;
#pragma unroll 4
  for (; c + V <= d; c += lanes * V) {
    float x[V], y[V], z[V];
    unpack16<DT>(*(const vec4f*)(h + c), x);
    unpack16<DT>(*(const vec4f*)(w[0] + c), y);
    unpack16<DT>(*(const vec4f*)(w[1] + c), z);
#pragma unroll
    for (int e = 0; e < V; ++e) s[0] = fmaf(x[e], y[e], s[0]), s[1] = fmaf(x[e], z[e], s[1]);
  }
  for (c = (vec ? d / V * V : 0) + l; c < d; c += lanes)
#pragma unroll
    for (int q = 0; q < 2; ++q) s[q] = fmaf((float)h[c], (float)w[q][c], s[q]);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
#pragma unroll
    for (int o = 32; o; o >>= 1)
      if (o < lanes) s[q] += __shfl_xor(s[q], o, 64);
    if (l == 0 && k + q < tg.k) zk[k + q] = at[q] < 0 ? 0.f : s[q] + (bias ? Elem<DT>::load(bias, at[q]) : 0.f);
  }
}

// Packs the hidden rows that count, a block each (rows behind the last one: zeros), and takes their targets' logits (zk; not
// where the logits are kept).
template <int DT>
__global__ __launch_bounds__(256) void head_pack_rows_kernel(const void* __restrict__ hidden, int64_t ldh, int64_t all, int two, int d,
                                                             const int* __restrict__ rows, const int* __restrict__ count,
                                                             void* __restrict__ dst, int ldd, const void* __restrict__ weight,
                                                             int64_t ldw, const void* __restrict__ bias, Targets tg,
                                                             float* __restrict__ zk) {
  typedef typename std::conditional<DT == NIF_F32, float, short>::type W;
  const int64_t i = row_block();
  if (i >= all) return;
  const int64_t row = two && i >= two && i < 2 * two ? i - two : i;  // once more for the second part of dz
  const bool have = row < *count;
  const int64_t src = have ? rows[row] : 0;
  const typename Elem<DT>::t* h = (const typename Elem<DT>::t*)hidden + src * ldh;
  pack_row<W>((const W*)h, have, d, (W*)dst + i * ldd, ldd);
  if (!have || !zk || row != i) return;
  for (int k0 = (threadIdx.x >> 6) * DOTS; k0 < tg.k; k0 += 4 * DOTS)
    target_dots<DT>(h, weight, ldw, bias, d, tg, src, k0, zk + i * tg.k, threadIdx.x & 63);
}

// ---- the loss of each row -------------------------------------------------------------------------------
// ROWS packed rows a block (16, a line of the statistics; two where there are at most FINISH_FEW rows, for more blocks: 41 rows
// of 2180 tiles 17 us to 8): joins the tiles' (maximum, sum) pairs, and writes each row's loss to its own place.  The
// block that is done last (`done`, cleared by head_rows_kernel) reduces the losses: sum or mean over the rows that count,
// in a fixed order and 64 bits.
constexpr int FINISH_NT = 1024;
constexpr int64_t FINISH_FEW = 512;
template <int ROWS>
__global__ __launch_bounds__(FINISH_NT) void head_finish_kernel(const float2* __restrict__ stats, int64_t stat_ld, int tiles, Targets tg,
                                                                const int* __restrict__ rows, const int* __restrict__ count,
                                                                float* __restrict__ tops, float* __restrict__ sums,
                                                                const float* __restrict__ zk, const float* __restrict__ z, int64_t ldz,
                                                                float* loss,
                                                                int64_t all_rows, int reduction, int* done, float* __restrict__ reduced) {
  constexpr int PARTS = FINISH_NT / ROWS;
  __shared__ float sh_top[ROWS][PARTS + 1], sh_sum[ROWS][PARTS + 1];
  __shared__ double sh[16];
  __shared__ int last;
  const int64_t i0 = row_block() * ROWS;
  const int n = *count, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (i0 < n) {
    const int r = threadIdx.x % ROWS, part = threadIdx.x / ROWS;
    float top = -INFINITY, sum = 0.f;
    if (i0 + r < n)
#pragma unroll 4
      for (int t = part; t < tiles; t += PARTS) {
        const float2 x = stats[(int64_t)t * stat_ld + i0 + r];
        join(top, sum, x.x, x.y, tg.inv_tau);
      }
    sh_top[r][part] = top;
    sh_sum[r][part] = sum;
    __syncthreads();
    const int64_t i = i0 + wave;  // a wave a row
    if (wave < ROWS && i < n) {
      top = sh_top[wave][lane], sum = sh_sum[wave][lane];
#pragma unroll
      for (int p = 64 + lane; p < PARTS; p += 64) join(top, sum, sh_top[wave][p], sh_sum[wave][p], tg.inv_tau);
      const float all = wave_max_f32(top);
      sum = wave_sum_f32(sum * expf((top - reference_of(all)) * tg.inv_tau));
      const float log_sum = logf(sum);
      const int64_t src = rows[i];
      double s = 0.0;
      for (int k = lane; k < tg.k; k += 64)
        s += target_term(tg, src, k,
                         ((double)(z ? z[i * ldz + max(0, tg.at[src * tg.k + k])] : zk[i * tg.k + k]) - (double)all) *
                             (double)tg.inv_tau,
                         log_sum);
      s = wave_sum_f64(s);
      if (lane == 0) {
        tops[i] = all;
        sums[i] = sum;
        loss[src] = (float)(s * tg.tau2);
      }
    }
  }
  if (reduction == NIF_REDUCE_NONE) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the losses have left, before the block counts as done
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(done, 1) == (int)(gridDim.x * gridDim.z) - 1;
    if (last) __threadfence();
  }
  __syncthreads();
  if (!last) return;
  double s = 0.0;
  for (int64_t r = threadIdx.x; r < all_rows; r += FINISH_NT) s += (double)loss[r];
  s = wave_sum_f64(s);
  if (lane == 0) sh[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < 16; ++w) s += sh[w];
    *reduced = (float)(reduction == NIF_REDUCE_MEAN ? s / max(1, n) : s);
  }
}

// First block: dz = coef[i] (P s - p) with cp[i] = coef[i] * P[i] / (the row's sum of exponentials), and what the products of
// dz are multiplied with.  Where one gradient arrives for all rows, dz goes without it and it joins at the end, in 32 bits:
// the row's largest entry, mostly near -1, then keeps its bits.  f16 holds nothing below 2^-24, so there dz is scaled by the power of two that takes
// the largest |coef| max(1, P) to [2^13, 2^14) (|dz| is no larger).  Where no row counts the arriving gradient is not read
// (there may be none, and zeros stay zeros whatever it holds).  inv_scale[1]: the power of two that takes that largest one
// to [2^37, 2^38), for `rest`.  The other blocks: gradient 0 for rows without a target, and `rest` cleared.
template <typename W>
__global__ __launch_bounds__(1024) void head_coef_kernel(const float* __restrict__ grad, int per_row, int mean, Targets tg,
                                                         const int* __restrict__ rows, const int* __restrict__ inv,
                                                         const int* __restrict__ count, const float* __restrict__ sums, int64_t rows_all,
                                                         int f16, float* __restrict__ coef,
                                                         float* __restrict__ cp, float* __restrict__ inv_scale, W* __restrict__ out,
                                                         int64_t ld, int d, int64_t clearing, long long* __restrict__ rest, int classes) {
  if (row_block() > clearing) {
    const int64_t c = (row_block() - 1 - clearing) * 1024 + threadIdx.x;
    if (rest && c < classes) rest[c] = 0;
    return;
  }
  if (row_block() > 0) {
    const int64_t r = (row_block() - 1) * 4 + (threadIdx.x >> 8);
    if (r < rows_all && inv[r] < 0)
      for (int c = threadIdx.x & 255; c < d; c += 256) out[r * ld + c] = 0;
    return;
  }
  __shared__ float sh[16];
  const int n = *count;
  const float w = tg.tau * (mean ? 1.f / max(1, n) : 1.f), all = per_row || n == 0 ? 1.f : grad[0] * w;
  float scale = 1.f;
  if (f16 || rest) {
    float top = 0.f;
    for (int i = threadIdx.x; i < n; i += 1024) {
      const float c = (per_row ? fabsf(grad[rows[i]] * w) : 1.f) * fmaxf(1.f, tg.P[rows[i]]);
      top = c < INFINITY ? fmaxf(top, c) : top;
    }
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int v = 0; v < 16; ++v) top = fmaxf(top, sh[v]);
    int e = 0;
    if (top > 0.f && top < INFINITY) {
      frexpf(top, &e);  // top in [2^(e-1), 2^e)
      if (f16) scale = ldexpf(1.f, max(-100, min(100, 14 - e)));
    }
    if (threadIdx.x == 0) inv_scale[1] = ldexpf(1.f, max(-100, min(100, 38 - (f16 ? 14 : e))));
  }
  if (threadIdx.x == 0) *inv_scale = all / scale;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float c = (per_row ? grad[rows[i]] * w : 1.f) * scale;
    coef[i] = c;
    cp[i] = c * tg.P[rows[i]] / sums[i];
  }
}

// The targets' entries of a piece of dz: coef (P s - sum of the row's p with that class).  The first of equal classes
// writes, with the sum over all of them in order; dz2: the second part, or null.  rest: what the rounding takes off, for
// dbias, added up over the rows in whole numbers of 1 / fix (whose order does not matter), or null.  One wave per packed row.
template <class W, class U>
__device__ __forceinline__ void target_entries(const Targets& tg, int64_t src, U&& z_of, float top, float coef, float cp, int v0,
                                               int v1, W* dz, W* dz2, long long* rest, float fix, int lane) {
  const int* at = tg.at + src * tg.k;
  const float* p = tg.p + src * tg.k;
  for (int k0 = 0; k0 < tg.k; k0 += 64) {
    const int k = k0 + lane, v = k < tg.k ? at[k] : -1;
    const bool mine = v >= v0 && v < v1;
    if (!__any(mine)) continue;
    float sum = 0.f;
    bool first = true;
    for (int q0 = 0; q0 < tg.k; q0 += 64) {
      const int aq = q0 + lane < tg.k ? at[q0 + lane] : -1;
      const float pq = q0 + lane < tg.k ? p[q0 + lane] : 0.f;
      const int n = min(64, tg.k - q0);
      for (int q = 0; q < n; ++q) {
        const bool same = __builtin_amdgcn_readlane(aq, q) == v;
        if (same && q0 + q < k) first = false;
        sum += same ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pq), q)) : 0.f;
      }
    }
    if (mine && first) {
      const float x = cp * expf((z_of(k, v) - top) * tg.inv_tau) - coef * sum;
      dz[v - v0] = (W)x;
      if (dz2) dz2[v - v0] = (W)(x - (float)(W)x);
      if (rest) {
        const float r = (x - (float)(W)x) * fix;
        if (fabsf(r) < 0x1p40f) atomicAdd((unsigned long long*)(rest + v - v0), (unsigned long long)llrintf(r));  // not NaN or inf
      }
    }
  }
}
template <class T>
__global__ __launch_bounds__(256) void head_targets_kernel(Targets tg, const int* __restrict__ rows, const int* __restrict__ count,
                                                           const float* __restrict__ zk, const float* __restrict__ tops,
                                                           const float* __restrict__ coef, const float* __restrict__ cp, int v0, int v1,
                                                           typename T::t* __restrict__ dz, int64_t ldz, int two, long long* rest,
                                                           const float* __restrict__ inv_scale) {
  const int64_t i = row_block() * 4 + (threadIdx.x >> 6);
  if (i >= *count) return;
  target_entries(tg, rows[i], [&](int k, int) { return zk[i * tg.k + k]; }, tops[i], coef[i], cp[i], v0, v1, dz + i * ldz,
                 two ? dz + (i + two) * ldz : nullptr, rest, inv_scale[1], threadIdx.x & 63);
}

// dbias of a piece: column sums of dz (of both parts, or with what the targets' entries lost, `rest`, which is left cleared for
// the next piece) over stretches of packed rows (256 columns a block, 8 a thread), joined in order by
// head_bias_join_kernel where there are several.  Bound by the read of dz (2048 x 32000 f16, 125 MB: 20 us).
__device__ __forceinline__ float take_rest(long long* rest, int c, const float* inv_scale) {
  if (!rest) return 0.f;
  const long long r = rest[c];
  rest[c] = 0;
  return (float)((double)r / (double)inv_scale[1]);
}
template <class T>
__global__ __launch_bounds__(256) void head_bias_kernel(const typename T::t* __restrict__ dz, int64_t ldz, int cols,
                                                        const int* __restrict__ count, int two, int stretch, float* __restrict__ part,
                                                        const float* __restrict__ inv_scale, typename T::t* __restrict__ out,
                                                        long long* __restrict__ rest) {
  typedef __attribute__((ext_vector_type(8))) typename T::t Eight;
  __shared__ float sh[8][256 + 8];
  const int c0 = blockIdx.x * 256 + (threadIdx.x & 31) * 8, group = threadIdx.x >> 5;
  const int r0 = blockIdx.y * stretch, r1 = min(*count, r0 + stretch);
  if (r0 >= r1 && gridDim.y > 1) return;
  float s[8] = {};
  if (c0 < ldz)
#pragma unroll 4
    for (int r = r0 + group; r < r1; r += 8) {
      const Eight x = *(const Eight*)(dz + (int64_t)r * ldz + c0);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += (float)x[e];
    }
  if (two && c0 < ldz)
    for (int r = r0 + group; r < r1; r += 8) {
      const Eight x = *(const Eight*)(dz + (int64_t)(r + two) * ldz + c0);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += (float)x[e];
    }
#pragma unroll
  for (int e = 0; e < 8; ++e) sh[group][(threadIdx.x & 31) * 8 + e] = s[e];
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int q = 0; q < 8; ++q) sum += sh[q][threadIdx.x];
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  if (gridDim.y > 1)
    part[(int64_t)blockIdx.y * cols + c] = sum;
  else
    out[c] = (typename T::t)((sum + take_rest(rest, c, inv_scale)) * *inv_scale);
}
template <class T>
__global__ __launch_bounds__(256) void head_bias_join_kernel(const float* __restrict__ part, int cols, const int* __restrict__ count, int stretch,
                                                             const float* __restrict__ inv_scale, void* __restrict__ out,
                                                             long long* __restrict__ rest) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  const int stretches = (*count + stretch - 1) / stretch;
  float s = 0.f;
#pragma unroll 8
  for (int q = 0; q < stretches; ++q) s += part[(int64_t)q * cols + c];
  s += take_rest(rest, c, inv_scale);
  s *= *inv_scale;
  ((typename T::t*)out)[c] = (typename T::t)s;
}

// out = (sum of the splits' partial sums, in order, + acc) * inv_scale, or acc = that sum: 4 columns a thread, 1024 a block
template <class T>
__global__ __launch_bounds__(256) void head_join_kernel(const float* __restrict__ part, int splits, int64_t part_split, int64_t part_ld,
                                                        int n, const int* __restrict__ n_dev, int m, float* __restrict__ acc, int first,
                                                        int last, void* __restrict__ out, int64_t out_ld, const int* __restrict__ rowmap,
                                                        const float* __restrict__ inv_scale) {
  const int64_t i = row_block();
  const int c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (i >= (n_dev ? min(n, *n_dev) : n) || c >= m) return;
  const float* p = part + i * part_ld + c;  // rows are padded to a multiple of 4
  f32x4 s = first ? f32x4{0.f, 0.f, 0.f, 0.f} : *(const f32x4*)(acc + i * part_ld + c);
#pragma unroll 8
  for (int q = 0; q < splits; ++q) s += *(const f32x4*)(p + q * part_split);
  if (!last) {
    *(f32x4*)(acc + i * part_ld + c) = s;
    return;
  }
  s *= *inv_scale;
  const int64_t o = (int64_t)(rowmap ? rowmap[i] : i) * out_ld + c;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < m) ((typename T::t*)out)[o + e] = (typename T::t)s[e];
}

// ---- kept logits ------------------------------------------------------------------------------------------------
// z = the splits' partial sums, in order, + bias, kept in 32 bits, and its (maximum, sum of exponentials) over
// stretches of KEPT classes: a block a stretch of one packed row.
constexpr int KEPT = 1024;
template <class T>
__global__ __launch_bounds__(256) void head_kept_kernel(const float* __restrict__ part, int splits, int64_t part_split, float* __restrict__ kept,
                                                        int64_t ldu, int v, const int* __restrict__ count, const void* __restrict__ bias,
                                                        float inv_tau, float2* __restrict__ stats, int64_t stat_ld) {
  __shared__ float sh_top[4], sh_sum[4];
  const int64_t i = blockIdx.x;
  if (i >= *count) return;
  const int c = blockIdx.y * KEPT + threadIdx.x * 4;
  f32x4 x = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (c < v) {  // rows are padded to a multiple of 4
    f32x4* at = (f32x4*)(kept + i * ldu + c);
    f32x4 z;
    if (splits > 1) {
      z = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
      for (int q = 0; q < splits; ++q) z += *(const f32x4*)(part + q * part_split + i * ldu + c);
    } else {
      z = *at;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < v) x[e] = z[e] + (bias ? (float)((const typename T::t*)bias)[c + e] : 0.f);
    *at = x;
  }
  float top = wave_max_f32(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum += expf((x[e] - ref) * inv_tau);  // a NaN stays in the sum
  sum = wave_sum_f32(sum);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) sh_top[wave] = top, sh_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    float s = sum;
    for (int w = 1; w < 4; ++w) join(top, s, sh_top[w], sh_sum[w], inv_tau);
    stats[blockIdx.y * stat_ld + i] = make_float2(top, s);
  }
}

// dz = cp exp((z - top) / tau) of a piece of the classes, 8 a thread, and the targets' entries; zeros up to a multiple of K_PAD rows
// and in the padding of the columns, where the products read them.  Rounded as head_gemm_kernel's, or in two parts.
constexpr int KEPT_DZ = 2048;
template <class T>
__global__ __launch_bounds__(256) void head_kept_dz_kernel(const float* __restrict__ z, int64_t ldu, int v0, int cols, Targets tg,
                                                           const int* __restrict__ rows, const int* __restrict__ count,
                                                           const float* __restrict__ tops, const float* __restrict__ coef,
                                                           const float* __restrict__ cp, typename T::t* dz, int64_t ldz, int two,
                                                           long long* rest, const float* __restrict__ inv_scale) {
  typedef __attribute__((ext_vector_type(8))) typename T::t Eight;
  const int n = *count, c0 = blockIdx.y * KEPT_DZ, c = c0 + threadIdx.x * 8;
  const int64_t i = blockIdx.x;
  if (i >= (two ? two : (n + K_PAD - 1) / K_PAD * K_PAD)) return;
  const bool live = i < n;
  const float top = live ? tops[i] : 0.f, k = live ? cp[i] : 0.f;
  const auto one = [&](float x) { return k * expf((x - top) * tg.inv_tau); };
  if (c < ldz) {
    float y[8];
    const float* x = z + i * ldu + v0 + c;
    if (live && c + 8 <= cols) {
      const f32x4 lo = *(const f32x4*)x, hi = *(const f32x4*)(x + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = one(e < 4 ? lo[e & 3] : hi[e & 3]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = live && c + e < cols ? one(x[e]) : 0.f;
    }
    Eight w;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = (typename T::t)y[e];
    *(Eight*)(dz + i * ldz + c) = w;
    if (two) {
      Eight w2;
#pragma unroll
      for (int e = 0; e < 8; ++e) w2[e] = (typename T::t)(y[e] - (float)w[e]);
      *(Eight*)(dz + (i + two) * ldz + c) = w2;
    }
  }
  if (!live) return;
  __syncthreads();  // the entries are stored again behind the others
  if (threadIdx.x < 64)
    target_entries(tg, rows[i], [&](int, int v) { return z[i * ldu + v]; }, top, coef[i], k, v0 + c0, v0 + min(cols, c0 + KEPT_DZ),
                   dz + i * ldz + c0, two ? dz + (i + two) * ldz + c0 : nullptr, rest ? rest + c0 : nullptr,
                   inv_scale[1], threadIdx.x);
}

// ---- small heads ----------------------------------------------------------------------------------------------
// A batch of a classifier's level fit (32 rows, 10 to 200 classes, 400 features) costs launches, not arithmetic: forward
// one block per row, which keeps the row's dz (n x classes f32, at most 1 MiB) for the backward pass, a single launch of
// dot products.  Sums in 32 bits, the row's loss in 64.
constexpr int SMALL_V = 2048;

template <int DT, int NT>
__global__ __launch_bounds__(NT) void head_small_forward_kernel(nif_head_desc h, Targets t, float* __restrict__ dz,
                                                                 float* __restrict__ row_loss) {
  typedef typename Elem<DT>::t E;
  constexpr int V = Elem<DT>::PER16, Q = 4;
  __shared__ float u[SMALL_V], sh[2 * NT / 64];
  __shared__ double sh_loss[NT / 64];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int classes = h.classes, d = h.features;
  __shared__ float sh_P;
  if (wave == 0) {
    if (h.labels) {
      if (lane == 0) label_target(h.labels[row], h.ignore_index, classes, t.p[row], t.at[row], sh_P), t.P[row] = sh_P;
    } else {
      const float P = top_targets(h.top_indices, h.top_values, h.top_lse, row, classes, t, lane);
      if (lane == 0) sh_P = P;
    }
  }
  __syncthreads();
  const float P = sh_P;
  if (P == NO_TARGET) {
    if (threadIdx.x == 0) row_loss[row] = 0.f;
    return;
  }
  const E* x = (const E*)h.hidden + row * h.ldh;
  const E* w = (const E*)h.weight;
  const bool vec = (((uintptr_t)x | (uintptr_t)w) & 15) == 0 && h.ldw % V == 0;
  for (int v0 = wave * Q; v0 < classes; v0 += NT / 64 * Q) {
    float s[Q];
    const E* wr[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) s[q] = 0.f, wr[q] = w + (int64_t)min(v0 + q, classes - 1) * h.ldw;
    int c = vec ? lane * V : d;
    for (; c + V <= d; c += 64 * V) {
      float a[V];
      unpack16<DT>(*(const vec4f*)(x + c), a);
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        float b[V];
        unpack16<DT>(*(const vec4f*)(wr[q] + c), b);
#pragma unroll
        for (int e = 0; e < V; ++e) s[q] = fmaf(a[e], b[e], s[q]);
      }
    }
    for (c = (vec ? d / V * V : 0) + lane; c < d; c += 64)
#pragma unroll
      for (int q = 0; q < Q; ++q) s[q] = fmaf((float)x[c], (float)wr[q][c], s[q]);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      s[q] = wave_sum_f32(s[q]);
      if (lane == 0 && v0 + q < classes) u[v0 + q] = s[q] + (h.bias ? Elem<DT>::load(h.bias, v0 + q) : 0.f);
    }
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int v = threadIdx.x; v < classes; v += NT) top = fmaxf(top, u[v]);
  top = wave_max_f32(top);
  const float ref = top == -INFINITY ? 0.f : top;
  for (int v = threadIdx.x; v < classes; v += NT) sum += expf((u[v] - ref) * t.inv_tau);
  sum = wave_sum_f32(sum);
  if (lane == 0) sh[2 * wave] = top, sh[2 * wave + 1] = sum;
  __syncthreads();
  top = sh[0], sum = sh[1];
  for (int q = 1; q < NT / 64; ++q) join(top, sum, sh[2 * q], sh[2 * q + 1], t.inv_tau);
  const float log_sum = logf(sum);
  double loss = 0.0;
  for (int k = threadIdx.x; k < t.k; k += NT) {
    const int at = t.at[row * t.k + k];
    if (at >= 0) loss += target_term(t, row, k, ((double)u[at] - (double)top) * (double)t.inv_tau, log_sum);
  }
  loss = wave_sum_f64(loss);
  if (lane == 0) sh_loss[wave] = loss;
  __syncthreads();
  if (threadIdx.x == 0) {
    loss = 0.0;
    for (int q = 0; q < NT / 64; ++q) loss += sh_loss[q];
    row_loss[row] = (float)(loss * t.tau2);
  }
  const float cp = t.tau * P / sum;
  for (int v = threadIdx.x; v < classes; v += NT) u[v] = cp * expf((u[v] - top) * t.inv_tau);
  __syncthreads();
  for (int k = threadIdx.x; k < t.k; k += NT) {
    const int v = t.at[row * t.k + k];
    if (v < 0) continue;
    float p = 0.f;
    bool first = true;
    for (int q = 0; q < t.k; ++q)
      if (t.at[row * t.k + q] == v) {
        first &= q >= k;
        p += t.p[row * t.k + q];
      }
    if (first) u[v] -= t.tau * p;
  }
  __syncthreads();
  for (int v = threadIdx.x; v < classes; v += NT) dz[row * classes + v] = u[v];
}

// Blocks of 64 columns x NT / 64 parts of a sum: first those of dhidden (a row each), then those of dweight (4 classes).
template <int DT, int NT>
__global__ __launch_bounds__(NT) void head_small_backward_kernel(nif_head_desc h, const float* __restrict__ P, const float* __restrict__ dz,
                                                                 const float* __restrict__ count, const float* __restrict__ grad,
                                                                 void* __restrict__ dhidden, int64_t lddh, void* __restrict__ dweight,
                                                                 int64_t lddw, void* __restrict__ dbias, int hidden_blocks, int stretches) {
  typedef typename Elem<DT>::t E;
  constexpr int PARTS = NT / 64;
  __shared__ float sh[4][PARTS][64], shb[4][PARTS];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
  const int n = (int)h.rows, classes = h.classes, d = h.features;
  const bool per_row = h.reduction == NIF_REDUCE_NONE;
  const float share = h.reduction == NIF_REDUCE_MEAN ? 1.f / *count : 1.f;
  const int block = (int)blockIdx.x < hidden_blocks ? blockIdx.x : blockIdx.x - hidden_blocks;
  const int c = block % stretches * 64 + lane;
  const auto total = [&](int q) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < PARTS; ++w) s += sh[q][w][lane];
    return s;
  };
  if ((int)blockIdx.x < hidden_blocks) {
    const int64_t row = block / stretches;
    E* out = (E*)dhidden + row * lddh;
    if (P[row] == NO_TARGET) {
      if (part == 0 && c < d) out[c] = (E)0.f;
      return;
    }
    const float coef = grad[per_row ? row : 0] * share;
    const E* w = (const E*)h.weight + min(c, d - 1);
    const float* z = dz + row * classes;
    float s = 0.f;
#pragma unroll 16
    for (int v = part; v < classes; v += PARTS) s = fmaf(z[v], (float)w[v * h.ldw], s);
    sh[0][part][lane] = s;
    __syncthreads();
    if (part == 0 && c < d) out[c] = (E)(coef * total(0));
    return;
  }
  const int v0 = block / stretches * 4;
  const bool bias = dbias && block % stretches == 0;
  const E* x = (const E*)h.hidden + min(c, d - 1);
  float s[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int r = part; r < n; r += PARTS) {
    if (P[r] == NO_TARGET) continue;  // whatever such a row holds
    const float coef = grad[per_row ? r : 0] * share, a = dweight ? (float)x[r * h.ldh] : 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float g = coef * dz[(int64_t)r * classes + min(v0 + q, classes - 1)];
      s[q] = fmaf(g, a, s[q]);
      sb[q] += g;
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    sh[q][part][lane] = s[q];
    if (lane == 0) shb[q][part] = sb[q];
  }
  __syncthreads();
  const int v = v0 + part;  // each of the first four waves writes one of the classes
  if (part >= 4 || v >= classes) return;
  if (dweight && c < d) ((E*)dweight)[v * lddw + c] = (E)total(part);
  if (bias && lane == 0) {
    float b = 0.f;
    for (int w = 0; w < PARTS; ++w) b += shb[part][w];
    ((E*)dbias)[v] = (E)b;
  }
}

// ---- host side ----------------------------------------------------------------------------------------------

static inline int64_t round_up(int64_t x, int64_t q) { return (x + q - 1) / q * q; }

struct Plan {
  int64_t n, cap;
  int d, ldd, v, k;
  int e;             // bytes of an operand's element
  // How the passes read the weight: head_gemm_any_kernel (f32; 16 bits with rows that direct loads cannot take, few rows of
  // hidden), or head_gemm_kernel, from a copy by pieces where the rows are such.
  bool any_f, any_b, pack_f, pack_b;
  bool small;        // the small heads' kernels
  bool keep;         // few rows: the logits are kept
  int two;           // very few rows of 16 bits: dz in two parts, so many rows apart; else 0
  int piece;         // classes per piece (multiple of 256, or all)
  // state: what the backward pass reads
  size_t s_p, s_at, s_P, s_dz, s_rows, s_inv, s_count, s_top, s_sum, s_zk, s_h, s_z, state;
  int64_t ldu;       // of the kept logits
};

// Rows up to which dz has two parts.  One rounding more of each element is 1.4 times the error where many count alike, but up
// to 2.3 times where few do (1 x 64 x 110210 bf16, 13 targets: dweight 1.7e-3 -> 3.0e-3 of its norm; in two parts 1.7e-3).
// For so few rows the products are bound by the weight's bytes and pad their rows to 32 or 64 anyway: a step of 2048 x 131072
// bf16 takes 475 -> 477 us with 1 row, 492 -> 509 with 32, 521 -> 559 with 64; 2050 x 100001 485 -> 508, 520 -> 535, 548 -> 620.
static constexpr int TWO_ROWS = 64;

static constexpr size_t PIECE_BYTES = (size_t)256 << 20;

static size_t take(size_t& at, size_t bytes) {
  const size_t r = at;
  at += (bytes + 255) / 256 * 256;
  return r;
}

struct Shape {
  bool any;  // of head_gemm_any_kernel
  int bm, bn, wm, splits;
  float us;  // what the model says
};
struct Tile {
  int bm, bn, wm, per_cu;
  float step, share, fixed, rate[3];
};
static const Tile TILES16[] = {
    {256, 256, 2, 1, 0.81f, 0.f, 11.f, {4.2f, 3.3f, 3.3f}},
    {128, 128, 2, 2, 0.06f, 0.295f, 5.9f, {4.5f, 3.6f, 3.1f}},
    {128, 64, 4, 3, 0.08f, 0.174f, 4.3f, {4.8f, 3.2f, 3.0f}},
};
static const Tile TILES_ANY16[] = {
    {128, 128, 2, 2, 0.4f, 0.35f, 4.f, {4.0f, 3.5f, 3.0f}},
    {128, 64, 4, 2, 0.35f, 0.25f, 4.f, {4.0f, 3.5f, 3.0f}},
};
static const Tile TILES32[] = {
    {128, 128, 2, 2, 1.05f, 0.85f, 4.f, {3.0f, 2.9f, 3.8f}},
    {128, 64, 4, 2, 0.8f, 0.53f, 4.f, {4.0f, 3.7f, 3.2f}},
};
enum { LOGITS = 0, DHIDDEN = 1, DWEIGHT = 2 };  // the products
// m x n results of a contraction over k, `e` bytes an element; `results`: bytes of one that is written (0: they are reduced)
static Shape shape_of(int product, int64_t m, int64_t n, int64_t k, int e, int results, bool may_split, bool any) {
  const int64_t steps = (k + BK - 1) / BK;
  Shape best = {true, 128, 128, 2, 1, INFINITY};
  const Tile* tiles = e == 4 ? TILES32 : any ? TILES_ANY16 : TILES16;
  any |= e == 4;
  for (int i = 0; i < (any ? 2 : 3); ++i) {
    const Tile& t = tiles[i];
    const int64_t count = ((m + t.bm - 1) / t.bm) * ((n + t.bn - 1) / t.bn);
    for (int splits = 1; splits <= (may_split ? 128 : 1); splits *= 2) {
      if (splits > 1 && steps / splits < 8) break;
      const int64_t blocks = count * splits, slots = 256 * t.per_cu, rest = blocks % slots;
      const float each = (float)((steps + splits - 1) / splits);
      float us = (float)(blocks / slots) * (each * (t.step + t.share * (float)t.per_cu) + t.fixed);
      if (rest) us += each * (t.step + t.share * (float)((rest + 255) / 256)) + t.fixed;
      const float in = (float)(m + n) * (float)k * (float)e;
      const float out = !results ? 0.f : (float)m * (float)n * (splits > 1 ? 4.f * (float)splits : (float)results);
      const float memory = (in + out) * 1e-6f / t.rate[product] + 2.f;
      us = us > memory ? us : memory;
      if (splits > 1) us += 4.f + out * 1e-6f / 4.f;
      if (us < best.us) best = {any, t.bm, t.bn, t.wm, splits, us};
    }
  }
  return best;
}

static Shape logit_shape(const Plan& p, int classes, bool any) { return shape_of(LOGITS, classes, p.n, p.d, p.e, 0, false, any); }

// Few rows: the product has few tiles, or is bound by the weight's bytes, which its repetition reads again.  Kept in 32 bits
// the logits cost their bytes three times over (forward: written, read with the splits joined; backward: read for dz), and
// the product may split its contraction.  bf16, forward and backward: 1 x 2048 x 131072 0.66 -> 0.50 ms, 300 x 2048 x 50000
// 0.50 -> 0.42 ms; f32: 32 x 2048 x 131072 1.9 -> 0.86 ms (with the 128 x 64 tiles' deeper prefetch).
constexpr int64_t KEEP_BYTES = 64 << 20;
static Shape kept_shape(const Plan& p, int classes) { return shape_of(LOGITS, classes, p.n, p.d, p.e, 4, true, p.any_f); }
static bool kept_logits_are_faster(const Plan& p, bool forward_only) {
  if (p.n == 0 || p.n * p.ldu * 4 > KEEP_BYTES) return false;
  // the same for both passes, whatever the weight's address and strides in each
  const Shape s = shape_of(LOGITS, p.v, p.n, p.d, p.e, 4, true, false);
  const float mb = (float)p.n * (float)p.v * 1e-6f, once = logit_shape(p, p.v, false).us;
  const float forward = s.us + (s.splits > 1 ? 0.f : 4.f + 8.f * mb / 4.f), backward = 4.f + (4.f + (float)p.e) * mb / 4.f;
  const float dots = (float)p.n * (float)p.k * (float)p.d * (float)p.e * 1e-6f / 6.f;  // the targets' logits, otherwise
  return forward_only ? forward < once + dots : forward + backward < 2.f * once + dots;
}

// Weights in 16 bits whose rows are off 16-byte borders: up to so many rows of hidden they go through registers, from there
// on a copy pays.  bf16, losses only: 300 x 1001 x 60000 106 us to 135, 1000 x 1001 x 60000 240 to 205; backward: 30 x 2050
// x 100001 313 us to 558, 100 x 1001 x 60000 298 to 220.
constexpr int64_t ANY_ROWS_F = 512, ANY_ROWS_B = 64;
static bool make_plan(const nif_head_desc* h, Plan& p) {
  if (!h || h->rows < 0 || h->features <= 0 || h->classes <= 0 || h->top < 0) return false;
  if (h->dtype != NIF_F32 && h->dtype != NIF_BF16 && h->dtype != NIF_F16) return false;
  if (h->rows > (1 << 30) || h->features > (1 << 20) || h->classes > (1 << 28) || h->top > NIF_TOP_MAX_K) return false;
  if (h->rows * h->classes > (int64_t)1 << 43) return false;  // tiles of a product are counted in 31 bits
  p.n = h->rows;
  p.cap = round_up(p.n > 0 ? p.n : 1, HEAD_PAD);
  p.d = h->features;
  p.ldd = (int)round_up(p.d, K_PAD);
  p.v = h->classes;
  p.k = h->top > 0 ? h->top : 1;
  p.e = h->dtype == NIF_F32 ? 4 : 2;
  const bool odd = p.e == 2 && (p.d % 8 != 0 || h->ldw % 8 != 0 || ((uintptr_t)h->weight & 15) != 0);
  const bool far = h->ldw > HEAD_MAX_LD;
  p.any_f = p.e == 4 || (odd && !far && p.n <= ANY_ROWS_F);
  p.two = p.e == 4 || p.n == 0 || p.n > TWO_ROWS ? 0 : p.n <= 16 ? 16 : p.n <= 32 ? 32 : TWO_ROWS;
  p.any_b = p.e == 4 || (odd && !far && p.n <= ANY_ROWS_B);
  p.pack_f = far || (odd && !p.any_f);
  p.pack_b = far || (odd && !p.any_b);
  const int64_t per = (p.pack_b && p.ldd > p.cap ? (int64_t)p.ldd : p.cap) * p.e;  // bytes of one class of a piece
  int64_t c = (int64_t)(PIECE_BYTES / per) / 256 * 256;
  if (c < 1024) c = 1024;
  if (c > p.v) c = p.v;
  p.piece = (int)c;
  // Small: the tiled path's launches cost 25 us more on the host than one block's read of the whole weight from L2 (32 x 1024 x
  // 1000 bf16, a training step: 83 us against 110; 4 x 128 x 8000: 307 against 111, its sums over the classes are too long).
  p.small = p.n <= 512 && p.v <= SMALL_V && (int64_t)p.v * p.d <= (1 << 20) && p.n * p.v <= (1 << 18) && p.n * p.v * p.d <= (1 << 25);
  size_t at = 0;
  p.s_p = take(at, (size_t)p.n * p.k * 4);
  p.s_at = take(at, (size_t)p.n * p.k * 4);
  p.s_P = take(at, (size_t)p.n * 4);
  p.s_count = take(at, 8);  // the rows that count; the blocks that are done
  p.s_dz = 0;
  if (p.small) {
    p.s_dz = take(at, (size_t)p.n * p.v * 4);
    p.state = at;
    return true;
  }
  p.s_rows = take(at, (size_t)p.cap * 4);
  p.s_inv = take(at, (size_t)p.cap * 4);
  p.s_top = take(at, (size_t)p.cap * 4);
  p.s_sum = take(at, (size_t)p.cap * 4);
  p.s_h = take(at, (size_t)p.cap * p.ldd * p.e);
  p.ldu = round_up(p.v, 4);
  p.keep = kept_logits_are_faster(p, h->forward_only != 0);
  p.s_z = take(at, p.keep ? (size_t)p.n * p.ldu * 4 : 0);
  p.s_zk = take(at, p.keep ? 0 : (size_t)p.cap * p.k * 4);
  p.state = at;
  return true;
}

static Targets targets_of(const nif_head_desc* h, const Plan& p, char* state) {
  Targets t;
  t.p = (float*)(state + p.s_p);
  t.at = (int*)(state + p.s_at);
  t.P = (float*)(state + p.s_P);
  t.k = p.k;
  t.tau = h->labels ? 1.f : h->temperature;
  t.inv_tau = 1.f / t.tau;
  t.tau2 = (double)t.tau * t.tau;
  return t;
}

// Tile and split of a product, by what it would take: rounds of as many blocks as run at once, each its steps of 32 along
// the contraction (`step` us and `share` more for each block on a CU) and a prologue and epilogue (`fixed` us), or its
// bytes at the rate that the tile reaches (`rate`, 10^6 bytes a us), whichever is more; a split adds its partial sums and
// the launch that joins them.  The constants are fitted to each tile's times on 32 products of 10^8 to 10^11 operations
// (20 to 4000 rows, 256 to 2048 features, 1000 to 100000 classes; 10 % off at the median, and the tile chosen costs 2 %
// over the best): 8192 x 4096 x 131072 takes 6.9 ms in tiles of 256 and 10.5 in tiles of 128; 1000 x 1024 x 4000 takes 27 and 15.5 us.
template <class T, bool TRA, bool TRB, int EPI>
static void run_gemm(const Shape& s, GemmArgs& g, hipStream_t st) {
  g.mt = (g.M + s.bm - 1) / s.bm;
  g.nt = (g.N + s.bn - 1) / s.bn;
  g.tiles = g.mt * g.nt * g.splits;
  // a launch takes fewer than 2^32 threads; multiples of eight blocks, so that a tile's XCD does not change
  constexpr int MOST = 1 << 20;
  for (g.first = 0; g.first < g.tiles; g.first += MOST) {
    const dim3 grid(g.tiles - g.first < MOST ? g.tiles - g.first : MOST);
    if (s.any && (T::WIDE || !TRB)) {
      if constexpr (T::WIDE || !TRB) {  // 16 bits: dweight does not read the weight
        if (s.bn == 64)
          hipLaunchKernelGGL((head_gemm_any_kernel<T, 128, 64, 4, 1, TRA, TRB, EPI>), grid, dim3(256), 0, st, g);
        else
          hipLaunchKernelGGL((head_gemm_any_kernel<T, 128, 128, 2, 2, TRA, TRB, EPI>), grid, dim3(256), 0, st, g);
      }
      continue;
    }
    if constexpr (!T::WIDE) {
      if (s.bn == 64)
        hipLaunchKernelGGL((head_gemm_kernel<T, 128, 64, 4, 1, TRA, TRB, EPI>), grid, dim3(256), 0, st, g);
      else if (s.bn == 256)
        hipLaunchKernelGGL((head_gemm_kernel<T, 256, 256, 2, 4, TRA, TRB, EPI>), grid, dim3(512), 0, st, g);
      else
        hipLaunchKernelGGL((head_gemm_kernel<T, 128, 128, 2, 2, TRA, TRB, EPI>), grid, dim3(256), 0, st, g);
    }
  }
}

// of the products that make logits of a piece of `classes`
struct FwdSpace {
  size_t stats, w, part, bytes;
};
static FwdSpace forward_space(const Plan& p) {
  FwdSpace f;
  size_t at = 0;
  const Shape s = logit_shape(p, p.pack_f ? p.piece : p.v, p.any_f);
  const int64_t tiles = p.keep ? (p.v + KEPT - 1) / KEPT : (p.v / s.bm + (p.pack_f ? p.v / p.piece : 0) + 2) * s.wm;
  f.stats = take(at, (size_t)tiles * p.cap * 8);
  const int splits = p.keep ? kept_shape(p, p.pack_f ? p.piece : p.v).splits : 1;
  f.part = take(at, splits > 1 ? (size_t)splits * p.n * p.ldu * 4 : 0);
  f.w = take(at, p.pack_f ? (size_t)p.piece * p.ldd * p.e : 0);
  f.bytes = at;
  return f;
}

// the weight rows of a piece as a side with classes along its rows
static Side weight_side(const nif_head_desc* h, const Plan& p, int v0, int vc, bool pack, void* packed, hipStream_t st) {
  const char* src = (const char*)h->weight + (size_t)v0 * h->ldw * p.e;
  if (!pack) return Side{src, h->ldw, vc, p.d};
  if (p.e == 4)
    hipLaunchKernelGGL(head_pack_kernel<float>, dim3(vc), dim3(256), 0, st, (const float*)src, h->ldw, p.d, (float*)packed, p.ldd);
  else
    hipLaunchKernelGGL(head_pack_kernel<short>, dim3(vc), dim3(256), 0, st, (const short*)src, h->ldw, p.d, (short*)packed, p.ldd);
  return Side{packed, p.ldd, vc, p.ldd};
}

static const void* bias_at(const nif_head_desc* h, int v0) {
  return h->bias ? (const char*)h->bias + (size_t)v0 * (h->dtype == NIF_F32 ? 4 : 2) : nullptr;
}

template <class T>
static void forward_products(const nif_head_desc* h, const Plan& p, char* state, char* ws, const FwdSpace& f, int& tiles, hipStream_t st) {
  const Shape s = logit_shape(p, p.pack_f ? p.piece : p.v, p.any_f);
  tiles = 0;
  for (int v0 = 0; v0 < p.v; v0 += p.pack_f ? p.piece : p.v) {
    const int vc = p.pack_f ? (p.v - v0 < p.piece ? p.v - v0 : p.piece) : p.v;
    GemmArgs g = {};
    g.A = weight_side(h, p, v0, vc, p.pack_f, ws + f.w, st);
    g.B = Side{state + p.s_h, p.ldd, (int)p.cap, p.ldd};
    g.M = vc;
    g.N = (int)p.n;
    g.n_dev = (const int*)(state + p.s_count);
    g.K = p.any_f ? p.d : p.ldd;
    g.splits = 1;
    g.bias = bias_at(h, v0);
    if (p.keep) {
      const Shape ks = kept_shape(p, p.pack_f ? p.piece : p.v);
      g.splits = ks.splits;
      g.out_kind = OUT_F32;
      g.acc = (float*)(ks.splits > 1 ? ws + f.part : state + p.s_z) + v0;
      g.acc_ld = p.ldu;
      g.acc_split = p.n * p.ldu;
      run_gemm<T, false, false, EPI_OUT>(ks, g, st);
      continue;
    }
    g.inv_tau = h->labels ? 1.f : 1.f / h->temperature;
    g.stats = (float2*)(ws + f.stats) + (int64_t)tiles * p.cap;
    g.stat_ld = p.cap;
    run_gemm<T, false, false, EPI_STATS>(s, g, st);
    tiles += g.mt * s.wm;
  }
  if (p.keep) {
    const int splits = kept_shape(p, p.pack_f ? p.piece : p.v).splits;
    tiles = (p.v + KEPT - 1) / KEPT;
    hipLaunchKernelGGL(head_kept_kernel<T>, dim3((unsigned)p.n, tiles), dim3(256), 0, st, (const float*)(ws + f.part), splits,
                       p.n * p.ldu, (float*)(state + p.s_z), p.ldu, p.v, (const int*)(state + p.s_count), h->bias,
                       h->labels ? 1.f : 1.f / h->temperature, (float2*)(ws + f.stats), p.cap);
  }
}

template <int DT>
static void pack_rows(const nif_head_desc* h, const Plan& p, char* state, hipStream_t st) {
  hipLaunchKernelGGL(head_pack_rows_kernel<DT>, row_grid(p.cap), dim3(256), 0, st, h->hidden, h->ldh, p.cap, p.two, p.d,
                     (const int*)(state + p.s_rows), (const int*)(state + p.s_count), state + p.s_h, p.ldd, h->weight, h->ldw, h->bias, targets_of(h, p, state), p.keep ? nullptr : (float*)(state + p.s_zk));
}

struct BwdSpace {
  size_t coef, cp, scale, dz, w, acc, part, rest, bytes;
  int64_t ldz, dh_ld, part_rows;  // part_rows: of a split's partial sums of dhidden
  int stretch;
  Shape dh, dw;
};
static BwdSpace backward_space(const Plan& p) {
  BwdSpace b;
  b.ldz = round_up(p.piece, DZ_PAD);
  b.dh_ld = round_up(p.d, 4);
  // Two parts: each in tiles of its own where the weight goes through registers (a step of 48 x 2050 x 100001 bf16: 600 us, in
  // 128 x 128 tiles over both 711).
  const int64_t rows = p.two ? 2 * p.two : p.n;
  b.dh = shape_of(DHIDDEN, p.d, p.two && p.any_b ? p.two : rows, p.piece, p.e, p.e, true, p.any_b);
  b.dw = shape_of(DWEIGHT, p.d, p.piece, rows, p.e, p.e, true, false);
  size_t at = 0;
  b.coef = take(at, (size_t)p.cap * 4);
  b.cp = take(at, (size_t)p.cap * 4);
  b.scale = take(at, 8);
  b.dz = take(at, (size_t)p.cap * b.ldz * p.e);
  b.w = take(at, p.pack_b ? (size_t)p.piece * p.ldd * p.e : 0);
  b.acc = take(at, p.piece < p.v ? (size_t)p.cap * b.dh_ld * 4 : 0);
  b.part_rows = p.two ? 2 * p.two : p.cap;
  const size_t part_h = b.dh.splits > 1 || p.two ? (size_t)b.dh.splits * b.part_rows * b.dh_ld * 4 : 0;
  const size_t part_w = b.dw.splits > 1 ? (size_t)b.dw.splits * p.piece * b.dh_ld * 4 : 0;
  b.stretch = p.n <= 64 ? 64 : 32;  // rows of a block of column sums: the fewest that leave at most 2048 blocks, up to 256
  while (b.stretch < 256 && (p.n + b.stretch - 1) / b.stretch * ((p.piece + 255) / 256) > 2048) b.stretch *= 2;
  while ((p.n + b.stretch - 1) / b.stretch > 65535) b.stretch *= 2;  // a grid takes no more along y
  const size_t part_b = (size_t)((p.n + b.stretch - 1) / b.stretch) * p.piece * 4;
  const size_t part = part_h > part_w ? part_h : part_w;
  b.part = take(at, part > part_b ? part : part_b);
  b.rest = take(at, p.e == 2 && !p.two ? (size_t)p.piece * 8 : 0);
  b.bytes = at;
  return b;
}

// where dbias keeps what the rounding of dz takes off the targets' entries; null where there is no need
static long long* rest_of(const Plan& p, const BwdSpace& b, char* ws, const void* dbias) {
  return dbias && p.e == 2 && !p.two ? (long long*)(ws + b.rest) : nullptr;
}

template <class T>
static void backward_products(const nif_head_desc* h, const Plan& p, const char* state, char* ws, const BwdSpace& b, void* dhidden,
                              int64_t lddh, void* dweight, int64_t lddw, void* dbias, hipStream_t st) {
  const int* count = (const int*)(state + p.s_count);
  const int* rows = (const int*)(state + p.s_rows);
  const void* hp = state + p.s_h;
  const Targets tg = targets_of(h, p, (char*)state);
  const float* tops = (const float*)(state + p.s_top);
  const float* zk = (const float*)(state + p.s_zk);
  const float* coef = (const float*)(ws + b.coef);
  const float* cp = (const float*)(ws + b.cp);
  const float* inv_scale = (const float*)(ws + b.scale);
  typedef typename T::t W;
  W* dz = (W*)(ws + b.dz);
  float* acc = (float*)(ws + b.acc);
  float* part = (float*)(ws + b.part);
  long long* rest = rest_of(p, b, ws, dbias);
  const int f32 = h->dtype == NIF_F32;
  for (int v0 = 0; v0 < p.v; v0 += p.piece) {
    const int vc = p.v - v0 < p.piece ? p.v - v0 : p.piece;
    const bool first = v0 == 0, last = v0 + vc == p.v;
    const Side w = weight_side(h, p, v0, vc, p.pack_b, ws + b.w, st);
    const int kz = p.any_b ? vc : (int)round_up(vc, K_PAD);  // the contraction over the piece's columns of dz
    if (p.keep) {
      hipLaunchKernelGGL(head_kept_dz_kernel<T>, dim3((unsigned)round_up(p.n, K_PAD), (unsigned)((b.ldz + KEPT_DZ - 1) / KEPT_DZ)), dim3(256),
                         0, st, (const float*)(state + p.s_z), p.ldu, v0, vc, tg, rows, count, tops, coef, cp, dz, b.ldz,
                         p.two, rest, inv_scale);
    } else {
      GemmArgs g = {};
      g.A = w;
      g.B = Side{hp, p.ldd, (int)p.cap, p.ldd};
      g.M = vc;
      g.N = (int)round_up(p.n, K_PAD);
      g.n_dev = count;
      g.K = p.any_b ? p.d : p.ldd;
      g.splits = 1;
      g.bias = bias_at(h, v0);
      g.inv_tau = tg.inv_tau;
      g.top = tops;
      g.cp = cp;
      g.dz = dz;
      g.ldz = b.ldz;
      g.two = p.two;
      run_gemm<T, false, false, EPI_DZ>(p.two ? Shape{p.any_b, 128, 64, 4, 1, 0.f} : logit_shape(p, vc, p.any_b), g, st);
    }
    if (p.n > 0 && !p.keep)
      hipLaunchKernelGGL(head_targets_kernel<T>, row_grid((p.n + 3) / 4), dim3(256), 0, st, tg, rows, count, zk, tops, coef, cp, v0,
                       v0 + vc, dz, b.ldz, p.two, rest, inv_scale);
    if (dbias) {
      W* out = (W*)dbias + v0;
      const unsigned stretches = (unsigned)((p.n + b.stretch - 1) / b.stretch);
      if (p.n > 0)
        hipLaunchKernelGGL(head_bias_kernel<T>, dim3((vc + 255) / 256, stretches), dim3(256), 0, st, dz, b.ldz, vc, count, p.two, b.stretch, part,
                           inv_scale, out, rest);
      if (stretches != 1)
        hipLaunchKernelGGL(head_bias_join_kernel<T>, dim3((vc + 255) / 256), dim3(256), 0, st, part, vc, count, b.stretch, inv_scale, out, rest);
    }
    if (dweight) {  // [classes of the piece][features] = dz^T hidden, contraction over the packed rows
      GemmArgs g = {};
      g.A = Side{hp, p.ldd, p.ldd, (int)p.cap};
      g.B = Side{dz, b.ldz, (int)round_up(vc, K_PAD), (int)p.cap};
      g.M = p.d;
      g.N = vc;
      g.K = p.two ? 2 * p.two : (int)p.cap;
      g.k_dev = count;
      g.two = p.two;
      g.splits = b.dw.splits;
      g.out = (char*)dweight + (size_t)v0 * lddw * (f32 ? 4 : 2);
      g.out_ld = lddw;
      g.inv_scale = inv_scale;
      g.out_kind = OUT_FINAL;
      if (g.splits > 1) {
        g.out_kind = OUT_F32;
        g.acc = part;
        g.acc_ld = b.dh_ld;
        g.acc_split = (int64_t)p.piece * b.dh_ld;
      }
      run_gemm<T, true, true, EPI_OUT>(b.dw, g, st);
      if (g.splits > 1)
        hipLaunchKernelGGL(head_join_kernel<T>, row_grid(vc, (p.d + 1023) / 1024), dim3(256), 0, st, part, g.splits, g.acc_split, b.dh_ld, vc,
                           nullptr, p.d, nullptr, 1, 1, g.out, lddw, nullptr, inv_scale);
    }
    if (dhidden) {  // [packed rows][features] += dz W, contraction over the classes of the piece
      GemmArgs g = {};
      g.A = w;
      g.A.klim = w.rlim;
      g.A.rlim = p.pack_b ? p.ldd : p.d;
      g.B = Side{dz, b.ldz, (int)p.cap, kz};
      g.M = p.d;
      g.N = p.two ? 2 * p.two : (int)p.n;
      g.n_dev = p.two ? nullptr : count;
      g.K = kz;
      g.splits = b.dh.splits;
      g.out = dhidden;
      g.out_ld = lddh;
      g.rowmap = rows;
      g.inv_scale = inv_scale;
      const bool join = g.splits > 1 || p.two;  // the two parts' results are joined like splits, of which they are two each
      if (join) {
        g.out_kind = OUT_F32;
        g.acc = part;
        g.acc_split = b.part_rows * b.dh_ld;
      } else {
        g.out_kind = last ? OUT_FINAL : first ? OUT_F32 : OUT_ADD;
        g.acc = first && last ? nullptr : acc;
      }
      g.acc_ld = b.dh_ld;
      run_gemm<T, true, false, EPI_OUT>(b.dh, g, st);
      if (join && p.n > 0)
        hipLaunchKernelGGL(head_join_kernel<T>, row_grid(p.n, (p.d + 1023) / 1024), dim3(256), 0, st, part,
                           p.two ? 2 * g.splits : g.splits, p.two ? p.two * b.dh_ld : g.acc_split, b.dh_ld, (int)p.n, count, p.d, acc, first, last, dhidden, lddh, rows, inv_scale);
    }
  }
}

template <int DT>
static void small_forward(const nif_head_desc* h, const Plan& p, const Targets& tg, float* dz, float* row_loss, hipStream_t st) {
  if (p.v > 64)
    hipLaunchKernelGGL((head_small_forward_kernel<DT, 1024>), dim3((unsigned)p.n), dim3(1024), 0, st, *h, tg, dz, row_loss);
  else
    hipLaunchKernelGGL((head_small_forward_kernel<DT, 256>), dim3((unsigned)p.n), dim3(256), 0, st, *h, tg, dz, row_loss);
}

static int check_desc(const nif_head_desc* h, Plan& p) {
  if (!make_plan(h, p)) return NIF_ERR_INVALID_ARG;
  if (!h->weight || (h->rows > 0 && !h->hidden) || h->ldh < h->features || h->ldw < h->features) return NIF_ERR_INVALID_ARG;
  if (h->reduction < NIF_REDUCE_NONE || h->reduction > NIF_REDUCE_SUM) return NIF_ERR_INVALID_ARG;
  if (h->rows > 0) {
    if (!h->labels == !h->top_indices) return NIF_ERR_INVALID_ARG;  // one of the two
    if (h->labels && h->top != 0) return NIF_ERR_INVALID_ARG;
    if (!h->labels && (h->top < 1 || !h->top_values || !(h->temperature > 0.f) || !(h->temperature < INFINITY))) return NIF_ERR_INVALID_ARG;
  }
  return NIF_OK;
}

}  // namespace nif

extern "C" size_t nif_head_state_bytes(const nif_head_desc* h) {
  nif::Plan p;
  return nif::make_plan(h, p) ? p.state : 0;
}

extern "C" size_t nif_head_forward_workspace_bytes(const nif_head_desc* h) {
  nif::Plan p;
  return nif::make_plan(h, p) ? (p.small ? 0 : nif::forward_space(p).bytes) + (size_t)p.cap * 4 : 0;
}

extern "C" size_t nif_head_backward_workspace_bytes(const nif_head_desc* h) {
  nif::Plan p;
  return !nif::make_plan(h, p) ? 0 : p.small ? 256 : nif::backward_space(p).bytes;
}

extern "C" int nif_head_forward(const nif_head_desc* h, float* loss, void* state, size_t state_bytes, void* ws, size_t ws_bytes,
                                void* stream) {
  nif::Range nif_range_("nif_head_forward");
  using namespace nif;
  Plan p;
  const int rc = check_desc(h, p);
  if (rc != NIF_OK) return rc;
  if (!loss && (h->rows > 0 || h->reduction != NIF_REDUCE_NONE)) return NIF_ERR_INVALID_ARG;
  if (!state || state_bytes < nif_head_state_bytes(h) || !ws || ws_bytes < nif_head_forward_workspace_bytes(h)) return NIF_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  char* s = (char*)state;
  clear_err();
  if (p.small) {
    Targets tg = targets_of(h, p, s);
    float* row_loss = h->reduction == NIF_REDUCE_NONE ? loss : (float*)ws;
    float* dz = (float*)(s + p.s_dz);
    if (p.n > 0) {
      if (h->dtype == NIF_F32)
        small_forward<NIF_F32>(h, p, tg, dz, row_loss, st);
      else if (h->dtype == NIF_BF16)
        small_forward<NIF_BF16>(h, p, tg, dz, row_loss, st);
      else
        small_forward<NIF_F16>(h, p, tg, dz, row_loss, st);
    }
    if (h->reduction != NIF_REDUCE_NONE)
      launch_reduce(row_loss, tg.P, p.n, h->reduction == NIF_REDUCE_MEAN, (float*)(s + p.s_count), loss, st);
    return launch_ok() ? NIF_OK : NIF_ERR_LAUNCH;
  }
  const FwdSpace f = forward_space(p);
  int* rows = (int*)(s + p.s_rows);
  int* inv = (int*)(s + p.s_inv);
  int* count = (int*)(s + p.s_count);
  float* row_loss = h->reduction == NIF_REDUCE_NONE ? loss : (float*)((char*)ws + f.bytes);
  if (p.n > 0) {
    const Targets tg = targets_of(h, p, s);
    if (!h->labels) launch_targets(h->top_indices, h->top_values, h->top_lse, p.n, p.v, tg, st);
    hipLaunchKernelGGL(head_rows_kernel, dim3(1), dim3(1024), 0, st, tg, h->labels, h->ignore_index, p.v, p.n, rows, inv, count, row_loss);
    if (h->dtype == NIF_F32)
      pack_rows<NIF_F32>(h, p, s, st);
    else if (h->dtype == NIF_BF16)
      pack_rows<NIF_BF16>(h, p, s, st);
    else
      pack_rows<NIF_F16>(h, p, s, st);
    int tiles = 0;
    if (h->dtype == NIF_F32)
      forward_products<F32>(h, p, s, (char*)ws, f, tiles, st);
    else if (h->dtype == NIF_BF16)
      forward_products<Bf16>(h, p, s, (char*)ws, f, tiles, st);
    else
      forward_products<F16>(h, p, s, (char*)ws, f, tiles, st);
    const float2* stats = (const float2*)((char*)ws + f.stats);
    const auto finish = [&](auto each) {
      hipLaunchKernelGGL(head_finish_kernel<each>, row_grid((p.n + each - 1) / each), dim3(FINISH_NT), 0, st, stats, p.cap, tiles, tg,
                         rows, count, (float*)(s + p.s_top), (float*)(s + p.s_sum), (const float*)(s + p.s_zk), p.keep ? (const float*)(s + p.s_z) : nullptr,
                         p.ldu, row_loss, p.n, h->reduction, count + 1, loss);
    };
    if (p.n <= FINISH_FEW)
      finish(std::integral_constant<int, 2>());
    else
      finish(std::integral_constant<int, 16>());
  } else {
    hipLaunchKernelGGL(head_rows_kernel, dim3(1), dim3(1024), 0, st, targets_of(h, p, s), nullptr, (int64_t)0, p.v, (int64_t)0, rows, inv,
                       count, nullptr);
    if (h->reduction != NIF_REDUCE_NONE) launch_reduce(row_loss, nullptr, 0, false, nullptr, loss, st);
  }
  return launch_ok() ? NIF_OK : NIF_ERR_LAUNCH;
}

extern "C" int nif_head_backward(const nif_head_desc* h, const float* grad_loss, const void* state, size_t state_bytes, void* dhidden,
                                 int64_t lddh, void* dweight, int64_t lddw, void* dbias, void* ws, size_t ws_bytes, void* stream) {
  nif::Range nif_range_("nif_head_backward");
  using namespace nif;
  Plan p;
  const int rc = check_desc(h, p);
  if (rc != NIF_OK) return rc;
  if (h->forward_only || (p.n > 0 && !grad_loss) || (dhidden && lddh < h->features) || (dweight && lddw < h->features)) return NIF_ERR_INVALID_ARG;
  if (!state || state_bytes < nif_head_state_bytes(h) || !ws || ws_bytes < nif_head_backward_workspace_bytes(h)) return NIF_ERR_WORKSPACE;
  if (!dhidden && !dweight && !dbias) return NIF_OK;
  hipStream_t st = (hipStream_t)stream;
  const char* s = (const char*)state;
  clear_err();
  if (p.small) {
    const int stretches = (p.d + 63) / 64;
    const int hb = dhidden ? (int)p.n * stretches : 0, wb = dweight ? (p.v + 3) / 4 * stretches : 0;
    const int bb = !dweight && dbias ? (p.v + 3) / 4 * stretches : 0;
    if (hb + wb + bb == 0) return NIF_OK;
    const float* P = (const float*)(s + p.s_P);
    const float* dz = (const float*)(s + p.s_dz);
    const float* count = (const float*)(s + p.s_count);
    const auto launch = [&](auto dt) {
      const dim3 grid((unsigned)(hb + wb + bb));
      if (p.v > 256)  // long sums over the classes
        hipLaunchKernelGGL((head_small_backward_kernel<dt, 1024>), grid, dim3(1024), 0, st, *h, P, dz, count, grad_loss, dhidden, lddh,
                           dweight, lddw, dbias, hb, stretches);
      else
        hipLaunchKernelGGL((head_small_backward_kernel<dt, 256>), grid, dim3(256), 0, st, *h, P, dz, count, grad_loss, dhidden, lddh,
                           dweight, lddw, dbias, hb, stretches);
    };
    if (h->dtype == NIF_F32)
      launch(std::integral_constant<int, NIF_F32>());
    else if (h->dtype == NIF_BF16)
      launch(std::integral_constant<int, NIF_BF16>());
    else
      launch(std::integral_constant<int, NIF_F16>());
    return launch_ok() ? NIF_OK : NIF_ERR_LAUNCH;
  }
  const BwdSpace b = backward_space(p);
  const auto prepare = [&](auto* out) {
    const int64_t clearing = out && p.n > 0 ? (p.n + 3) / 4 : 0;
    long long* rest = rest_of(p, b, (char*)ws, dbias);
    hipLaunchKernelGGL(head_coef_kernel, row_grid(1 + clearing + (rest ? (p.piece + 1023) / 1024 : 0)), dim3(1024), 0, st, grad_loss, h->reduction == NIF_REDUCE_NONE,
                       h->reduction == NIF_REDUCE_MEAN, targets_of(h, p, (char*)s), (const int*)(s + p.s_rows), (const int*)(s + p.s_inv),
                       (const int*)(s + p.s_count), (const float*)(s + p.s_sum), p.n, h->dtype == NIF_F16, (float*)((char*)ws + b.coef), (float*)((char*)ws + b.cp),
                       (float*)((char*)ws + b.scale), out, lddh, p.d, clearing, rest, p.piece);
  };
  if (h->dtype == NIF_F32)
    prepare((float*)dhidden);
  else
    prepare((short*)dhidden);
  if (h->dtype == NIF_F32)
    backward_products<F32>(h, p, s, (char*)ws, b, dhidden, lddh, dweight, lddw, dbias, st);
  else if (h->dtype == NIF_BF16)
    backward_products<Bf16>(h, p, s, (char*)ws, b, dhidden, lddh, dweight, lddw, dbias, st);
  else
    backward_products<F16>(h, p, s, (char*)ws, b, dhidden, lddh, dweight, lddw, dbias, st);
  return launch_ok() ? NIF_OK : NIF_ERR_LAUNCH;
}
