// head.hpp -- operators around a learned head over q categories: the launchers,
// and the device helpers that their kernels share.  Rows of bf16, f16 or f32
// values may start at any multiple of their element size: a lane loads 8
// neighbouring values as 16-byte pieces at the element's own alignment (global
// loads and stores need no more on gfx950).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "internal.hpp"

namespace thrml {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// thrml_logits with its pointers typed; a row's parameters that are NULL leave
// their step out.
struct LogitRows {
  const void *z;
  int64_t z_stride;
  uint64_t rows;
  uint32_t q;
  const int32_t *history;
  int64_t history_stride;
  uint32_t history_len;
  const int32_t *lengths, *prompt_lengths;
  const float *repetition, *presence, *frequency;
  const int32_t *bias_ids;
  const float *bias_values;
  int64_t bias_stride;
  uint32_t n_bias;
  const float *temperature;
  const uint32_t *mask;
  int64_t mask_stride;  // 0: one mask for all rows
};

struct DistillArgs {
  const void *z;
  int64_t z_stride;
  uint64_t rows;
  uint32_t q, k;
  const int32_t *ids;
  const float *teacher;
  int64_t ids_stride, teacher_stride;
  float tau;
  const float *weight;  // null: the loss alone
  float *loss;
  void *grad;
  int64_t grad_stride;
};

struct LinearArgs {
  const void *x;
  int64_t x_stride;
  uint64_t rows;
  uint32_t k, q;
  const int8_t *w;
  int64_t w_stride;
  const float *w_scale, *bias;
  void *y;
  int64_t y_stride;
};

constexpr uint32_t HEAD_MAX_HISTORY = (1u << 29) - 1;  // the counter bits of a table word
constexpr uint32_t DISTILL_MAX_K = 4096;               // candidates kept in LDS
constexpr uint32_t LINEAR_MAX_K = 131072;              // 127 * 128 * k stays below 2^31

int launch_process_logits(thrml_ctx *ctx, const LogitRows &a, int dtype, void *out, int out_dtype,
                          int64_t out_stride);
uint64_t sample_logits_work(thrml_ctx *ctx, uint64_t rows, uint32_t q);
int launch_sample_logits(thrml_ctx *ctx, const LogitRows &a, int dtype, const float *u, int64_t u_stride,
                         int32_t *index, float *logprob, void *work);
uint64_t distill_work(thrml_ctx *ctx, int dtype, uint64_t rows, uint32_t q);
int launch_distill(thrml_ctx *ctx, const DistillArgs &a, int dtype, void *work);
uint64_t linear_i8_work(thrml_ctx *ctx, uint64_t rows, uint32_t k, uint32_t q);
int launch_linear_i8(thrml_ctx *ctx, const LinearArgs &a, int dtype, int out_dtype, void *work);

// ---------------------------------------------------------------------------
// Device helpers
template <class T>
struct Raw8 {  // 8 values as they lie in memory
  static constexpr int W = (int)sizeof(T) * 2;
  uint32_t w[W];
};

typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
template <class T>
struct Vec4 {
  typedef std::conditional_t<sizeof(T) == 2, u32x4_a2, u32x4_a4> type;
};

template <class T>
__device__ __forceinline__ void load8(const T *p, Raw8<T> &r) {
  const typename Vec4<T>::type *v = reinterpret_cast<const typename Vec4<T>::type *>(p);
#pragma unroll
  for (int i = 0; i < Raw8<T>::W / 4; ++i) {
    const typename Vec4<T>::type t = v[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) r.w[4 * i + j] = t[j];
  }
}

// n where it is used: its comparisons are made there and not kept in registers from
// far before
__device__ __forceinline__ uint32_t here(uint32_t n) {
  asm volatile("" : "+v"(n));
  return n;
}

// vmcnt(0), once in a loop over rows where nothing is under way any more.  The compiler,
// with a load and its use under conditions of their own, takes the load to be under way
// still at the next row, and there puts a wait before every load.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// p[0 .. n-1], and the bits `fill` for the rest, n < 8
template <class T>
__device__ __forceinline__ void load8_part(const T *p, uint32_t n_, Raw8<T> &r, uint32_t fill = 0) {
  const uint32_t n = here(n_);
#pragma unroll
  for (int i = 0; i < Raw8<T>::W; ++i) r.w[i] = sizeof(T) == 4 ? fill : fill | fill << 16;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j)
    if (j < n) {
      if constexpr (sizeof(T) == 4) {
        r.w[j] = __builtin_bit_cast(uint32_t, p[j]);
      } else {
        const uint32_t b = __builtin_bit_cast(uint16_t, p[j]);
        r.w[j / 2] = (j & 1u) ? (r.w[j / 2] & 0xffffu) | b << 16 : (r.w[j / 2] & 0xffff0000u) | b;
      }
    }
}

template <class T>
__device__ __forceinline__ float value(const Raw8<T> &r, int j) {
  if constexpr (sizeof(T) == 4)
    return __builtin_bit_cast(float, r.w[j]);
  else if constexpr (__is_same(T, bf16_t))
    return __builtin_bit_cast(float, (j & 1) ? r.w[j / 2] & 0xffff0000u : r.w[j / 2] << 16);
  else
    return (float)__builtin_bit_cast(f16_t, (uint16_t)(r.w[j / 2] >> (16 * (j & 1))));
}

// N values rounded to nearest, ties to even, as they lie in memory
template <class T, int N>
struct Rounded {
  uint32_t w[N * (int)sizeof(T) / 4];
};
template <class T, int N>
__device__ __forceinline__ Rounded<T, N> rounded(const float (&v)[N]) {
  Rounded<T, N> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < N; ++j) r.w[j] = __builtin_bit_cast(uint32_t, v[j]);
  } else {
    typedef T pair __attribute__((ext_vector_type(2)));
    typedef float fpair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const fpair f = {v[j], v[j + 1]};
      r.w[j / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, pair));
    }
  }
  return r;
}

template <class T, int N>
__device__ __forceinline__ void store_part(T *p, uint32_t n_, const Rounded<T, N> &r) {
  const uint32_t n = here(n_);
#pragma unroll
  for (uint32_t j = 0; j < N; ++j)
    if (j < n) {
      if constexpr (sizeof(T) == 4)
        p[j] = __builtin_bit_cast(T, r.w[j]);
      else
        p[j] = __builtin_bit_cast(T, (uint16_t)(r.w[j / 2] >> (16u * (j & 1u))));
    }
}

// The first n (at most 8) of v to p.
template <class T>
__device__ __forceinline__ void store8(T *p, uint32_t n, const float (&v)[8]) {
  const Rounded<T, 8> r = rounded<T>(v);
  if (n >= 8) {
    typename Vec4<T>::type *o = reinterpret_cast<typename Vec4<T>::type *>(p);
#pragma unroll
    for (int i = 0; i < Raw8<T>::W / 4; ++i) o[i] = typename Vec4<T>::type{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]};
  } else {
    store_part<T, 8>(p, n, r);
  }
}

// The first n (at most 4) of v to p.
template <class T>
__device__ __forceinline__ void store4(T *p, uint32_t n, const float (&v)[4]) {
  const Rounded<T, 4> r = rounded<T>(v);
  if (n >= 4) {
    typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<u32x4_a4 *>(p) = u32x4_a4{r.w[0], r.w[1], r.w[2], r.w[3]};
    else
      *reinterpret_cast<u32x2_a2 *>(p) = u32x2_a2{r.w[0], r.w[1]};
  } else {
    store_part<T, 4>(p, n, r);
  }
}

// a / b for many a: q = a r with r = 1 / b rounded, and one step of the remainder,
// which an fma gives exactly, leave the correctly rounded quotient (Markstein 1990)
// for |b| within 2^-100 .. 2^100 and |a| from 2^-100 on, but for one within a step of
// overflow, and elsewhere one a step off it at most; infinities, zeros and NaN divide as
// they should.  5 operations instead of the 10 of a full division, in line.  Not for a b
// below 2^-128, whose reciprocal is infinite (0 would give NaN, small dividends infinities).
struct Divisor {
  float b, r, m;  // m: b, or 1 for an infinite one
  bool plain;     // b is within 2^-100 .. 2^100
  __device__ __forceinline__ explicit Divisor(float b_)
      : b(b_), r(1.0f / b_), m(__builtin_isinf(b_) ? 1.0f : b_), plain(b_ >= 0x1p-100f && b_ <= 0x1p100f) {}
  __device__ __forceinline__ bool fine() const { return !__builtin_isinf(r); }
  __device__ __forceinline__ float fast(float a) const {  // where fine()
    const float q = a * r;
    return __builtin_isinf(q) ? q : __builtin_fmaf(__builtin_fmaf(-q, m, a), r, q);
  }
  // r and m, the same in all lanes of the wave, in scalar registers (where it is called: b
  // has to be there)
  __device__ __forceinline__ void scalar() {
    r = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, r)));
    m = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, m)));
  }
};

// f(the element type of dtype); an unknown dtype is the caller's to refuse
template <class F>
int with_type(int dtype, F &&f) {
  if (dtype == THRML_DTYPE_BF16) return f(bf16_t{});
  if (dtype == THRML_DTYPE_F16) return f(f16_t{});
  return f(float{});
}

}  // namespace thrml
