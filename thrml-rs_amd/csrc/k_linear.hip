// k_linear.hip -- the product of a learned head in 8-bit integers: rows of
// activations, quantised with a scale each, times weights with a scale for each
// output channel.
//   s_r = max |x_r| / 127,  a_r = round(x_r / s_r)   (ties to even)
//   y[r][c] = (sum_k a[r][k] w[c][k]) s_r w_scale[c] + bias[c]
// The sum is exact in 32-bit integers (k <= 131072).  A row of zeros has zeros
// for integers; a row with an infinity or a NaN has the scale NaN.
#include "head.hpp"

namespace thrml {

static inline uint32_t cdiv(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef int32_t i32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));

// Workspace: the scales of the rows, then their integers in rows of kp (k rounded
// up to 64, zeros behind k).
static inline uint32_t padded_k(uint32_t k) { return (k + 63u) & ~63u; }
static inline uint64_t scales_bytes(uint64_t rows) { return (rows * 4 + 255) & ~(uint64_t)255; }
uint64_t linear_i8_work(thrml_ctx *, uint64_t rows, uint32_t k, uint32_t) {
  return scales_bytes(rows) + rows * padded_k(k);
}

// A workgroup quantises one row.
template <class T>
__global__ __launch_bounds__(256) void quantise_kernel(const T *__restrict__ x, int64_t x_stride, uint64_t rows,
                                                       uint32_t k, uint32_t kp, float *__restrict__ scale,
                                                       int8_t *__restrict__ xq) {
  __shared__ float buf[4];
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + (int64_t)row * x_stride;
    float m = 0.0f;
    int bad = 0;
    for (uint32_t c = threadIdx.x * 8u; c < k; c += 2048u) {
      Raw8<T> r;
      if (c + 8u <= k)
        load8(xr + c, r);
      else
        load8_part(xr + c, k - c, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = fabsf(value(r, j));
        bad |= !(v < INFINITY);
        m = fmaxf(m, v);
      }
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
    if ((threadIdx.x & 63u) == 0) buf[threadIdx.x / 64u] = m;
    bad = __syncthreads_or(bad);
    m = fmaxf(fmaxf(buf[0], buf[1]), fmaxf(buf[2], buf[3]));
    const float s = m / 127.0f, d = s > 0.0f ? s : 1.0f;
    if (threadIdx.x == 0) scale[row] = bad ? __builtin_nanf("") : s;
    int8_t *o = xq + row * kp;
    for (uint32_t c = threadIdx.x * 8u; c < kp; c += 2048u) {
      Raw8<T> r;
      if (c + 8u <= k)
        load8(xr + c, r);
      else
        load8_part(xr + c, c < k ? k - c : 0u, r);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int v = bad ? 0 : (int)rintf(value(r, j) / d);
        w[j / 4] |= ((uint32_t)v & 255u) << (8 * (j & 3));
      }
      *reinterpret_cast<uint2 *>(o + c) = make_uint2(w[0], w[1]);
    }
    __syncthreads();
  }
}

// 16 weights from column c0 on; zeros behind k
__device__ __forceinline__ i32x4 load_w16(const int8_t *wr, uint32_t c0, uint32_t k) {
  if (c0 + 16u <= k) return *reinterpret_cast<const i32x4_a1 *>(wr + c0);
  i32x4 r = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (c0 + j < k) r[j / 4] |= (int32_t)((uint32_t)(uint8_t)wr[c0 + j] << (8 * (j & 3)));
  return r;
}

// A wave multiplies 32 output channels by 32 rows.
template <class TO>
__global__ __launch_bounds__(64) void linear_kernel(LinearArgs a, const float *__restrict__ scale,
                                                    const int8_t *__restrict__ xq, uint32_t kp) {
  const uint32_t l = threadIdx.x, lo = l & 31u, hi = l >> 5;
  const uint32_t c0 = blockIdx.x * 32u;
  for (uint64_t r0 = (uint64_t)blockIdx.y * 32u; r0 < a.rows; r0 += (uint64_t)gridDim.y * 32u) {
    const int8_t *wr = a.w + (int64_t)min(c0 + lo, a.q - 1u) * a.w_stride;
    const uint64_t row = min(r0 + lo, a.rows - 1u);
    const int8_t *xr = xq + row * kp;
    i32x16 acc = {};
    for (uint32_t k0 = 0; k0 < kp; k0 += 32u) {
      const i32x4 w = load_w16(wr, k0 + hi * 16u, a.k);
      const i32x4 x = *reinterpret_cast<const i32x4 *>(xr + k0 + hi * 16u);
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(w, x, acc, 0, 0, 0);
    }
    if (r0 + lo < a.rows) {
      const float s = scale[row];
      TO *y = reinterpret_cast<TO *>(a.y) + (int64_t)row * a.y_stride;
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        const uint32_t c = c0 + 8u * (i / 4u) + 4u * hi + i % 4u;
        if (c < a.q) {
          // (the sum times a weight's scale: a row's scale may be near the ends of f32)
          const float v = (float)acc[i] * a.w_scale[c] * s;
          y[c] = (TO)(a.bias ? v + a.bias[c] : v);
        }
      }
    }
  }
}

int launch_linear_i8(thrml_ctx *ctx, const LinearArgs &a, int dtype, int out_dtype, void *work) {
  if (a.rows == 0 || a.q == 0) return THRML_OK;
  const uint32_t kp = padded_k(a.k);
  float *scale = reinterpret_cast<float *>(work);
  int8_t *xq = reinterpret_cast<int8_t *>(work) + scales_bytes(a.rows);
  int rc = with_type(dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    hipLaunchKernelGGL((quantise_kernel<T>), dim3((uint32_t)std::min<uint64_t>(a.rows, 1u << 20)), dim3(256), 0,
                       ctx->stream, reinterpret_cast<const T *>(a.x), a.x_stride, a.rows, a.k, kp, scale, xq);
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
  if (rc) return rc;
  return with_type(out_dtype, [&](auto t) -> int {
    typedef decltype(t) TO;
    hipLaunchKernelGGL((linear_kernel<TO>), dim3(cdiv(a.q, 32), (uint32_t)std::min<uint64_t>(cdiv(a.rows, 32), 256)),
                       dim3(64), 0, ctx->stream, a, scale, xq, kp);
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
}

}  // namespace thrml
