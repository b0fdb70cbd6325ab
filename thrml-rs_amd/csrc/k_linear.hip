// k_linear.hip -- the product of a learned head in 8-bit integers: rows of
// activations, quantised with a scale each, times weights with a scale for each
// output channel.
//   s_r = max |x_r| (1 / 127),  a_r = round(x_r / s_r)   (ties to even)
//   y[r][c] = (sum_k a[r][k] w[c][k]) s_r w_scale[c] + bias[c]
// A subnormal scale is rounded up, so that |a| <= 127 (127 s >= max |x_r|).
// The sum is exact in 32-bit integers (k <= 131072).  A row of zeros has zeros
// for integers; a row with an infinity or a NaN has the scale NaN.  1 / 127 is rounded
// to 32 bits first, as torch on the device divides by a number: in one row of 22 a true
// quotient is a step off that, and now and then an integer with it.
#include "dev_util.hpp"
#include "head.hpp"

namespace thrml {

static inline uint32_t cdiv(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef int32_t i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int32_t i32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));

// Workspace: the scales of the rows, then their integers in rows of kp (k rounded
// up to 64, zeros behind k).
static inline uint32_t padded_k(uint32_t k) { return (k + 63u) & ~63u; }
static inline uint64_t scales_bytes(uint64_t rows) { return (rows * 4 + 255) & ~(uint64_t)255; }
// x / d, rounded to integers; |x| is at most 127 d but for roundings of d, so that the
// integers fit 8 bits and only d decides whether Divisor::fast is exact (a quotient below
// 2^-50 may be off and rounds to 0 either way).
__device__ __forceinline__ uint32_t integers4(const float *v, const Divisor &d) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= ((uint32_t)(int)rintf(d.plain ? d.fast(v[j]) : v[j] / d.b) & 255u) << (8 * j);
  return w;
}
template <class T>
__device__ __forceinline__ uint2 integers8(const Raw8<T> &r, const Divisor &d) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = value(r, j);
  return make_uint2(integers4(v, d), integers4(v + 4, d));
}
// A row's scale.  Where it is subnormal the product may lose up to all of its bits and
// leave quotients far above 127 (190 for a peak of 190 x 2^-149): such scales are rounded up.
__device__ __forceinline__ float scale_of(float peak) {
  const float s = peak * (1.0f / 127.0f);
  return s < 0x1p-126f && s * 127.0f < peak ? s + 0x1p-149f : s;
}
// a row's largest magnitude and whether it has an infinity or NaN
struct Peak {
  float m = 0.0f;
  int bad = 0;
  template <class T>
  __device__ __forceinline__ void take(const Raw8<T> &r) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = fabsf(value(r, j));
      bad |= !(v < INFINITY);
      m = fmaxf(m, v);
    }
  }
  __device__ __forceinline__ void join_wave() {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
    bad = __any(bad);
  }
};

template <class T>
__device__ __forceinline__ void load_x(const T *xr, uint32_t c, uint32_t k, Raw8<T> &r) {
  if (c + 8u <= k)
    load8(xr + c, r);
  else
    load8_part(xr + c, c < k ? k - c : 0u, r);
}

// A workgroup quantises one row; one of at most 8192 values stays in registers between
// its maximum and its integers.
template <class T>
__global__ __launch_bounds__(256) void quantise_kernel(const T *__restrict__ x, int64_t x_stride, uint64_t rows,
                                                       uint32_t k, uint32_t kp, float *__restrict__ scale,
                                                       int8_t *__restrict__ xq) {
  __shared__ float peak[4];
  __shared__ int bads[4];
  constexpr int KEPT = 4;
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + (int64_t)row * x_stride;
    Raw8<T> r[KEPT];
    Peak p;
#pragma unroll
    for (int g = 0; g < KEPT; ++g)
      if ((uint32_t)g * 2048u < kp) load_x(xr, (uint32_t)g * 2048u + threadIdx.x * 8u, k, r[g]);
#pragma unroll
    for (int g = 0; g < KEPT; ++g)
      if ((uint32_t)g * 2048u < kp) p.take(r[g]);
    for (uint32_t c = KEPT * 2048u + threadIdx.x * 8u; c < k; c += 2048u) {
      Raw8<T> t;
      load_x(xr, c, k, t);
      p.take(t);
    }
    p.join_wave();
    if ((threadIdx.x & 63u) == 0) {
      peak[threadIdx.x / 64u] = p.m;
      bads[threadIdx.x / 64u] = p.bad;
    }
    __syncthreads();
    const float m = fmaxf(fmaxf(peak[0], peak[1]), fmaxf(peak[2], peak[3]));
    const int bad = bads[0] | bads[1] | bads[2] | bads[3];
    const float s = scale_of(m);
    const Divisor d(s > 0.0f ? s : 1.0f);
    if (threadIdx.x == 0) scale[row] = bad ? __builtin_nanf("") : s;
    int8_t *o = xq + row * kp;
    auto put = [&](uint32_t c, const Raw8<T> &t) {
      if (c < kp) *reinterpret_cast<uint2 *>(o + c) = bad ? make_uint2(0, 0) : integers8(t, d);
    };
#pragma unroll
    for (int g = 0; g < KEPT; ++g)
      if ((uint32_t)g * 2048u < kp) put((uint32_t)g * 2048u + threadIdx.x * 8u, r[g]);
    for (uint32_t c = KEPT * 2048u + threadIdx.x * 8u; c < kp; c += 2048u) {
      Raw8<T> t;
      load_x(xr, c, k, t);
      put(c, t);
    }
    __syncthreads();
  }
}

// 16 weights of a row from column c0 on, any weights behind k (x is zero there): as
// they lie in memory up to `end`, the end of the last row's weights.
//
// ODD: rows that do not start at multiples of 4, for a wave that waits for its loads.
// A 16-byte load from such an address takes longer (27 x 7806 x 64: 18.7 us against 9.7 at
// k = 7808), so the words that hold them are loaded, 5 where they start within one, and
// shifted at their use (13 us).  Tiles through LDS take such loads as they are (1245 x 2834
// x 1467: 28 us, 39 by words).
template <bool ODD>
struct Weights16 {
  i32x4 w = {0, 0, 0, 0};
  int32_t next = 0;
  uint32_t shift = 0;
  __device__ __forceinline__ void load(const int8_t *wr, uint32_t c0, uint32_t k, const int8_t *end) {
    const int8_t *p = wr + c0;
    shift = ODD ? (uint32_t)(uintptr_t)p & 3u : 0u;
    if (p + (ODD ? 20 : 16) <= end) {
      if (ODD) {
        const i32x4_a4 *v = reinterpret_cast<const i32x4_a4 *>(p - shift);
        w = *v;
        next = reinterpret_cast<const int32_t *>(v)[shift ? 4 : 0];
      } else {
        w = *reinterpret_cast<const i32x4_a1 *>(p);
      }
    } else {
      w = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c0 + j < k) w[j / 4] |= (int32_t)((uint32_t)(uint8_t)p[j] << (8 * (j & 3)));
      shift = 0;
      next = 0;
    }
  }
  __device__ __forceinline__ i32x4 get() const {
    if (!ODD) return w;
    return i32x4{(int32_t)__builtin_amdgcn_alignbyte(w[1], w[0], shift), (int32_t)__builtin_amdgcn_alignbyte(w[2], w[1], shift),
                 (int32_t)__builtin_amdgcn_alignbyte(w[3], w[2], shift), (int32_t)__builtin_amdgcn_alignbyte(next, w[3], shift)};
  }
};
__device__ __forceinline__ const int8_t *weights_end(const LinearArgs &a) {
  return a.w + (int64_t)(a.q - 1u) * a.w_stride + a.k;
}

// ---------------------------------------------------------------------------
// Little work: the chain of loads is what it costs.  A workgroup takes 16 output
// channels and 16 rows; its four waves take turns in 64-column steps of k, straight
// from memory into the operand registers of v_mfma_i32_16x16x64_i8 (lane l: row l % 16,
// columns 16 (l / 16) .. + 15), U steps at a time, and their sums, exact integers, meet
// in LDS.  (More waves, or 32 x 32 tiles, were no faster where this kernel is taken; where
// there is much to read, its 64 neighbouring bytes a row at a time reach 4 TB/s
// against 6 through LDS.)
//
// OWN (at most 16 rows of at most 8192 values together): each workgroup quantises the
// rows itself, into LDS, while its first weights load: one launch for a call.  1: one
// row, by all waves, from registers; 2: a wave takes every fourth row.
constexpr uint32_t LF_WAVES = 4;
constexpr uint32_t OWN_GROUPS = 4;  // of 8 values a lane, for one row
constexpr uint32_t OWN_VALUES = OWN_GROUPS * 8 * 64 * LF_WAVES;
// (more than one row and many channels: tiles read the weights faster; 4 x 2048 x 40000
// takes 20 us with them, 25 so)
static bool own_rows(const thrml_ctx *ctx, uint64_t rows, uint32_t kp, uint32_t q) {
  return rows <= 16 && rows * kp <= OWN_VALUES && (rows == 1 || q <= 64u * (uint32_t)ctx->cu_count);
}

template <class T, class TO, int OWN, bool ODD>
__global__ __launch_bounds__(64 * LF_WAVES) void linear_few_kernel(LinearArgs a, const float *__restrict__ scale_,
                                                                   const int8_t *__restrict__ xq_, uint32_t kp) {
  __shared__ i32x4 part[LF_WAVES][64];
  __shared__ float own_peak[LF_WAVES];
  __shared__ int own_bad[LF_WAVES];
  __shared__ float own_scales[16];
  extern __shared__ __attribute__((aligned(16))) int8_t own_x[];
  const uint32_t l = threadIdx.x & 63u, wave = threadIdx.x / 64u, lo = l & 15u, hi = l >> 4;
  const uint32_t r0 = blockIdx.y * 16u, steps = kp / 64u, row = min(r0 + lo, (uint32_t)a.rows - 1u);
  const int8_t *end = weights_end(a);
  constexpr int U = 8;
  const int8_t *xr = OWN ? own_x + row * kp : xq_ + (uint64_t)row * kp;
  bool quantised = !OWN;
  float own_scale = 0.0f;
  for (uint32_t c0 = blockIdx.x * 16u; c0 < a.q; c0 += gridDim.x * 16u) {
    const int8_t *wr = a.w + (int64_t)min(c0 + lo, a.q - 1u) * a.w_stride;
    i32x4 acc = {};
    for (uint32_t s = wave; s < steps || !quantised; s += LF_WAVES * U) {
      Weights16<ODD> w[U];
      i32x4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t st = s + LF_WAVES * u, k0 = st * 64u + hi * 16u;
        if (st < steps)
          w[u].load(wr, k0, a.k, end);
        else
          w[u] = Weights16<ODD>{};
        if (!OWN) x[u] = st < steps ? *reinterpret_cast<const i32x4 *>(xr + k0) : i32x4{0, 0, 0, 0};
      }
      if constexpr (OWN == 2) {
        if (!quantised) {
          for (uint32_t i = wave; i < (uint32_t)a.rows; i += LF_WAVES) {
            const T *x_row = reinterpret_cast<const T *>(a.x) + (int64_t)i * a.x_stride;
            Peak p;
            for (uint32_t c = l * 8u; c < a.k; c += 512u) {
              Raw8<T> r;
              load_x(x_row, c, a.k, r);
              p.take(r);
            }
            p.join_wave();
            const float sx = scale_of(p.m);
            const Divisor d(sx > 0.0f ? sx : 1.0f);
            if (l == 0) own_scales[i] = p.bad ? __builtin_nanf("") : sx;
            for (uint32_t c = l * 8u; c < kp; c += 512u) {
              Raw8<T> r;
              load_x(x_row, c, a.k, r);
              *reinterpret_cast<uint2 *>(own_x + i * kp + c) = p.bad ? make_uint2(0, 0) : integers8(r, d);
            }
          }
          quantised = true;
          __syncthreads();
        }
      }
      if constexpr (OWN == 1) {
        if (!quantised) {
          Raw8<T> r[OWN_GROUPS];
          Peak p;
#pragma unroll
          for (uint32_t g = 0; g < OWN_GROUPS; ++g)
            if (g * 2048u < kp) load_x(reinterpret_cast<const T *>(a.x), g * 2048u + threadIdx.x * 8u, a.k, r[g]);
#pragma unroll
          for (uint32_t g = 0; g < OWN_GROUPS; ++g)
            if (g * 2048u < kp) p.take(r[g]);
          p.join_wave();
          if (l == 0) {
            own_peak[wave] = p.m;
            own_bad[wave] = p.bad;
          }
          __syncthreads();
          p.m = fmaxf(fmaxf(own_peak[0], own_peak[1]), fmaxf(own_peak[2], own_peak[3]));
          p.bad = own_bad[0] | own_bad[1] | own_bad[2] | own_bad[3];
          own_scale = p.bad ? __builtin_nanf("") : scale_of(p.m);
          const Divisor d(own_scale > 0.0f ? own_scale : 1.0f);
#pragma unroll
          for (uint32_t g = 0; g < OWN_GROUPS; ++g) {
            const uint32_t c = g * 2048u + threadIdx.x * 8u;
            if (c < kp) *reinterpret_cast<uint2 *>(own_x + c) = p.bad ? make_uint2(0, 0) : integers8(r[g], d);
          }
          quantised = true;
          __syncthreads();
        }
      }
      if constexpr (OWN != 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t st = s + LF_WAVES * u;
          x[u] = st < steps ? *reinterpret_cast<const i32x4 *>(xr + st * 64u + hi * 16u) : i32x4{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u].get(), x[u], acc, 0, 0, 0);
    }
    part[wave][l] = acc;
    __syncthreads();
    const uint32_t c = c0 + 4u * hi;
    if (wave == 0 && r0 + lo < a.rows && c < a.q) {
      i32x4 v = part[0][l];
#pragma unroll
      for (uint32_t o = 1; o < LF_WAVES; ++o) v += part[o][l];
      const float sx = OWN == 1 ? own_scale : OWN == 2 ? own_scales[row] : scale_[row];
      float f[4];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        // (the sum times a weight's scale first: a row's scale may be near the ends of f32)
        const uint32_t ci = min(c + i, a.q - 1u);
        f[i] = (float)v[i] * a.w_scale[ci] * sx;
        if (a.bias) f[i] = f[i] + a.bias[ci];
      }
      store4(reinterpret_cast<TO *>(a.y) + (int64_t)row * a.y_stride + c, a.q - c, f);
    }
    __syncthreads();  // the sums of the next channels
  }
}

// ---------------------------------------------------------------------------
// Many rows: tiles through LDS, v_mfma_i32_32x32x32_i8.
//
// A workgroup of WM x WN waves takes BM = 32 TM WM rows by BN = 32 TN WN
// channels; a stage is 64 columns of k of both operands, in LDS as rows of 64
// bytes whose four 16-byte pieces are permuted by the row (tile_swz), so that the
// 32 rows that a wave reads at a time fall on all banks.  A wave multiplies a stage
// in two halves of 32 columns, reading the next half's operands before it
// multiplies the present one's.
//
// DIRECT (weight rows at multiples of 16 bytes): stages are loaded straight into
// LDS, three ahead, with explicit waits; one barrier a stage, between the two
// halves of the one before, where the matrix unit has work queued.  Otherwise the
// pieces go through registers, one stage ahead.
//
// 4096 x 4096 x 16384 in tiles of 256 x 256: 283-300 us, 1.8-1.9 10^15 operations a second,
// as the vendor's int8 product of that shape (291 us).  The matrix unit is busy for half of
// 533 thousand cycles; the clock falls to 1.95 GHz under that load (on zeros, at 2.4 GHz, the
// same cycles take 227 us).  Tiles of 128 x 128 for each of four waves, three stages instead
// of four and a raised wave priority around the products were 2 to 9 % slower.
//
// A 16-byte LDS read takes 16 lanes at a time, four quads of lanes: 0, 3, 5, 6 of a half
// wave, then 1, 2, 4, 7; four rows of 64 bytes fill the banks, so that the rows r, r + 12,
// r + 20, r + 24 that meet have to differ in their permutation (by bits 1 and 2 of r
// instead, two and two met: 99 of 210 thousand LDS cycles per compute unit at 4096 x 4096
// x 16384).
__device__ __forceinline__ uint32_t tile_swz(uint32_t r) { return (r >> 3) & 3u; }

// lane l's 16 bytes from g to LDS address lds + 16 l (lds wave-uniform); counted by
// the explicit waits alone
__device__ __forceinline__ void to_lds16(const int8_t *g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(g), "s"(lds) : "memory", "m0");
}

// all but the last N of this wave's loads into LDS have ended, and so have its LDS
// reads; then every wave's
template <int N>
__device__ __forceinline__ void wait_loads_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "i"(N) : "memory");
}

template <int TM_, int TN_, int WM_, int WN_>
struct TileShape {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int STAGE = (BM + BN) * 64;           // bytes
  static constexpr int PIECES = STAGE / 16 / THREADS;    // 16-byte pieces of a stage per lane
  static_assert(PIECES * 16 * THREADS == STAGE, "a stage is whole pieces of every lane");
};

template <class S, class TO, bool DIRECT>
__global__ __launch_bounds__(S::THREADS) void linear_tile_kernel(LinearArgs a, const float *__restrict__ scale,
                                                                 const int8_t *__restrict__ xq, uint32_t kp,
                                                                 uint32_t tiles_m) {
  constexpr int TM = S::TM, TN = S::TN, BM = S::BM, PIECES = S::PIECES;
  constexpr uint32_t STAGES = DIRECT ? 4 : 2;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const uint32_t tid = threadIdx.x, l = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid / 64u);
  const uint32_t lo = l & 31u, hi = l >> 5;
  const uint32_t tile = xcd_remap(blockIdx.x, gridDim.x);
  const uint32_t r0 = (tile % tiles_m) * BM, c0 = (tile / tiles_m) * S::BN;
  const uint32_t steps = kp / 64u;

  // this lane's pieces: piece p of the stage is LDS bytes 16 (p THREADS + tid) ..,
  // row (p THREADS + tid) / 4, first the BM rows of x, then the BN of w
  const int8_t *src[PIECES];
  uint32_t col[PIECES];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const uint32_t e = (uint32_t)p * S::THREADS + tid, r = e / 4u;
    col[p] = ((e & 3u) ^ tile_swz(r)) * 16u;
    if (r < BM)
      src[p] = xq + (uint64_t)min(r0 + r, (uint32_t)a.rows - 1u) * kp;
    else
      src[p] = a.w + (int64_t)min(c0 + r - BM, a.q - 1u) * a.w_stride;
  }
  // wave-uniform: a wave's 16 rows of a piece are all x's or all w's
  auto is_x = [&](int p) { return ((uint32_t)p * S::THREADS + wave * 64u) / 4u < BM; };

  i32x16 acc[TM][TN] = {};
  i32x4 fx[2][TM], fw[2][TN];
  const uint32_t xrow = (wave / S::WN) * 32u * TM + lo, wrow = BM + (wave % S::WN) * 32u * TN + lo;
  auto read = [&](uint32_t base, int half, i32x4 (&vx)[TM], i32x4 (&vw)[TN]) {
    const uint32_t c = 2u * half + hi;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const uint32_t r = xrow + 32u * i;
      vx[i] = *reinterpret_cast<const i32x4 *>(lds + base + r * 64u + ((c ^ tile_swz(r)) * 16u));
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const uint32_t r = wrow + 32u * j;
      vw[j] = *reinterpret_cast<const i32x4 *>(lds + base + r * 64u + ((c ^ tile_swz(r)) * 16u));
    }
  };
  auto multiply = [&](const i32x4 (&vx)[TM], const i32x4 (&vw)[TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(vx[i], vw[j], acc[i][j], 0, 0, 0);
  };

  if constexpr (DIRECT) {
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    // (columns behind k: any weights, x is zero there)
    auto fetch = [&](uint32_t s) {
      const uint32_t k0 = s * 64u, base = lds0 + (s % STAGES) * S::STAGE + wave * 1024u;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const uint32_t k = k0 + col[p];
        to_lds16(src[p] + (is_x(p) || k < a.k ? k : 0u), base + (uint32_t)p * S::THREADS * 16u);
      }
    };
    // fetches past the end re-read the last stage, so that every wait counts alike
#pragma unroll
    for (uint32_t s = 0; s < STAGES - 1; ++s) {
      const uint32_t k0 = min(s, steps - 1u) * 64u, base = lds0 + s * S::STAGE + wave * 1024u;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const uint32_t k = k0 + col[p];
        to_lds16(src[p] + (is_x(p) || k < a.k ? k : 0u), base + (uint32_t)p * S::THREADS * 16u);
      }
    }
    wait_loads_barrier<(STAGES - 2) * PIECES>();
    read(0, 0, fx[0], fw[0]);
    for (uint32_t s = 0; s < steps; ++s) {
      const uint32_t base = (s % STAGES) * S::STAGE;
      read(base, 1, fx[1], fw[1]);
      // stage s + 3 takes the place of stage s - 1, which all waves have read
      // (their operands of its last half were in registers before the barrier below)
      if (s + STAGES - 1 < steps) {
        fetch(s + STAGES - 1);
      } else {
        const uint32_t b = lds0 + ((s + STAGES - 1) % STAGES) * S::STAGE + wave * 1024u;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) to_lds16(src[p], b + (uint32_t)p * S::THREADS * 16u);
      }
      multiply(fx[0], fw[0]);
      // the last reads of stage s have ended, stage s + 1 is in LDS
      wait_loads_barrier<(STAGES - 2) * PIECES>();
      read(((s + 1) % STAGES) * S::STAGE, 0, fx[0], fw[0]);  // (behind the last stage: not used)
      multiply(fx[1], fw[1]);
    }
    wait_loads_barrier<0>();
  } else {
    // (two stages ahead, in twice the registers, was no faster)
    Weights16<false> reg[PIECES];
    const int8_t *end = weights_end(a);
    auto load = [&](uint32_t s) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const uint32_t k = s * 64u + col[p];
        if (is_x(p))
          reg[p].w = *reinterpret_cast<const i32x4 *>(src[p] + k);
        else
          reg[p].load(src[p], k, a.k, end);
      }
    };
    auto put = [&](uint32_t s) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
        *reinterpret_cast<i32x4 *>(lds + (s & 1u) * S::STAGE + ((uint32_t)p * S::THREADS + tid) * 16u) = reg[p].get();
    };
    load(0);
    put(0);
    if (steps > 1) load(1);
    __syncthreads();
    for (uint32_t s = 0; s < steps; ++s) {
      const uint32_t base = (s & 1u) * S::STAGE;
      if (s + 1 < steps) put(s + 1);
      if (s + 2 < steps) load(s + 2);
      read(base, 0, fx[0], fw[0]);
      read(base, 1, fx[1], fw[1]);
      multiply(fx[0], fw[0]);
      multiply(fx[1], fw[1]);
      __syncthreads();
    }
  }
  __syncthreads();

  // Epilogue: a wave turns 32 rows x 32 TN channels at a time through its part of
  // LDS, so that it writes whole runs of a row: lane l has 4 channels of rows l /
  // (8 TN), ...
  constexpr uint32_t WB = 32u * TN, LPR = WB / 4u, RPI = 64u / LPR;  // channels, lanes per row, rows at a time
  int32_t *mine = reinterpret_cast<int32_t *>(lds) + wave * 32u * WB;
  const uint32_t cl = (l % LPR) * 4u, c = c0 + (wave % S::WN) * WB + cl;
  float ws[4], b[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    ws[i] = c + i < a.q ? a.w_scale[c + i] : 0.0f;
    b[i] = a.bias && c + i < a.q ? a.bias[c + i] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (uint32_t t = 0; t < 16; ++t)
        mine[(8u * (t / 4u) + 4u * hi + t % 4u) * WB + 32u * j + lo] = acc[i][j][t];
    __builtin_amdgcn_wave_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (uint32_t t = 0; t < 32u / RPI; ++t) {
      const uint32_t rl = t * RPI + l / LPR;
      const i32x4 v = *reinterpret_cast<const i32x4 *>(mine + rl * WB + cl);
      const uint32_t row = r0 + (wave / S::WN) * 32u * TM + 32u * i + rl;
      if (row < a.rows) {
        const float sx = scale[row];
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[e] = (float)v[e] * ws[e] * sx;
          if (a.bias) f[e] = f[e] + b[e];
        }
        store4(reinterpret_cast<TO *>(a.y) + (int64_t)row * a.y_stride + c, c < a.q ? a.q - c : 0u, f);
      }
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// weight rows at multiples of n bytes
static bool weights_at(const LinearArgs &a, uint32_t n) {
  return (a.q == 1 || a.w_stride % n == 0) && reinterpret_cast<uintptr_t>(a.w) % n == 0;
}

template <class S, class TO>
static int launch_tiles(thrml_ctx *ctx, const LinearArgs &a, const float *scale, const int8_t *xq, uint32_t kp) {
  const uint32_t tm = cdiv(a.rows, S::BM), tn = cdiv(a.q, S::BN);
  const bool direct = weights_at(a, 16) && a.k % 16u == 0;
  const size_t turn = (size_t)S::WAVES * 32 * 32 * S::TN * 4;
  const size_t lds = std::max<size_t>((direct ? 4 : 2) * (size_t)S::STAGE, turn);
  auto *f = direct ? &linear_tile_kernel<S, TO, true> : &linear_tile_kernel<S, TO, false>;
  if (lds > 65536)
    THRML_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(f), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(f, dim3(tm * tn), dim3(S::THREADS), lds, ctx->stream, a, scale, xq, kp, tm);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

template <class T, class TO, int OWN>
static int launch_few(thrml_ctx *ctx, const LinearArgs &a, const float *scale, const int8_t *xq, uint32_t kp) {
  const dim3 grid(std::min(cdiv(a.q, 16), 1u << 20), cdiv(a.rows, 16));
  auto *f = weights_at(a, 4) ? &linear_few_kernel<T, TO, OWN, false> : &linear_few_kernel<T, TO, OWN, true>;
  hipLaunchKernelGGL(f, grid, dim3(64 * LF_WAVES), OWN ? a.rows * kp : 0, ctx->stream, a, scale, xq, kp);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

uint64_t linear_i8_work(thrml_ctx *ctx, uint64_t rows, uint32_t k, uint32_t q) {
  return own_rows(ctx, rows, padded_k(k), q) ? 0 : scales_bytes(rows) + rows * padded_k(k);
}

int launch_linear_i8(thrml_ctx *ctx, const LinearArgs &a, int dtype, int out_dtype, void *work) {
  if (a.rows == 0) return THRML_OK;
  const uint32_t kp = padded_k(a.k);
  // one launch (1 x 4096 x 32768, weights from memory: 33 us against 36 with the
  // quantisation's own launch and tiles)
  if (own_rows(ctx, a.rows, kp, a.q))
    return with_type(dtype, [&](auto ti) {
      return with_type(out_dtype, [&](auto to) {
        return a.rows == 1 ? launch_few<decltype(ti), decltype(to), 1>(ctx, a, nullptr, nullptr, kp)
                           : launch_few<decltype(ti), decltype(to), 2>(ctx, a, nullptr, nullptr, kp);
      });
    });
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
    // The kind of tile by an estimate of each one's time: steps of k, and about 6 more
    // for beginning and end, at its time for a step, which is that of a tile alone on a
    // compute unit or, where a unit has several, their number times that of one of many.
    // In us a step, measured (alone / of many): 16 x 16 without LDS 0.078 / 0.063, 64 x 64
    // 0.195 / 0.164, 64 x 128 0.21 / 0.25, 128 x 256 0.45 / 0.67, 256 x 256 0.69 / 1.13.
    // The kind taken and the next best of calls (us, quantisation included):
    //    65 x 1000 x 700     16 x 16: 8      64 x 64: 14     512 x 4096 x 4096   64 x 128: 25    64 x 64: 27
    //   128 x 8192 x 512     16 x 16: 16     64 x 64: 29    2000 x 8192 x 4096  128 x 256: 93  256 x 256: 112
    //     4 x 2048 x 40000   64 x 64: 19     16 x 16: 21    4096 x 1000 x 65536 256 x 256: 512 128 x 256: 585
    struct Kind {
      uint32_t bm, bn;
      float alone, many;
    };
    static constexpr Kind kinds[] = {
        {16, 16, 0.078f, 0.063f}, {64, 64, 0.195f, 0.164f}, {64, 128, 0.21f, 0.25f}, {128, 256, 0.45f, 0.67f}, {256, 256, 0.69f, 1.13f}};
    int best = 0;
    double best_t = 0.0;
    for (int i = 0; i < 5; ++i) {
      const uint64_t tiles = (uint64_t)cdiv(a.rows, kinds[i].bm) * cdiv(a.q, kinds[i].bn);
      const double t = std::max<double>(kinds[i].alone, (double)kinds[i].many * (double)cdiv(tiles, ctx->cu_count));
      if (i == 0 || t < best_t) {
        best = i;
        best_t = t;
      }
    }
    switch (best) {
      case 0: return launch_few<float, TO, 0>(ctx, a, scale, xq, kp);
      case 1: return launch_tiles<TileShape<1, 1, 2, 2>, TO>(ctx, a, scale, xq, kp);
      case 2: return launch_tiles<TileShape<1, 2, 2, 2>, TO>(ctx, a, scale, xq, kp);
      case 3: return launch_tiles<TileShape<2, 2, 2, 4>, TO>(ctx, a, scale, xq, kp);
      default: return launch_tiles<TileShape<4, 2, 2, 4>, TO>(ctx, a, scale, xq, kp);
    }
  });
}

}  // namespace thrml
