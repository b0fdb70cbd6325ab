// k_linear.hip -- the product of a learned head in 8-bit integers: rows of
// activations, quantised with a scale each, times weights with a scale for each
// output channel.
//   s_r = max |x_r| / 127,  a_r = round(x_r / s_r)   (ties to even)
//   y[r][c] = (sum_k a[r][k] w[c][k]) s_r w_scale[c] + bias[c]
// The sum is exact in 32-bit integers (k <= 131072).  A row of zeros has zeros
// for integers; a row with an infinity or a NaN has the scale NaN.
#include "dev_util.hpp"
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

// ---------------------------------------------------------------------------
// Few rows: the weights are read once and that is what it costs.  A workgroup takes
// 16 CT output channels and all rows (16 RT of them at most); its four waves take
// every fourth 64-column step of k, so that together they read 256 neighbouring
// bytes of each weight row, straight into the operand registers of
// v_mfma_i32_16x16x64_i8 (lane l: row l % 16, columns 16 (l / 16) .. + 15), and
// their sums, exact integers, meet in LDS.
constexpr uint32_t LF_WAVES = 4;
constexpr uint32_t FEW_ROWS = 64;

template <class TO, int CT, int RT>
__global__ __launch_bounds__(64 * LF_WAVES) void linear_few_kernel(LinearArgs a, const float *__restrict__ scale,
                                                                   const int8_t *__restrict__ xq, uint32_t kp) {
  __shared__ i32x4 part[LF_WAVES][CT * RT][64];
  const uint32_t l = threadIdx.x & 63u, wave = threadIdx.x / 64u, lo = l & 15u, hi = l >> 4;
  for (uint32_t c0 = blockIdx.x * 16u * CT; c0 < a.q; c0 += gridDim.x * 16u * CT) {
    const int8_t *wr[CT], *xr[RT];
#pragma unroll
    for (int i = 0; i < CT; ++i) wr[i] = a.w + (int64_t)min(c0 + 16u * i + lo, a.q - 1u) * a.w_stride;
#pragma unroll
    for (int j = 0; j < RT; ++j) xr[j] = xq + (uint64_t)min(16u * j + lo, (uint32_t)a.rows - 1u) * kp;
    i32x4 acc[CT][RT] = {};
    // steps that lie within the weight rows, U at a time so that their loads are in
    // flight together
    constexpr int U = CT * RT <= 2 ? 8 : 4;
    const uint32_t whole = a.k / 64u, steps = kp / 64u;
    uint32_t s = wave;
    for (; s + LF_WAVES * (U - 1) < whole; s += LF_WAVES * U) {
      i32x4 w[U][CT], x[U][RT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t k0 = (s + LF_WAVES * u) * 64u + hi * 16u;
#pragma unroll
        for (int i = 0; i < CT; ++i) w[u][i] = *reinterpret_cast<const i32x4_a1 *>(wr[i] + k0);
#pragma unroll
        for (int j = 0; j < RT; ++j) x[u][j] = *reinterpret_cast<const i32x4 *>(xr[j] + k0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
          for (int j = 0; j < RT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][i], x[u][j], acc[i][j], 0, 0, 0);
    }
    for (; s < steps; s += LF_WAVES) {
      const uint32_t k0 = s * 64u + hi * 16u;
      i32x4 w[CT];
#pragma unroll
      for (int i = 0; i < CT; ++i) w[i] = load_w16(wr[i], k0, a.k);
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        const i32x4 x = *reinterpret_cast<const i32x4 *>(xr[j] + k0);
#pragma unroll
        for (int i = 0; i < CT; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x, acc[i][j], 0, 0, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < CT * RT; ++t) part[wave][t][l] = acc[t / RT][t % RT];
    __syncthreads();
#pragma unroll 1
    for (uint32_t t = wave; t < CT * RT; t += LF_WAVES) {
      i32x4 v = part[0][t][l];
#pragma unroll
      for (uint32_t o = 1; o < LF_WAVES; ++o) v += part[o][t][l];
      const uint32_t row = 16u * (t % RT) + lo, c = c0 + 16u * (t / RT) + 4u * hi;
      if (row < a.rows && c < a.q) {
        const float sx = scale[row];
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
__device__ __forceinline__ uint32_t tile_swz(uint32_t r) { return ((r >> 1) ^ (r >> 3)) & 3u; }

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
    i32x4 reg[PIECES];
    auto load = [&](uint32_t s) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const uint32_t k = s * 64u + col[p];
        if (is_x(p))
          reg[p] = *reinterpret_cast<const i32x4 *>(src[p] + k);
        else
          reg[p] = load_w16(src[p], k, a.k);
      }
    };
    auto put = [&](uint32_t s) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
        *reinterpret_cast<i32x4 *>(lds + (s & 1u) * S::STAGE + ((uint32_t)p * S::THREADS + tid) * 16u) = reg[p];
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

template <class S, class TO>
static int launch_tiles(thrml_ctx *ctx, const LinearArgs &a, const float *scale, const int8_t *xq, uint32_t kp) {
  const uint32_t tm = cdiv(a.rows, S::BM), tn = cdiv(a.q, S::BN);
  const bool direct = a.w_stride % 16 == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0 && a.k % 16u == 0;
  const size_t turn = (size_t)S::WAVES * 32 * 32 * S::TN * 4;
  const size_t lds = std::max<size_t>((direct ? 4 : 2) * (size_t)S::STAGE, turn);
  auto *f = direct ? &linear_tile_kernel<S, TO, true> : &linear_tile_kernel<S, TO, false>;
  if (lds > 65536)
    THRML_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(f), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(f, dim3(tm * tn), dim3(S::THREADS), lds, ctx->stream, a, scale, xq, kp, tm);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

template <class TO, int CT, int RT>
static int launch_few(thrml_ctx *ctx, const LinearArgs &a, const float *scale, const int8_t *xq, uint32_t kp) {
  hipLaunchKernelGGL((linear_few_kernel<TO, CT, RT>), dim3(std::min(cdiv(a.q, 16 * CT), 1u << 20)), dim3(64 * LF_WAVES), 0, ctx->stream, a,
                     scale, xq, kp);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

int launch_linear_i8(thrml_ctx *ctx, const LinearArgs &a, int dtype, int out_dtype, void *work) {
  if (a.rows == 0) return THRML_OK;
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
    if (a.rows <= 16) return launch_few<TO, 1, 1>(ctx, a, scale, xq, kp);
    if (a.rows <= 32) return launch_few<TO, 2, 2>(ctx, a, scale, xq, kp);
    if (a.rows <= 48) return launch_few<TO, 2, 3>(ctx, a, scale, xq, kp);
    if (a.rows <= FEW_ROWS) return launch_few<TO, 2, 4>(ctx, a, scale, xq, kp);
    const uint64_t cu = ctx->cu_count;
    if ((uint64_t)cdiv(a.rows, 256) * cdiv(a.q, 256) >= cu)
      return launch_tiles<TileShape<4, 2, 2, 4>, TO>(ctx, a, scale, xq, kp);
    if ((uint64_t)cdiv(a.rows, 128) * cdiv(a.q, 128) >= cu)
      return launch_tiles<TileShape<2, 2, 2, 2>, TO>(ctx, a, scale, xq, kp);
    return launch_tiles<TileShape<1, 1, 2, 2>, TO>(ctx, a, scale, xq, kp);
  });
}

}  // namespace thrml
