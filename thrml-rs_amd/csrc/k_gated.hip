// k_gated.hip -- the hidden block of a learned head: h = act(z) u with z = x w_gate^T,
// u = x w_up^T, and its gradient,
//   dz = dh u act'(z), du = dh act(z)
//   dx = dz w_gate + du w_up,  dw_gate = dz^T x,  dw_up = du^T x.
//
// Operands are 16-bit, sums f32, on v_mfma_f32_32x32x16.  Forward is one product with a
// fused end: a tile has the same channels of both weights.  Backward is one pass that
// writes dz and du, rounded to 16 bits as operands of the two products behind it have to
// be (half a step of 2^-8 or 2^-11, as is every operand), and those products, whose
// operands lie across the reduction and are transposed on their way from LDS.
// z and u are kept between the two in f32 (rounded to 16 bits they would put as much error
// again into the gradients as dz, du and the results' own rounding have together: 3.1e-3 of the
// norm in bf16, not 2.4e-3; at 4096 x 8192 it would save 60 us of a step's 1450).
#include "tile.hpp"

namespace thrml {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <class T>
struct Frag;
template <>
struct Frag<bf16_t> {
  typedef bf16x8 type;
  __device__ static __forceinline__ f32x16 mul(type a, type b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<f16_t> {
  typedef f16x8 type;
  __device__ static __forceinline__ f32x16 mul(type a, type b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// ---------------------------------------------------------------------------
// The activation and its derivative

// The normal distribution function at z, and e = exp(-z^2 / 2), for gelu: below 0, where 1 +
// erf(z / sqrt 2) loses its bits, it is e Q(t) t with t = 1 / (1 + 0.345 |z|), above 0
// 1 less that of -z.  Q is the polynomial of degree 8 of least relative error over |z| up to 13.5 (2e-8;
// weighted least squares).  In all within (8 + 2 z^2) 2^-24 of its value, the second part from
// the rounded exponent; 0 from about z = -13.2 down.  A forward product of 4096 x 4096 x 8192
// takes 427 us with it, 435 with erff and 438 with erfcf.
__device__ __forceinline__ float normal_cdf(float z, float &e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(z), 0.345f, 1.0f));
  e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
  float q = -0.028427219f;
  q = __builtin_fmaf(q, t, 0.14548801f);
  q = __builtin_fmaf(q, t, -0.27156994f);
  q = __builtin_fmaf(q, t, 0.18761782f);
  q = __builtin_fmaf(q, t, -0.037870139f);
  q = __builtin_fmaf(q, t, 0.11190453f);
  q = __builtin_fmaf(q, t, 0.11721380f);
  q = __builtin_fmaf(q, t, 0.13802400f);
  q = __builtin_fmaf(q, t, 0.13761912f);
  q *= t * e;
  return z < 0.0f ? q : 1.0f - q;
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == THRML_ACT_RELU) return z < 0.0f ? 0.0f : z;  // (NaN stays)
  // (hardware exponential and reciprocal: the exponent is rounded, and its factor's 2^-26, so
  // that the value is off by (1.3 |z| + 8) 2^-24 of it at most, where it is rounded to 16
  // bits; with expf and a division the end of a tile took 17 of 200 thousand cycles.  0 from
  // about z = -88 down)
  if constexpr (ACT == THRML_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950f));
  float e;
  return z * normal_cdf(z, e);
}
template <int ACT>
__device__ __forceinline__ void act_both(float z, float &value, float &slope) {
  if constexpr (ACT == THRML_ACT_RELU) {
    value = z < 0.0f ? 0.0f : z;
    slope = z > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (ACT == THRML_ACT_SILU) {
    const float e = expf(-fabsf(z)), r = 1.0f / (1.0f + e);
    const float sig = z < 0.0f ? e * r : r, other = z < 0.0f ? r : e * r;  // sig and 1 - sig
    value = z * sig;
    slope = sig * (1.0f + z * other);
  } else {
    float e;
    const float cdf = normal_cdf(z, e);
    value = z * cdf;
    slope = cdf + z * e * 0.39894228f;
  }
}

// ---------------------------------------------------------------------------
// The products
enum { G_FORWARD = 0, G_INPUT = 1, G_WEIGHT = 2 };  // h; dx; dw_gate and dw_up

struct GatedTiles {
  const void *a0, *a1;  // G_FORWARD, G_INPUT: w_gate, w_up; G_WEIGHT: x
  const void *b;        // G_FORWARD: x; else dz and du, a row's du behind its dz
  const void *b_units;  // G_WEIGHT in f16: the same, where some passed the type's range
  uint64_t a_stride, b_stride;  // bytes
  uint64_t rows;        // of x
  uint32_t k, n;
  uint32_t np;          // columns from a row's dz to its du
  uint32_t ta, tb;      // tiles
  uint32_t splits, steps;  // of the reduction; stages in all
  bool small_b;         // side B stays in the caches
  // G_FORWARD: h and, unless null, z and u; G_INPUT: dx; G_WEIGHT: dw_gate and dw_up
  void *out, *out1, *out2;
  int64_t out_stride;   // elements
  float *part;          // sums of the splits, [split][row][column], in place of the above
  // f16 gradients: whether dz or du passed the type's range, and then the factors of dx's rows,
  // or of dw_gate's and, from np on, dw_up's
  const uint32_t *passed;
  const float *factor;
  // and what dz and du are computed from
  const f16_t *grad;
  int64_t grad_stride;
  const float *z, *u;
  int32_t act;
};

// dz and du of one unit
template <int ACT>
__device__ __forceinline__ void slopes(float dh, float z, float u, float &dz, float &du) {
  float value, slope;
  act_both<ACT>(z, value, slope);
  dz = dh * u * slope;
  du = dh * value;
}

// A gradient that comes out near f16's border (65520: what is rounded from there on is
// infinite) says nothing of which side it is on: the rounding of dz and du to 11 bits moved
// it by a rms of 0.4 2^-11 of a term times the root of the terms' number, 2e-4 of what is a
// typical result of its row.  Such results are summed again, dz and du in f32 and the sum in
// 64 bits.  Near is within 2^-10 of the border, or 2^-9 of a large result of the row's 64
// columns here, which is about 1.2 typical ones: 12 times the rms.  (Among 8 lanes'
// largest, the smaller one of pairs, the larger one of two pairs, the smaller one of those: a
// column that is far larger than the others does not make these near.)  Results far from
// the border pay comparisons: a step of 1021 x 2001 x 5003 takes 257 us with them
// and without.  One of 5 x 7040 x 8000 takes 280 where 1.5 % of the weights' gradients pass the
// border and 17 thousand are near it, 193 without these sums.
__device__ __forceinline__ void slopes_of(const GatedTiles &g, float dh, float z, float u, float &dz, float &du) {
  if (g.act == THRML_ACT_RELU)
    slopes<THRML_ACT_RELU>(dh, z, u, dz, du);
  else if (g.act == THRML_ACT_GELU)
    slopes<THRML_ACT_GELU>(dh, z, u, dz, du);
  else
    slopes<THRML_ACT_SILU>(dh, z, u, dz, du);
}

// One result by a workgroup of 256, of row `row` (G_WEIGHT: dw_up's come behind dw_gate's) and
// column c; the loads of U turns are under way together
template <int OP>
__device__ __forceinline__ double gated_again(const GatedTiles &g, uint32_t row, uint32_t c, double *part) {
  constexpr uint32_t U = 8;
  const bool up = OP == G_WEIGHT && row >= g.n;
  const uint64_t all = OP == G_WEIGHT ? g.rows : g.n;
  double sum = 0.0;
  for (uint64_t i0 = threadIdx.x; i0 < all; i0 += 256u * U) {
    float dh[U], z[U], u[U], a0[U], a1[U];
#pragma unroll
    for (uint32_t e = 0; e < U; ++e) {
      const uint64_t i = min(i0 + 256u * e, all - 1u), r = OP == G_WEIGHT ? i : row;
      const uint32_t unit = OP == G_WEIGHT ? (up ? row - g.n : row) : (uint32_t)i;
      auto operand = [&](const void *p) {
        return (float)*reinterpret_cast<const f16_t *>(reinterpret_cast<const uint8_t *>(p) + i * g.a_stride + c * 2ull);
      };
      dh[e] = (float)g.grad[(int64_t)r * g.grad_stride + unit];
      z[e] = g.z[r * g.n + unit];
      u[e] = g.u[r * g.n + unit];
      a0[e] = operand(g.a0);
      if (OP == G_INPUT) a1[e] = operand(g.a1);
    }
#pragma unroll
    for (uint32_t e = 0; e < U; ++e) {
      if (i0 + 256u * e >= all) break;
      float dz, du;
      slopes_of(g, dh[e], z[e], u[e], dz, du);
      if (OP == G_WEIGHT)
        sum += (double)(up ? du : dz) * (double)a0[e];
      else
        sum += (double)dz * (double)a0[e] + (double)du * (double)a1[e];
    }
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
  if ((threadIdx.x & 63u) == 0) part[threadIdx.x / 64u] = sum;
  __syncthreads();
  return (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ float larger_finite(float m, float v) {
  v = fabsf(v);
  return v < INFINITY ? fmaxf(m, v) : m;
}

constexpr float BORDER = 65520.0f;

// what a lane has seen of results: the largest, and how near one came to the border
struct Border {
  float most = 0.0f, nearest = INFINITY;
  template <bool FINITE>  // whether infinite ones do not count as large
  __device__ __forceinline__ void see(const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      most = FINITE ? larger_finite(most, v[e]) : fmaxf(most, fabsf(v[e]));
      nearest = fminf(nearest, fabsf(fabsf(v[e]) - BORDER));
    }
  }
  // whether a lane of the wave has seen one that is near; band: the distance that is, from
  // what 8 lanes have seen.  MIXED (in a join, where they may be of two rows): and half as far
  // from what this one has
  template <bool MIXED>
  __device__ __forceinline__ bool any_near(float &band) const {
    if (!__any(most >= 0.99f * BORDER)) return false;  // (a band over 0.01 of the border comes from one beyond it)
    float m = fminf(most, __shfl_xor(most, 1));
    m = fmaxf(m, __shfl_xor(m, 2));
    m = fminf(m, __shfl_xor(m, 4));
    band = fmaxf(0x1p-9f * m, 0x1p-10f * BORDER);
    if (MIXED) band = fmaxf(band, 0x1p-10f * most);
    return __any(nearest <= band);
  }
};

// which of 8 results are near, m of them that count (all lanes of the wave come here)
template <bool MIXED>
__device__ __forceinline__ uint32_t border_bits(const float (&v)[8], uint32_t m) {
  Border b;
  b.see<true>(v);  // (those of no column or row are as large as the others)
  float band;
  if (!b.any_near<MIXED>(band)) return 0;
  uint32_t bits = 0;
#pragma unroll
  for (uint32_t e = 0; e < 8; ++e) bits |= (uint32_t)(e < m && fabsf(fabsf(v[e]) - BORDER) <= band) << e;
  return bits;
}

// The results v of row `row` from column c on, of which m count (0 in a thread that has none),
// one after another: the few of a join.  All threads of the workgroup come here.
template <int OP>
__device__ __forceinline__ void settle_each(const GatedTiles &g, float (&v)[8], uint32_t m, uint32_t row, uint32_t c) {
  __shared__ double part[4];
  __shared__ uint32_t first, first_row, first_c;
  uint32_t bits = border_bits<true>(v, m);
  if (!__syncthreads_or(bits != 0)) return;
  do {
    if (threadIdx.x == 0) first = 256;
    __syncthreads();
    if (bits) atomicMin(&first, threadIdx.x);  // (which comes first does not change a sum)
    __syncthreads();
    const bool mine = first == threadIdx.x;
    const uint32_t at = mine ? (uint32_t)__builtin_ctz(bits) : 0u;
    if (mine) {
      first_row = row;
      first_c = c + at;
    }
    __syncthreads();
    const float sum = (float)gated_again<OP>(g, first_row, first_c, part);
    if (mine) {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) v[e] = e == at ? sum : v[e];
      bits &= bits - 1u;
    }
  } while (__syncthreads_or(bits != 0));
}

// Those of a wave's 32 rows (from row0 on, of `limit`) x MA columns (from c0 on) at the end of
// a tile, which lie in `mine` before their factors and have been stored: each lane sums one, 64
// at a time, of operands that come through LDS, DEEP of the reduction at a time: 32 rows' dz
// or du (dx: both) and MA columns of the other side.  The gradient of 4096 x 4096 x 8192 with 87 %
// of the weights' results infinite takes 7.7 ms (1.06 where none is near); each by the wave, it
// took 122.
template <int OP, int MA, uint32_t LPR>
__device__ __forceinline__ void settle_slab(const GatedTiles &g, bool passed, float *mine, uint64_t row0, uint32_t up, uint64_t limit,
                                            uint32_t c0, uint32_t cols, f16_t *out) {
  constexpr uint32_t PITCH = MA + 4, RPI = 64u / LPR, DEEP = 16, DP = 33, SIDES = OP == G_INPUT ? 2 : 1;
  static_assert(256u + SIDES * DEEP * (DP * 4u + MA * 2u) <= 32u * PITCH * 4u, "fits where the results were");
  const uint32_t l = here(threadIdx.x) & 63u;
  uint64_t marks = 0;
#pragma unroll 1
  for (uint32_t t = 0; t < 32u / RPI; ++t) {
    const uint32_t rl = t * RPI + l / LPR, cl = l % LPR * 8u;
    const uint64_t row = row0 + rl;
    const float f = passed && row < limit ? g.factor[row + up * g.np] : 1.0f;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = mine[rl * PITCH + cl + e] * f;
    marks |= (uint64_t)border_bits<false>(v, row < limit && c0 + cl < cols ? cols - c0 - cl : 0u) << (8u * t);
  }
  wait_loads<0>();  // (the stores of these results have ended)
  uint32_t *list = reinterpret_cast<uint32_t *>(mine);
  float *d = mine + 64;
  uint32_t *a = reinterpret_cast<uint32_t *>(d + SIDES * DEEP * DP);
  auto fence = [] {
    __builtin_amdgcn_wave_barrier();
    wait_reads();
  };
  while (__ballot(marks != 0)) {
    // the next 64 of the wave's
    uint32_t scan = (uint32_t)__popcll(marks);
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const uint32_t o = (uint32_t)__shfl_up((int)scan, s);
      if (l >= (uint32_t)s) scan += o;
    }
    const uint32_t total = min((uint32_t)__builtin_amdgcn_readlane((int)scan, 63), 64u);
    uint32_t at = scan - (uint32_t)__popcll(marks);
    fence();
    while (marks && at < 64u) {
      const uint32_t bit = (uint32_t)__builtin_ctzll(marks);
      marks &= marks - 1u;
      list[at++] = (bit / 8u * RPI + l / LPR) << 16 | (l % LPR * 8u + bit % 8u);
    }
    fence();
    const uint32_t code = list[min(l, total - 1u)], rl = code >> 16, cl = code & 0xffffu;
    const uint64_t all = OP == G_WEIGHT ? g.rows : g.n;
    double sum = 0.0;
    for (uint64_t i0 = 0; i0 < all; i0 += DEEP) {
      constexpr uint32_t D_TURNS = DEEP / 2, A_ROWS = 128 / MA, A_TURNS = DEEP / A_ROWS;
      float dh[D_TURNS], z[D_TURNS], u[D_TURNS];
      uint32_t w[SIDES][A_TURNS];
      // lanes along what is contiguous: units
      auto place = [&](uint32_t e, uint32_t &i, uint32_t &r) {  // of the reduction, of the rows
        i = OP == G_WEIGHT ? 2u * e + l / 32u : l % DEEP;
        r = OP == G_WEIGHT ? l % 32u : 4u * e + l / DEEP;
      };
#pragma unroll
      for (uint32_t e = 0; e < D_TURNS; ++e) {
        uint32_t i, r;
        place(e, i, r);
        const uint64_t red = min(i0 + i, all - 1u), own = min(row0 + r, limit - 1u);
        const uint64_t row = OP == G_WEIGHT ? red : own, unit = OP == G_WEIGHT ? own : red;
        dh[e] = (float)g.grad[(int64_t)row * g.grad_stride + (int64_t)unit];
        z[e] = g.z[row * g.n + unit];
        u[e] = g.u[row * g.n + unit];
      }
#pragma unroll
      for (uint32_t e = 0; e < A_TURNS; ++e) {
        const uint64_t red = min(i0 + e * A_ROWS + l / (MA / 2u), all - 1u);
        const uint32_t c = min(c0 + l % (MA / 2u) * 2u, ((g.k + 7u) & ~7u) - 2u);
        w[0][e] = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint8_t *>(g.a0) + red * g.a_stride + c * 2ull);
        if (SIDES == 2) w[1][e] = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint8_t *>(g.a1) + red * g.a_stride + c * 2ull);
      }
      fence();
#pragma unroll
      for (uint32_t e = 0; e < D_TURNS; ++e) {
        uint32_t i, r;
        place(e, i, r);
        float dz, du;
        slopes_of(g, dh[e], z[e], u[e], dz, du);
        d[i * DP + r] = OP == G_WEIGHT && up ? du : dz;
        if (SIDES == 2) d[(DEEP + i) * DP + r] = du;
      }
#pragma unroll
      for (uint32_t e = 0; e < A_TURNS; ++e)
#pragma unroll
        for (uint32_t o = 0; o < SIDES; ++o) a[(o * DEEP + e * A_ROWS) * (MA / 2u) + l] = w[o][e];
      fence();
      const uint32_t left = (uint32_t)min((uint64_t)DEEP, all - i0);
#pragma unroll
      for (uint32_t o = 0; o < SIDES; ++o)
#pragma unroll 4
        for (uint32_t i = 0; i < left; ++i)
          sum += (double)d[(o * DEEP + i) * DP + rl] * (double)(float)reinterpret_cast<const f16_t *>(a)[(o * DEEP + i) * MA + cl];
    }
    if (l < total) out[(int64_t)(row0 + rl) * g.out_stride + c0 + cl] = (f16_t)(float)sum;
  }
}

template <class S, int OP, class T, int ACT, bool PART>
__global__ __launch_bounds__(S::THREADS) void gated_tile_kernel(GatedTiles g) {
  constexpr bool A_CROSS = OP != G_FORWARD, B_CROSS = OP == G_WEIGHT;
  constexpr uint32_t HALF = OP == G_FORWARD ? S::NA / 2 : S::NA;  // channels of a tile
  constexpr int TA = S::MA / 32, TB = S::MB / 32, SLICES = S::KB / 32 / S::WK;
  constexpr uint32_t ROWS = S::KB / 2;  // reduction indices of a stage
  typedef typename Frag<T>::type V;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
  const uint32_t wk = wave / (S::WA * S::WB), wa = wave % (S::WA * S::WB) / S::WB, wb = wave % S::WB;
  uint32_t ia, ib;
  tile_place(blockIdx.x, gridDim.x, g.ta, g.tb, ia, ib);
  const uint32_t c0 = ia * HALF;
  // G_WEIGHT: the tiles of dw_up's rows come behind those of dw_gate's
  const uint32_t up = OP == G_WEIGHT && ib >= g.tb / 2u ? 1u : 0u;
  const uint64_t r0 = (uint64_t)(ib - up * (g.tb / 2u)) * S::NB;
  const uint32_t s0 = (uint32_t)((uint64_t)g.steps * blockIdx.y / g.splits);
  const uint32_t s1 = (uint32_t)((uint64_t)g.steps * (blockIdx.y + 1u) / g.splits);

  // (across, rows come in eights: k is padded to them, np is a multiple of 128)
  typedef Side<S, S::NA, A_CROSS> SideA;
  typedef Side<S, S::NB, B_CROSS> SideB;
  const SideA sa{(uint32_t)g.a_stride, OP == G_FORWARD ? g.n - 1u - c0 : ((g.k + 7u) & ~7u) - 1u - c0};
  const SideB sb{(uint32_t)g.b_stride, OP == G_WEIGHT ? (uint32_t)(g.np - 1u - r0) : (uint32_t)min(g.rows - 1u - r0, (uint64_t)S::NB)};
  // G_FORWARD: a wave's MA rows of side A are half w_gate's, half w_up's, the same channels
  static_assert(OP != G_FORWARD || S::MA / 2 % SideA::STEP == 0, "a piece is one weight's");
  auto a_first = [&](int p) { return OP == G_FORWARD ? (p * SideA::STEP) / S::MA * (S::MA / 2u) + p * SideA::STEP % (S::MA / 2u) : p * SideA::STEP; };
  auto b_first = [&](int p) { return p * SideB::STEP; };
  const uint32_t half_steps = g.steps / 2u;  // G_INPUT: the stages of w_gate
  const uint8_t *a0 = reinterpret_cast<const uint8_t *>(g.a0), *a1 = reinterpret_cast<const uint8_t *>(g.a1);
  const uint8_t *b0 = reinterpret_cast<const uint8_t *>(g.b);
  if constexpr (OP == G_WEIGHT && __is_same(T, f16_t))
    if (*g.passed) b0 = reinterpret_cast<const uint8_t *>(g.b_units);
  if (OP == G_FORWARD) {
    a0 += (uint64_t)c0 * g.a_stride;
    a1 += (uint64_t)c0 * g.a_stride;
  } else {
    a0 += (uint64_t)c0 * 2u;
    a1 += (uint64_t)c0 * 2u;
  }
  b0 += OP == G_WEIGHT ? (r0 + (uint64_t)up * g.np) * 2u : r0 * g.b_stride;
  // G_INPUT: the stage's number among its weight's
  auto in_half = [&](uint32_t s) { return OP == G_INPUT && s >= half_steps ? s - half_steps : s; };
  // what is left of the reduction: bytes of a row, or indices
  auto left = [&](uint32_t s) -> uint64_t {
    return OP == G_FORWARD ? (uint64_t)g.k * 2u - (uint64_t)s * S::KB
           : OP == G_INPUT ? (uint64_t)g.n - min((uint64_t)in_half(s) * ROWS, (uint64_t)g.n)
                           : g.rows - (uint64_t)s * ROWS;
  };
  auto whole = [&](uint32_t s) { return left(s) >= (OP == G_FORWARD ? S::KB : ROWS); };
  auto a_base = [&](uint32_t s) {
    return [&, s](int p) {
      const uint64_t at = A_CROSS ? (uint64_t)in_half(s) * ROWS * g.a_stride : (uint64_t)s * S::KB;
      if (OP == G_FORWARD) return (p * SideA::STEP % S::MA >= S::MA / 2u ? a1 : a0) + at;
      return (OP == G_INPUT && s >= half_steps ? a1 : a0) + at;
    };
  };
  auto b_base = [&](uint32_t s) {
    return [&, s](int) { return b0 + (B_CROSS ? (uint64_t)s * ROWS * g.b_stride : (uint64_t)s * S::KB); };
  };
  const uint32_t lds0 = lds_address(lds) + wave % (S::LOADERS / 64u) * 1024u;
  const uint32_t start = tile_start(ia, s1 - s0, g.small_b);
  auto ring = [&](uint32_t s) { return s + start < s1 ? s + start : s + start - (s1 - s0); };
  auto fetch_a = [&](uint32_t s_, uint32_t slot) {
    const uint32_t s = ring(s_);
    if (whole(s))
      sa.fetch(a_base(s), a_first, lds0 + S::a_at(slot));
    else
      sa.fetch_end(a_base(s), a_first, lds0 + S::a_at(slot), (uint32_t)left(s));
  };
  auto fetch_b = [&](uint32_t s_, uint32_t slot) {
    const uint32_t s = ring(s_);
    if (OP == G_INPUT || whole(s))  // (dz and du have zeros behind their ends)
      sb.fetch(b_base(s), b_first, lds0 + S::b_at(slot));
    else
      sb.fetch_end(b_base(s), b_first, lds0 + S::b_at(slot), (uint32_t)left(s));
  };

  V va[SLICES][TA], vb[SLICES][TB];
  f32x16 acc[TA][TB] = {};
  // 8 reduction indices of a slice of 16 (the lane's half of it) for 32 rows of a side, of
  // lane l
  auto take = [&](uint32_t l, uint32_t base, uint32_t ks) -> V {
    const uint32_t lo = l & 31u, hi = l >> 5;
    return *reinterpret_cast<const V *>(lds + base + lo * S::KB + (((2u * ks + hi) ^ tile_turn<S>(lo)) * 16u));
  };
  auto take_cross = [&](uint32_t l, uint32_t base, uint32_t pitch, uint32_t chunks, uint32_t chunk, uint32_t ks) -> V {
    const uint32_t q = (l & 15u) / 4u, turn = chunks >= 4 ? q : chunks == 2 ? q >> 1 : 0u;
    const uint32_t at = base + (16u * ks + 8u * (l >> 5) + q) * pitch + ((chunk ^ turn) * 64u) + (l >> 4 & 1u) * 32u + (l & 3u) * 8u;
    typedef __attribute__((address_space(3))) s16x4 *P;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lds + at));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lds + at + 4u * pitch));
    return __builtin_bit_cast(V, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto read = [&](uint32_t slot_a, uint32_t slot_b) {
    const uint32_t base = S::a_at(slot_a), base_b = S::b_at(slot_b), l = here(threadIdx.x) & 63u;
#pragma unroll
    for (int k = 0; k < SLICES; ++k) {
      const uint32_t ks = wk * SLICES + k;
#pragma unroll
      for (int i = 0; i < TA; ++i)
        va[k][i] = A_CROSS ? take_cross(l, base, S::NA * 2u, S::NA / 32, wa * TA + i, ks) : take(l, base + (wa * S::MA + 32u * i) * S::KB, ks);
#pragma unroll
      for (int j = 0; j < TB; ++j)
        vb[k][j] = B_CROSS ? take_cross(l, base_b, S::NB * 2u, S::NB / 32, wb * TB + j, ks) : take(l, base_b + (wb * S::MB + 32u * j) * S::KB, ks);
    }
  };
  auto multiply = [&]() {
#pragma unroll
    for (int k = 0; k < SLICES; ++k)
#pragma unroll
      for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) acc[i][j] = Frag<T>::mul(va[k][i], vb[k][j], acc[i][j]);
  };
  tile_loop<S, S::PB>(s0, s1, fetch_a, fetch_b, read, multiply, [] {});

  // The end: a wave turns 32 rows x MA columns at a time through its part of LDS, so that
  // 8 neighbouring columns come to a lane (rows are padded by 16 bytes: 16 lanes that write
  // together fall on all banks).
  constexpr uint32_t PITCH = S::MA + 4, LPR = HALF / S::WA / 8u, RPI = 64u / LPR;  // floats; lanes per row, rows at a time
  constexpr uint32_t PARTS = S::WA * S::WB;
  const uint32_t l = here(threadIdx.x) & 63u, lo = l & 31u, hi = l >> 5;
  float *mine = reinterpret_cast<float *>(lds) + (wave % PARTS) * 32u * PITCH;
  T *out = reinterpret_cast<T *>(up ? g.out1 : g.out);
  const uint64_t limit = OP == G_WEIGHT ? g.n : g.rows;  // rows of the output
  const uint32_t cols = OP == G_FORWARD ? g.n : g.k;
  const uint32_t cl = (l % LPR) * 8u, c = c0 + wa * (HALF / S::WA) + cl;
  constexpr bool SETTLE = !PART && OP != G_FORWARD && __is_same(T, f16_t);
  uint32_t passed = 0;
  if constexpr (SETTLE) passed = *g.passed;
#pragma unroll
  for (int j = 0; j < TB; ++j) {
    // (the waves that share a tile add their sums one after another)
    for (int turn = 0; turn < S::WK; ++turn) {
      if (S::WK == 1 || wk == (uint32_t)turn) {
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
          for (uint32_t q = 0; q < 4; ++q) {
            f32x4 *p = reinterpret_cast<f32x4 *>(mine + lo * PITCH + 32u * i + 8u * q + 4u * hi);
            f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            if (turn) v += *p;
            *p = v;
          }
      }
      if (S::WK > 1) __syncthreads();
    }
    __builtin_amdgcn_wave_barrier();
    wait_reads();
    if (S::WK == 1 || wk == 0) {
      Border seen;
#pragma unroll
      for (uint32_t t = 0; t < 32u / RPI; ++t) {
        const uint32_t rl = t * RPI + l / LPR;
        const uint64_t row = r0 + wb * S::MB + 32u * j + rl;
        const uint32_t m = row < limit && c < cols ? cols - c : 0u;
        if (!SETTLE && m == 0) continue;
        float v[8], w[8];
        const float *at = mine + rl * PITCH + cl;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = at[e];
          if (OP == G_FORWARD) w[e] = at[S::MA / 2 + e];
        }
        if constexpr (PART) {
          const uint64_t all = OP == G_WEIGHT ? 2ull * g.n : g.rows, vr = row + (uint64_t)up * g.n;
          float *to = g.part + ((uint64_t)blockIdx.y * all + vr) * (OP == G_FORWARD ? 2ull * g.n : g.k) + c;
          store8(to, m, v);
          if (OP == G_FORWARD) store8(to + g.n, m, w);
        } else if constexpr (OP == G_FORWARD) {
          const int64_t saved = (int64_t)row * g.n + c;
          if (g.out1) {
            store8(reinterpret_cast<float *>(g.out1) + saved, m, v);
            store8(reinterpret_cast<float *>(g.out2) + saved, m, w);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = act_value<ACT>(v[e]) * w[e];
          store8(out + (int64_t)row * g.out_stride + c, m, v);
        } else {
          if (SETTLE && passed) {
            const float f = row < limit ? g.factor[row + up * g.np] : 1.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= f;
          }
          if constexpr (SETTLE) {
            seen.see<false>(v);  // (those of no column, too: they repeat others)
            if (m == 0) continue;
          }
          store8(out + (int64_t)row * g.out_stride + c, m, v);
        }
      }
      if constexpr (SETTLE) {
        float band;
        if (seen.template any_near<false>(band))
          settle_slab<OP, S::MA, LPR>(g, passed != 0, mine, r0 + wb * S::MB + 32u * j, up, limit, c0 + wa * (HALF / S::WA), cols, out);
      }
    }
    if (S::WK > 1)
      __syncthreads();
    else
      __builtin_amdgcn_wave_barrier();
    wait_reads();
  }
}

// Few rows, operands at any alignment (tile.hpp): a workgroup takes 16 units and up to 32
// rows; its four waves take turns in the stages of 128 bytes, and their sums meet in LDS.
// One row of 4095 x 16384 in bf16: 75 us, by tiles from a copy 165 (50 at 4096); 32 of 4095 x
// 8192: 64, from a copy 83.
template <class T>
struct FewFrag;
template <>
struct FewFrag<bf16_t> {
  __device__ static __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct FewFrag<f16_t> {
  __device__ static __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

template <class T, int ACT, int ROWS16>
__global__ __launch_bounds__(256) void gated_few_kernel(GatedTiles g, int64_t gate_stride, int64_t up_stride, int64_t x_stride) {
  __shared__ f32x4 part[4][2][ROWS16][64];
  const uint32_t l = threadIdx.x & 63u, wave = threadIdx.x / 64u, lo = l & 15u, hi = l >> 4;
  const uint32_t c0 = blockIdx.x * 16u, c = min(c0 + lo, g.n - 1u), bytes = g.k * 2u, steps = (bytes + 127u) / 128u;
  const uint8_t *wg = reinterpret_cast<const uint8_t *>(g.a0) + (int64_t)c * gate_stride * 2;
  const uint8_t *wu = reinterpret_cast<const uint8_t *>(g.a1) + (int64_t)c * up_stride * 2;
  const uint8_t *x[ROWS16];
#pragma unroll
  for (int j = 0; j < ROWS16; ++j)
    x[j] = reinterpret_cast<const uint8_t *>(g.b) + (int64_t)min(16u * j + lo, (uint32_t)g.rows - 1u) * x_stride * 2;
  f32x4 z[ROWS16] = {}, u[ROWS16] = {};
#pragma unroll 2
  for (uint32_t s = wave; s < steps; s += 4u) {
    RowPiece a[2][2], b[ROWS16][2];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t at = s * 128u + hi * 16u + h * 64u;
      a[0][h].load(wg, at, bytes);
      a[1][h].load(wu, at, bytes);
#pragma unroll
      for (int j = 0; j < ROWS16; ++j) b[j][h].load(x[j], at, bytes);
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < ROWS16; ++j) {
        const u32x4 xs = b[j][h].get();
        z[j] = FewFrag<T>::mul(a[0][h].get(), xs, z[j]);
        u[j] = FewFrag<T>::mul(a[1][h].get(), xs, u[j]);
      }
  }
#pragma unroll
  for (int j = 0; j < ROWS16; ++j) {
    part[wave][0][j][l] = z[j];
    part[wave][1][j][l] = u[j];
  }
  __syncthreads();
  for (uint32_t j = wave; j < ROWS16; j += 4u) {
    f32x4 zs = part[0][0][j][l], us = part[0][1][j][l];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      zs += part[w][0][j][l];
      us += part[w][1][j][l];
    }
    const uint32_t row = 16u * j + lo;
    const uint32_t cc = c0 + 4u * hi;
    if (row >= g.rows || cc >= g.n) continue;
    float v[4], w[4], h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = zs[e];
      w[e] = us[e];
      h[e] = act_value<ACT>(v[e]) * w[e];
    }
    const int64_t saved = (int64_t)row * g.n + cc;
    if (g.out1) {
      store4(reinterpret_cast<float *>(g.out1) + saved, g.n - cc, v);
      store4(reinterpret_cast<float *>(g.out2) + saved, g.n - cc, w);
    }
    store4(reinterpret_cast<T *>(g.out) + (int64_t)row * g.out_stride + cc, g.n - cc, h);
  }
}

// The sums of the splits, added in their order.
__host__ __device__ static inline uint32_t join_groups(uint64_t all) { return all < 65536u ? 32u : 256u; }

template <int OP, class T, int ACT>
__global__ __launch_bounds__(256) void gated_join_kernel(GatedTiles g) {
  const uint32_t cols = OP == G_FORWARD ? g.n : g.k, groups = (cols + 7u) / 8u;
  const uint64_t rows = OP == G_WEIGHT ? 2ull * g.n : g.rows, pitch = OP == G_FORWARD ? 2ull * g.n : g.k;
  constexpr bool SETTLE = OP != G_FORWARD && __is_same(T, f16_t);
  // SETTLE: whole workgroups, of few groups each where there are few, so that their long sums are
  // in many; threads behind the end repeat the last group and store nothing
  const uint64_t all = rows * groups;
  const uint32_t own = SETTLE ? join_groups(all) : 256u;
  for (uint64_t at = (uint64_t)blockIdx.x * own; at < all; at += (uint64_t)gridDim.x * own) {
    const uint64_t i_ = at + threadIdx.x, i = SETTLE ? min(i_, min(at + own, all) - 1u) : i_;
    if (!SETTLE && i >= all) break;
    const uint64_t row = i / groups;
    const uint32_t c = (uint32_t)(i - row * groups) * 8u, m = cols - c;
    float v[8], w[8];
    const float *p = g.part + row * pitch + c;
    join8(p, rows * pitch, g.splits, m, v);
    if (OP == G_FORWARD) join8(p + g.n, rows * pitch, g.splits, m, w);
    if constexpr (SETTLE) {
      const float f = *g.passed ? g.factor[OP == G_WEIGHT && row >= g.n ? row - g.n + g.np : row] : 1.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= f;
      settle_each<OP>(g, v, i == i_ ? m : 0u, (uint32_t)row, c);
      if (i != i_) continue;
    }
    if constexpr (OP == G_FORWARD) {
      const int64_t saved = (int64_t)row * g.n + c;
      if (g.out1) {
        store8(reinterpret_cast<float *>(g.out1) + saved, m, v);
        store8(reinterpret_cast<float *>(g.out2) + saved, m, w);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = act_value<ACT>(v[e]) * w[e];
      store8(reinterpret_cast<T *>(g.out) + (int64_t)row * g.out_stride + c, m, v);
    } else if constexpr (OP == G_INPUT) {
      store8(reinterpret_cast<T *>(g.out) + (int64_t)row * g.out_stride + c, m, v);
    } else {
      T *out = reinterpret_cast<T *>(row < g.n ? g.out : g.out1);
      store8(out + (int64_t)(row < g.n ? row : row - g.n) * g.out_stride + c, m, v);
    }
  }
}

// dz and du from dh and the z and u that the forward pass kept (14 bytes a unit): rows of 2
// np elements, zeros behind the n of each half.  f16: each workgroup leaves the largest
// finite magnitude that it wrote.
constexpr uint32_t SLOPE_GROUPS = 2048;  // workgroups, with f16

// of the workgroup
__device__ __forceinline__ float slope_max(float m, float *shared) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) shared[threadIdx.x / 64u] = m;
  __syncthreads();
  return fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
}

template <class T, int ACT>
__global__ __launch_bounds__(256) void gated_slope_kernel(const T *__restrict__ grad, int64_t grad_stride,
                                                          const float *__restrict__ z, const float *__restrict__ u, uint64_t rows,
                                                          uint32_t n, uint32_t np, T *__restrict__ d, float *maxima) {
  constexpr bool SCALED = __is_same(T, f16_t);
  __shared__ float shared[4];
  float most = 0.0f;
  const uint32_t groups = np / 8u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < rows * groups; i += (uint64_t)gridDim.x * 256u) {
    const uint64_t row = i / groups;
    const uint32_t c = (uint32_t)(i - row * groups) * 8u;
    float a[8], b[8];
    if (c < n) {
      Raw8<T> rg;
      Raw8<float> rz, ru;
      const T *pg = grad + (int64_t)row * grad_stride + c;
      const float *pz = z + row * n + c, *pu = u + row * n + c;
      if (c + 8u <= n) {
        load8(pg, rg);
        load8(pz, rz);
        load8(pu, ru);
      } else {
        load8_part(pg, n - c, rg);
        load8_part(pz, n - c, rz);
        load8_part(pu, n - c, ru);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float dz, du;
        slopes<ACT>(value(rg, e), value(rz, e), value(ru, e), dz, du);
        // (behind the end: zeros)
        a[e] = c + e < n ? dz : 0.0f;
        b[e] = c + e < n ? du : 0.0f;
        if constexpr (SCALED) most = larger_finite(larger_finite(most, a[e]), b[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = b[e] = 0.0f;
    }
    T *o = d + row * 2u * np + c;
    store8(o, 8, a);
    store8(o + np, 8, b);
  }
  if constexpr (SCALED) {
    most = slope_max(most, shared);
    if (threadIdx.x == 0) maxima[blockIdx.x] = most;
  }
}

// f16 gradients that carry a loss scale may pass its 65504 in dz and du, where neither dh nor
// the results do.  Where one did (else this launch ends at once, 4.7 us), they are
// written once more, for dx with each row divided by a power of two that takes its
// largest below 2^15, and for dw_gate and dw_up, into d_units, with each unit's dz and du
// so: a result depends on its own row, or unit, and the others' sizes take none of its
// bits.  The products' results are multiplied by the powers.
__device__ __forceinline__ int passed_by(float largest) { return largest > 65504.0f ? ilogbf(largest) - 14 : 0; }

template <int ACT>
__global__ __launch_bounds__(256) void gated_rescale_kernel(const f16_t *__restrict__ grad, int64_t grad_stride,
                                                            const float *__restrict__ z, const float *__restrict__ u, uint64_t rows,
                                                            uint32_t n, uint32_t np, f16_t *__restrict__ d, f16_t *__restrict__ d_units,
                                                            const float *__restrict__ maxima, uint32_t groups, uint32_t *passed,
                                                            float *__restrict__ row_factor, float *__restrict__ unit_factor) {
  constexpr uint32_t COLS = 32, DEEP = 256 / COLS;  // units of a workgroup, rows at a time
  __shared__ float shared[4], tall[2][DEEP][COLS];
  float m = 0.0f;
  for (uint32_t i = threadIdx.x; i < groups; i += 256u) m = fmaxf(m, maxima[i]);
  m = slope_max(m, shared);
  if (blockIdx.x == 0 && threadIdx.x == 0) *passed = m > 65504.0f;
  if (!(m > 65504.0f)) return;
  auto pair = [&](uint64_t row, uint32_t c, float &dz, float &du) {
    slopes<ACT>((float)grad[(int64_t)row * grad_stride + c], z[row * n + c], u[row * n + c], dz, du);
  };
  float dz, du;
  // rows first, then units
  for (uint64_t item = blockIdx.x; item < rows + np / COLS; item += gridDim.x) {
    if (item < rows) {
      float most = 0.0f;
      auto units = [&](uint32_t c, float (&a)[8], float (&b)[8]) {
        Raw8<f16_t> rg;
        Raw8<float> rz, ru;
        const f16_t *pg = grad + (int64_t)item * grad_stride + c;
        const float *pz = z + item * n + c, *pu = u + item * n + c;
        if (c + 8u <= n) {
          load8(pg, rg);
          load8(pz, rz);
          load8(pu, ru);
        } else {
          load8_part(pg, n - c, rg);
          load8_part(pz, n - c, rz);
          load8_part(pu, n - c, ru);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          slopes<ACT>(value(rg, e), value(rz, e), value(ru, e), a[e], b[e]);
          if (c + e >= n) a[e] = b[e] = 0.0f;
        }
      };
      float a[8], b[8];
      for (uint32_t c = threadIdx.x * 8u; c < n; c += 2048u) {
        units(c, a, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = larger_finite(larger_finite(most, a[e]), b[e]);
      }
      const int down = passed_by(slope_max(most, shared));
      if (threadIdx.x == 0) row_factor[item] = ldexpf(1.0f, down);
      if (down == 0) continue;  // (written so already)
      const float f = ldexpf(1.0f, -down);
      for (uint32_t c = threadIdx.x * 8u; c < n; c += 2048u) {
        units(c, a, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] *= f;
          b[e] *= f;
        }
        f16_t *o = d + item * 2u * np + c;
        store8(o, 8, a);
        store8(o + np, 8, b);
      }
    } else {
      const uint32_t lo = threadIdx.x % COLS, hi = threadIdx.x / COLS, c = (uint32_t)(item - rows) * COLS + lo;
      float za = 0.0f, ua = 0.0f;
      if (c < n) {
#pragma unroll 4
        for (uint64_t row = hi; row < rows; row += DEEP) {
          pair(row, c, dz, du);
          za = larger_finite(za, dz);
          ua = larger_finite(ua, du);
        }
      }
      __syncthreads();
      tall[0][hi][lo] = za;
      tall[1][hi][lo] = ua;
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < DEEP; ++i) {
        za = fmaxf(za, tall[0][i][lo]);
        ua = fmaxf(ua, tall[1][i][lo]);
      }
      const int zd = passed_by(za), ud = passed_by(ua);
      if (hi == 0) {
        unit_factor[c] = ldexpf(1.0f, zd);
        unit_factor[np + c] = ldexpf(1.0f, ud);
      }
      const float zf = ldexpf(1.0f, -zd), uf = ldexpf(1.0f, -ud);
#pragma unroll 4
      for (uint64_t row = hi; row < rows; row += DEEP) {
        dz = du = 0.0f;
        if (c < n) pair(row, c, dz, du);
        f16_t *o = d_units + row * 2u * np + c;
        o[0] = (f16_t)(dz * zf);
        o[np] = (f16_t)(du * uf);
      }
    }
  }
}

// Rows of k elements to rows of kp, zeros behind k.
__global__ __launch_bounds__(256) void gated_pack_kernel(const uint16_t *__restrict__ x, int64_t stride, uint64_t rows, uint32_t k,
                                                         uint32_t kp, uint16_t *__restrict__ out) {
  const uint32_t groups = kp / 8u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < rows * groups; i += (uint64_t)gridDim.x * 256u) {
    const uint64_t row = i / groups;
    const uint32_t c = (uint32_t)(i - row * groups) * 8u;
    const f16_t *p = reinterpret_cast<const f16_t *>(x) + (int64_t)row * stride + c;
    Raw8<f16_t> r;
    if (c + 8u <= k)
      load8(p, r);
    else
      load8_part(p, c < k ? k - c : 0u, r);
    *reinterpret_cast<u32x4 *>(out + row * kp + c) = u32x4{r.w[0], r.w[1], r.w[2], r.w[3]};
  }
}

// n 16-bit zeros to each of a and b
__global__ __launch_bounds__(256) void gated_zero_kernel(uint16_t *a, uint16_t *b, uint64_t n) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256u) a[i] = b[i] = 0;
}

// ---------------------------------------------------------------------------
// Calls
static uint32_t padded(uint32_t n, uint32_t to) { return (n + to - 1u) / to * to; }

// rows that tiles load as they lie: whole 16-byte pieces, and 256 rows within 32 bits
static bool tile_rows(const void *p, int64_t stride, uint64_t rows, uint32_t k) {
  return k % 8u == 0 && reinterpret_cast<uintptr_t>(p) % 16u == 0 &&
         (rows <= 1 || (stride % 8 == 0 && stride < (1 << 22)));
}

// Taken and next best (us a call):
//    16 x 4096 x 8192   64 x 32: 23.7  64 x 64: 24.0               512 x 4096 x 8192  256 x 256: 81  128 x 128: 93
//    64 x 4096 x 8192   64 x 64: 25    64 x 32: 30                1024 x 2048 x 2048  128 x 128: 25   64 x 64: 33
//   300 x 8192 x 256    64 x 64 in 8 parts: 20  in one: 38        1024 x 4096 x 8192  256 x 256: 114  128 x 128: 178
// and of the gradient in x:
//  1024 x 1024 x 4096   128 x 128 in 4 parts: 39  64 x 64: 57     2048 x 4096 x 4096  256 x 256 in 2 parts: 145  in one: 178
static constexpr TileKind gated_kinds[] = {{64, 32, 256, 0.56f, 0.38f}, {64, 64, 128, 0.36f, 0.23f}, {128, 128, 128, 0.57f, 0.62f}, {256, 256, 128, 0.9f, 1.5f}};
// (stages of 256 bytes for the fewest rows: with 128, rows that are no whole lines have each
// line on two of them; one row of 4104 x 16384: 53 -> 49.5 us, of 4096 x 16384: 51.5 -> 47.  With 64
// rows such stages take 34 us for 38 at 3544 x 8192, but 38 for 31 at 4096 x 8192)
typedef TileShape<64, 32, 1, 1, 4, 256, 3, false> Tile32;
typedef TileShape<64, 32, 1, 2, 2, 128, 4, false> Tile64;
typedef TileShape<64, 64, 2, 2, 1, 128, 3, false> Tile128;
typedef TileShape<128, 64, 2, 4, 1, 128, 2, true> Tile256;

struct GatedPlan {
  bool few;  // the forward pass reads the operands as they lie
  bool pack_x, pack_w;
  bool scaled;  // dz and du may pass the type's range
  uint32_t kp, np;
  // packed x, each packed weight, dz and du; f16: their maxima, whether one passed, and factors
  uint64_t x_bytes, w_bytes, d_bytes, m_bytes;
  TilePlan forward, input, weight;
  GatedPlan(const thrml_ctx *ctx, const thrml_gated &g) {
    // (whole lines of memory: rows of 7088 bytes take 34 us where rows of 7168 take 26, at 121 x
    // 3544 x 4952)
    kp = padded(g.k, 64);
    np = padded(g.n, 128);  // whole stages of each weight
    pack_x = !tile_rows(g.x, g.x_stride, g.rows, g.k);
    pack_w = !tile_rows(g.w_gate, g.gate_stride, g.n, g.k) || !tile_rows(g.w_up, g.up_stride, g.n, g.k) || (g.n > 1 && g.gate_stride != g.up_stride);
    x_bytes = pack_x ? tile_bytes(g.rows * kp * 2u) : 0;
    w_bytes = pack_w ? tile_bytes((uint64_t)g.n * kp * 2u) : 0;
    d_bytes = tile_bytes(g.rows * 2u * np * 2u);
    scaled = g.dtype == THRML_DTYPE_F16;
    m_bytes = scaled ? tile_bytes((SLOPE_GROUPS + 1 + g.rows + 2ull * np) * 4) : 0;
    few = (pack_x || pack_w) && g.rows <= 32;
    forward = plan_tiles(ctx, gated_kinds, 4, 2ull * g.n, g.rows, false, g.k * 2ull, g.rows * 2u * g.n);
    input = plan_tiles(ctx, gated_kinds, 4, g.k, g.rows, false, np * 4ull, g.rows * g.k);
    weight = plan_tiles(ctx, gated_kinds, 4, g.k, g.n, true, g.rows * 2ull, 2ull * g.n * g.k);
  }
};

uint64_t gated_work(thrml_ctx *ctx, const thrml_gated &g, bool backward) {
  const GatedPlan p(ctx, g);
  if (p.few && !backward) return 0;
  return p.x_bytes + 2 * p.w_bytes + (backward ? p.d_bytes * (p.scaled ? 2 : 1) + p.m_bytes + std::max(p.input.part, p.weight.part) : p.forward.part);
}

static int launch_pack(thrml_ctx *ctx, const void *x, int64_t stride, uint64_t rows, uint32_t k, uint32_t kp, void *out) {
  const uint64_t n = rows * (kp / 8u);
  hipLaunchKernelGGL(gated_pack_kernel, dim3((uint32_t)std::min<uint64_t>(tile_cdiv(n, 256), 1u << 16)), dim3(256), 0, ctx->stream,
                     reinterpret_cast<const uint16_t *>(x), stride, rows, k, kp, reinterpret_cast<uint16_t *>(out));
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

template <class S, int OP, class T, int ACT>
static int launch_kind(thrml_ctx *ctx, const GatedTiles &g) {
  const size_t lds = std::max<size_t>(S::BYTES, (size_t)S::WA * S::WB * 32 * (S::MA + 4) * 4);
  // (the sums of splits do not use the activation)
  auto *f = g.splits > 1 ? &gated_tile_kernel<S, OP, T, THRML_ACT_RELU, true> : &gated_tile_kernel<S, OP, T, ACT, false>;
  return launch_tiles(ctx, f, g, S::THREADS, lds);
}

template <int OP, class T, int ACT>
static int launch_product(thrml_ctx *ctx, const TilePlan &p, GatedTiles g) {
  g.ta = p.ta;
  g.tb = p.tb;
  g.splits = p.splits;
  g.steps = p.steps;
  g.small_b = OP == G_WEIGHT ? tile_small(g.rows, g.np * 4ull) : tile_small(g.rows, g.b_stride);
  int rc;
  switch (p.kind) {
    case 0: rc = launch_kind<Tile32, OP, T, ACT>(ctx, g); break;
    case 1: rc = launch_kind<Tile64, OP, T, ACT>(ctx, g); break;
    case 2: rc = launch_kind<Tile128, OP, T, ACT>(ctx, g); break;
    default: rc = launch_kind<Tile256, OP, T, ACT>(ctx, g); break;
  }
  if (rc || p.splits == 1) return rc;
  const uint64_t n = (OP == G_WEIGHT ? 2ull * g.n : g.rows) * tile_cdiv(OP == G_FORWARD ? g.n : g.k, 8);
  auto *f = &gated_join_kernel<OP, T, ACT>;
  const uint32_t own = OP != G_FORWARD && __is_same(T, f16_t) ? join_groups(n) : 256u;
  hipLaunchKernelGGL(f, dim3((uint32_t)std::min<uint64_t>(tile_cdiv(n, own), 1u << 16)), dim3(256), 0, ctx->stream, g);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

// f(an element, std::integral_constant of the activation)
template <class F>
static int with_gated(const thrml_gated &g, F &&f) {
  auto typed = [&](auto t) {
    if (g.act == THRML_ACT_RELU) return f(t, std::integral_constant<int, THRML_ACT_RELU>{});
    if (g.act == THRML_ACT_GELU) return f(t, std::integral_constant<int, THRML_ACT_GELU>{});
    return f(t, std::integral_constant<int, THRML_ACT_SILU>{});
  };
  return g.dtype == THRML_DTYPE_F16 ? typed(f16_t{}) : typed(bf16_t{});
}

// The operands as the tiles read them, packed into work where they have to be.
static int operands(thrml_ctx *ctx, const thrml_gated &g, const GatedPlan &p, uint8_t *&work, GatedTiles &t, const void *&x, uint64_t &x_stride) {
  t = GatedTiles{};
  t.rows = g.rows;
  t.k = g.k;
  t.n = g.n;
  t.np = p.np;
  x = g.x;
  x_stride = (uint64_t)(g.rows > 1 ? g.x_stride : p.kp) * 2u;
  if (p.pack_x) {
    if (int rc = launch_pack(ctx, g.x, g.x_stride, g.rows, g.k, p.kp, work)) return rc;
    x = work;
    x_stride = (uint64_t)p.kp * 2u;
    work += p.x_bytes;
  }
  t.a0 = g.w_gate;
  t.a1 = g.w_up;
  t.a_stride = (uint64_t)(g.n > 1 ? g.gate_stride : p.kp) * 2u;
  if (p.pack_w) {
    if (int rc = launch_pack(ctx, g.w_gate, g.gate_stride, g.n, g.k, p.kp, work)) return rc;
    if (int rc = launch_pack(ctx, g.w_up, g.up_stride, g.n, g.k, p.kp, work + p.w_bytes)) return rc;
    t.a0 = work;
    t.a1 = work + p.w_bytes;
    t.a_stride = (uint64_t)p.kp * 2u;
    work += 2 * p.w_bytes;
  }
  return THRML_OK;
}

int launch_gated(thrml_ctx *ctx, const thrml_gated &g, void *h, int64_t h_stride, float *gate, float *up, void *work) {
  if (g.rows == 0) return THRML_OK;
  const GatedPlan p(ctx, g);
  uint8_t *w = reinterpret_cast<uint8_t *>(work);
  GatedTiles t;
  if (p.few) {
    t = GatedTiles{};
    t.rows = g.rows;
    t.k = g.k;
    t.n = g.n;
    t.a0 = g.w_gate;
    t.a1 = g.w_up;
    t.b = g.x;
    t.out = h;
    t.out_stride = h_stride;
    t.out1 = gate;
    t.out2 = up;
    return with_gated(g, [&](auto e, auto act) -> int {
      typedef decltype(e) T;
      constexpr int ACT = decltype(act)::value;
      auto *f = g.rows <= 16 ? &gated_few_kernel<T, ACT, 1> : &gated_few_kernel<T, ACT, 2>;
      hipLaunchKernelGGL(f, dim3(tile_cdiv(g.n, 16)), dim3(256), 0, ctx->stream, t, g.gate_stride, g.up_stride, g.x_stride);
      THRML_HIP(hipGetLastError());
      return THRML_OK;
    });
  }
  const void *x;
  uint64_t x_stride;
  if (int rc = operands(ctx, g, p, w, t, x, x_stride)) return rc;
  t.b = x;
  t.b_stride = x_stride;
  t.out = h;
  t.out_stride = h_stride;
  t.out1 = gate;
  t.out2 = up;
  t.part = reinterpret_cast<float *>(w);
  return with_gated(g, [&](auto e, auto act) { return launch_product<G_FORWARD, decltype(e), decltype(act)::value>(ctx, p.forward, t); });
}

int launch_gated_grad(thrml_ctx *ctx, const thrml_gated &g, const void *grad, int64_t grad_stride, const float *gate,
                      const float *up, void *dx, int64_t dx_stride, void *dw_gate, void *dw_up, void *work) {
  if (g.rows == 0) {
    const uint64_t n = (uint64_t)g.n * g.k;
    hipLaunchKernelGGL(gated_zero_kernel, dim3((uint32_t)std::min<uint64_t>(tile_cdiv(n, 256), 1u << 16)), dim3(256), 0, ctx->stream,
                       reinterpret_cast<uint16_t *>(dw_gate), reinterpret_cast<uint16_t *>(dw_up), n);
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  }
  const GatedPlan p(ctx, g);
  uint8_t *w = reinterpret_cast<uint8_t *>(work);
  GatedTiles t;
  const void *x;
  uint64_t x_stride;
  if (int rc = operands(ctx, g, p, w, t, x, x_stride)) return rc;
  t.b = w;
  t.b_stride = (uint64_t)p.np * 4u;
  w += p.d_bytes;
  t.b_units = w;
  if (p.scaled) w += p.d_bytes;
  float *maxima = reinterpret_cast<float *>(w), *row_factor = maxima + SLOPE_GROUPS + 1, *unit_factor = row_factor + g.rows;
  uint32_t *passed = reinterpret_cast<uint32_t *>(maxima + SLOPE_GROUPS);
  t.passed = passed;
  t.grad = reinterpret_cast<const f16_t *>(grad);
  t.grad_stride = grad_stride;
  t.z = gate;
  t.u = up;
  t.act = g.act;
  w += p.m_bytes;
  t.part = reinterpret_cast<float *>(w);
  return with_gated(g, [&](auto e, auto act) -> int {
    typedef decltype(e) T;
    constexpr int ACT = decltype(act)::value;
    const uint64_t n = g.rows * (p.np / 8u);
    const dim3 grid((uint32_t)std::min<uint64_t>(tile_cdiv(n, 256), p.scaled ? SLOPE_GROUPS : 1u << 16));
    const T *dh = reinterpret_cast<const T *>(grad);
    T *d = reinterpret_cast<T *>(const_cast<void *>(t.b)), *d_units = reinterpret_cast<T *>(const_cast<void *>(t.b_units));
    hipLaunchKernelGGL((gated_slope_kernel<T, ACT>), grid, dim3(256), 0, ctx->stream, dh, grad_stride, gate, up, g.rows, g.n, p.np, d,
                       p.scaled ? maxima : nullptr);
    THRML_HIP(hipGetLastError());
    if constexpr (__is_same(T, f16_t)) {
      const dim3 items((uint32_t)std::min<uint64_t>(g.rows + p.np / 32u, SLOPE_GROUPS));
      hipLaunchKernelGGL((gated_rescale_kernel<ACT>), items, dim3(256), 0, ctx->stream, dh, grad_stride, gate, up, g.rows, g.n, p.np, d,
                         d_units, maxima, grid.x, passed, row_factor, unit_factor);
      THRML_HIP(hipGetLastError());
    }
    // (the products do not use the activation)
    if (dx) {
      GatedTiles i = t;
      i.factor = row_factor;
      i.out = dx;
      i.out_stride = dx_stride;
      if (int rc = launch_product<G_INPUT, T, THRML_ACT_RELU>(ctx, p.input, i)) return rc;
    }
    GatedTiles i = t;
    i.factor = unit_factor;
    i.a0 = i.a1 = x;
    i.a_stride = x_stride;
    i.out = dw_gate;
    i.out1 = dw_up;
    i.out_stride = g.k;
    return launch_product<G_WEIGHT, T, THRML_ACT_RELU>(ctx, p.weight, i);
  });
}

}  // namespace thrml
