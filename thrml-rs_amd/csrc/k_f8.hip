// k_f8.hip -- the product of a learned head in 8-bit floating point (e4m3), with a scale
// for each 128 of a row of activations and each 128 x 128 of the weights.
//   s[r][b] = max(2^-126, max |x[r][128 b ..]| (1 / 448)),  a = x / s rounded to e4m3
//   y[r][c] = sum_b (sum_j a[r][j] w[c][j]) s[r][b] w_scale[c / 128][b] + bias[c]
//
// A stage of the tiles (tile.hpp) is one block of 128, and so is one
// v_mfma_f32_16x16x128_f8f6f4: its result times the two scales is added in f32.  The
// weights are side A, so that a wave's 128 channels have one scale and a lane's column is
// one row of activations with another.
//
// The 8-bit matrix unit keeps of the sum of a block what lies within about 2^-16 of its
// largest product (against 64 bits, 1.5e-5 of the norm).  That is far below the rounding of
// a result in 16 bits.  For results in f32, EXACT widens the operands to bf16, which holds
// every e4m3 value, and uses v_mfma_f32_16x16x32_bf16 (8e-9), at half the rate.
#include "tile.hpp"

namespace thrml {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// rows of the scales of one block, so that any tile's 256 are there
static uint64_t scale_rows(uint64_t rows) { return ((rows + 255u) & ~(uint64_t)255u) + 64u; }

// A wave quantises the 512 values of a row from part * 512 on, 8 in a lane, 16 lanes to a
// block; a lane's 8 bytes, its block's scale (NaN where a value is not finite).
template <class T>
__device__ __forceinline__ void f8_load(const T *row, uint32_t c, uint32_t k, Raw8<T> &r) {
  if (c + 8u <= k)
    load8(row + c, r);
  else
    load8_part(row + c, c < k ? k - c : 0u, r);
}
template <class T>
__device__ __forceinline__ uint2 f8_quantise(const Raw8<T> &r, float &scale) {
  float v[8], m = 0.0f;
  int bad = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = value(r, j);
    bad |= !(fabsf(v[j]) < INFINITY);
    m = fmaxf(m, fabsf(v[j]));
  }
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) {
    m = fmaxf(m, __shfl_xor(m, s));
    bad |= __shfl_xor(bad, s);
  }
  // 1 / 448 is rounded first, as a division by a number is on the device; a scale below
  // 2^-126 would be rounded to so few bits that quotients leave e4m3's range
  const float s = fmaxf(m * (1.0f / 448.0f), 0x1p-126f);
  scale = bad ? __builtin_nanf("") : s;
  uint32_t w[2] = {0, 0};
  if (!bad) {
    const Divisor d(s);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = d.plain ? d.fast(v[j]) : v[j] / s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h], f[4 * h + 1], 0, false);
      w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h + 2], f[4 * h + 3], t, true);
    }
  }
  return make_uint2(w[0], w[1]);
}

template <class T>
__global__ __launch_bounds__(256) void f8_quantise_kernel(const T *__restrict__ x, int64_t x_stride, uint64_t rows, uint32_t k,
                                                          uint32_t kp, float *__restrict__ scale, uint64_t scale_pitch,
                                                          uint8_t *__restrict__ xq) {
  const uint32_t l = threadIdx.x & 63u, parts = (kp + 511u) / 512u;
  const uint64_t waves = (uint64_t)gridDim.x * 4u;
  for (uint64_t i = (uint64_t)blockIdx.x * 4u + threadIdx.x / 64u; i < rows * parts; i += waves) {
    const uint64_t row = i / parts;
    const uint32_t c = (uint32_t)(i - row * parts) * 512u + l * 8u;
    Raw8<T> r;
    f8_load(x + (int64_t)row * x_stride, c, k, r);
    float s;
    const uint2 w = f8_quantise(r, s);
    if (c < kp) {
      *reinterpret_cast<uint2 *>(xq + row * kp + c) = w;
      if ((l & 15u) == 0) scale[(uint64_t)(c / 128u) * scale_pitch + row] = s;
    }
  }
}

// ---------------------------------------------------------------------------
struct F8Tiles {
  const uint8_t *w, *x;   // x: quantised, rows of kp
  const float *scale;     // [block][scale_pitch]
  const float *w_scale, *bias;
  uint64_t w_stride, scale_pitch, rows;
  uint32_t k, kp, q;
  uint32_t ta, tb, splits, steps;
  bool small_b;           // x stays in the caches
  void *y;
  int64_t y_stride;
  float *part;            // [split][row][column]
  const void *x_own;      // the rows themselves, where each workgroup quantises them
  int64_t x_own_stride;
};

__device__ __forceinline__ bf16x8 widen8(uint32_t a, uint32_t b) {
  const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false), s = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
  return bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

// what a wave holds of 16 rows of a side: 32 reduction indices a lane
template <bool EXACT>
struct F8Frag {
  i32x8 v;
  __device__ __forceinline__ void set(u32x4 a, u32x4 b) { v = i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]}; }
  __device__ static __forceinline__ f32x4 mul(const F8Frag &a, const F8Frag &b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
  }
};
template <>
struct F8Frag<true> {
  bf16x8 v[4];
  __device__ __forceinline__ void set(u32x4 a, u32x4 b) {
    v[0] = widen8(a[0], a[1]);
    v[1] = widen8(a[2], a[3]);
    v[2] = widen8(b[0], b[1]);
    v[3] = widen8(b[2], b[3]);
  }
  __device__ static __forceinline__ f32x4 mul(const F8Frag &a, const F8Frag &b) {
    f32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
  }
};

// The rows' scales of a stage: floats in LDS behind the stages, loaded with side B.  With
// PING, whose stages fill LDS, a wave keeps those of four stages in its four groups of 16
// lanes and hands them around: the compiler waits for all loads under way before it uses
// one of its own, so that these are loaded every fourth stage, four stages ahead.  The weights'
// scales of 64 stages lie in a wave's 64 lanes (a scalar load in each stage: 25 of 306 us at
// 4096 x 4096 x 16384).
template <class S>
constexpr uint32_t f8_scales() {
  return S::PING ? 0 : S::NB < 64 ? 64 : S::NB;
}

// OWN (few values in all): each workgroup quantises the rows itself, of the type OWN, into
// LDS behind the stages of side A, while its first weights load: one launch for a call.
template <class S, class TO, bool EXACT, bool PART, class OWN = void>
__global__ __launch_bounds__(S::THREADS) void f8_tile_kernel(F8Tiles g) {
  constexpr bool IS_OWN = !std::is_void<OWN>::value;
  constexpr int TA = S::MA / 16, TB = S::MB / 16;
  constexpr uint32_t SCALES = f8_scales<S>();
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), wa = wave / S::WB, wb = wave % S::WB;
  uint32_t ia, ib;
  tile_place(blockIdx.x, gridDim.x, g.ta, g.tb, ia, ib);
  const uint32_t c0 = ia * S::NA;
  const uint64_t r0 = (uint64_t)ib * S::NB;
  const uint32_t s0 = (uint32_t)((uint64_t)g.steps * blockIdx.y / g.splits);
  const uint32_t s1 = (uint32_t)((uint64_t)g.steps * (blockIdx.y + 1u) / g.splits);

  typedef Side<S, S::NA, false> SideA;
  typedef Side<S, S::NB, false> SideB;
  const SideA sa{(uint32_t)g.w_stride, g.q - 1u - c0};
  const SideB sb{g.kp, (uint32_t)min(g.rows - 1u - r0, (uint64_t)S::NB)};
  auto a_first = [&](int p) { return p * SideA::STEP; };
  auto b_first = [&](int p) { return p * SideB::STEP; };
  const uint8_t *a0 = g.w + (uint64_t)c0 * g.w_stride, *b0 = g.x + r0 * g.kp;
  // the wave's block of channels (of 128: MA divides it)
  const float *sw0 = g.w_scale + (uint64_t)(min(c0 + wa * S::MA, g.q - 1u) / 128u) * g.steps;
  const uint32_t lds0 = lds_address(lds) + wave % (S::LOADERS / 64u) * 1024u;
  auto a_base = [&](uint32_t s) { return [&, s](int) { return a0 + s * 128u; }; };
  auto b_base = [&](uint32_t s) { return [&, s](int) { return b0 + s * 128u; }; };
  const uint32_t start = tile_start(ia, s1 - s0, g.small_b);
  auto ring = [&](uint32_t s) { return s + start < s1 ? s + start : s + start - (s1 - s0); };
  auto fetch_a = [&](uint32_t s_, uint32_t slot) {
    const uint32_t s = ring(s_);
    const uint32_t left = g.k - s * 128u;
    if (left >= 128u)
      sa.fetch(a_base(s), a_first, lds0 + S::a_at(slot));
    else
      sa.fetch_end(a_base(s), a_first, lds0 + S::a_at(slot), left);
  };
  auto fetch_b = [&](uint32_t s_, uint32_t slot) {
    const uint32_t s = ring(s_);
    if constexpr (IS_OWN) return;
    if constexpr (!S::PING) {
      const uint32_t part = wave % (SCALES / 64u) * 64u;
      word_to_lds(g.scale + s * g.scale_pitch + r0 + part, (here(threadIdx.x) & 63u) * 4u,
                  lds_address(lds) + S::BYTES + (slot * SCALES + part) * 4u);
    }
    sb.fetch(b_base(s), b_first, lds0 + S::b_at(slot));  // (rows of kp, zeros behind k)
  };
  F8Frag<EXACT> va[TA], vb[TB];
  float sx[TB], quad[S::PING ? TB : 1], next_quad[S::PING ? TB : 1], sw64 = 0.0f, sw = 0.0f;
  f32x4 acc[TA][TB] = {};
  uint32_t turn = 0;  // stages read
  auto scales = [&](uint32_t i) {  // PING: of turns i .. i + 3
    const uint32_t l = here(threadIdx.x) & 63u;
    const float *p = g.scale + (uint64_t)ring(min(s0 + i + (l >> 4), s1 - 1u)) * g.scale_pitch + r0 + wb * S::MB + (l & 15u);
#pragma unroll
    for (int j = 0; j < TB; ++j) next_quad[j] = p[16 * j];
  };
  if constexpr (S::PING) scales(0);
  auto take = [&](uint32_t l, uint32_t base, F8Frag<EXACT> &f) {
    // (pieces hi and hi + 4 of the row: any order of the block's indices, the same on both sides)
    const uint32_t lo = l & 15u, hi = l >> 4, at = base + lo * 128u + ((hi ^ tile_turn<S>(lo)) * 16u);
    f.set(*reinterpret_cast<const u32x4 *>(lds + at), *reinterpret_cast<const u32x4 *>(lds + (at ^ 64u)));
  };
  auto read = [&](uint32_t slot_a, uint32_t slot_b) {
    const uint32_t l = here(threadIdx.x) & 63u;
    const uint32_t stage_at = ring(s0 + turn), row = wb * S::MB + (l & 15u);
    if (turn % 64u == 0) {
      sw64 = sw0[ring(min(s0 + turn + l, s1 - 1u))];
      asm volatile("" : "+v"(sw64));  // (waited for here, not in every stage)
    }
    sw = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sw64), turn % 64u));
    if constexpr (IS_OWN) {
      const float *own_s = reinterpret_cast<const float *>(lds + S::B_AT + (uint32_t)g.rows * g.kp);
#pragma unroll
      for (int j = 0; j < TB; ++j) sx[j] = own_s[min(row + 16u * j, (uint32_t)g.rows - 1u) * g.steps + stage_at];
    } else if constexpr (S::PING) {
      if (turn % 4u == 0) {
#pragma unroll
        for (int j = 0; j < TB; ++j) {
          quad[j] = next_quad[j];
          asm volatile("" : "+v"(quad[j]));
        }
        scales(turn + 4u);
      }
#pragma unroll
      for (int j = 0; j < TB; ++j)
        sx[j] = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute((int)((turn % 4u * 16u + (l & 15u)) * 4u), __builtin_bit_cast(int, quad[j])));
    } else {
#pragma unroll
      for (int j = 0; j < TB; ++j)
        sx[j] = *reinterpret_cast<const float *>(lds + S::BYTES + (slot_b * SCALES + row + 16u * j) * 4u);
    }
    ++turn;
#pragma unroll
    for (int j = 0; j < TB; ++j) {
      if constexpr (IS_OWN) {
        const uint8_t *at = lds + S::B_AT + min(row + 16u * j, (uint32_t)g.rows - 1u) * g.kp + stage_at * 128u + (l >> 4) * 16u;
        vb[j].set(*reinterpret_cast<const u32x4 *>(at), *reinterpret_cast<const u32x4 *>(at + 64u));
      } else {
        take(l, S::b_at(slot_b) + (wb * S::MB + 16u * j) * 128u, vb[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < TA; ++i) take(l, S::a_at(slot_a) + (wa * S::MA + 16u * i) * 128u, va[i]);
  };
  // A product's result is added three products later, when the matrix unit has it.  (The
  // fences keep the compiler from other orders: it would add each result at once, with a
  // wait, or hold more of them than the 256 registers of a 256 x 256 tile have room for
  // beside 224 of operands and sums.)
  auto multiply = [&]() {
    constexpr int LAG = 3;
    f32x4 t[LAG + 1];
#pragma unroll
    for (int j = 0; j < TB; ++j) sx[j] *= sw;
#pragma unroll
    for (int n = 0; n < TA * TB + LAG; ++n) {
      if (n < TA * TB) t[n % (LAG + 1)] = F8Frag<EXACT>::mul(va[n % TA], vb[n / TA]);
      if (S::PING) __builtin_amdgcn_sched_barrier(0);
      if (n >= LAG) {
        const int m = n - LAG;
        f32x4 &to = acc[m % TA][m / TA];
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = __builtin_fmaf(t[m % (LAG + 1)][e], sx[m / TA], to[e]);
        if (S::PING) asm volatile("" : "+v"(to));
        if (S::PING) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto begin = [&]() {
    if constexpr (IS_OWN) {
      // (four parts of 512 values of a row at a time, their loads together)
      constexpr uint32_t U = 4;
      const uint32_t parts = (g.kp + 511u) / 512u, all = (uint32_t)g.rows * parts, l = threadIdx.x & 63u;
      float *own_s = reinterpret_cast<float *>(lds + S::B_AT + (uint32_t)g.rows * g.kp);
      for (uint32_t i = threadIdx.x / 64u; i < all; i += S::WAVES * U) {
        Raw8<OWN> r[U];
#pragma unroll
        for (uint32_t e = 0; e < U; ++e) {
          const uint32_t n = min(i + e * S::WAVES, all - 1u), row = n / parts, c = (n - row * parts) * 512u + l * 8u;
          f8_load(reinterpret_cast<const OWN *>(g.x_own) + (int64_t)row * g.x_own_stride, c, g.k, r[e]);
        }
#pragma unroll
        for (uint32_t e = 0; e < U; ++e) {
          const uint32_t n = i + e * S::WAVES;
          if (n >= all) break;
          const uint32_t row = n / parts, c = (n - row * parts) * 512u + l * 8u;
          float s;
          const uint2 w = f8_quantise(r[e], s);
          if (c < g.kp) {
            *reinterpret_cast<uint2 *>(lds + S::B_AT + row * g.kp + c) = w;
            if ((l & 15u) == 0) own_s[row * g.steps + c / 128u] = s;
          }
        }
      }
      __syncthreads();
    }
  };
  tile_loop<S, IS_OWN ? 0 : S::PB + (S::PING ? 0 : 1)>(s0, s1, fetch_a, fetch_b, read, multiply, begin);

  // The end: 16 rows x MA channels at a time through LDS, 8 neighbouring channels to a lane.
  constexpr uint32_t PITCH = S::MA + 4, LPR = S::MA / 8u;
  const uint32_t l = here(threadIdx.x) & 63u, lo = l & 15u, hi = l >> 4;
  float *mine = reinterpret_cast<float *>(lds) + wave * 16u * PITCH;
  static_assert(64u % LPR == 0, "a lane's channels are the same in every row");
  const uint32_t cl = l % LPR * 8u, c = c0 + wa * S::MA + cl, m = c < g.q ? g.q - c : 0u;
  float bias[8];
#pragma unroll
  for (uint32_t e = 0; e < 8; ++e) bias[e] = !PART && g.bias && e < m ? g.bias[c + e] : 0.0f;
#pragma unroll
  for (int j = 0; j < TB; ++j) {
#pragma unroll
    for (int i = 0; i < TA; ++i) *reinterpret_cast<f32x4 *>(mine + lo * PITCH + 16u * i + 4u * hi) = acc[i][j];
    __builtin_amdgcn_wave_barrier();
    wait_reads();
#pragma unroll
    for (uint32_t t = 0; t < (16u * LPR + 63u) / 64u; ++t) {
      const uint32_t rl = (t * 64u + l) / LPR;
      const uint64_t row = r0 + wb * S::MB + 16u * j + rl;
      if (rl >= 16u || row >= g.rows || m == 0) continue;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = mine[rl * PITCH + cl + e];
      if constexpr (PART) {
        store8(g.part + ((uint64_t)blockIdx.y * g.rows + row) * g.q + c, m, v);
      } else {
        if (g.bias) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += bias[e];
        }
        store8(reinterpret_cast<TO *>(g.y) + (int64_t)row * g.y_stride + c, m, v);
      }
    }
    __builtin_amdgcn_wave_barrier();
    wait_reads();
  }
}

// Few rows, weights at any alignment (tile.hpp): a workgroup takes 16 channels and up to 64
// rows; its four waves take turns in the blocks of 128, and their sums meet in LDS.  33 x
// 1000 x 50001 to f32: 32 us, by tiles from a copy 47.
template <class TO, bool EXACT, int ROWS16>
__global__ __launch_bounds__(256) void f8_few_kernel(F8Tiles g) {
  __shared__ f32x4 part[4][ROWS16][64];
  const uint32_t l = threadIdx.x & 63u, wave = threadIdx.x / 64u, lo = l & 15u, hi = l >> 4;
  const uint32_t c0 = blockIdx.x * 16u;
  const uint8_t *w = g.w + (uint64_t)min(c0 + lo, g.q - 1u) * g.w_stride;
  const float *sw = g.w_scale + (uint64_t)(c0 / 128u) * g.steps;
  uint32_t row[ROWS16];
#pragma unroll
  for (int j = 0; j < ROWS16; ++j) row[j] = min(16u * j + lo, (uint32_t)g.rows - 1u);
  f32x4 acc[ROWS16] = {};
#pragma unroll 2
  for (uint32_t s = wave; s < g.steps; s += 4u) {
    const uint32_t at = s * 128u + hi * 16u;
    F8Frag<EXACT> a, b[ROWS16];
    RowPiece a0, a1;
    a0.load(w, at, g.k);
    a1.load(w, at + 64u, g.k);
    float sx[ROWS16];
#pragma unroll
    for (int j = 0; j < ROWS16; ++j) {
      const uint8_t *p = g.x + (uint64_t)row[j] * g.kp + at;
      b[j].set(*reinterpret_cast<const u32x4 *>(p), *reinterpret_cast<const u32x4 *>(p + 64));
      sx[j] = g.scale[s * g.scale_pitch + row[j]] * sw[s];
    }
    a.set(a0.get(), a1.get());
#pragma unroll
    for (int j = 0; j < ROWS16; ++j) {
      const f32x4 t = F8Frag<EXACT>::mul(a, b[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = __builtin_fmaf(t[e], sx[j], acc[j][e]);
    }
  }
#pragma unroll
  for (int j = 0; j < ROWS16; ++j) part[wave][j][l] = acc[j];
  __syncthreads();
  for (uint32_t j = wave; j < ROWS16; j += 4u) {
    f32x4 v = part[0][j][l];
#pragma unroll
    for (int o = 1; o < 4; ++o) v += part[o][j][l];
    const uint32_t r = 16u * j + lo, c = c0 + 4u * hi;
    if (r >= g.rows || c >= g.q) continue;
    float f[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) f[e] = v[e] + (g.bias && c + e < g.q ? g.bias[c + e] : 0.0f);
    store4(reinterpret_cast<TO *>(g.y) + (int64_t)r * g.y_stride + c, g.q - c, f);
  }
}

// The sums of the splits, added in their order.
template <class TO>
__global__ __launch_bounds__(256) void f8_join_kernel(F8Tiles g) {
  const uint32_t groups = (g.q + 7u) / 8u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < g.rows * groups; i += (uint64_t)gridDim.x * 256u) {
    const uint64_t row = i / groups;
    const uint32_t c = (uint32_t)(i - row * groups) * 8u, m = g.q - c;
    float v[8];
    join8(g.part + row * g.q + c, g.rows * g.q, g.splits, m, v);
    if (g.bias) {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e)
        if (e < m) v[e] += g.bias[c + e];
    }
    store8(reinterpret_cast<TO *>(g.y) + (int64_t)row * g.y_stride + c, m, v);
  }
}

// Weight rows of k bytes to rows of kp, zeros behind k.
__global__ __launch_bounds__(256) void f8_pack_kernel(const uint8_t *__restrict__ w, int64_t stride, uint32_t q, uint32_t k, uint32_t kp,
                                                      uint8_t *__restrict__ out) {
  typedef uint32_t u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));
  const uint32_t groups = kp / 16u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < (uint64_t)q * groups; i += (uint64_t)gridDim.x * 256u) {
    const uint64_t row = i / groups;
    const uint32_t c = (uint32_t)(i - row * groups) * 16u;
    const uint8_t *p = w + (int64_t)row * stride + c;
    u32x4 v = {0, 0, 0, 0};
    if (c + 16u <= k) {
      v = *reinterpret_cast<const u32x4_a1 *>(p);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 16; ++j)
        if (c + j < k) v[j / 4u] |= (uint32_t)p[j] << (8u * (j & 3u));
    }
    *reinterpret_cast<u32x4 *>(out + row * kp + c) = v;
  }
}

// ---------------------------------------------------------------------------
// Calls
// Taken and next best (us a call):
//     1 x 4096 x 4096   64 x 32 in 8 parts: 18.9  in one: 19.6      128 x 4096 x 16384  64 x 64: 28    128 x 128: 33
//    16 x 8192 x 8192   64 x 32 in 4 parts: 23    in one: 32       1024 x 4096 x 8192  128 x 128: 67  256 x 256: 69
//    64 x 4096 x 16384  64 x 64: 23.6  64 x 32: 24.0               2048 x 1024 x 2048  128 x 128: 19   64 x 64: 22
// For results in f32 (the products at half the rate; 256 x 256 would need more registers):
//   256 x 4096 x 4096   64 x 64: 30  64 x 32: 32                  1024 x 4096 x 8192  128 x 128: 104  64 x 64: 121
static constexpr TileKind f8_kinds[] = {{64, 32, 128, 0.33f, 0.21f}, {64, 64, 128, 0.40f, 0.26f}, {128, 128, 128, 0.65f, 0.77f}, {256, 256, 128, 1.5f, 1.75f}};
static constexpr TileKind f8_exact_kinds[] = {{64, 32, 128, 0.40f, 0.26f}, {64, 64, 128, 0.55f, 0.37f}, {128, 128, 128, 1.2f, 1.26f}};
typedef TileShape<16, 32, 4, 1, 1, 128, 6, false> F8Tile32;
typedef TileShape<32, 32, 2, 2, 1, 128, 4, false> F8Tile64;
typedef TileShape<64, 64, 2, 2, 1, 128, 3, false> F8Tile128;
typedef TileShape<128, 64, 2, 4, 1, 128, 2, true> F8Tile256;

struct F8Plan {
  bool few, pack, own;
  uint32_t kp;
  uint64_t scale_bytes, x_bytes, w_bytes;
  TilePlan tiles;
  F8Plan(const thrml_ctx *ctx, const F8Args &a, int out_dtype) {
    kp = (a.k + 127u) & ~127u;
    pack = a.k % 16u != 0 || reinterpret_cast<uintptr_t>(a.w) % 16u != 0 ||
           (a.q > 1 && (a.w_stride % 16 != 0 || a.w_stride >= (1 << 23)));
    few = pack && a.rows <= 64;
    pack = pack && !few;
    scale_bytes = tile_bytes(scale_rows(a.rows) * (kp / 128u) * 4u);
    x_bytes = tile_bytes(a.rows * kp);
    w_bytes = pack ? tile_bytes((uint64_t)a.q * kp) : 0;
    const bool exact = out_dtype == THRML_DTYPE_F32;
    tiles = plan_tiles(ctx, exact ? f8_exact_kinds : f8_kinds, exact ? 3 : 4, a.q, a.rows, false, kp, a.rows * a.q);
    // (the quantisation's own launch: 4 us and the gap behind it)
    own = !few && !pack && tiles.kind == 0 && tiles.tb == 1 && tiles.splits == 1 && a.rows * kp <= 16384;
    if (own) scale_bytes = x_bytes = 0;
    if (few) tiles.part = 0;
  }
};

uint64_t linear_f8_work(thrml_ctx *ctx, const F8Args &a, int out_dtype) {
  const F8Plan p(ctx, a, out_dtype);
  return p.scale_bytes + p.x_bytes + p.w_bytes + p.tiles.part;
}

template <class TO, bool EXACT, class T>
static int launch_f8_own(thrml_ctx *ctx, const F8Tiles &g) {
  typedef F8Tile32 S;
  const size_t lds = std::max<size_t>(S::B_AT + g.rows * (g.kp + g.steps * 4), (size_t)S::WAVES * 16 * (S::MA + 4) * 4);
  return launch_tiles(ctx, &f8_tile_kernel<S, TO, EXACT, false, T>, g, S::THREADS, lds);
}

template <class S, class TO, bool EXACT>
static int launch_f8_kind(thrml_ctx *ctx, const F8Tiles &g) {
  const size_t lds = std::max<size_t>(S::BYTES + S::STAGES_B * f8_scales<S>() * 4, (size_t)S::WAVES * 16 * (S::MA + 4) * 4);
  auto *f = g.splits > 1 ? &f8_tile_kernel<S, TO, EXACT, true> : &f8_tile_kernel<S, TO, EXACT, false>;
  return launch_tiles(ctx, f, g, S::THREADS, lds);
}

int launch_linear_f8(thrml_ctx *ctx, const F8Args &a, int dtype, int out_dtype, void *work) {
  if (a.rows == 0) return THRML_OK;
  const F8Plan p(ctx, a, out_dtype);
  uint8_t *at = reinterpret_cast<uint8_t *>(work);
  F8Tiles g{};
  g.rows = a.rows;
  g.k = a.k;
  g.kp = p.kp;
  g.q = a.q;
  g.scale = reinterpret_cast<const float *>(at);
  g.scale_pitch = scale_rows(a.rows);
  at += p.scale_bytes;
  g.x = at;
  at += p.x_bytes;
  const int rc = p.own ? THRML_OK : with_type(dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    const uint64_t n = a.rows * ((p.kp + 511u) / 512u);
    hipLaunchKernelGGL((f8_quantise_kernel<T>), dim3((uint32_t)std::min<uint64_t>((n + 3u) / 4u, 1u << 16)), dim3(256), 0, ctx->stream,
                       reinterpret_cast<const T *>(a.x), a.x_stride, a.rows, a.k, p.kp, const_cast<float *>(g.scale), g.scale_pitch,
                       const_cast<uint8_t *>(g.x));
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
  if (rc) return rc;
  g.w = a.w;
  g.w_stride = a.q > 1 ? (uint64_t)a.w_stride : p.kp;
  if (p.pack) {
    const uint64_t n = (uint64_t)a.q * (p.kp / 16u);
    hipLaunchKernelGGL(f8_pack_kernel, dim3((uint32_t)std::min<uint64_t>(tile_cdiv(n, 256), 1u << 16)), dim3(256), 0, ctx->stream,
                       a.w, a.w_stride, a.q, a.k, p.kp, at);
    THRML_HIP(hipGetLastError());
    g.w = at;
    g.w_stride = p.kp;
    at += p.w_bytes;
  }
  g.part = reinterpret_cast<float *>(at);
  g.w_scale = a.w_scale;
  g.bias = a.bias;
  g.y = a.y;
  g.y_stride = a.y_stride;
  g.ta = p.tiles.ta;
  g.tb = p.tiles.tb;
  g.splits = p.tiles.splits;
  g.steps = p.tiles.steps;
  g.small_b = tile_small(a.rows, p.kp);
  return with_type(out_dtype, [&](auto t) -> int {
    typedef decltype(t) TO;
    constexpr bool EXACT = sizeof(TO) == 4;
    if (p.own) {
      g.x_own = a.x;
      g.x_own_stride = a.x_stride;
      return with_type(dtype, [&](auto t) { return launch_f8_own<TO, EXACT, decltype(t)>(ctx, g); });
    }
    if (p.few) {
      auto *f = a.rows <= 16 ? &f8_few_kernel<TO, EXACT, 1> : a.rows <= 32 ? &f8_few_kernel<TO, EXACT, 2> : a.rows <= 48 ? &f8_few_kernel<TO, EXACT, 3> : &f8_few_kernel<TO, EXACT, 4>;
      g.splits = 1;
      g.steps = p.kp / 128u;
      hipLaunchKernelGGL(f, dim3(tile_cdiv(a.q, 16)), dim3(256), 0, ctx->stream, g);
      THRML_HIP(hipGetLastError());
      return THRML_OK;
    }
    int rc = THRML_OK;
    switch (p.tiles.kind) {
      case 0: rc = launch_f8_kind<F8Tile32, TO, EXACT>(ctx, g); break;
      case 1: rc = launch_f8_kind<F8Tile64, TO, EXACT>(ctx, g); break;
      case 2: rc = launch_f8_kind<F8Tile128, TO, EXACT>(ctx, g); break;
      default:
        if constexpr (!EXACT) rc = launch_f8_kind<F8Tile256, TO, false>(ctx, g);
        break;
    }
    if (rc || g.splits == 1) return rc;
    const uint64_t n = a.rows * tile_cdiv(a.q, 8);
    hipLaunchKernelGGL((f8_join_kernel<TO>), dim3((uint32_t)std::min<uint64_t>(tile_cdiv(n, 256), 1u << 16)), dim3(256), 0, ctx->stream, g);
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
}

}  // namespace thrml
