// tile.hpp -- products in tiles through LDS, for the kernels of a learned head's
// hidden block (k_gated.hip) and its 8-bit product (k_f8.hip).
//
// out[r][c] = sum over j of B[r][j] A[c][j]: side A are the output's columns (its
// contiguous direction), side B its rows.  A stage is 128 bytes of the reduction of
// every row of both sides.  An operand lies in memory either with the reduction
// contiguous (a row of a side is a row in memory), or across (CROSS: a row in memory
// holds one reduction index for all rows of the side), as a gradient's operands do.
//
// In LDS, 16-byte pieces:
//   along   rows of 128 bytes, a row's 8 pieces permuted by (row >> 1) & 7.  A 16-byte
//           read takes 16 lanes at a time, four quads of lanes: 0, 3, 5, 6 of a half wave,
//           then 1, 2, 4, 7; two rows of 128 bytes fill the banks, and the rows of one
//           parity that meet (0, 2, 12, 14, 20, 22, 24, 26 of 32) differ in those bits.
//   across  64 rows, one for each reduction index, of the side's rows in chunks of 32
//           (64 bytes), permuted so that the 4 neighbouring indices that the transposing
//           read takes together fall on different banks.
// Both permutations are made in the addresses that the loads into LDS read from: these
// write 16 bytes a lane in order.
//
// Reduction indices behind the end are read from a piece of zeros, on both sides (an
// infinity times zero would be NaN); rows behind the end repeat a valid row, and their
// sums are not stored.
#pragma once
#include "dev_util.hpp"
#include "head.hpp"

namespace thrml {

static inline uint32_t tile_cdiv(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

static __device__ const u32x4 zero_piece = {0, 0, 0, 0};

// Lane l's 16 bytes from base + off to LDS address lds + 16 l (lds and base are the wave's);
// counted by the explicit waits alone.
__device__ __forceinline__ void piece_to_lds(const void *base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void piece_to_lds(const void *p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(lds) : "memory", "m0");
}
// the same with 4 bytes a lane
__device__ __forceinline__ void word_to_lds(const void *base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)p;
}
template <int N>
__device__ __forceinline__ void wait_loads() {  // all but this wave's last N loads into LDS have ended
  asm volatile("s_waitcnt vmcnt(%0)" : : "i"(N) : "memory");
}
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// nothing moves across it, matrix instructions neither
__device__ __forceinline__ void tile_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A workgroup of WA x WB x WK waves; a wave takes MA rows of side A by MB of side B
// and, of each stage, one of WK parts of the reduction.
template <int MA_, int MB_, int WA_, int WB_, int WK_, int STAGES_, bool PING_>
struct TileShape {
  static constexpr int MA = MA_, MB = MB_, WA = WA_, WB = WB_, WK = WK_, STAGES = STAGES_;
  static constexpr bool PING = PING_;
  static constexpr int NA = MA * WA, NB = MB * WB, WAVES = WA * WB * WK, THREADS = 64 * WAVES;
  static constexpr int PA = NA * 8 / THREADS, PB = NB * 8 / THREADS;  // pieces per lane
  static_assert(PA * THREADS == NA * 8 && PB * THREADS == NB * 8, "a stage is whole pieces of every lane");
  static_assert(!PING || (WAVES == 8 && WK == 1 && STAGES == 2), "two waves of a SIMD take turns");
};

// What a lane loads of one side.
template <class S, int N, bool CROSS>
struct Side {
  static constexpr int P = N * 8 / S::THREADS;
  static constexpr int CHUNKS = N / 32;  // of a row in LDS, where CROSS
  uint32_t off[P];                       // bytes from the stage's first

  __device__ static uint32_t turn(uint32_t kk) { return CHUNKS >= 4 ? kk & 3u : CHUNKS == 2 ? kk >> 1 & 1u : 0u; }
  // piece p's place: (row, first byte in the row) along, (first row, reduction index) across
  __device__ static uint32_t element(int p) { return (uint32_t)p * S::THREADS + threadIdx.x; }
  __device__ static uint32_t row(int p) {
    const uint32_t e = element(p);
    if (!CROSS) return e / 8u;
    const uint32_t pos = e % (N / 8u);
    return ((pos / 4u ^ turn(index(p))) * 4u + pos % 4u) * 8u;
  }
  __device__ static uint32_t index(int p) {  // bytes along, an index across
    const uint32_t e = element(p);
    return CROSS ? e / (N / 8u) : ((e & 7u) ^ (e / 8u >> 1 & 7u)) * 16u;
  }
  // src(row): a valid row of the operand, from the tile's first on
  template <class F>
  __device__ __forceinline__ void init(uint32_t stride, F src) {
#pragma unroll
    for (int p = 0; p < P; ++p) off[p] = CROSS ? index(p) * stride + src(row(p)) * 2u : src(row(p)) * stride + index(p);
  }
  // base(p): where the stage begins in memory, the wave's
  template <class F>
  __device__ __forceinline__ void fetch(F base, uint32_t lds) const {
#pragma unroll
    for (int p = 0; p < P; ++p) piece_to_lds(base(p), off[p], lds + (uint32_t)p * S::THREADS * 16u);
  }
  // the same where only `left` of the stage's bytes (along) or indices (across) are left
  template <class F>
  __device__ __forceinline__ void fetch_end(F base, uint32_t lds, uint32_t left) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint8_t *at = reinterpret_cast<const uint8_t *>(base(p)) + off[p];
      piece_to_lds(index(p) < left ? at : reinterpret_cast<const uint8_t *>(&zero_piece), lds + (uint32_t)p * S::THREADS * 16u);
    }
  }
};

// The loop over the stages s0 .. s1 - 1.  fetch(s, buffer) begins the loads of stage s,
// of LOADS instructions a wave, read(buffer) takes a wave's operands from LDS, multiply()
// multiplies them.
//
// PING: a SIMD's two waves take turns: one reads its operands of a stage while the other
// multiplies, so that the matrix unit always has a wave that needs nothing but registers.
// The second wave is one phase, half a stage, behind.  A stage's loads have two phases to
// arrive.
template <class S, int LOADS, class Fetch, class Read, class Multiply>
__device__ __forceinline__ void tile_loop(uint32_t s0, uint32_t s1, Fetch fetch, Read read, Multiply multiply) {
  if constexpr (S::PING) {
    const bool second = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u) >= 4u;
    fetch(s0, 0);
    wait_loads<0>();
    tile_barrier();
    if (second) {
      if (s0 + 1 < s1) fetch(s0 + 1, 1);
      tile_barrier();
    }
    for (uint32_t s = s0; s < s1; ++s) {
      const uint32_t b = (s - s0) & 1u;
      read(b);
      if (!second && s + 1 < s1) fetch(s + 1, b ^ 1u);
      wait_reads();
      if (second) wait_loads<0>();
      tile_barrier();
      if (second && s + 2 < s1) fetch(s + 2, b);
      __builtin_amdgcn_s_setprio(1);
      multiply();
      __builtin_amdgcn_s_setprio(0);
      if (!second) wait_loads<0>();
      if (!second || s + 1 < s1) tile_barrier();
    }
    tile_barrier();
  } else {
    // fetches past the end repeat the last stage, so that every wait counts alike
    constexpr uint32_t AHEAD = S::STAGES - 1;
    for (uint32_t i = 0; i < AHEAD; ++i) fetch(min(s0 + i, s1 - 1u), i);
    uint32_t b = 0;
    for (uint32_t s = s0; s < s1; ++s) {
      // (a wave's reads of the stage before have ended: its products have been issued)
      wait_loads<(S::STAGES - 2) * LOADS>();
      tile_barrier();
      const uint32_t into = b == 0 ? AHEAD : b - 1u;
      fetch(min(s + AHEAD, s1 - 1u), into);
      read(b);
      wait_reads();
      multiply();
      b = b == AHEAD ? 0 : b + 1u;
    }
    wait_loads<0>();
    tile_barrier();
  }
}

// Tiles in an order in which those that run together share operands: workgroups of one
// XCD take neighbouring tiles, 8 of side B at a time.
__device__ __forceinline__ void tile_place(uint32_t index, uint32_t tiles, uint32_t ta, uint32_t tb, uint32_t &a, uint32_t &b) {
  const uint32_t i = xcd_remap(index, tiles), group = i / (8u * ta), first = group * 8u;
  const uint32_t n = min(8u, tb - first), j = i - group * 8u * ta;
  b = first + j % n;
  a = j / n;
}

// ---------------------------------------------------------------------------
// On the host: which tiles a call takes
static inline uint64_t tile_bytes(uint64_t n) { return (n + 255u) & ~(uint64_t)255u; }

struct TileKind {
  uint32_t na, nb;
  float alone, many;  // us a stage: of a tile alone on a compute unit, and of one of several
};

struct TilePlan {
  int kind = 0;
  uint32_t ta = 0, tb = 0, splits = 1, steps = 0;
  uint64_t part = 0;  // bytes of the splits' sums
};

// The kind of tile, and into how many parts the reduction goes, by an estimate of each
// one's time: its stages, and about 6 more for beginning and end, at its time for one.
// cols: the rows of side A; rows: those of side B, of two matrices where `halves`.
static inline TilePlan plan_tiles(const thrml_ctx *ctx, const TileKind *kinds, int n, uint64_t cols, uint64_t rows, bool halves,
                                  uint32_t steps, uint64_t out_values) {
  TilePlan best;
  double best_t = 0.0;
  for (int i = 0; i < n; ++i) {
    const TileKind &kd = kinds[i];
    const uint32_t ta = tile_cdiv(cols, kd.na), tb = tile_cdiv(rows, kd.nb) * (halves ? 2u : 1u);
    const uint64_t tiles = (uint64_t)ta * tb;
    for (uint32_t splits = 1; splits <= 16; splits *= 2) {
      if (splits > 1 && (steps < 8 * splits || tiles * splits > 2u * (uint32_t)ctx->cu_count)) break;
      const double one = std::max<double>(kd.alone, (double)kd.many * (double)tile_cdiv(tiles * splits, ctx->cu_count));
      // a join reads what the splits wrote, 3 bytes a ps, and is a launch
      const double t = one * (tile_cdiv(steps, splits) + 6) + (splits > 1 ? 5.0 + (double)out_values * 4 * 2 * splits / 3e6 : 0.0);
      if (best_t == 0.0 || t < best_t) {
        best_t = t;
        best.kind = i;
        best.ta = ta;
        best.tb = tb;
        best.splits = splits;
        best.steps = steps;
        best.part = splits > 1 ? tile_bytes(out_values * 4 * splits) : 0;
      }
    }
  }
  return best;
}

// One workgroup for each tile and split.
template <class G>
static int launch_tiles(thrml_ctx *ctx, void (*f)(G), const G &g, uint32_t threads, size_t lds) {
  if ((uint64_t)g.ta * g.tb * threads >> 32) {
    set_error("more tiles than a launch takes");
    return THRML_EUNSUPPORTED;
  }
  if (lds > 65536)
    THRML_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(f), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(f, dim3(g.ta * g.tb, g.splits), dim3(threads), lds, ctx->stream, g);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

}  // namespace thrml
