// tile.hpp -- products in tiles through LDS, for the kernels of a learned head's
// hidden block (k_gated.hip) and its 8-bit product (k_f8.hip).
//
// out[r][c] = sum over j of B[r][j] A[c][j]: side A are the output's columns (its
// contiguous direction), side B its rows.  A stage is KB (128 or 256) bytes of the reduction of
// every row of both sides.  An operand lies in memory either with the reduction
// contiguous (a row of a side is a row in memory), or across (CROSS: a row in memory
// holds one reduction index for all rows of the side), as a gradient's operands do.
//
// In LDS, 16-byte pieces:
//   along   rows of KB bytes, a row's pieces permuted by bits of the row: (row >> 1) & 7 for
//           128 bytes, row & 15 for 256 (among 16 pieces).  A 16-byte read takes 16 lanes at a
//           time, four quads of lanes: 0, 3, 5, 6 of a half wave, then 1, 2, 4, 7; two rows of 128
//           bytes fill the banks, and the rows of one parity that meet (0, 2, 12, 14, 20, 22, 24,
//           26 of 32) differ in those bits.
//   across  KB / 2 rows, one for each reduction index, of the side's rows in chunks of 32
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
// and, of each stage, one of WK parts of the reduction.  STAGES: those in LDS; PING (below)
// has three of side A and two of side B.
template <int MA_, int MB_, int WA_, int WB_, int WK_, int KB_, int STAGES_, bool PING_>
struct TileShape {
  static constexpr int MA = MA_, MB = MB_, WA = WA_, WB = WB_, WK = WK_, KB = KB_;
  static constexpr int STAGES_A = PING_ ? 3 : STAGES_, STAGES_B = PING_ ? 2 : STAGES_;
  static constexpr bool PING = PING_;
  static constexpr int NA = MA * WA, NB = MB * WB, WAVES = WA * WB * WK, THREADS = 64 * WAVES;
  static constexpr int LOADERS = PING_ ? THREADS / 2 : THREADS;       // threads that load a side
  static constexpr int PIECES = KB / 16;                              // of a row
  static constexpr int PA = NA * PIECES / LOADERS, PB = NB * PIECES / LOADERS;  // for each of them
  static constexpr int B_AT = STAGES_A * NA * KB, BYTES = B_AT + STAGES_B * NB * KB;  // in LDS: side A's stages, then B's
  static_assert(PA * LOADERS == NA * PIECES && PB * LOADERS == NB * PIECES, "a stage is whole pieces of every lane");
  static_assert(!PING || (WAVES == 8 && WK == 1), "two waves of a SIMD take turns");
  __device__ static __forceinline__ uint32_t a_at(uint32_t slot) { return slot * (NA * KB); }
  __device__ static __forceinline__ uint32_t b_at(uint32_t slot) { return B_AT + slot * (NB * KB); }
};

// a row's permutation of its pieces
template <class S>
__device__ __forceinline__ uint32_t tile_turn(uint32_t row) {
  static_assert(S::KB == 128 || S::KB == 256, "8 or 16 pieces");
  return S::KB == 256 ? row & 15u : row >> 1 & 7u;
}

// What a lane loads of one side, in P pieces.  Along, its pieces lie STEP rows apart, at
// the same bytes of a row; across, STEP indices apart, at the same rows.  Where they lie in
// memory is computed from the thread's number at each stage (here() keeps the compiler from
// doing it once): kept, it was what did not fit into the registers of a 256 x 256 tile.
template <class S, int N, bool CROSS>
struct Side {
  static constexpr int P = N * S::PIECES / S::LOADERS;
  static constexpr int CHUNKS = N / 32;                              // of a row in LDS, where CROSS
  static constexpr uint32_t STEP = CROSS ? S::LOADERS / (N / 8) : S::LOADERS / S::PIECES;
  static_assert(CROSS ? STEP % 4 == 0 || P == 1 : STEP % 16 == 0 || P == 1, "pieces are permuted alike");
  uint32_t stride, last;    // bytes between rows in memory (below 2^24), the last valid row

  struct Place {            // of piece 0
    uint32_t row, index;    // along: row and first byte in it; across: first row and index
  };
  __device__ __forceinline__ Place place() const {
    const uint32_t e = here(threadIdx.x) % S::LOADERS;
    Place a;
    if (CROSS) {
      const uint32_t pos = e % (N / 8u);
      a.index = e / (N / 8u);
      const uint32_t turn = CHUNKS >= 4 ? a.index & 3u : CHUNKS == 2 ? a.index >> 1 & 1u : 0u;
      a.row = ((pos / 4u ^ turn) * 4u + pos % 4u) * 8u;
      if (a.row > last) a.row = 0;  // (8 rows: last is 7 mod 8)
    } else {
      a.row = e / S::PIECES;
      a.index = (e % S::PIECES ^ tile_turn<S>(a.row)) * 16u;
    }
    return a;
  }
  // piece p's bytes from base(p) on.  first(p): along, the row in memory of the side's row
  // p STEP
  template <class F>
  __device__ __forceinline__ uint32_t offset(int p, Place a, F first) const {
    if (CROSS) return __umul24(a.index, stride) + a.row * 2u;
    return __umul24(min(a.row + first(p), last), stride) + a.index;
  }
  template <class B, class F>
  __device__ __forceinline__ void fetch(B base, F first, uint32_t lds) const {
    const Place a = place();
#pragma unroll
    for (int p = 0; p < P; ++p)
      piece_to_lds(base(p) + (CROSS ? (uint64_t)p * STEP * stride : 0u), offset(p, a, first), lds + (uint32_t)p * S::LOADERS * 16u);
  }
  // the same where only `left` of the stage's bytes (along) or indices (across) are left
  template <class B, class F>
  __device__ __forceinline__ void fetch_end(B base, F first, uint32_t lds, uint32_t left) const {
    const Place a = place();
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint8_t *at = base(p) + (CROSS ? (uint64_t)p * STEP * stride : 0u) + offset(p, a, first);
      const bool in = CROSS ? a.index + p * STEP < left : a.index < left;
      piece_to_lds(in ? at : reinterpret_cast<const uint8_t *>(&zero_piece), lds + (uint32_t)p * S::LOADERS * 16u);
    }
  }
};

// The loop over the stages s0 .. s1 - 1.  fetch_a(s, slot) and fetch_b begin the loads of
// a side's stage s, of S::PA and LOADS_B instructions a wave, read(slot of A, of B) takes a
// wave's operands from LDS, multiply() multiplies them.  begin() is called when the loads
// of the first stage are under way (not with PING; it may wait for all that are).
//
// PING: a SIMD's two waves take turns: one reads its operands of a stage while the other
// multiplies, so that the matrix unit always has a wave that needs nothing but registers.
// The second wave is one phase, half a stage, behind.  Behind its reads, the first loads
// the next stage of side B, the second the next but one of side A.  A load into LDS
// holds its wave up for some 40 cycles, also between products: so each phase has half of
// them, and none is among the products.  Cycles of a phase at 4096 x 4096 x 16384 in bf16:
// 1055 multiply (of 1024 that the products take), 650 read, 400 load; a stage, two phases,
// takes 2460.  With all loads from the first wave it took 2830, with all among the
// second's products 3350.
template <class S, int LOADS_B, class FetchA, class FetchB, class Read, class Multiply, class Begin>
__device__ __forceinline__ void tile_loop(uint32_t s0, uint32_t s1, FetchA fetch_a, FetchB fetch_b, Read read, Multiply multiply, Begin begin) {
  if constexpr (S::PING) {
    const bool second = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u) >= 4u;
    if (second) {
      fetch_a(s0, 0);
      if (s0 + 1 < s1) fetch_a(s0 + 1, 1);
    } else {
      fetch_b(s0, 0);
    }
    wait_loads<0>();
    tile_barrier();
    if (second) tile_barrier();
    uint32_t a = 0, b = 0;
    for (uint32_t s = s0; s < s1; ++s) {
      read(a, b);
      // (A's slot held stage s - 1, B's too, which everyone has read)
      const bool more = s + (second ? 2u : 1u) < s1;
      if (more) {
        if (second)
          fetch_a(s + 2, a == 0 ? 2u : a - 1u);
        else
          fetch_b(s + 1, b ^ 1u);
      }
      wait_reads();
      // side A's stage s + 1 has come
      if (second) {
        if (more)
          wait_loads<S::PA>();
        else
          wait_loads<0>();
      }
      tile_barrier();
      __builtin_amdgcn_s_setprio(1);
      multiply();
      __builtin_amdgcn_s_setprio(0);
      if (!second) wait_loads<0>();  // side B's
      if (!second || s + 1 < s1) tile_barrier();
      a = a == 2 ? 0 : a + 1u;
      b ^= 1u;
    }
    tile_barrier();
  } else {
    // fetches past the end repeat the last stage, so that every wait counts alike
    constexpr uint32_t AHEAD = S::STAGES_A - 1;
    for (uint32_t i = 0; i < AHEAD; ++i) {
      fetch_a(min(s0 + i, s1 - 1u), i);
      fetch_b(min(s0 + i, s1 - 1u), i);
      if (i == 0) begin();
    }
    uint32_t b = 0;
    for (uint32_t s = s0; s < s1; ++s) {
      // (a wave's reads of the stage before have ended: its products have been issued)
      wait_loads<(S::STAGES_A - 2) * (S::PA + LOADS_B)>();
      tile_barrier();
      const uint32_t into = b == 0 ? AHEAD : b - 1u;
      fetch_a(min(s + AHEAD, s1 - 1u), into);
      fetch_b(min(s + AHEAD, s1 - 1u), into);
      read(b, b);
      wait_reads();
      multiply();
      b = b == AHEAD ? 0 : b + 1u;
    }
    wait_loads<0>();
    tile_barrier();
  }
}

// ---------------------------------------------------------------------------
// Few rows whose operands do not start at 16 bytes: straight from memory into the operand
// registers of 16 x 16 products, without a copy.  16 bytes of a row from byte c on, zeros
// from byte n on; p at any address.  The words that hold them are loaded and shifted: loads
// from addresses within a word take longer.
struct RowPiece {
  u32x4 v = {0, 0, 0, 0};
  uint32_t next = 0, shift = 0;
  __device__ __forceinline__ void load(const uint8_t *p, uint32_t c, uint32_t n) {
    typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
    if (c + 20u <= n) {
      shift = (uint32_t)(uintptr_t)p & 3u;
      const uint8_t *at = p + c - shift;
      v = *reinterpret_cast<const u32x4_a4 *>(at);
      next = reinterpret_cast<const uint32_t *>(at)[shift ? 4 : 0];
    } else {
      v = u32x4{0, 0, 0, 0};
      shift = 0;
      if (c < n) {
        const uint32_t left = here(n - c);
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j)
          if (j < left) v[j / 4u] |= (uint32_t)p[c + j] << (8u * (j & 3u));
      }
    }
  }
  __device__ __forceinline__ u32x4 get() const {
    return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], shift), __builtin_amdgcn_alignbyte(v[2], v[1], shift),
                 __builtin_amdgcn_alignbyte(v[3], v[2], shift), __builtin_amdgcn_alignbyte(next, v[3], shift)};
  }
};

// Tiles in an order in which those that run together share operands: workgroups of one
// XCD take neighbouring tiles, 8 of side B at a time.
__device__ __forceinline__ void tile_place(uint32_t index, uint32_t tiles, uint32_t ta, uint32_t tb, uint32_t &a, uint32_t &b) {
  const uint32_t i = xcd_remap(index, tiles), group = i / (8u * ta), first = group * 8u;
  const uint32_t n = min(8u, tb - first), j = i - group * 8u * ta;
  b = first + j % n;
  a = j / n;
}

// Where a tile begins in its stages, of which it takes n in a ring.  Rows of a power of two
// bytes have the same columns on few channels of memory, and tiles that all begin at the
// first column ask those for everything.  Where side B is small enough to stay in the caches,
// each tile of side A begins elsewhere (one row by 4096 x 32768 in bf16: 54 us, not 65; 49
// either way at 4160); otherwise the tiles of an XCD, which share what they load, begin
// together.
__device__ __forceinline__ uint32_t tile_start(uint32_t ia, uint32_t n, bool small_b) {
  return small_b ? ia * 5u % n : (blockIdx.x & 7u) * n / 8u;
}

// The sums of the splits for 8 neighbouring values (n of them, at most 8), added in their
// order; several loads are under way together.
__device__ __forceinline__ void join8(const float *p, uint64_t pitch, uint32_t splits, uint32_t n, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.0f;
#pragma unroll 4
  for (uint32_t s = 0; s < splits; ++s) {
    Raw8<float> r;
    if (n >= 8u)
      load8(p + s * pitch, r);
    else
      load8_part(p + s * pitch, n, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += value(r, e);
  }
}

// ---------------------------------------------------------------------------
// On the host: which tiles a call takes
static inline uint64_t tile_bytes(uint64_t n) { return (n + 255u) & ~(uint64_t)255u; }

struct TileKind {
  uint32_t na, nb;
  uint32_t kb;        // bytes of a row in a stage
  float alone, many;  // us a stage: of a tile where few compute units have one, and where each has one or several
};

struct TilePlan {
  int kind = 0;
  uint32_t ta = 0, tb = 0, splits = 1, steps = 0;
  uint64_t part = 0;  // bytes of the splits' sums
};

// The kind of tile, and into how many parts the reduction goes, by an estimate of each
// one's time: its stages, and about 6 more of 128 bytes for beginning and end, at its time
// for one.
// row_bytes: of the reduction, in a row; cols: the rows of side A; rows: those of side B, of two matrices where `halves`.
static inline TilePlan plan_tiles(const thrml_ctx *ctx, const TileKind *kinds, int n, uint64_t cols, uint64_t rows, bool halves,
                                  uint64_t row_bytes, uint64_t out_values) {
  TilePlan best;
  double best_t = 0.0;
  for (int i = 0; i < n; ++i) {
    const TileKind &kd = kinds[i];
    const uint32_t ta = tile_cdiv(cols, kd.na), tb = tile_cdiv(rows, kd.nb) * (halves ? 2u : 1u);
    const uint64_t tiles = (uint64_t)ta * tb;
    const uint32_t steps = tile_cdiv(row_bytes, kd.kb);
    // (a split has two stages or more: an empty one would have no last stage to repeat)
    for (uint32_t splits = 1; splits <= 16; splits *= 2) {
      if (splits > 1 && (steps * (uint64_t)kd.kb < 512u * splits || tiles * splits > 2u * (uint32_t)ctx->cu_count)) break;
      const uint64_t groups = tiles * splits, cus = (uint64_t)ctx->cu_count;
      const double one = groups > cus ? (double)kd.many * (double)tile_cdiv(groups, cus)
                                      : kd.alone + std::max(0.0f, kd.many - kd.alone) * (double)groups / (double)cus;
      // a join reads what the splits wrote, together 4.5 bytes a ps, and is a launch
      const double t = one * (tile_cdiv(steps, splits) + 768.0 / kd.kb) + (splits > 1 ? 7.0 + (double)out_values * 4 * 2 * splits / 4.5e6 : 0.0);
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

static inline bool tile_small(uint64_t rows, uint64_t row_bytes) { return rows * row_bytes <= (2u << 20); }

// One workgroup for each tile and split, which all have a stage or more: one without would repeat
// stage -1.
template <class G>
static int launch_tiles(thrml_ctx *ctx, void (*f)(G), const G &g, uint32_t threads, size_t lds) {
  if ((uint64_t)g.ta * g.tb * threads >> 32) {
    set_error("more tiles than a launch takes");
    return THRML_EUNSUPPORTED;
  }
  if (g.splits == 0 || g.splits > g.steps) {
    set_error("a split of the reduction without a stage");
    return THRML_EUNSUPPORTED;
  }
  if (lds > 65536)
    THRML_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(f), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(f, dim3(g.ta * g.tb, g.splits), dim3(threads), lds, ctx->stream, g);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

}  // namespace thrml
