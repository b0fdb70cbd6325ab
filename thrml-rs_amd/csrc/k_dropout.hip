// k_dropout.hip -- units kept or zeroed by the bits of a key's ChaCha8 stream; the mask is
// never stored, the gradient's way back computes it again.
//   i = (first_row + row) cols + col
//   y[row][col] = (residual[row][col] +) (half word i of the stream >= border ? x[row][col] scale : 0)
// A block of the stream, 400 integer operations, serves 32 units.  A lane computes one
// block and keeps its 32 comparisons as one word; then a lane takes 8 neighbouring units at
// a time, so that a wave reads and writes whole lines, and fetches their bits from the
// lane that has them.  What the span reads is under way before the block is computed.
#include "head.hpp"
#include "thrml_rng.hpp"

namespace thrml {

// FLAT: one row.  Otherwise the row of a group of 8 units is found by a division, and a
// group may lie across rows.
template <class T, bool RESIDUAL, bool FLAT>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
  const uint32_t l = threadIdx.x & 63u;
  const Key8 key = seed_from_u64(a.seed_at ? (uint64_t)*a.seed_at : a.seed);
  uint32_t pre[KEY_WORDS];
  key_expand(key.k, pre);
  const T *x = reinterpret_cast<const T *>(a.x), *res = reinterpret_cast<const T *>(a.residual);
  T *y = reinterpret_cast<T *>(a.y);
  const uint64_t n = a.rows * a.cols, end = a.begin + n, first = a.begin & ~(uint64_t)31u;
  const bool small = n >> 32 == 0;
  // spans of 2048 units from a multiple of 32 on, one for a wave at a time
  const uint64_t stride = (uint64_t)gridDim.x * 4u * 2048u;
  for (uint64_t span = first + ((uint64_t)blockIdx.x * 4u + threadIdx.x / 64u) * 2048u; span < end; span += stride) {
    int64_t at[4];  // the group's first unit, counted from row 0's first: may be negative, or behind the end
    int64_t row[4], col[4];
    bool whole[4];
    Raw8<T> rx[4], rr[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      at[g] = (int64_t)(span + (uint32_t)g * 512u + l * 8u - a.begin);
      row[g] = 0;
      col[g] = at[g];
      if (!FLAT && at[g] > 0) {
        row[g] = (int64_t)(small ? (uint32_t)at[g] / (uint32_t)a.cols : (uint64_t)at[g] / a.cols);
        col[g] = at[g] - row[g] * (int64_t)a.cols;
      }
      whole[g] = at[g] >= 0 && col[g] + 8 <= (int64_t)a.cols && (FLAT || row[g] < (int64_t)a.rows);
      if (whole[g]) {
        load8(x + row[g] * a.x_stride + col[g], rx[g]);
        if (RESIDUAL) load8(res + row[g] * a.residual_stride + col[g], rr[g]);
      }
    }
    uint32_t words[16], kept = 0;
    chacha_block_pre<8>(pre, (uint32_t)(span / 32u) + l, words);  // (blocks are fewer than 2^32)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      kept |= (uint32_t)((words[j] & 0xffffu) >= a.border) << (2 * j);
      kept |= (uint32_t)((words[j] >> 16) >= a.border) << (2 * j + 1);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t bits = (uint32_t)__shfl((int)kept, (int)(16u * g + l / 4u)) >> (8u * (l & 3u));
      if (whole[g]) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = bits >> e & 1u ? value(rx[g], e) * a.scale : 0.0f;
          if (RESIDUAL) v[e] = value(rr[g], e) + v[e];
        }
        store8(y + row[g] * a.y_stride + col[g], 8, v);
      } else {
        int64_t r = row[g], c = col[g];
        for (uint32_t e = 0; e < 8; ++e, ++c) {
          if (c == (int64_t)a.cols) {
            c = 0;
            ++r;
          }
          if (c < 0 || c >= (int64_t)a.cols || r >= (int64_t)a.rows) continue;  // (a group behind the end begins there)
          float f = bits >> e & 1u ? (float)x[r * a.x_stride + c] * a.scale : 0.0f;
          if (RESIDUAL) f = (float)res[r * a.residual_stride + c] + f;
          y[r * a.y_stride + c] = (T)f;
        }
      }
    }
  }
}

int launch_dropout(thrml_ctx *ctx, DropoutArgs a, int dtype) {
  if (a.rows == 0 || a.cols == 0) return THRML_OK;
  const int64_t cols = (int64_t)a.cols;
  if (a.rows == 1 || (a.x_stride == cols && a.y_stride == cols && (!a.residual || a.residual_stride == cols))) {
    a.cols *= a.rows;
    a.rows = 1;
  }
  const uint64_t spans = (a.rows * a.cols + 31u) / 2048u + 1u;
  const uint32_t grid = (uint32_t)std::min<uint64_t>((spans + 3u) / 4u, 8u * (uint64_t)ctx->cu_count);
  return with_type(dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    auto *f = a.residual ? (a.rows == 1 ? &dropout_kernel<T, true, true> : &dropout_kernel<T, true, false>)
                         : (a.rows == 1 ? &dropout_kernel<T, false, true> : &dropout_kernel<T, false, false>);
    hipLaunchKernelGGL(f, dim3(grid), dim3(256), 0, ctx->stream, a);
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
}

}  // namespace thrml
