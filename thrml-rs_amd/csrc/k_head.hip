// k_head.hip -- rows of logits of a learned head: processing, sampling, and
// distillation from a teacher's top candidates.
#include "head.hpp"

namespace thrml {

static inline uint32_t cdiv(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// ---------------------------------------------------------------------------
// What a row's history and biases say of the categories c0 .. c0 + n - 1: a word
// for each category in LDS,
//   bit 31   the category occurs in the prompt part of the history
//   bit 30   it has a bias (its value in the second table)
//   bits 0-28  how often it was drawn after the prompt
// and, where rows have biases, the sum of its bias entries, in list order.  A
// workgroup scans the row's whole history (it is short beside the row, and all
// workgroups of a row share it in L2) and keeps what falls into its categories.
constexpr uint32_t T_PROMPT = 1u << 31, T_BIAS = 1u << 30, T_COUNT = (1u << 29) - 1u;

struct RowParams {
  float theta, presence, frequency, t;
  uint32_t len, prompt;
};

__device__ __forceinline__ RowParams row_params(const LogitRows &a, uint64_t row) {
  RowParams p;
  p.theta = a.repetition ? a.repetition[row] : 1.0f;
  p.presence = a.presence ? a.presence[row] : 0.0f;
  p.frequency = a.frequency ? a.frequency[row] : 0.0f;
  p.t = a.temperature ? a.temperature[row] : 0.0f;
  const int32_t h = (int32_t)a.history_len;
  const int32_t len = a.lengths ? a.lengths[row] : h, pr = a.prompt_lengths ? a.prompt_lengths[row] : 0;
  p.len = (uint32_t)(len < 0 ? 0 : len > h ? h : len);
  p.prompt = (uint32_t)(pr < 0 ? 0 : pr);
  return p;
}

// tab: n words, then n floats where there are biases.  All threads of the
// workgroup call it; it ends with a barrier.
__device__ __forceinline__ void build_table(const LogitRows &a, const RowParams &p, uint64_t row, uint32_t c0,
                                            uint32_t n, uint32_t *tab, float *btab) {
  const uint32_t tid = threadIdx.x, nt = blockDim.x;
  for (uint32_t i = tid; i < n; i += nt) tab[i] = 0;
  __syncthreads();
  if (a.history) {
    const int32_t *h = a.history + (int64_t)row * a.history_stride;
    for (uint32_t i = tid; i < p.len; i += nt) {
      const uint32_t d = (uint32_t)h[i] - c0;
      if (d < n) {
        if (i < p.prompt)
          atomicOr(&tab[d], T_PROMPT);
        else
          atomicAdd(&tab[d], 1u);
      }
    }
  }
  if (a.n_bias) {
    const int32_t *ids = a.bias_ids + (int64_t)row * a.bias_stride;
    const float *vals = a.bias_values + (int64_t)row * a.bias_stride;
    int again = 0;
    for (uint32_t i = tid; i < a.n_bias; i += nt) {
      const uint32_t d = (uint32_t)ids[i] - c0;
      if (d < n) {
        if (atomicOr(&tab[d], T_BIAS) & T_BIAS) again = 1;
        btab[d] = vals[i];
      }
    }
    // a category named more than once: its entries are added in list order by
    // the thread of the first one
    if (__syncthreads_or(again)) {
      for (uint32_t i = tid; i < a.n_bias; i += nt) {
        const int32_t id = ids[i];
        if ((uint32_t)id - c0 >= n) continue;
        bool first = true;
        for (uint32_t j = 0; j < i && first; ++j) first = ids[j] != id;
        if (!first) continue;
        float s = vals[i];
        for (uint32_t j = i + 1; j < a.n_bias; ++j)
          if (ids[j] == id) s += vals[j];
        btab[(uint32_t)id - c0] = s;
      }
    }
  }
  __syncthreads();
}

// A logit with its row's penalties and its bias, each step rounded to f32.
__device__ __forceinline__ float penalised(float z, uint32_t w, float bias, const RowParams &p) {
  const uint32_t n = w & T_COUNT;
  if (n || (w & T_PROMPT)) z = z > 0.0f ? z / p.theta : z * p.theta;
  if (n) {
    z = z - p.frequency * (float)n;
    z = z - p.presence;
  }
  if (w & T_BIAS) z = z + bias;
  return z;
}

// y[j] = the 8 logits from c0 + d on with penalties and biases
template <class T>
__device__ __forceinline__ void row_values(const Raw8<T> &r, const uint32_t *tab, const float *btab, uint32_t d,
                                           const RowParams &p, float (&y)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = value(r, j);
  if (tab) {
    const uint4 t0 = *reinterpret_cast<const uint4 *>(tab + d), t1 = *reinterpret_cast<const uint4 *>(tab + d + 4);
    const uint32_t w[8] = {t0.x, t0.y, t0.z, t0.w, t1.x, t1.y, t1.z, t1.w};
    if ((t0.x | t0.y | t0.z | t0.w | t1.x | t1.y | t1.z | t1.w) != 0u) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (w[j]) y[j] = penalised(y[j], w[j], (w[j] & T_BIAS) ? btab[d + j] : 0.0f, p);
    }
  }
}

// ---------------------------------------------------------------------------
// Processing: a workgroup writes `chunk` categories of one row.
template <class TI, class TO>
__global__ __launch_bounds__(256) void process_kernel(LogitRows a, TO *__restrict__ out, int64_t out_stride,
                                                      uint32_t chunk, uint32_t n_chunks, uint64_t n_tasks) {
  extern __shared__ uint32_t lds[];
  const bool table = a.history || a.n_bias;
  float *btab = reinterpret_cast<float *>(lds + chunk);
  for (uint64_t task = blockIdx.x; task < n_tasks; task += gridDim.x) {
    const uint64_t row = task / n_chunks;
    const uint32_t c0 = (uint32_t)(task % n_chunks) * chunk;
    const uint32_t n = min(chunk, a.q - c0);
    const RowParams p = row_params(a, row);
    if (table) build_table(a, p, row, c0, (n + 7u) & ~7u, lds, btab);
    const TI *z = reinterpret_cast<const TI *>(a.z) + (int64_t)row * a.z_stride + c0;
    TO *o = out + (int64_t)row * out_stride + c0;
    const uint8_t *mask =
        a.mask ? reinterpret_cast<const uint8_t *>(a.mask + (int64_t)row * a.mask_stride) + c0 / 8u : nullptr;
    for (uint32_t d = threadIdx.x * 8u; d < n; d += 256u * 8u) {
      Raw8<TI> r;
      if (d + 8u <= n)
        load8(z + d, r);
      else
        load8_part(z + d, n - d, r);
      float y[8];
      row_values(r, table ? lds : nullptr, btab, d, p, y);
      if (p.t > 0.0f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = y[j] / p.t;
      }
      if (mask) {
        const uint32_t m = mask[d / 8u];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (m >> j & 1u) ? y[j] : -INFINITY;
      }
      store8(o + d, n - d, y);
    }
    if (table) __syncthreads();  // the next task builds its own
  }
}

int launch_process_logits(thrml_ctx *ctx, const LogitRows &a, int dtype, void *out, int out_dtype,
                          int64_t out_stride) {
  if (a.rows == 0) return THRML_OK;
  uint32_t chunk = 8192;
  while (chunk > 2048 && a.rows * cdiv(a.q, chunk) < 4ull * ctx->cu_count) chunk /= 2;
  const uint32_t nc = cdiv(a.q, chunk);
  const uint64_t tasks = a.rows * nc;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(tasks, 1u << 20);
  const size_t lds = (a.n_bias ? 2 : a.history ? 1 : 0) * (size_t)chunk * 4;
  return with_type(dtype, [&](auto ti) {
    return with_type(out_dtype, [&](auto to) -> int {
      typedef decltype(ti) TI;
      typedef decltype(to) TO;
      hipLaunchKernelGGL((process_kernel<TI, TO>), dim3(grid), dim3(256), lds, ctx->stream, a,
                         reinterpret_cast<TO *>(out), out_stride, chunk, nc, tasks);
      THRML_HIP(hipGetLastError());
      return THRML_OK;
    });
  });
}

// ---------------------------------------------------------------------------
// Sampling.  With x the processed logits, a row's category is the first argmax
// over the allowed ones of x - log(-log u) (Gumbel-max), or of x for a greedy
// row, and its log-probability is x - m - log(sum exp(x - m)), all in one pass
// over the row: the running maximum and sum of a softmax per lane, and the pick.
//
// The pick is exact in 64 bits at f32 cost.  v, the score from hardware
// logarithms and x from a reciprocal of the temperature, is within S_MARGIN +
// |v| S_REL of the score in 64 bits; only a lane whose v exceeds its wave's best
// exact score less that margin computes the score in 64 bits (from x as the
// steps in f32 give it), a few times per wave and row.  A score of u below 2^-126 is
// that of 2^-126 in v, which is no less than its own.  An allowed category
// whose own score is -inf (u = 0) is taken only where there is no other, a
// masked one never.
constexpr float S_MARGIN = 1e-4f, S_REL = 0x1p-18f;
constexpr float LOG2E = 1.44269504f;

struct SamplePart {
  double best;
  float m, sum, x;
  int32_t arg;
};

__device__ __forceinline__ void part_merge(SamplePart &a, const SamplePart &b) {
  const float m = fmaxf(a.m, b.m);
  a.sum = a.sum * __builtin_amdgcn_exp2f((a.m - m) * LOG2E) + b.sum * __builtin_amdgcn_exp2f((b.m - m) * LOG2E);
  a.m = m;
  if (b.best > a.best || (b.best == a.best && (uint32_t)b.arg < (uint32_t)a.arg)) {
    a.best = b.best;
    a.arg = b.arg;
    a.x = b.x;
  }
}

__device__ __forceinline__ SamplePart part_xor(const SamplePart &a, int s) {
  SamplePart b;
  b.best = __shfl_xor(a.best, s);
  b.m = __shfl_xor(a.m, s);
  b.sum = __shfl_xor(a.sum, s);
  b.x = __shfl_xor(a.x, s);
  b.arg = __shfl_xor(a.arg, s);
  return b;
}

__device__ __forceinline__ void part_write(const SamplePart &s, uint64_t row, int32_t *index, float *logprob) {
  // no sum: nothing is allowed; NaN: a NaN or +inf among the logits
  const bool ok = s.sum > 0.0f && s.arg >= 0;
  index[row] = ok ? s.arg : -1;
  logprob[row] = ok ? (s.x - s.m) - logf(s.sum) : __builtin_nanf("");
}

constexpr int S_BLOCK = 512;

template <class T>
__global__ __launch_bounds__(S_BLOCK) void sample_kernel(LogitRows a, const float *__restrict__ u,
                                                         int64_t u_stride, uint32_t seg, uint32_t n_seg,
                                                         uint32_t chunk, SamplePart *__restrict__ parts,
                                                         int32_t *__restrict__ index,
                                                         float *__restrict__ logprob) {
  extern __shared__ uint32_t lds[];
  __shared__ SamplePart wave_part[S_BLOCK / 64];
  const bool table = a.history || a.n_bias;
  float *btab = reinterpret_cast<float *>(lds + chunk);
  const uint64_t n_tasks = a.rows * n_seg;
  for (uint64_t task = blockIdx.x; task < n_tasks; task += gridDim.x) {
    const uint64_t row = task / n_seg;
    const uint32_t s0 = (uint32_t)(task % n_seg) * seg, s1 = min(s0 + seg, a.q);
    const RowParams p = row_params(a, row);
    const bool scaled = p.t > 0.0f, noisy = u && (scaled || !a.temperature);
    const float rt = scaled ? 1.0f / p.t : 1.0f;
    const T *z = reinterpret_cast<const T *>(a.z) + (int64_t)row * a.z_stride;
    const float *ur = noisy ? u + (int64_t)row * u_stride : nullptr;
    const uint8_t *mask = a.mask ? reinterpret_cast<const uint8_t *>(a.mask + (int64_t)row * a.mask_stride) : nullptr;
    SamplePart s{-INFINITY, -__FLT_MAX__, 0.0f, 0.0f, -1};
    float thr = -INFINITY;  // of the wave
    for (uint32_t c0 = s0; c0 < s1; c0 += chunk) {
      const uint32_t n = min(chunk, s1 - c0);
      if (table) build_table(a, p, row, c0, (n + 7u) & ~7u, lds, btab);
      // whole waves stay in the loop: the threshold is the wave's
      for (uint32_t d0 = (threadIdx.x & ~63u) * 8u; d0 < n; d0 += S_BLOCK * 8u) {
        const uint32_t d = d0 + (threadIdx.x & 63u) * 8u, c = c0 + d;
        float x[8], y[8] = {}, v[8];
        Raw8<T> r{};
        Raw8<float> ru{};
        uint32_t live = 0;
        if (d + 8u <= n) {
          load8(z + c, r);
          if (noisy) load8(ur + c, ru);
          live = mask ? mask[c / 8u] : 255u;
        } else if (d < n) {
          load8_part(z + c, n - d, r);
          if (noisy) load8_part(ur + c, n - d, ru);
          live = (mask ? mask[c / 8u] : 255u) & ((1u << (n - d)) - 1u);
        }
        if (live) row_values(r, table ? lds : nullptr, btab, d, p, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (live >> j & 1u) ? y[j] * rt : -INFINITY;
        float m = s.m;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, x[j]);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += __builtin_amdgcn_exp2f((x[j] - m) * LOG2E);
        s.sum = s.sum * __builtin_amdgcn_exp2f((s.m - m) * LOG2E) + sum;
        s.m = m;
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = x[j];
          if (noisy) {
            const float l = __builtin_amdgcn_logf(fmaxf(__builtin_bit_cast(float, ru.w[j]), 0x1p-126f));
            v[j] = x[j] + __builtin_fmaf(__builtin_amdgcn_logf(-l), -0.693147182f, 0.366512921f);
          }
          top = fmaxf(top, v[j]);
        }
        if (__any(top > thr)) {
          uint32_t todo = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) todo |= (v[j] > thr ? 1u : 0u) << j;
          while (todo) {
            const int j = __builtin_ctz(todo);
            todo &= todo - 1u;
            float yj = y[0];
            uint32_t uj = ru.w[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) {
              yj = i == j ? y[i] : yj;
              uj = i == j ? ru.w[i] : uj;
            }
            const float xj = scaled ? yj / p.t : yj;
            double e = xj;
            if (noisy) {
              e = xj - log(-log((double)__builtin_bit_cast(float, uj)));
              e = e == -INFINITY && xj > -INFINITY ? -__DBL_MAX__ : e;
            }
            if (e > s.best) {
              s.best = e;
              s.x = xj;
              s.arg = (int32_t)(c + j);
            }
          }
          float b = (float)s.best;
#pragma unroll
          for (int k = 32; k > 0; k >>= 1) b = fmaxf(b, __shfl_xor(b, k));
          thr = noisy || scaled ? b - (S_MARGIN + fabsf(b) * S_REL) : b;
        }
      }
      if (table) __syncthreads();
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) part_merge(s, part_xor(s, k));
    if ((threadIdx.x & 63u) == 0) wave_part[threadIdx.x / 64u] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < S_BLOCK / 64; ++w) part_merge(s, wave_part[w]);
      if (n_seg > 1)
        parts[task] = s;
      else
        part_write(s, row, index, logprob);
    }
    __syncthreads();
  }
}

// one wave per row
__global__ __launch_bounds__(64) void sample_join_kernel(const SamplePart *__restrict__ parts, uint64_t rows,
                                                         uint32_t n_seg, int32_t *__restrict__ index,
                                                         float *__restrict__ logprob) {
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    SamplePart s{-INFINITY, -__FLT_MAX__, 0.0f, 0.0f, -1};
    for (uint32_t i = threadIdx.x; i < n_seg; i += 64u) part_merge(s, parts[row * n_seg + i]);
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) part_merge(s, part_xor(s, k));
    if (threadIdx.x == 0) part_write(s, row, index, logprob);
  }
}

// Segments of a row: enough workgroups for the device, none shorter than a pass of a workgroup.
static void sample_split(thrml_ctx *ctx, uint64_t rows, uint32_t q, uint32_t *seg, uint32_t *n_seg) {
  constexpr uint32_t unit = S_BLOCK * 8;
  uint32_t n = 1;
  while (rows * n * 2 <= 2ull * ctx->cu_count && cdiv(q, n * 2) >= unit) n *= 2;
  *seg = cdiv(cdiv(q, n), unit) * unit;
  *n_seg = cdiv(q, *seg);
}

uint64_t sample_logits_work(thrml_ctx *ctx, uint64_t rows, uint32_t q) {
  uint32_t seg, n;
  sample_split(ctx, rows, q, &seg, &n);
  return n > 1 ? rows * n * sizeof(SamplePart) : 0;
}

int launch_sample_logits(thrml_ctx *ctx, const LogitRows &a, int dtype, const float *u, int64_t u_stride,
                         int32_t *index, float *logprob, void *work) {
  if (a.rows == 0) return THRML_OK;
  uint32_t seg, n_seg;
  sample_split(ctx, a.rows, a.q, &seg, &n_seg);
  const uint32_t chunk = 4096;
  const size_t lds = (a.n_bias ? 2 : a.history ? 1 : 0) * (size_t)chunk * 4;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(a.rows * n_seg, 1u << 20);
  SamplePart *parts = reinterpret_cast<SamplePart *>(work);
  const int rc = with_type(dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    hipLaunchKernelGGL((sample_kernel<T>), dim3(grid), dim3(S_BLOCK), lds, ctx->stream, a, u, u_stride, seg, n_seg,
                       chunk, parts, index, logprob);
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
  if (rc || n_seg == 1) return rc;
  hipLaunchKernelGGL(sample_join_kernel, dim3((uint32_t)std::min<uint64_t>(a.rows, 1u << 20)), dim3(64), 0, ctx->stream,
                     parts, a.rows, n_seg, index, logprob);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

// ---------------------------------------------------------------------------
// Distillation from a teacher's top k candidates.  With z = logits / tau, lse =
// log sum exp z, p = softmax(teacher / tau) over the row's entries,
//   loss = tau^2 sum_i p_i (log p_i - z[id_i] + lse)
//   d(weight loss)/d logits = weight tau (softmax(z) - p)
// Two passes over a row: the running maximum and sum, then the gradient.
constexpr int D_BLOCK = 512;

template <class Op>
__device__ __forceinline__ float block_reduce(float v, float *buf, Op op) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) v = op(v, __shfl_xor(v, k));
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) buf[threadIdx.x / 64u] = v;
  __syncthreads();
  float r = buf[0];
  for (uint32_t w = 1; w < blockDim.x / 64u; ++w) r = op(r, buf[w]);
  return r;
}
struct MaxOp {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct AddOp {
  __device__ float operator()(float a, float b) const { return a + b; }
};

// e^x: the hardware's 2^x of the rounded product, times what the rounding left
// out (the relative error stays at 2 in 10^7 for x down to -100, 2 in 10^6 without)
__device__ __forceinline__ float exp_wide(float x) {
  const float p = x * LOG2E;
  const float e = __builtin_fmaf(x, LOG2E, -p) + x * 1.92596299e-8f;
  const float r = __builtin_amdgcn_exp2f(p);
  return p == -INFINITY ? 0.0f : __builtin_fmaf(r, e * 0.693147182f, r);
}

template <class T>
__global__ __launch_bounds__(D_BLOCK) void distill_kernel(DistillArgs a) {
  extern __shared__ uint32_t lds[];
  __shared__ float buf[D_BLOCK / 64];
  int32_t *ids = reinterpret_cast<int32_t *>(lds);
  float *pr = reinterpret_cast<float *>(lds + a.k);
  const float rtau = 1.0f / a.tau;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *z = reinterpret_cast<const T *>(a.z) + (int64_t)row * a.z_stride;
    float m = -__FLT_MAX__, sum = 0.0f;
    for (uint32_t c = threadIdx.x * 8u; c < a.q; c += D_BLOCK * 8u) {
      Raw8<T> r;
      float x[8];
      const uint32_t n = a.q - c;
      if (n >= 8u)
        load8(z + c, r);
      else
        load8_part(z + c, n, r);
      float mn = m, t = 0.0f;
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        x[j] = j < n ? value(r, j) * rtau : -INFINITY;
        mn = fmaxf(mn, x[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) t += __builtin_amdgcn_exp2f((x[j] - mn) * LOG2E);
      sum = sum * __builtin_amdgcn_exp2f((m - mn) * LOG2E) + t;
      m = mn;
    }
    const float top = block_reduce(m, buf, MaxOp());
    sum = block_reduce(sum * __builtin_amdgcn_exp2f((m - top) * LOG2E), buf, AddOp());
    // log softmax(z) = (z - top) - ls: the two parts stay apart, so that logits of
    // any size lose nothing
    const float ls = logf(sum);
    // the teacher's entries; those out of range do not count
    const int32_t *id_row = a.ids + (int64_t)row * a.ids_stride;
    const float *t_row = a.teacher + (int64_t)row * a.teacher_stride;
    float tm = -INFINITY;
    for (uint32_t i = threadIdx.x; i < a.k; i += D_BLOCK) {
      const int32_t id = id_row[i];
      const bool ok = (uint32_t)id < a.q;
      const float t = ok ? t_row[i] / a.tau : -INFINITY;
      ids[i] = ok ? id : -1;
      pr[i] = t;
      tm = fmaxf(tm, t);
    }
    tm = block_reduce(tm, buf, MaxOp());
    if (!(tm > -INFINITY)) tm = 0.0f;
    float ts = 0.0f;
    for (uint32_t i = threadIdx.x; i < a.k; i += D_BLOCK) ts += expf(pr[i] - tm);
    ts = block_reduce(ts, buf, AddOp());
    const float lts = logf(ts), rts = 1.0f / ts;
    float l = 0.0f;
    for (uint32_t i = threadIdx.x; i < a.k; i += D_BLOCK) {
      const float lp = (pr[i] - tm) - lts;
      const float p = expf(pr[i] - tm) * rts;
      if (p != 0.0f && ids[i] >= 0) l += p * (lp - (((float)z[ids[i]] * rtau - top) - ls));
      pr[i] = p;
    }
    l = block_reduce(l, buf, AddOp());
    const bool none = ts == 0.0f;  // no entry
    if (threadIdx.x == 0) a.loss[row] = none ? 0.0f : a.tau * a.tau * l;
    if (a.weight) {
      const float f = a.tau * a.weight[row];
      T *g = reinterpret_cast<T *>(a.grad) + (int64_t)row * a.grad_stride;
      for (uint32_t c = threadIdx.x * 8u; c < a.q; c += D_BLOCK * 8u) {
        Raw8<T> r;
        float x[8];
        const uint32_t n = a.q - c;
        if (n >= 8u)
          load8(z + c, r);
        else
          load8_part(z + c, n, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = none ? 0.0f : f * exp_wide((value(r, j) * rtau - top) - ls);
        store8(g + c, n, x);
      }
      __syncthreads();
      if (!none)
        for (uint32_t i = threadIdx.x; i < a.k; i += D_BLOCK) {
          const int32_t id = ids[i];
          if (id < 0) continue;
          bool first = true;
          for (uint32_t j = 0; j < i && first; ++j) first = ids[j] != id;
          if (!first) continue;
          float p = pr[i];
          for (uint32_t j = i + 1; j < a.k; ++j)
            if (ids[j] == id) p += pr[j];
          g[id] = (T)(f * (exp_wide(((float)z[id] * rtau - top) - ls) - p));
        }
    }
    __syncthreads();
  }
}

uint64_t distill_work(thrml_ctx *, uint64_t, uint32_t) { return 0; }

int launch_distill(thrml_ctx *ctx, const DistillArgs &a, int dtype, void *) {
  if (a.rows == 0) return THRML_OK;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(a.rows, 1u << 20);
  return with_type(dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    hipLaunchKernelGGL((distill_kernel<T>), dim3(grid), dim3(D_BLOCK), (size_t)a.k * 8, ctx->stream, a);
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
}

}  // namespace thrml
