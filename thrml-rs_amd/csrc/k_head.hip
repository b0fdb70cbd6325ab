// k_head.hip -- rows of logits of a learned head: processing, sampling, and
// distillation from a teacher's top candidates.
#include "dev_util.hpp"
#include "head.hpp"

namespace thrml {

static inline uint32_t cdiv(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// a launch of f with that much LDS of its own choice
static int lds_limit(const void *f, size_t bytes) {
  if (bytes > 65536) THRML_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return THRML_OK;
}

// ---------------------------------------------------------------------------
// What a row's history and biases say of a chunk of categories: a word for each in LDS,
//   bit 31   the category occurs in the prompt part of the history
//   bit 30   it has a bias, which a small hash table holds under its place in the
//            chunk (the sum of its entries, in list order)
//   bits 0-28  how often it was drawn after the prompt
// A workgroup scans the row's whole history for each chunk: it is short beside the
// row, its first entries stay in registers, and the rest lies in L2.
constexpr uint32_t T_PROMPT = 1u << 31, T_BIAS = 1u << 30, T_COUNT = (1u << 29) - 1u;
constexpr uint32_t NO_KEY = 0xffffffffu;

struct RowParams {
  Divisor theta;
  float presence, frequency, t;
  uint32_t len, prompt;
};

__device__ __forceinline__ RowParams row_params(const LogitRows &a, uint64_t row) {
  RowParams p{Divisor(a.repetition ? a.repetition[row] : 1.0f)};
  p.presence = a.presence ? a.presence[row] : 0.0f;
  p.frequency = a.frequency ? a.frequency[row] : 0.0f;
  p.t = a.temperature ? a.temperature[row] : 0.0f;
  const int32_t h = (int32_t)a.history_len;
  const int32_t len = a.lengths ? a.lengths[row] : h, pr = a.prompt_lengths ? a.prompt_lengths[row] : 0;
  p.len = (uint32_t)(len < 0 ? 0 : len > h ? h : len);
  p.prompt = (uint32_t)(pr < 0 ? 0 : pr);
  return p;
}

// The table's place in LDS: `chunk` words, then `hash` keys and values.
struct Table {
  uint32_t *tab, *keys;
  float *vals;
  uint32_t chunk, hash;
};

// Slots of the hash table for n biases: at least twice as many as a chunk can have.
static uint32_t hash_slots(uint32_t n_bias, uint32_t chunk) {
  if (!n_bias) return 0;
  uint32_t h = 64;
  while (h < 2 * std::min(n_bias, chunk)) h *= 2;
  return h;
}
static size_t table_bytes(const LogitRows &a, uint32_t chunk) {
  return a.history || a.n_bias ? (size_t)chunk * 4 + (size_t)hash_slots(a.n_bias, chunk) * 8 : 0;
}

__device__ __forceinline__ uint32_t hash_at(uint32_t d, uint32_t hash) { return (d * 2654435761u >> 12) & (hash - 1u); }

// The biases' hash table: a value for each place; bias_put is false where the place
// has one already.
__device__ __forceinline__ bool bias_put(uint32_t *keys, float *vals, uint32_t hash, uint32_t d, float v) {
  uint32_t h = hash_at(d, hash);
  for (;;) {  // (at most half of the slots are ever taken)
    const uint32_t old = atomicCAS(&keys[h], NO_KEY, d);
    if (old == NO_KEY) vals[h] = v;
    if (old == NO_KEY || old == d) return old != d;
    h = (h + 1u) & (hash - 1u);
  }
}
// a key's slot in a hash table that has it
__device__ __forceinline__ uint32_t slot_of(const uint32_t *keys, uint32_t hash, uint32_t d) {
  uint32_t h = hash_at(d, hash);
  while (keys[h] != d) h = (h + 1u) & (hash - 1u);
  return h;
}
__device__ __forceinline__ float bias_of(const uint32_t *keys, const float *vals, uint32_t hash, uint32_t d) {
  return vals[slot_of(keys, hash, d)];
}
// Where a category is named more than once, its entries are added in list order by the
// thread of the first one.
__device__ __forceinline__ void bias_sums(const LogitRows &a, const int32_t *ids, const float *vals, uint32_t c0,
                                          uint32_t n, const uint32_t *keys, float *sums, uint32_t hash,
                                          uint32_t block) {
  for (uint32_t i = threadIdx.x; i < a.n_bias; i += block) {
    const int32_t id = ids[i];
    if ((uint32_t)id - c0 >= n) continue;
    bool first = true;
    for (uint32_t j = 0; j < i && first; ++j) first = ids[j] != id;
    if (!first) continue;
    float s = vals[i];
    for (uint32_t j = i + 1; j < a.n_bias; ++j)
      if (ids[j] == id) s += vals[j];
    sums[slot_of(keys, hash, (uint32_t)id - c0)] = s;
  }
}

// What a lane keeps of its row's lists: of the first 4096 history entries, 4
// neighbouring ones at a time (the row's length is applied at their use, so that
// these loads wait for nothing; behind the history's end: -1, which no chunk holds),
// and of the first BLOCK biases.
template <int BLOCK>
struct RowLists {
  static constexpr int KEPT = BLOCK == 1024 ? 1 : 2;
  int32_t id[KEPT][4], bias_id;
  float bias;
  __device__ __forceinline__ void load(const LogitRows &a, uint64_t row, uint32_t tid) {
    if (a.history) {
      const int32_t *h = a.history + (int64_t)row * a.history_stride;
#pragma unroll
      for (int k = 0; k < KEPT; ++k) get(h, a.history_len, (uint32_t)k * BLOCK * 4u + tid * 4u, id[k]);
    }
    bias_id = -1;
    bias = 0.0f;
    if (tid < a.n_bias) {
      bias_id = a.bias_ids[(int64_t)row * a.bias_stride + tid];
      bias = a.bias_values[(int64_t)row * a.bias_stride + tid];
    }
  }
  static __device__ __forceinline__ void get(const int32_t *h, uint32_t len, uint32_t i, int32_t (&v)[4]) {
    typedef int32_t i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
    if (i + 4u <= len) {
      const i32x4_a4 x = *reinterpret_cast<const i32x4_a4 *>(h + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = x[j];
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) v[j] = i + j < len ? h[i + j] : -1;
    }
  }
};

__device__ __forceinline__ void table_clear(const Table &t, uint32_t block) {
  for (uint32_t i = here(threadIdx.x) * 4u; i < t.chunk; i += block * 4u)
    *reinterpret_cast<uint4 *>(t.tab + i) = make_uint4(0, 0, 0, 0);
}

// Fills the (cleared) table for categories c0 .. c0 + chunk - 1.  The workgroup calls
// it together; it begins and ends with a barrier.
template <int BLOCK>
__device__ __forceinline__ void table_fill(const LogitRows &a, const RowParams &p, const RowLists<BLOCK> &lists,
                                           uint64_t row, uint32_t c0, const Table &t) {
  constexpr int KEPT = RowLists<BLOCK>::KEPT;
  const uint32_t tid = here(threadIdx.x);
  __syncthreads();
  if (t.hash) {
    for (uint32_t i = tid; i < t.hash; i += BLOCK) t.keys[i] = NO_KEY;
    __syncthreads();
  }
  auto note = [&](uint32_t i, const int32_t (&v)[4]) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t d = (uint32_t)v[j] - c0;
      if (d < t.chunk && i + j < p.len) {
        if (i + j < p.prompt)
          atomicOr(&t.tab[d], T_PROMPT);
        else
          atomicAdd(&t.tab[d], 1u);
      }
    }
  };
  if (p.len) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k)
      if ((uint32_t)k * BLOCK * 4u < p.len) note((uint32_t)k * BLOCK * 4u + tid * 4u, lists.id[k]);
    const int32_t *h = a.history + (int64_t)row * a.history_stride;
    for (uint32_t i = KEPT * BLOCK * 4u + tid * 4u; i < p.len; i += 2u * BLOCK * 4u) {
      int32_t v[2][4];
      RowLists<BLOCK>::get(h, p.len, i, v[0]);
      RowLists<BLOCK>::get(h, p.len, i + BLOCK * 4u, v[1]);
      note(i, v[0]);
      note(i + BLOCK * 4u, v[1]);
    }
  }
  if (a.n_bias) {
    const int32_t *ids = a.bias_ids + (int64_t)row * a.bias_stride;
    const float *vals = a.bias_values + (int64_t)row * a.bias_stride;
    int again = 0;
    const uint32_t n = min(t.chunk, a.q - c0);
    for (uint32_t i = tid; i < a.n_bias; i += BLOCK) {
      const uint32_t d = (uint32_t)(i == tid ? lists.bias_id : ids[i]) - c0;
      if (d < n) {
        atomicOr(&t.tab[d], T_BIAS);
        again |= bias_put(t.keys, t.vals, t.hash, d, i == tid ? lists.bias : vals[i]) ? 0 : 1;
      }
    }
    if (__syncthreads_or(again)) bias_sums(a, ids, vals, c0, n, t.keys, t.vals, t.hash, BLOCK);
  }
  __syncthreads();
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// z with its row's penalties, each step rounded to f32 (w = 0: none); ANY: for a repetition
// penalty that is not fine(), too
template <bool ANY>
__device__ __forceinline__ float penalised(float z, uint32_t w, const RowParams &p) {
  const uint32_t n = w & T_COUNT;
  const float fn = (float)n;
  float y = z > 0.0f ? ANY ? z / p.theta.b : p.theta.fast(z) : z * p.theta.b;
  y = (w & ~T_BIAS) ? y : z;
  const float less = (y - p.frequency * fn) - p.presence;
  return n ? less : y;
}

// y[j] = the 8 logits at place d of the chunk with penalties and biases; their table
// words are cleared for the next chunk
template <class T>
__device__ __forceinline__ void row_values(const Raw8<T> &r, bool table, const Table &t, uint32_t d,
                                           const RowParams &p, float (&y)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = value(r, j);
  if (table) {
    uint4 *w4 = reinterpret_cast<uint4 *>(t.tab + d);
    const uint4 t0 = w4[0], t1 = w4[1];
    if ((t0.x | t0.y | t0.z | t0.w | t1.x | t1.y | t1.z | t1.w) != 0u) {
      const uint32_t w[8] = {t0.x, t0.y, t0.z, t0.w, t1.x, t1.y, t1.z, t1.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = penalised<false>(y[j], w[j], p);
      if (((w[0] | w[1] | w[2] | w[3] | w[4] | w[5] | w[6] | w[7]) & T_BIAS) != 0u) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (w[j] & T_BIAS) y[j] = y[j] + bias_of(t.keys, t.vals, t.hash, d + j);
      }
      w4[0] = w4[1] = make_uint4(0, 0, 0, 0);
    }
  }
}

// Eight logits at place d of n; what lies behind them has the bits `fill`.
template <class T>
__device__ __forceinline__ void load_place(const T *z, uint32_t d, uint32_t n, Raw8<T> &r, uint32_t fill = 0) {
  if (d + 8u <= n)
    load8(z + d, r);
  else
    load8_part(z + d, d < n ? n - d : 0u, r, fill);
}
template <class T>
constexpr uint32_t LOWEST = sizeof(T) == 4 ? 0xff800000u : __is_same(T, bf16_t) ? 0xff80u : 0xfc00u;  // -inf

// Values computed from r so far are not kept for later uses of r.
template <class T>
__device__ __forceinline__ void hide(Raw8<T> &r) {
#pragma unroll
  for (int i = 0; i < Raw8<T>::W; ++i) asm volatile("" : "+v"(r.w[i]));
}

// ---------------------------------------------------------------------------
// Processing: a workgroup writes P_BLOCK * 8 V categories of one row.  Their logits
// are on their way while it fills its table.
//
// Memory bounds it: 512 x 65536 f32 without lists take 47 us (5.7 TB/s, part of it from
// the last-level cache).  Histories of 6144 entries on average bring that to 69 us (285
// MB, 4.1 TB/s): each of a row's 8 workgroups scans them, 0.75 entries per logit, and
// waits for the scan at two barriers.  At 80 registers three workgroups of a compute
// unit cover each other's waits (two, at 128 registers: 76 us).  A call whose workgroups are
// all there at once has no such cover: 48 x 131071 f16 in 768 of them take 14.2 us, and 10.3
// without lists.
constexpr int P_BLOCK = 512;

template <class TI, class TO, int V>
__global__ __launch_bounds__(P_BLOCK, 6) void process_kernel(LogitRows a, TO *__restrict__ out, int64_t out_stride,
                                                          uint32_t n_chunks, uint64_t n_tasks, uint32_t hash) {
  extern __shared__ __align__(16) uint32_t lds[];
  constexpr uint32_t CHUNK = P_BLOCK * 8 * V;
  const bool table = a.history || a.n_bias;
  const Table tab{lds, lds + CHUNK, reinterpret_cast<float *>(lds + CHUNK + hash), CHUNK, hash};
  if (table) table_clear(tab, P_BLOCK);
  // neighbouring chunks on one XCD: its L2 then reads a row's lists once
  for (uint64_t task = xcd_remap(blockIdx.x, gridDim.x); task < n_tasks; task += gridDim.x) {
    const uint32_t tid = here(threadIdx.x);  // (what follows from it is not kept over the loop)
    const uint64_t row = task / n_chunks;
    const uint32_t c0 = (uint32_t)(task % n_chunks) * CHUNK;
    const uint32_t n = min(CHUNK, a.q - c0);
    const TI *z = reinterpret_cast<const TI *>(a.z) + (int64_t)row * a.z_stride + c0;
    TO *o = out + (int64_t)row * out_stride + c0;
    const uint8_t *mask =
        a.mask ? reinterpret_cast<const uint8_t *>(a.mask + (int64_t)row * a.mask_stride) + c0 / 8u : nullptr;
    // the lists first: loads end in their order, and the table waits for these alone
    RowLists<P_BLOCK> lists;
    if (table) lists.load(a, row, tid);
    RowParams p = row_params(a, row);
    p.theta.scalar();
    Raw8<TI> r[V];
    uint32_t m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t d = ((uint32_t)v * P_BLOCK + tid) * 8u;
      load_place(z, d, n, r[v]);
      m[v] = mask && d < n ? mask[d / 8u] : 255u;
    }
    Divisor t(p.t > 0.0f ? p.t : 1.0f);
    t.scalar();
    if (table) table_fill(a, p, lists, row, c0, tab);
    loads_done();
    if (__builtin_expect(!p.theta.fine() || !t.fine(), 0)) {
      // a subnormal divisor: full divisions, one category at a time, from pointers of its own
      // (a second form of the divisions in the loop below, or its pointers kept for this one,
      // cost the rows of other divisors: 512 x 65536 takes 69 us, and took 76 to 102)
      const int64_t row_ = opaque((uint32_t)row);
      const TI *z_ = reinterpret_cast<const TI *>(a.z) + row_ * a.z_stride;
      const uint8_t *mask_ = reinterpret_cast<const uint8_t *>(a.mask + row_ * a.mask_stride);
#pragma unroll 1
      for (uint32_t d = tid; d < n; d += P_BLOCK) {
        const uint32_t w = table ? tab.tab[d] : 0u, c = c0 + d;
        float y = penalised<true>((float)z_[c], w, p);
        if (w & T_BIAS) y = y + bias_of(tab.keys, tab.vals, hash, d);
        if (p.t > 0.0f) y = y / p.t;
        if (a.mask && !(mask_[c / 8u] >> (c % 8u) & 1u)) y = -INFINITY;
        o[d] = (TO)y;
        if (table) tab.tab[d] = 0;
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const uint32_t d = ((uint32_t)v * P_BLOCK + tid) * 8u;
        if (d >= n) break;
        float y[8];
        row_values(r[v], table, tab, d, p, y);
        if (p.t > 0.0f) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = t.fast(y[j]);
        }
        if (mask) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = (m[v] >> j & 1u) ? y[j] : -INFINITY;
        }
        store8(o + d, n - d, y);
      }
    }
    // (the last chunk's words behind the row's end belong to no one)
    if (table && gridDim.x < n_tasks) {
      __syncthreads();
      table_clear(tab, P_BLOCK);
    }
  }
}

int launch_process_logits(thrml_ctx *ctx, const LogitRows &a, int dtype, void *out, int out_dtype,
                          int64_t out_stride) {
  if (a.rows == 0) return THRML_OK;
  // two groups of 8 per lane where that leaves two workgroups for each compute unit, and
  // LDS for many biases (one, two and four groups, of which the last spill registers: 48 x
  // 131071 17.7, 14.2 and 16.8 us, 512 x 65536 83.5, 68.5 and 115)
  const bool two = a.rows * cdiv(a.q, P_BLOCK * 16) >= 2ull * ctx->cu_count && a.n_bias <= 1024;
  const uint32_t chunk = P_BLOCK * (two ? 16 : 8), nc = cdiv(a.q, chunk);
  const uint64_t tasks = a.rows * nc;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(tasks, 1u << 20), hash = hash_slots(a.n_bias, chunk);
  return with_type(dtype, [&](auto ti) {
    return with_type(out_dtype, [&](auto to) -> int {
      typedef decltype(ti) TI;
      typedef decltype(to) TO;
      auto *f = two ? &process_kernel<TI, TO, 2> : &process_kernel<TI, TO, 1>;
      if (int rc = lds_limit(reinterpret_cast<const void *>(f), table_bytes(a, chunk))) return rc;
      hipLaunchKernelGGL(f, dim3(grid), dim3(P_BLOCK), table_bytes(a, chunk), ctx->stream, a,
                         reinterpret_cast<TO *>(out), out_stride, nc, tasks, hash);
      THRML_HIP(hipGetLastError());
      return THRML_OK;
    });
  });
}

// ---------------------------------------------------------------------------
// Sampling.  With x the processed logits, a row's category is the first argmax
// over the allowed ones of x - log(-log u) (Gumbel-max), or of x for a greedy
// row, all in one pass over the row: the running maximum and sum of a softmax per lane,
// and the pick.  With y the logits before the temperature t and m the largest of them,
// the log-probability is (y - m) / t - log(sum exp((y - m) / t)): its error follows the
// distance from the largest logit, and it is never above 0.
//
// The pick is exact in 64 bits at f32 cost.  v, the score from hardware logarithms and
// y times a reciprocal of the temperature, is within S_MARGIN / 2 + |v| S_REL / 2 of the
// score in 64 bits; picks are compared by v where that decides and in 64 bits, from x as
// the steps in f32 give it, where it does not.  A lane keeps its best group of 8 by v
// and the best v of its other groups; at the end of a part of the row the workgroup's
// best v less the margin says which lanes look at their group again (or, if their
// second is that close, at all their groups): mostly one.  v of a u below 2^-126 is that
// of 2^-126, no less than its own: where one comes into play, the row is done again
// without a bound.  An allowed category whose own score is -inf (u = 0) is taken only
// where there is no other, a masked one never.
// (The noise from hardware logarithms is within 1.98e-6 of -log(-log u) for every f32 u from
// 2^-126 to 1, all of them tried.)
constexpr float S_MARGIN = 1e-4f, S_REL = 0x1p-18f;
constexpr float LOG2E = 1.44269504f;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
  return v;
}

// What multiplies a row's logits (exact, but for overflows that their quotients share) and
// the divisor that is left of its temperature, with a reciprocal that is finite and above 0.
// A subnormal temperature is brought up by 2^64; over an infinite one a logit is 0, or NaN.
// A temperature that is not above 0 leaves the logits as they are.
struct Scaled {
  float by, d;
  __device__ __forceinline__ explicit Scaled(float t) {  // (no branches: loads behind it would wait for t)
    const bool tiny = t > 0.0f && t < 0x1p-126f, endless = t == INFINITY;
    by = tiny ? 0x1p64f : endless ? 0.0f : 1.0f;
    d = tiny ? t * 0x1p64f : t > 0.0f && !endless ? t : 1.0f;
  }
};

// Here and below y is a logit as Scaled::by makes it: x = y / d.
struct SamplePart {
  float m, sum;   // running maximum of y, and sum of exp((y - m) / d)
  float v, y, u;  // of the pick: its score in 32 bits, logit and uniform (-1: the logit is the score)
  int32_t arg;    // -1: none yet
};
constexpr float U_MIN = 0x1p-126f;

__device__ __forceinline__ double exact_score(float x, float u) {
  if (u < 0.0f) return x;
  const double e = x - log(-log((double)u));
  return e == -INFINITY && x > -INFINITY ? -__DBL_MAX__ : e;
}
// b's pick comes before a's: by v where that decides, else in 64 bits.
__device__ __forceinline__ bool beats(const SamplePart &b, const SamplePart &a, float d) {
  if (b.arg < 0 || a.arg < 0) return b.arg >= 0;
  const float margin = 2.0f * S_MARGIN + (fabsf(a.v) + fabsf(b.v)) * S_REL, lead = b.v - a.v;
  if (lead > margin && b.u >= U_MIN) return true;
  if (lead < -margin && a.u >= U_MIN) return false;
  const double ea = exact_score(a.y / d, a.u), eb = exact_score(b.y / d, b.u);
  return eb > ea || (eb == ea && b.arg < a.arg);
}

// c: log2 e / d
__device__ __forceinline__ void part_merge(SamplePart &a, const SamplePart &b, float d, float c) {
  const float m = fmaxf(a.m, b.m);
  a.sum = a.sum * __builtin_amdgcn_exp2f((a.m - m) * c) + b.sum * __builtin_amdgcn_exp2f((b.m - m) * c);
  a.m = m;
  if (beats(b, a, d)) {
    a.v = b.v;
    a.y = b.y;
    a.u = b.u;
    a.arg = b.arg;
  }
}

// of all lanes of a wave, in lane 0 (a loop, so that there is one merge to compile)
__device__ __forceinline__ void part_join_wave(SamplePart &a, float d, float c) {
#pragma unroll 1
  for (int s = 32; s > 0; s >>= 1) {
    SamplePart b;
    b.m = __shfl_xor(a.m, s);
    b.sum = __shfl_xor(a.sum, s);
    b.v = __shfl_xor(a.v, s);
    b.y = __shfl_xor(a.y, s);
    b.u = __shfl_xor(a.u, s);
    b.arg = __shfl_xor(a.arg, s);
    part_merge(a, b, d, c);
  }
}

__device__ __forceinline__ void part_write(const SamplePart &s, float d, uint64_t row, int32_t *index, float *logprob) {
  // no sum: nothing is allowed; NaN: a NaN or +inf among the logits; and the largest
  // quotient may be infinite where the logit is not
  const bool ok = s.sum > 0.0f && s.arg >= 0 && fabsf(s.m / d) < INFINITY;
  index[row] = ok ? s.arg : -1;
  logprob[row] = ok ? (s.y - s.m) / d - logf(s.sum) : __builtin_nanf("");
}

// What the lists name is few beside the row and goes apart: a hash table in LDS holds
// the words (T_PROMPT, T_BIAS, count) of the categories named in a part of the row,
// a bitmap says which these are, and a list has them in the bitmap's order.  The pass
// over the part leaves them out, and lanes score them from the list.  So the lists of
// the row are scanned once for a part, as large as LDS allows, and the waves go over it
// without a barrier.  (Their places in the table depend on which lane came first; the
// list does not, and with it the order in which exponentials are added.)
struct Named {
  uint32_t *keys, *words, *flags, *list, *bias_keys;
  float *bias_vals;
  uint32_t slots, hash;  // of the table, of the biases' table
};
constexpr uint32_t PART_MAX = 131072;  // categories that a bitmap of 16 KB holds

struct NamedPlan {
  uint32_t part, slots, list, hash;
  size_t bytes;
};
// The largest part (a multiple of unit, at least unit) whose tables take `limit` bytes.
static NamedPlan named_plan(const LogitRows &a, uint32_t seg, uint32_t unit, size_t limit) {
  NamedPlan p{std::min(seg, PART_MAX), 0, 0, 0, 0};
  if (!a.history && !a.n_bias) {
    p.part = seg;
    return p;
  }
  for (;;) {
    const uint64_t n = std::min<uint64_t>((uint64_t)a.history_len * (a.history ? 1 : 0) + a.n_bias, p.part);
    p.slots = (uint32_t)std::max<uint64_t>(512, (n * 4 / 3 + 4) & ~(uint64_t)3);  // at most three quarters are taken
    p.list = (uint32_t)(n + 3) & ~3u;
    p.hash = hash_slots(a.n_bias, p.part);
    p.bytes = (size_t)p.slots * 8 + p.part / 8 + (size_t)p.list * 4 + (size_t)p.hash * 8;
    if (p.bytes <= limit || p.part <= unit) return p;
    p.part = std::max(unit, p.part / 2 / unit * unit);
  }
}

// (any number of slots: a power of two would not fit 8192 entries beside the list)
__device__ __forceinline__ uint32_t named_first(const Named &t, uint32_t d) { return __umulhi(d * 2654435761u, t.slots); }
__device__ __forceinline__ uint32_t named_next(const Named &t, uint32_t h) { return h + 1u < t.slots ? h + 1u : 0u; }

__device__ __forceinline__ uint32_t named_slot(const Named &t, uint32_t d, bool *fresh) {
  uint32_t h = named_first(t, d);
  for (;;) {
    const uint32_t old = atomicCAS(&t.keys[h], NO_KEY, d);
    *fresh = old == NO_KEY;
    if (old == NO_KEY || old == d) return h;
    h = named_next(t, h);
  }
}
__device__ __forceinline__ uint32_t named_word(const Named &t, uint32_t d) {
  uint32_t h = named_first(t, d);
  while (t.keys[h] != d) h = named_next(t, h);  // it is there
  return t.words[h];
}

// Fills the tables for the n categories from c0 on, and gives the length of the list;
// begins and ends with a barrier.
template <int BLOCK>
__device__ __forceinline__ uint32_t named_fill(const LogitRows &a, const RowParams &p, const RowLists<BLOCK> &lists,
                                               uint64_t row, uint32_t c0, uint32_t n, const Named &t,
                                               uint32_t *wave_count) {
  constexpr int KEPT = RowLists<BLOCK>::KEPT;
  const uint32_t tid = here(threadIdx.x);
  __syncthreads();
  for (uint32_t i = tid; i < t.slots; i += BLOCK) {
    t.keys[i] = NO_KEY;
    t.words[i] = 0;
  }
  for (uint32_t i = tid; i < (n + 31u) / 32u; i += BLOCK) t.flags[i] = 0;
  for (uint32_t i = tid; i < t.hash; i += BLOCK) t.bias_keys[i] = NO_KEY;
  __syncthreads();
  auto name = [&](uint32_t d) {
    bool fresh;
    const uint32_t h = named_slot(t, d, &fresh);
    if (fresh) atomicOr(&t.flags[d / 32u], 1u << (d % 32u));
    return h;
  };
  auto note = [&](uint32_t i, const int32_t (&v)[4]) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t d = (uint32_t)v[j] - c0;
      if (i + j < p.len && d < n) {
        const uint32_t h = name(d);
        if (i + j < p.prompt)
          atomicOr(&t.words[h], T_PROMPT);
        else
          atomicAdd(&t.words[h], 1u);
      }
    }
  };
  if (a.history) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k)
      if ((uint32_t)k * BLOCK * 4u < p.len) note((uint32_t)k * BLOCK * 4u + tid * 4u, lists.id[k]);
    const int32_t *h = a.history + (int64_t)row * a.history_stride;
    for (uint32_t i = KEPT * BLOCK * 4u + tid * 4u; i < p.len; i += BLOCK * 4u) {
      int32_t v[4];
      RowLists<BLOCK>::get(h, p.len, i, v);
      note(i, v);
    }
  }
  if (a.n_bias) {
    const int32_t *ids = a.bias_ids + (int64_t)row * a.bias_stride;
    const float *vals = a.bias_values + (int64_t)row * a.bias_stride;
    int again = 0;
    for (uint32_t i = tid; i < a.n_bias; i += BLOCK) {
      const uint32_t d = (uint32_t)(i == tid ? lists.bias_id : ids[i]) - c0;
      if (d < n) {
        atomicOr(&t.words[name(d)], T_BIAS);
        again |= bias_put(t.bias_keys, t.bias_vals, t.hash, d, i == tid ? lists.bias : vals[i]) ? 0 : 1;
      }
    }
    if (__syncthreads_or(again)) bias_sums(a, ids, vals, c0, n, t.bias_keys, t.bias_vals, t.hash, BLOCK);
  }
  __syncthreads();
  const uint32_t words = (n + 31u) / 32u, lane = tid & 63u;
  uint32_t count = 0;
  for (uint32_t i = tid; i < words; i += BLOCK) count += __popc(t.flags[i]);
  uint32_t upto = count;
#pragma unroll
  for (uint32_t s = 1; s < 64; s *= 2) {
    const uint32_t v = __shfl_up(upto, s);
    if (lane >= s) upto += v;
  }
  if (lane == 63u) wave_count[tid / 64u] = upto;
  __syncthreads();
  uint32_t at = upto - count, total = 0;
#pragma unroll
  for (uint32_t w = 0; w < BLOCK / 64; ++w) {
    const uint32_t c = wave_count[w];
    at += w < tid / 64u ? c : 0u;
    total += c;
  }
  for (uint32_t i = tid; i < words; i += BLOCK)
    for (uint32_t bits = t.flags[i]; bits; bits &= bits - 1u) t.list[at++] = i * 32u + (uint32_t)__builtin_ctz(bits);
  __syncthreads();
  return total;
}

// One row's state in a lane.
struct Sampler {
  SamplePart s{-__FLT_MAX__, 0.0f, -INFINITY, 0.0f, -1.0f, -1};
  // of a part's groups: the best v, the place of its group, the best v of the others
  float first, second;
  uint32_t at;
  float t, rd;  // the temperature, 1 / Scaled::d (what follows from them is not kept in registers)
  bool scaled, noisy, odd = false;

  __device__ __forceinline__ float d() const { return Scaled(t).d; }
  __device__ __forceinline__ float c() const { return rd * LOG2E; }
  __device__ __forceinline__ void begin(const RowParams &p, const float *u, const float *temperature) {
    t = p.t;
    scaled = t > 0.0f;
    noisy = u && (scaled || !temperature);
    rd = 1.0f / Scaled(t).d;
  }

  // What v has to reach where the best is b.  Greedy rows without a temperature have
  // x exactly, and of equal ones the lowest category counts.
  __device__ __forceinline__ float bound(float b) const {
    return noisy || scaled ? b - (S_MARGIN + fabsf(b) * S_REL) : b;
  }

  // v of N logits with penalties and biases, which become y, -inf where the bit in live is
  // clear
  template <int N>
  __device__ __forceinline__ void scores(float (&y)[N], const uint32_t (&u)[N], uint32_t live, float (&v)[N]) const {
    if (__builtin_expect(__builtin_amdgcn_classf(t, 0x280), 0)) {  // a subnormal or infinite temperature
      const float by = Scaled(t).by;
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] *= by;
    }
    if (__any(live != (1u << N) - 1u)) {
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = (live >> j & 1u) ? y[j] : -INFINITY;
    }
    if (noisy) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float l =
            __builtin_amdgcn_logf(__builtin_amdgcn_fmed3f(__builtin_bit_cast(float, u[j]), U_MIN, INFINITY));
        v[j] = __builtin_fmaf(y[j], rd, __builtin_fmaf(__builtin_amdgcn_logf(-l), -0.693147182f, 0.366512921f));
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = y[j] * rd;
    }
  }

  template <int N>
  __device__ __forceinline__ void add(const float (&y)[N]) {
    float m = s.m;
    const float c = this->c();
#pragma unroll
    for (int j = 0; j < N; j += 2) m = max3(m, y[j], y[j + 1]);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) sum += __builtin_amdgcn_exp2f((y[j] - m) * c);
    s.sum = s.sum * __builtin_amdgcn_exp2f((s.m - m) * c) + sum;
    s.m = m;
  }

  // Eight logits from place d on.
  __device__ __forceinline__ void take(float (&y)[8], const uint32_t (&u)[8], uint32_t live, uint32_t place) {
    float v[8];
    scores(y, u, live, v);
    add(y);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; j += 2) top = max3(top, v[j], v[j + 1]);
    second = __builtin_amdgcn_fmed3f(second, first, top);
    at = top > first ? place : at;
    first = fmaxf(first, top);
  }

  // Those of N logits that `todo` names against the lane's pick; id(j): category.
  template <int N, class Id>
  __device__ __forceinline__ void settle(const float (&y)[N], const uint32_t (&u)[N], const float (&v)[N],
                                         uint32_t todo, Id id) {
    while (todo) {
      const int j = __builtin_ctz(todo);
      todo &= todo - 1u;
      float yj = y[0], vj = v[0];
      uint32_t uj = u[0];
#pragma unroll
      for (int i = 1; i < N; ++i) {
        yj = i == j ? y[i] : yj;
        uj = i == j ? u[i] : uj;
        vj = i == j ? v[i] : vj;
      }
      SamplePart b;
      b.v = vj;
      b.y = yj;
      b.u = noisy ? __builtin_bit_cast(float, uj) : -1.0f;
      b.arg = id(j);
      // (v of a u below 2^-126 is too high, and so are bounds that come from it)
      odd = odd || (noisy && b.u < U_MIN);
      if (beats(b, s, d())) {
        s.v = b.v;
        s.y = b.y;
        s.u = b.u;
        s.arg = b.arg;
      }
    }
  }

  template <int N>
  static __device__ __forceinline__ uint32_t reach(const float (&v)[N], const float (&y)[N], float cut) {
    uint32_t todo = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) todo |= (y[j] > -INFINITY && !(v[j] < cut) ? 1u : 0u) << j;
    return todo;
  }
};

// A lane's next 8 logits and uniforms.
//
// 256 x 131072 bf16, a workgroup of 1024 for a row: 40 us without lists (201 MB, 5.0 TB/s),
// 60 us with histories of 3000 entries on average.  The difference is a row's own: the
// table is filled before the pass over it begins, and the 2 % of categories that it names
// are fetched again one by one, with half a kilobyte of cache lines for 8 of them.  One
// instance does it all, at 128 registers, with up to 6 of them and about 110 scalars spilled
// (32 or 48 bytes of scratch a lane).
template <class T>
struct SampleGroup {
  Raw8<T> z;
  Raw8<float> u;
  uint32_t in, allowed;  // not joined before use: that would wait for all of the loads
  __device__ __forceinline__ void load(const T *z_, const float *u_, const uint8_t *mask, uint32_t c, uint32_t end) {
    load_place(z_, c, end, z);
    if (u_) load_place(u_, c, end, u);
    in = c >= end ? 0u : c + 8u <= end ? 255u : (1u << (end - c)) - 1u;
    allowed = mask && in ? mask[c / 8u] : 255u;
  }
};

template <class T, int BLOCK>
__global__ __launch_bounds__(BLOCK, 4) void sample_kernel(LogitRows a, const float *__restrict__ u, int64_t u_stride,
                                                          uint32_t seg, uint32_t n_seg, NamedPlan plan,
                                                          SamplePart *__restrict__ parts, int32_t *__restrict__ index,
                                                          float *__restrict__ logprob) {
  extern __shared__ __align__(16) uint32_t lds[];
  __shared__ SamplePart wave_part[BLOCK / 64];
  __shared__ float wave_best[BLOCK / 64];
  __shared__ uint32_t wave_count[BLOCK / 64];
  const bool table = a.history || a.n_bias;
  Named named;
  named.keys = lds;
  named.words = named.keys + plan.slots;
  named.flags = named.words + plan.slots;
  named.list = named.flags + plan.part / 32u;
  named.bias_keys = named.list + plan.list;
  named.bias_vals = reinterpret_cast<float *>(named.bias_keys + plan.hash);
  named.slots = plan.slots;
  named.hash = plan.hash;
  const uint8_t *flags = reinterpret_cast<const uint8_t *>(named.flags);
  const uint64_t n_tasks = a.rows * n_seg;
  for (uint64_t task = xcd_remap(blockIdx.x, gridDim.x); task < n_tasks; task += gridDim.x) {
    const uint32_t tid = here(threadIdx.x);
    const uint64_t row = task / n_seg;
    const uint32_t s0 = (uint32_t)(task % n_seg) * seg, s1 = min(s0 + seg, a.q);
    RowLists<BLOCK> lists;
    if (table) lists.load(a, row, tid);
    const RowParams p = row_params(a, row);
    Sampler s;
    s.begin(p, u, a.temperature);
    const T *z = reinterpret_cast<const T *>(a.z) + (int64_t)row * a.z_stride;
    const float *ur = s.noisy ? u + (int64_t)row * u_stride : nullptr;
    const uint8_t *mask = a.mask ? reinterpret_cast<const uint8_t *>(a.mask + (int64_t)row * a.mask_stride) : nullptr;
    for (bool bounded = true;; bounded = false) {
      SampleGroup<T> next{};
      next.load(z, ur, mask, s0 + tid * 8u, s1);
      for (uint32_t c0 = s0; c0 < s1; c0 += plan.part) {
        const uint32_t end = min(c0 + plan.part, s1);
        const uint32_t n_named = table ? named_fill(a, p, lists, row, c0, end - c0, named, wave_count) : 0u;
        auto group = [&](const SampleGroup<T> &k, uint32_t d, float (&y)[8]) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = value(k.z, j);
          const uint32_t live = k.in & k.allowed;
          return table && d < end ? live & ~(uint32_t)flags[(d - c0) / 8u] : live;
        };
        s.first = s.second = -INFINITY;
        s.at = c0;
        for (uint32_t d0 = c0 + (tid & ~63u) * 8u; d0 < end; d0 += BLOCK * 8u) {
          const uint32_t d = d0 + (tid & 63u) * 8u;
          const SampleGroup<T> k = next;
          // the next one: in this part, or this wave's first in the next part
          const uint32_t ahead = d0 + BLOCK * 8u < end ? d0 + BLOCK * 8u : end + (tid & ~63u) * 8u;
          if (ahead < s1) next.load(z, ur, mask, ahead + (tid & 63u) * 8u, s1);
          float y[8];
          const uint32_t live = group(k, d, y);
          s.take(y, k.u.w, live, d);
        }
        const float w = wave_max(s.first);
        if ((tid & 63u) == 0) wave_best[tid / 64u] = w;
        __syncthreads();
        float cut = -INFINITY;
        if (bounded) {
#pragma unroll
          for (int i = 0; i < BLOCK / 64; ++i) cut = fmaxf(cut, wave_best[i]);
          cut = s.bound(cut);
        }
        if (!(s.first < cut) && (s.first > -INFINITY || !bounded)) {
          const bool all = !(s.second < cut);
          for (uint32_t d = all ? c0 + tid * 8u : s.at; d < end; d += all ? BLOCK * 8u : end) {
            SampleGroup<T> k{};
            k.load(z, ur, mask, d, s1);
            float y[8], v[8];
            const uint32_t live = group(k, d, y);
            s.scores(y, k.u.w, live, v);
            s.settle(y, k.u.w, v, Sampler::reach(v, y, cut), [&](int j) { return (int32_t)(d + j); });
          }
        }
        // the named ones
        constexpr int N = 4;
        for (uint32_t b = 0; b < n_named; b += BLOCK * N) {
          float y[N], v[N];
          uint32_t c[N], n[N], r[N], live = 0;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const uint32_t i = b + (uint32_t)j * BLOCK + tid;
            c[j] = c0;
            n[j] = 0;
            if (i < n_named) {
              const uint32_t d = named.list[i];
              c[j] = c0 + d;
              n[j] = named_word(named, d);
              live |= 1u << j;
            }
          }
          if (!__any(live != 0u)) continue;
          // (places without one read the part's first: all loads are under way at once)
          T zc[N];
          uint32_t m[N];
#pragma unroll
          for (int j = 0; j < N; ++j) {
            zc[j] = z[c[j]];
            r[j] = 0;
            m[j] = 255u;
          }
          if (ur) {
#pragma unroll
            for (int j = 0; j < N; ++j) r[j] = __builtin_bit_cast(uint32_t, ur[c[j]]);
          }
          if (mask) {
#pragma unroll
            for (int j = 0; j < N; ++j) m[j] = mask[c[j] / 8u];
          }
#pragma unroll
          for (int j = 0; j < N; ++j) {
            if (!(m[j] >> (c[j] % 8u) & 1u)) live &= ~(1u << j);
            y[j] = penalised<true>((float)zc[j], n[j], p);
            if (n[j] & T_BIAS) y[j] = y[j] + bias_of(named.bias_keys, named.bias_vals, plan.hash, c[j] - c0);
          }
          s.scores(y, r, live, v);
          s.add(y);
          // (no bound but the other categories': few of these reach it)
          s.settle(y, r, v, Sampler::reach(v, y, cut), [&](int j) {
            uint32_t cj = c[0];
#pragma unroll
            for (int i = 1; i < N; ++i) cj = i == j ? c[i] : cj;
            return (int32_t)cj;
          });
        }
      }
      if (!__syncthreads_or(bounded && s.odd)) break;
      const Sampler again = s;
      s = Sampler{};
      s.t = again.t;
      s.rd = again.rd;
      s.scaled = again.scaled;
      s.noisy = again.noisy;
    }
    SamplePart o = s.s;
    part_join_wave(o, s.d(), s.c());
    if ((tid & 63u) == 0) wave_part[tid / 64u] = o;
    __syncthreads();
    if (tid == 0) {
#pragma unroll 1
      for (int w = 1; w < BLOCK / 64; ++w) part_merge(o, wave_part[w], s.d(), s.c());
      if (n_seg > 1)
        parts[task] = o;
      else
        part_write(o, s.d(), row, index, logprob);
    }
    __syncthreads();
    loads_done();
  }
}

// one wave per row
__global__ __launch_bounds__(64) void sample_join_kernel(const SamplePart *__restrict__ parts, uint64_t rows,
                                                         uint32_t n_seg, const float *__restrict__ temperature,
                                                         int32_t *__restrict__ index, float *__restrict__ logprob) {
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float d = Scaled(temperature ? temperature[row] : 0.0f).d, c = 1.0f / d * LOG2E;
    SamplePart s{-__FLT_MAX__, 0.0f, -INFINITY, 0.0f, -1.0f, -1};
    for (uint32_t i = threadIdx.x; i < n_seg; i += 64u) part_merge(s, parts[row * n_seg + i], d, c);
    part_join_wave(s, d, c);
    if (threadIdx.x == 0) part_write(s, d, row, index, logprob);
  }
}

// How a call is laid out: a workgroup of 1024 per row where there are about as many
// rows as compute units (two rows at a time would leave half of them idle at the
// end), of 512 for more rows, and segments of rows, joined by a second kernel, for
// few.
struct SamplePlan {
  bool wide;  // 1024 threads
  uint32_t seg, n_seg;
};
static SamplePlan sample_plan(thrml_ctx *ctx, uint64_t rows, uint32_t q) {
  SamplePlan p;
  p.wide = rows < 2ull * ctx->cu_count && rows * 2 > (uint64_t)ctx->cu_count && q > 8192;
  const uint32_t pass = p.wide ? 8192 : 4096;  // categories that a workgroup takes at a time
  uint32_t n = 1;
  if (!p.wide)
    while (rows * n * 2 <= 2ull * ctx->cu_count && cdiv(q, n * 2) >= pass) n *= 2;
  p.seg = cdiv(cdiv(q, n), pass) * pass;
  p.n_seg = cdiv(q, p.seg);
  return p;
}

uint64_t sample_logits_work(thrml_ctx *ctx, uint64_t rows, uint32_t q) {
  const SamplePlan p = sample_plan(ctx, rows, q);
  return p.n_seg > 1 ? rows * p.n_seg * sizeof(SamplePart) : 0;
}

int launch_sample_logits(thrml_ctx *ctx, const LogitRows &a, int dtype, const float *u, int64_t u_stride,
                         int32_t *index, float *logprob, void *work) {
  if (a.rows == 0) return THRML_OK;
  const SamplePlan p = sample_plan(ctx, a.rows, a.q);
  // Two workgroups of 512 in a compute unit's LDS, or one of 1024, which also takes the
  // segments whose lists would leave those several parts (512 x 65536 with histories of
  // 8192: 257 us in 16 parts each).
  NamedPlan named = named_plan(a, p.seg, 4096, 76 << 10);
  bool wide = p.wide || named.part < std::min(p.seg, PART_MAX);
  if (wide) {
    const NamedPlan one = named_plan(a, p.seg, 8192, 150 << 10);
    if (one.bytes <= 150 << 10)
      named = one;
    else
      wide = false;
  }
  const uint32_t grid = (uint32_t)std::min<uint64_t>(a.rows * p.n_seg, 1u << 20);
  SamplePart *parts = reinterpret_cast<SamplePart *>(work);
  const int rc = with_type(dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    auto *f = wide ? &sample_kernel<T, 1024> : &sample_kernel<T, 512>;
    if (int rc = lds_limit(reinterpret_cast<const void *>(f), named.bytes)) return rc;
    hipLaunchKernelGGL(f, dim3(grid), dim3(wide ? 1024 : 512), named.bytes, ctx->stream, a, u, u_stride, p.seg, p.n_seg,
                       named, parts, index, logprob);
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
  if (rc || p.n_seg == 1) return rc;
  hipLaunchKernelGGL(sample_join_kernel, dim3((uint32_t)std::min<uint64_t>(a.rows, 1u << 20)), dim3(64), 0, ctx->stream,
                     parts, a.rows, p.n_seg, a.temperature, index, logprob);
  THRML_HIP(hipGetLastError());
  return THRML_OK;
}

// ---------------------------------------------------------------------------
// Distillation from a teacher's top k candidates.  With z = logits / tau, p =
// softmax(teacher / tau) over the row's entries,
//   loss = tau^2 sum_i p_i (log p_i - log softmax(z)[id_i])
//   d(weight loss)/d logits = weight tau (softmax(z) - p)
// log softmax(z) = (z - m) - log(sum exp(z - m)) keeps its two parts apart, so that
// logits of any size lose nothing.
//
// A workgroup takes a row.  Its first wave does the teacher's part, with the
// candidates in LDS, while the row's logits load; the other waves need its result
// only behind the barrier that joins the maxima and sums.  The gradient is written
// without p first, and at the candidates' places once more behind a barrier.
//
// Where the row fits the workgroup's registers, the gradient reads it there: one
// read and one write of memory.  2048 x 131072 bf16: 247 us (1.07 GB, 4.4 TB/s; a copy
// reaches 4.8), 363 us reading the row twice.  Two exponentials and about 14 other
// operations for a logit keep the vector unit busy for 160 us of that.
// e^x: the hardware's 2^x of the rounded product, times what the rounding left
// out (the relative error stays at 1.4 in 10^7 down to e^x = 2^-125, 3.9 in 10^6 without)
__device__ __forceinline__ float exp_wide(float x) {
  const float p = x * LOG2E;
  const float e = __builtin_fmaf(x, LOG2E, -p) + x * 1.92596299e-8f;
  const float r = __builtin_amdgcn_exp2f(p);
  return p == -INFINITY ? 0.0f : __builtin_fmaf(r, e * 0.693147182f, r);
}

// The scaled logit's exponential against the row's sum, for the gradient.  16-bit
// gradients take the hardware's 2^x as it is: with the roundings of its exponent, up to 125,
// it is within 2 in 10^5, where half of a step of theirs is 5 in 10^4 or more.
template <class T>
__device__ __forceinline__ float softmax_of(float z, float m, float rtau, float ls) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(__builtin_fmaf(z - m, rtau * LOG2E, -(ls * LOG2E)));
  return exp_wide(__builtin_fmaf(z - m, rtau, -ls));
}

// The teacher's candidates of a row in LDS: ids (-1: does not count), probabilities,
// log p, the logits at the ids, and a hash table that finds ids named twice.
struct Candidates {
  int32_t *ids;
  float *p, *logp, *z;
  int32_t *keys;
  uint32_t k, hash;
  bool some, again;  // of the first wave: there is an entry; an id comes twice
};
static uint32_t candidate_slots(uint32_t k) {
  uint32_t h = 64;
  while (h < 2 * k) h *= 2;
  return h;
}
static size_t candidate_bytes(uint32_t k) { return (size_t)k * 16 + (size_t)candidate_slots(k) * 4; }

// By the first wave alone: its LDS accesses are in order.
template <class T>
__device__ __forceinline__ void teacher_part(const DistillArgs &a, uint64_t row, const T *z, Candidates &c) {
  const uint32_t l = here(threadIdx.x);
  const int32_t *id_row = a.ids + (int64_t)row * a.ids_stride;
  const float *t_row = a.teacher + (int64_t)row * a.teacher_stride;
  for (uint32_t i = l; i < c.hash; i += 64u) c.keys[i] = -1;
  float tm = -INFINITY;
  for (uint32_t i = l; i < c.k; i += 64u) {
    int32_t id = id_row[i];
    float t = t_row[i] / a.tau;
    if ((uint32_t)id >= a.q) {
      id = -1;
      t = -INFINITY;
    }
    c.ids[i] = id;
    c.logp[i] = t;
    c.z[i] = id >= 0 ? (float)z[id] : 0.0f;
    tm = fmaxf(tm, t);
  }
  tm = wave_max(tm);
  if (!(tm > -INFINITY)) tm = 0.0f;
  float ts = 0.0f;
  bool again = false;
  for (uint32_t i = l; i < c.k; i += 64u) {
    const float e = expf(c.logp[i] - tm);
    c.p[i] = e;
    ts += e;
    const int32_t id = c.ids[i];
    if (id >= 0) {
      uint32_t h = hash_at((uint32_t)id, c.hash);
      for (;;) {  // (at most half of the slots are ever taken)
        const int32_t old = atomicCAS(&c.keys[h], -1, id);
        again = again || old == id;
        if (old == -1 || old == id) break;
        h = (h + 1u) & (c.hash - 1u);
      }
    }
  }
  ts = wave_sum(ts);
  const float lts = logf(ts), rts = 1.0f / ts;
  for (uint32_t i = l; i < c.k; i += 64u) {
    c.logp[i] = (c.logp[i] - tm) - lts;
    c.p[i] *= rts;
  }
  c.some = !(ts == 0.0f);
  c.again = __any(again);
}

// By the first wave: the loss, from the row's maximum (a logit) and log sum.
__device__ __forceinline__ void teacher_loss(const DistillArgs &a, uint64_t row, const Candidates &c, float m,
                                             float ls, float rtau) {
  float l = 0.0f;
  for (uint32_t i = here(threadIdx.x); i < c.k; i += 64u) {
    const float p = c.p[i];
    if (c.ids[i] >= 0 && p != 0.0f) l += p * (c.logp[i] - ((c.z[i] - m) * rtau - ls));
  }
  l = wave_sum(l);
  if (threadIdx.x == 0) a.loss[row] = c.some ? a.tau * a.tau * l : 0.0f;
}

// The candidates that count as (id, place), sorted, where their hash table was; behind them
// ones.  By the whole workgroup, a bitonic network.
__device__ __forceinline__ uint64_t *sort_candidates(const Candidates &c) {
  static_assert(DISTILL_MAX_K <= 4096, "12 bits for the place");
  uint64_t *s = reinterpret_cast<uint64_t *>(c.keys);
  const uint32_t n = c.hash / 2, tid = here(threadIdx.x);  // a power of two, k or more
  for (uint32_t i = tid; i < n; i += blockDim.x) {
    const int32_t id = i < c.k ? c.ids[i] : -1;
    s[i] = id >= 0 ? (uint64_t)id << 12 | i : ~0ull;
  }
  for (uint32_t size = 2; size <= n; size *= 2)
    for (uint32_t step = size / 2; step > 0; step /= 2) {
      __syncthreads();
      for (uint32_t i = tid; i < n / 2; i += blockDim.x) {
        const uint32_t lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const uint64_t x = s[lo], y = s[hi];
        if ((x > y) == !(lo & size)) {
          s[lo] = y;
          s[hi] = x;
        }
      }
    }
  __syncthreads();
  return s;
}

// The gradient at the candidates' places from s0 to s1 - 1, by the whole workgroup: an id that comes
// more than once has the sum of its probabilities, in the order of the list.  Such lists
// are sorted first: 32 rows of 20000 categories with one repeat in 1024 candidates take
// 50 us (without 31), where a search of the list for each entry took 317; with one in 64
// 15, and 19.
template <class T>
__device__ __forceinline__ void candidate_grads(const Candidates &c, bool again, uint32_t s0, uint32_t s1, T *g, float f,
                                                float m, float ls, float rtau) {
  const uint64_t *s = nullptr;
  if (again) s = sort_candidates(c);
  for (uint32_t e = here(threadIdx.x); e < c.k; e += blockDim.x) {
    const uint32_t i = again ? (uint32_t)s[e] & 4095u : e;
    const int32_t id = again ? (int32_t)(s[e] >> 12) : c.ids[e];  // (ones: -1)
    if (id < 0 || (uint32_t)id - s0 >= s1 - s0) continue;
    float p = 0.0f;
    if (again) {
      if (e > 0 && (int32_t)(s[e - 1] >> 12) == id) continue;
      for (uint32_t j = e; j < c.k && (int32_t)(s[j] >> 12) == id; ++j) p += c.p[(uint32_t)s[j] & 4095u];
    } else {
      p = c.p[e];
    }
    g[id] = (T)(f * (softmax_of<T>(c.z[i], m, rtau, ls) - p));
  }
}

// Maximum and sum of exponentials of z rtau, of lanes and waves.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum max_sum_merge(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * __builtin_amdgcn_exp2f((a.m - m) * c) + b.s * __builtin_amdgcn_exp2f((b.m - m) * c)};
}
template <int BLOCK>
__device__ __forceinline__ MaxSum max_sum_block(MaxSum v, float c, MaxSum *buf) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) v = max_sum_merge(v, {__shfl_xor(v.m, k), __shfl_xor(v.s, k)}, c);
  if ((threadIdx.x & 63u) == 0) buf[threadIdx.x / 64u] = v;
  __syncthreads();
  v = buf[0];
#pragma unroll
  for (int w = 1; w < BLOCK / 64; ++w) v = max_sum_merge(v, buf[w], c);
  return v;
}

// A lane's maximum and sum over the logits from d0 to end - 1.
template <class T, int BLOCK>
__device__ __forceinline__ MaxSum lane_max_sum(const T *z, uint32_t d0, uint32_t end, uint32_t tid, float l2) {
  MaxSum t{-__FLT_MAX__, 0.0f};
  for (uint32_t d = d0 + tid * 8u; d < end; d += BLOCK * 8u) {
    Raw8<T> r;
    load_place(z, d, end, r, LOWEST<T>);
    float x[8], m = t.m, s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = value(r, j);
#pragma unroll
    for (int j = 0; j < 8; j += 2) m = max3(m, x[j], x[j + 1]);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += __builtin_amdgcn_exp2f((x[j] - m) * l2);
    t.s = t.s * __builtin_amdgcn_exp2f((t.m - m) * l2) + s;
    t.m = m;
  }
  return t;
}

// Eight places of the gradient but for p; n: how many of them there are.
template <class T>
__device__ __forceinline__ void write_grad(T *o, uint32_t n, const Raw8<T> &v, bool some, float f, float m, float ls,
                                           float rtau) {
  float x[8];
  if (some) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = f * softmax_of<T>(value(v, j), m, rtau, ls);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.0f;
  }
  store8(o, n, x);
}

__device__ __forceinline__ Candidates candidates_in(uint32_t *lds, uint32_t k, uint32_t hash) {
  Candidates c;
  c.ids = reinterpret_cast<int32_t *>(lds);
  c.p = reinterpret_cast<float *>(lds) + k;
  c.logp = c.p + k;
  c.z = c.logp + k;
  c.keys = reinterpret_cast<int32_t *>(c.z + k);
  c.k = k;
  c.hash = hash;
  return c;
}

// GROUPS > 0: the row, of 8 to BLOCK * 8 GROUPS logits, stays in registers; 0: it is
// read twice.  In registers a place behind the last eight logits stands for those eight:
// the maximum does not mind, the sum leaves out what another lane has, and the gradient
// there is written twice with the same bits.  With all loads under way at once 1021 rows of
// 50001 f16 take 46 us and 200 of 20000 bf16 15; loads that wait for one another: 50, 19.
template <class T, int BLOCK, int GROUPS>
__global__ __launch_bounds__(BLOCK, GROUPS ? 4 : 1) void distill_kernel(DistillArgs a, uint32_t hash) {
  extern __shared__ __align__(16) uint32_t lds[];
  __shared__ MaxSum buf[BLOCK / 64];
  __shared__ uint32_t flags;  // 1: there is an entry, 2: an id comes twice
  Candidates c = candidates_in(lds, a.k, hash);
  const float rtau = 1.0f / a.tau, l2 = rtau * LOG2E;
  constexpr int G = GROUPS ? GROUPS : 1;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const uint32_t tid = here(threadIdx.x);
    const T *z = reinterpret_cast<const T *>(a.z) + (int64_t)row * a.z_stride;
    Raw8<T> r[G];
    if constexpr (GROUPS > 0) {
#pragma unroll
      for (int g = 0; g < G; ++g)
        if ((uint32_t)g * BLOCK * 8u < a.q) load8(z + min(((uint32_t)g * BLOCK + tid) * 8u, a.q - 8u), r[g]);
    }
    if (tid < 64u) {
      teacher_part(a, row, z, c);
      if (tid == 0) flags = (c.some ? 1u : 0u) | (c.again ? 2u : 0u);
    }
    MaxSum t{-__FLT_MAX__, 0.0f};
    if constexpr (GROUPS > 0) {
#pragma unroll
      for (int g = 0; g < G; ++g)
        if ((uint32_t)g * BLOCK * 8u < a.q) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) t.m = max3(t.m, value(r[g], j), value(r[g], j + 1));
          hide(r[g]);
        }
      loads_done();
#pragma unroll
      for (int g = 0; g < G; ++g)
        if ((uint32_t)g * BLOCK * 8u < a.q) {
          float s = 0.0f;
          if ((uint32_t)(g + 1) * BLOCK * 8u <= a.q) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s += __builtin_amdgcn_exp2f((value(r[g], j) - t.m) * l2);
          } else {
            const uint32_t d = ((uint32_t)g * BLOCK + tid) * 8u, before = d - min(d, a.q - 8u);
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
              const float e = __builtin_amdgcn_exp2f((value(r[g], j) - t.m) * l2);
              s += j >= before ? e : 0.0f;
            }
          }
          t.s += s;
          hide(r[g]);
        }
    } else {
      t = lane_max_sum<T, BLOCK>(z, 0, a.q, tid, l2);
    }
    t = max_sum_block<BLOCK>(t, l2, buf);
    const float ls = logf(t.s);
    if (tid < 64u) teacher_loss(a, row, c, t.m, ls, rtau);
    if (a.weight) {
      const uint32_t fl = flags;
      const bool some = fl & 1u;
      const float f = a.tau * a.weight[row];
      T *o = reinterpret_cast<T *>(a.grad) + (int64_t)row * a.grad_stride;
      if constexpr (GROUPS > 0) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t d = ((uint32_t)g * BLOCK + tid) * 8u;
          if (d < a.q) write_grad(o + min(d, a.q - 8u), 8, r[g], some, f, t.m, ls, rtau);
        }
      } else {
        for (uint32_t d = tid * 8u; d < a.q; d += BLOCK * 8u) {
          load_place(z, d, a.q, r[0]);
          write_grad(o + d, a.q - d, r[0], some, f, t.m, ls, rtau);
        }
      }
      __syncthreads();
      if (some) candidate_grads(c, fl & 2u, 0, a.q, o, f, t.m, ls, rtau);
    }
    __syncthreads();
  }
}

// Few long rows: a row's segments in workgroups of their own, first their maxima and
// sums, then, from all of a row's, their part of the gradient (and, in the first one,
// the loss).
constexpr int DS_BLOCK = 512;

template <class T>
__global__ __launch_bounds__(DS_BLOCK) void distill_sum_kernel(DistillArgs a, uint32_t seg, uint32_t n_seg,
                                                               MaxSum *__restrict__ parts) {
  __shared__ MaxSum buf[DS_BLOCK / 64];
  const uint32_t row = blockIdx.x / n_seg, s0 = blockIdx.x % n_seg * seg;
  const float l2 = (1.0f / a.tau) * LOG2E;
  const T *z = reinterpret_cast<const T *>(a.z) + (int64_t)row * a.z_stride;
  MaxSum t = lane_max_sum<T, DS_BLOCK>(z, s0, min(s0 + seg, a.q), threadIdx.x, l2);
  t = max_sum_block<DS_BLOCK>(t, l2, buf);
  if (threadIdx.x == 0) parts[blockIdx.x] = t;
}

template <class T>
__global__ __launch_bounds__(DS_BLOCK) void distill_segment_kernel(DistillArgs a, uint32_t hash, uint32_t seg,
                                                                   uint32_t n_seg, const MaxSum *__restrict__ parts) {
  extern __shared__ __align__(16) uint32_t lds[];
  __shared__ uint32_t flags;
  Candidates c = candidates_in(lds, a.k, hash);
  const uint32_t row = blockIdx.x / n_seg, s0 = blockIdx.x % n_seg * seg, s1 = min(s0 + seg, a.q), tid = threadIdx.x;
  const float rtau = 1.0f / a.tau, l2 = rtau * LOG2E;
  const T *z = reinterpret_cast<const T *>(a.z) + (int64_t)row * a.z_stride;
  if (tid < 64u) {
    teacher_part(a, row, z, c);
    if (tid == 0) flags = (c.some ? 1u : 0u) | (c.again ? 2u : 0u);
  }
  // every wave joins the row's parts in the same order
  MaxSum t{-__FLT_MAX__, 0.0f};
  for (uint32_t i = tid & 63u; i < n_seg; i += 64u) t = max_sum_merge(t, parts[row * n_seg + i], l2);
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) t = max_sum_merge(t, {__shfl_xor(t.m, k), __shfl_xor(t.s, k)}, l2);
  const float ls = logf(t.s);
  if (tid < 64u && s0 == 0) teacher_loss(a, row, c, t.m, ls, rtau);
  __syncthreads();
  const bool some = flags & 1u;
  const float f = a.tau * a.weight[row];
  T *o = reinterpret_cast<T *>(a.grad) + (int64_t)row * a.grad_stride;
  for (uint32_t d = s0 + tid * 8u; d < s1; d += DS_BLOCK * 8u) {
    Raw8<T> r;
    load_place(z, d, s1, r);
    write_grad(o + d, s1 - d, r, some, f, t.m, ls, rtau);
  }
  __syncthreads();
  if (some) candidate_grads(c, flags & 2u, s0, s1, o, f, t.m, ls, rtau);
}

// Segments of a row where they pay: 0 for a workgroup per row.  One and two launches (us):
//   16 x 65536 bf16 (128 KB a row) 12.5 / 15.4    32 rows: 16.7 / 15.8    64: 17.5 / 15.8
//    8 x 131072 bf16 (256 KB)      18.9 / 15.6    32 rows: 19.9 / 15.5    64: 21.3 / 18.2
//    8 x 131072 f32 (512 KB)       24.2 / 15.8    32 rows: 25.7 / 15.1    64: 34.0 / 20.6
static uint32_t distill_segments(const thrml_ctx *ctx, int dtype, uint64_t rows, uint32_t q) {
  const uint64_t bytes = (uint64_t)q * (dtype == THRML_DTYPE_F32 ? 4 : 2);
  if (rows * 4 > (uint64_t)ctx->cu_count || bytes < (rows < 32 ? 256u << 10 : 128u << 10)) return 0;
  return std::min<uint32_t>(64, std::min<uint32_t>(cdiv(q, 2 * DS_BLOCK * 8), 2 * ctx->cu_count / (uint32_t)rows));
}
uint64_t distill_work(thrml_ctx *ctx, int dtype, uint64_t rows, uint32_t q) {
  return rows * distill_segments(ctx, dtype, rows, q) * sizeof(MaxSum);
}

int launch_distill(thrml_ctx *ctx, const DistillArgs &a, int dtype, void *work) {
  if (a.rows == 0) return THRML_OK;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(a.rows, 1u << 20);
  if (const uint32_t n = a.weight ? distill_segments(ctx, dtype, a.rows, a.q) : 0) {
    const uint32_t seg = cdiv(cdiv(a.q, n), 8) * 8, n_seg = cdiv(a.q, seg);
    MaxSum *parts = reinterpret_cast<MaxSum *>(work);
    return with_type(dtype, [&](auto t) -> int {
      typedef decltype(t) T;
      hipLaunchKernelGGL((distill_sum_kernel<T>), dim3((uint32_t)a.rows * n_seg), dim3(DS_BLOCK), 0, ctx->stream, a, seg,
                         n_seg, parts);
      THRML_HIP(hipGetLastError());
      auto *f = &distill_segment_kernel<T>;
      const size_t lds = candidate_bytes(a.k);
      if (int rc = lds_limit(reinterpret_cast<const void *>(f), lds)) return rc;
      hipLaunchKernelGGL(f, dim3((uint32_t)a.rows * n_seg), dim3(DS_BLOCK), lds, ctx->stream, a, candidate_slots(a.k), seg,
                         n_seg, parts);
      THRML_HIP(hipGetLastError());
      return THRML_OK;
    });
  }
  return with_type(dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    // 64 registers of logits a lane
    constexpr int G = sizeof(T) == 2 ? 16 : 8;
    // rows that have a compute unit each: 16 waves for one (256 losses over 131072
    // categories in bf16 14.8 us, with 8 waves 19.2); more rows: several workgroups in a
    // compute unit
    uint32_t block = a.rows <= (uint64_t)ctx->cu_count && a.q > 8192 ? 1024 : 512;
    auto *f = block == 1024 ? &distill_kernel<T, 1024, 0> : &distill_kernel<T, 512, 0>;
    if (a.weight && a.q >= 8 && a.q <= 1024 * 8 * G) {
      block = a.q <= 256 * 8 * G ? 256 : a.q <= 512 * 8 * G ? 512 : 1024;
      f = block == 256 ? &distill_kernel<T, 256, G> : block == 512 ? &distill_kernel<T, 512, G> : &distill_kernel<T, 1024, G>;
    }
    const size_t lds = candidate_bytes(a.k);
    if (int rc = lds_limit(reinterpret_cast<const void *>(f), lds)) return rc;
    hipLaunchKernelGGL(f, dim3(grid), dim3(block), lds, ctx->stream, a, candidate_slots(a.k));
    THRML_HIP(hipGetLastError());
    return THRML_OK;
  });
}

}  // namespace thrml
