// Log probability of a given token, entropy and the most likely alternatives
// of each row of logits, in one pass over the logits; and the gradient of the
// first two, in one more.
//
// With m the running maximum of what a thread has read, it keeps
//   s = sum e^(x - m),   a = sum e^(x - m) (x - m)
// and moves both to a new maximum m' = m + t:  a' = e^-t (a - t s),
// s' = e^-t s.  Joined over the row:
//   log p = (x - m) - log s,  entropy = log s - a / s,
// where m and log s stay apart: next to a large m (a row of the type's lowest
// values) their sum would lose log s.
// Gradient, with p = e^(log p), g and h the gradients of the two results:
//   dx_j = g (1[j = token] - p_j) - h p_j (log p_j + entropy)
//
// What bounds it is reading the logits.  A row goes to one workgroup, or, when
// there are few rows, to several that take a share of the vocabulary each and
// whose results a second kernel joins.

#include "model_ops.h"

namespace sofa_model {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

__device__ __forceinline__ int64_t place(int64_t row, int64_t inner,
                                         int64_t outer_stride,
                                         int64_t inner_stride) {
  return row / inner * outer_stride + row % inner * inner_stride;
}

// A launch has less than 2^32 threads in a dimension, so rows go on in the next.
constexpr int64_t kRowsInX = 1 << 22;

__device__ __forceinline__ int64_t row_of(const LogprobArgs& a) {
  return blockIdx.y * kRowsInX + blockIdx.x / a.parts;
}

inline dim3 grid_of(const LogprobArgs& a) {
  return dim3((unsigned) (a.rows < kRowsInX ? a.rows : kRowsInX) * a.parts,
              (unsigned) ((a.rows + kRowsInX - 1) / kRowsInX));
}

struct Sums {
  float m, s, a;
};

// A part that holds nothing but -inf has m = -inf and s = a = 0.
__device__ __forceinline__ Sums join(Sums x, Sums y) {
  Sums r;
  r.m = fmaxf(x.m, y.m);
  const float base = r.m == -INFINITY ? 0.f : r.m;
  // max() keeps a part of -inf, or of the type's lowest value, from 0 * -inf
  // (or an overflow); e^-1e4 is 0 already
  const float tx = fmaxf(x.m - base, -1e4f), ty = fmaxf(y.m - base, -1e4f);
  const float ex = exp2_fast(tx * kLog2e), ey = exp2_fast(ty * kLog2e);
  r.s = x.s * ex + y.s * ey;
  r.a = ex * (x.a + tx * x.s) + ey * (y.a + ty * y.s);
  return r;
}

__device__ __forceinline__ Sums wave_join(Sums x) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) {
    Sums y{__shfl_xor(x.m, o), __shfl_xor(x.s, o), __shfl_xor(x.a, o)};
    x = join(x, y);
  }
  return x;
}

// Takes 8 more logits and returns the largest; absent ones are -inf.  A NaN or
// +inf makes s NaN, and with it every result of the row, as the definition has
// it.
__device__ __forceinline__ float take(Sums& t, const float (&x)[8]) {
  float most = x[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) most = fmaxf(most, x[j]);
  if (most > t.m) {
    const float step = fmaxf(t.m - most, -1e4f);
    const float e = exp2_fast(step * kLog2e);
    t.a = e * (t.a + step * t.s);
    t.s *= e;
    t.m = most;
  }
  const float base = t.m == -INFINITY ? 0.f : t.m;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float d = x[j] - base;
    const float e = exp2_fast(d * kLog2e);
    t.s += e;
    t.a += e * fmaxf(d, -1e4f);
  }
  return most;
}

// ------------------------------------------------------------ alternatives
//
// A candidate is one 64-bit number: the logit in an order-keeping integer form
// above, the inverted token below, so that the largest numbers are the largest
// logits and among equals the lowest tokens.  NaN counts as the largest, -0 as
// 0.  No candidate is 0.
__device__ __forceinline__ uint32_t ordered(float x) {
  const float z = x + 0.f;  // -0 becomes 0
  uint32_t u = __float_as_uint(z);
  if (z != z) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float unordered(uint32_t u) {
  return u == 0xffffffffu ? __uint_as_float(0x7fc00000u)
         : u & 0x80000000u ? __uint_as_float(u & 0x7fffffffu)
                           : __uint_as_float(~u);
}

__device__ __forceinline__ uint64_t candidate(float x, int token) {
  return (uint64_t) ordered(x) << 32 | (uint32_t) ~token;
}

// Orders this wave's accesses to LDS between its lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Each wave collects the candidates that reach a threshold: at first the
// `top`-th best of what its lanes have each seen best in their first loads,
// which at least `top` logits reach and, in random order, about one in a
// hundred.  A list of more than 2 top + 16 is cut to its best `top`, and the last
// of those is the threshold from then on: a row of 128256 takes a few such
// cuts.  In the worst (rising) order every step fills the list, which costs
// time but no result.
constexpr int kListSize = 640;  // 2 top + 16, and what 8 logits a lane may add
constexpr int kPerLane = kListSize / kWave;

struct Best {
  uint64_t* list;  // kListSize in LDS, this wave's
  int count;       // the same in every lane
  uint64_t least;  // the threshold
  float floor;     // and its logit, below which nothing has to be looked at
  int top;

  __device__ __forceinline__ void raise(uint64_t to) {
    if (to <= least) return;
    least = to;
    floor = unordered((uint32_t) (to >> 32));
  }
};

__device__ __forceinline__ uint64_t read_lane(uint64_t x, int lane) {
  return (uint64_t) __builtin_amdgcn_readlane((uint32_t) (x >> 32), lane) << 32 |
         (uint32_t) __builtin_amdgcn_readlane((uint32_t) x, lane);
}

// Raises the threshold to the `top`-th best of the lanes' best, 0 where a lane
// has none: as many candidates reach that.  All differ, so their ranks do.
__device__ __forceinline__ void raise_by_lanes(Best& b, uint64_t most) {
  int rank = 0;
#pragma unroll
  for (int i = 0; i < kWave; ++i) rank += read_lane(most, i) > most;
  const uint64_t who = __ballot(rank == b.top - 1 && most);
  if (who) b.raise(read_lane(most, __ffsll((unsigned long long) who) - 1));
}

// Appends the lanes' candidates that pass.
__device__ __forceinline__ void append(Best& b, uint64_t c, bool passes) {
  const uint64_t below = (1ull << threadIdx.x % kWave) - 1;
  const uint64_t who = __ballot(passes);
  if (passes) b.list[b.count + __popcll(who & below)] = c;
  b.count += __popcll(who);
}

// Cuts a list to its best `top`, in falling order, with zeros where there are
// fewer.
__device__ __forceinline__ void keep_best(Best& b) {
  const int lane = threadIdx.x % kWave;
  wave_sync();
  // A long one first loses what is below the `top`-th best of 64 parts of it:
  // with `top` at most 32 of 64 parts, at least half.
  while (b.count > 2 * kWave) {
    uint64_t mine[kPerLane], most = 0;
#pragma unroll
    for (int k = 0; k < kPerLane; ++k) {
      const int at = k * kWave + lane;
      mine[k] = at < b.count ? b.list[at] : 0;
      most = mine[k] > most ? mine[k] : most;
    }
    raise_by_lanes(b, most);
    wave_sync();
    b.count = 0;
#pragma unroll
    for (int k = 0; k < kPerLane; ++k)
      append(b, mine[k], mine[k] && mine[k] >= b.least);
    wave_sync();
  }
  // the place of a candidate is the number of those above it
  if (b.count <= kWave) {
    const uint64_t mine = lane < b.count ? b.list[lane] : 0;
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < b.count; ++i) rank += b.list[i] > mine;
    wave_sync();
    if (lane < b.count ? rank < b.top : lane < b.top)
      b.list[lane < b.count ? rank : lane] = mine;
  } else {
    uint64_t mine[2];
    int rank[2] = {};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int at = k * kWave + lane;
      mine[k] = at < b.count ? b.list[at] : 0;
    }
#pragma unroll 8
    for (int i = 0; i < b.count; ++i) {
      const uint64_t other = b.list[i];
#pragma unroll
      for (int k = 0; k < 2; ++k) rank[k] += other > mine[k];
    }
    wave_sync();
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (k * kWave + lane < b.count && rank[k] < b.top)
        b.list[rank[k]] = mine[k];
  }
  wave_sync();
  if (b.count > b.top) b.count = b.top;
  if (b.count == b.top) b.raise(b.list[b.top - 1]);
}

// `most`: the largest of them; `all`: one of the row may be NaN, which is above
// every threshold but not found by comparing
__device__ __forceinline__ void offer(Best& b, const float (&x)[8], float most,
                                      bool all, int first, int n) {
  if (!__ballot(n > 0 && (most >= b.floor || all))) return;
  uint32_t may = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    may |= (j < n && (x[j] >= b.floor || all) ? 1u : 0u) << j;
  // one of each lane's at a time: rarely more than twice in a row
  while (__ballot(may != 0)) {
    const int pick = __ffs(may) - 1;
    float value = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) value = pick == j ? x[j] : value;
    const uint64_t c = candidate(value, first + pick);
    append(b, c, may && c >= b.least);
    may &= may - 1;
  }
  if (b.count > 2 * b.top + 16) keep_best(b);
}

// The best candidate of 8 logits of which n are there, or `most`
__device__ __forceinline__ uint64_t better(uint64_t most, const float (&x)[8],
                                           int first, int n) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint64_t c = j < n ? candidate(x[j], first + j) : 0;
    most = c > most ? c : most;
  }
  return most;
}

template <typename T>
__device__ __forceinline__ void finish(const LogprobArgs& a, int64_t row,
                                       Sums t) {
  const float log_s = log2_fast(t.s) * kLn2;
  // a row without one allowed token: no distribution, and no NaN either
  const bool empty = t.s == 0.f;
  const int64_t token =
      a.tokens[place(row, a.inner, a.token_outer_stride, a.token_inner_stride)];
  float logprob = 0.f;
  if (token != a.ignore_index) {
    if (token < 0 || token >= a.vocab) {
      logprob = __uint_as_float(0x7fc00000u);  // not a token
    } else if (empty) {
      logprob = -INFINITY;
    } else {
      const T* x = static_cast<const T*>(a.logits) +
                   place(row, a.inner, a.outer_stride, a.inner_stride);
      logprob = ((float) x[token] - t.m) - log_s;
    }
  }
  a.logprob[row] = logprob;
  a.entropy[row] = empty ? 0.f : log_s - t.a / t.s;
  a.norm[row * 2] = empty ? -INFINITY : t.m;
  a.norm[row * 2 + 1] = log_s;
}

__device__ __forceinline__ void put_top(const LogprobArgs& a, int64_t row,
                                        int i, uint64_t c, Sums t) {
  const float x = unordered((uint32_t) (c >> 32));
  const float log_s = log2_fast(t.s) * kLn2;
  a.top_ids[row * a.top + i] = (int64_t) (int32_t) ~(uint32_t) c;
  a.top_logprobs[row * a.top + i] =
      t.s == 0.f ? -INFINITY : (x - t.m) - log_s;
}

// `part` of `parts` of a row.  TOP: with alternatives; looking for those leaves
// memory idle unless the next loads are on their way and there are four workgroups
// on a compute unit (8192 x 128256 bf16, 5 alternatives: 403 us, without 365; one
// load after the other 502).
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads, 4) void logprob_kernel(LogprobArgs a) {
  __shared__ float sums[kWaves][3];
  __shared__ uint64_t lists[TOP ? kWaves * kListSize : 1];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t row = row_of(a);
  if (row >= a.rows) return;
  const int part = blockIdx.x % a.parts;
  const T* x = static_cast<const T*>(a.logits) +
               place(row, a.inner, a.outer_stride, a.inner_stride);
  const int begin = part * a.part_size;
  const int end = min(a.vocab, begin + a.part_size);

  Sums t{-INFINITY, 0.f, 0.f};
  Best best{lists + (TOP ? wave * kListSize : 0), 0, 0, -INFINITY, a.top};
  constexpr int kLoads = TOP ? 2 : 4;  // vectors a thread loads at a time
  constexpr int kStep = kThreads * 8;
  constexpr int kStride = kLoads * kStep;
  int at = begin;
  auto fetch = [&](float (&v)[kLoads][8], int at) {
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      load8(x + at + k * kStep + threadIdx.x * 8, v[k]);
  };
  auto process = [&](const float (&v)[kLoads][8], int at) {
    if constexpr (TOP) {
      if (at == begin) {
        uint64_t most = 0;
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
          most = better(most, v[k], at + k * kStep + threadIdx.x * 8, 8);
        raise_by_lanes(best, most);
      }
    }
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const float most = take(t, v[k]);
      if constexpr (TOP)
        offer(best, v[k], most, t.s != t.s, at + k * kStep + threadIdx.x * 8, 8);
    }
  };
  if constexpr (TOP) {
    // the next loads are on their way while candidates are looked at
    if (at + kStride <= end) {
      float v[kLoads][8], next[kLoads][8];
      fetch(v, at);
      for (; at + 2 * kStride <= end; at += kStride) {
        fetch(next, at + kStride);
        process(v, at);
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] = next[k][j];
      }
      process(v, at);
      at += kStride;
    }
  } else {
    for (; at + kStride <= end; at += kStride) {
      float v[kLoads][8];
      fetch(v, at);
      process(v, at);
    }
  }
  for (; at < end; at += kStep) {
    const int first = at + threadIdx.x * 8;
    float v[8];
    load8(x + first, v, end - first, -INFINITY);
    const float most = take(t, v);
    if constexpr (TOP) {
      if (at == begin) raise_by_lanes(best, better(0, v, first, end - first));
      offer(best, v, most, t.s != t.s, first, end - first);
    }
  }

  t = wave_join(t);
  if (lane == 0) {
    sums[wave][0] = t.m;
    sums[wave][1] = t.s;
    sums[wave][2] = t.a;
  }
  if constexpr (TOP) keep_best(best);
  __syncthreads();
  if (wave) return;
  t = Sums{sums[0][0], sums[0][1], sums[0][2]};
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
    t = join(t, Sums{sums[w][0], sums[w][1], sums[w][2]});
  if (lane == 0) {
    if (a.parts == 1) {
      finish<T>(a, row, t);
    } else {
      float* out = a.part_sums + (row * a.parts + part) * 3;
      out[0] = t.m;
      out[1] = t.s;
      out[2] = t.a;
    }
  }
  if constexpr (TOP) {
    // the waves' lists follow each other at kListSize; gather them at the front
    const int all = kWaves * a.top;
    uint64_t mine[kWaves * kMaxTop / kWave];
#pragma unroll
    for (int k = 0; k < kWaves * kMaxTop / kWave; ++k) {
      const int i = k * kWave + lane;
      mine[k] = i < all ? lists[i / a.top * kListSize + i % a.top] : 0;
    }
    wave_sync();
    Best joined{lists, 0, 0, -INFINITY, a.top};
    raise_by_lanes(joined, mine[0] > mine[1] ? mine[0] : mine[1]);
#pragma unroll
    for (int k = 0; k < kWaves * kMaxTop / kWave; ++k)
      append(joined, mine[k], mine[k] && mine[k] >= joined.least);
    keep_best(joined);
    if (lane < a.top) {
      if (a.parts == 1)
        put_top(a, row, lane, lists[lane], t);
      else
        a.part_top[(row * a.parts + part) * a.top + lane] = lists[lane];
    }
  }
}

// Joins the parts of a row; one wave a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(kWave) void logprob_join_kernel(LogprobArgs a) {
  __shared__ uint64_t list[TOP ? kListSize : 1];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  Sums t{-INFINITY, 0.f, 0.f};
  if (lane < a.parts) {
    const float* in = a.part_sums + (row * a.parts + lane) * 3;
    t = Sums{in[0], in[1], in[2]};
  }
  t = wave_join(t);
  if (lane == 0) finish<T>(a, row, t);
  if constexpr (TOP) {
    Best best{list, 0, 0, -INFINITY, a.top};
    const uint64_t* in = a.part_top + row * a.parts * a.top;
    const int all = a.parts * a.top;
    // each part's best come first
    raise_by_lanes(best, lane < a.parts ? in[lane * a.top] : 0);
    for (int at = 0; at < all; at += kWave) {
      const int i = at + lane;
      const uint64_t c = i < all ? in[i] : 0;
      append(best, c, c && c >= best.least);
      if (best.count > kListSize - kWave) keep_best(best);
    }
    keep_best(best);
    if (lane < a.top) put_top(a, row, lane, list[lane], t);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logprob_backward_kernel(
    LogprobArgs a) {
  const int64_t row = row_of(a);
  if (row >= a.rows) return;
  const int part = blockIdx.x % a.parts;
  const T* x = static_cast<const T*>(a.logits) +
               place(row, a.inner, a.outer_stride, a.inner_stride);
  T* dx = static_cast<T*>(a.dlogits) + row * a.vocab;
  const int begin = part * a.part_size;
  const int end = min(a.vocab, begin + a.part_size);
  const float m = a.norm[row * 2], log_s = a.norm[row * 2 + 1];
  const float entropy = a.entropy[row];
  int64_t token =
      a.tokens[place(row, a.inner, a.token_outer_stride, a.token_inner_stride)];
  float g = 0.f, h = 0.f;
  if (a.dlogprob && token != a.ignore_index)
    g = a.dlogprob[place(row, a.inner, a.grad_outer_stride,
                         a.grad_inner_stride)];
  // a log probability of what is no token is NaN, and so is the gradient through it
  const bool wrong = g != 0.f && (token < 0 || token >= a.vocab);
  if (wrong) g = __uint_as_float(0x7fc00000u);
  if (a.dentropy)
    h = a.dentropy[place(row, a.inner, a.grad2_outer_stride,
                         a.grad2_inner_stride)];
  // nothing to pass on, or an empty row (no sum, while m is -inf in a row of NaN
  // and -inf too): zeros, and nothing is read
  const bool zero = (g == 0.f && h == 0.f) || (log_s == -INFINITY && !wrong);
  // dx = g 1[token] - p (g + h entropy + h log p)
  const float base = g + h * entropy;

  constexpr int kLoads = 4;
  constexpr int kStep = kThreads * 8;
  auto gradient = [&](float (&v)[8], int first) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float logp = (v[j] - m) - log_s;
      const float p = exp2_fast(logp * kLog2e);
      // a masked logit has p = 0 and log p = -inf
      float d = -p * (base + h * fmaxf(logp, -1e4f));
      if (first + j == token) d += g;
      v[j] = zero ? 0.f : d;
    }
  };
  int at = begin;
  for (; at + kLoads * kStep <= end; at += kLoads * kStep) {
    float v[kLoads][8];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      if (!zero) load8(x + at + k * kStep + threadIdx.x * 8, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int first = at + k * kStep + threadIdx.x * 8;
      gradient(v[k], first);
      store8(dx + first, v[k]);
    }
  }
  for (; at < end; at += kStep) {
    const int first = at + threadIdx.x * 8;
    float v[8];
    load8(x + first, v, zero ? 0 : end - first);
    gradient(v, first);
    store8(dx + first, v, end - first);
  }
}

template <typename T>
int forward(const LogprobArgs& a) {
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  const dim3 grid = grid_of(a);
  if (a.top)
    hipLaunchKernelGGL((logprob_kernel<T, true>), grid, dim3(kThreads), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((logprob_kernel<T, false>), grid, dim3(kThreads), 0,
                       stream, a);
  int status = (int) hipGetLastError();
  if (status || a.parts == 1) return status;
  if (a.top)
    hipLaunchKernelGGL((logprob_join_kernel<T, true>), dim3((unsigned) a.rows),
                       dim3(kWave), 0, stream, a);
  else
    hipLaunchKernelGGL((logprob_join_kernel<T, false>), dim3((unsigned) a.rows),
                       dim3(kWave), 0, stream, a);
  return (int) hipGetLastError();
}

template <typename T>
int backward(const LogprobArgs& a) {
  hipLaunchKernelGGL(logprob_backward_kernel<T>,
                     grid_of(a), dim3(kThreads), 0,
                     static_cast<hipStream_t>(a.stream), a);
  return (int) hipGetLastError();
}

bool sound(const LogprobArgs* a) {
  return a && a->logits && a->tokens && a->logprob && a->entropy && a->norm &&
         a->rows > 0 && a->inner > 0 && a->vocab > 0 && a->vocab <= kMaxVocab &&
         a->parts > 0 &&
         a->parts <= kMaxVocabParts && a->part_size > 0 &&
         (int64_t) a->parts * a->part_size >= a->vocab &&
         (int64_t) (a->parts - 1) * a->part_size < a->vocab &&
         a->rows <= INT32_MAX && (a->parts == 1 || a->rows <= kMaxBlocks / a->parts);
}

}  // namespace
}  // namespace sofa_model

extern "C" {

int sofa_logprob_forward(const sofa_model::LogprobArgs* a) {
  using namespace sofa_model;
  if (!sound(a) || a->top < 0 || a->top > kMaxTop || a->top > a->vocab ||
      (a->top && !(a->top_ids && a->top_logprobs)) ||
      (a->parts > 1 && !(a->part_sums && (a->part_top || !a->top))))
    return kBadArgument;
  DeviceGuard guard(a->device);
  if (guard.status()) return guard.status();
  if (a->type == kFloat32) return forward<float>(*a);
  if (a->type == kBFloat16) return forward<bf16>(*a);
  if (a->type == kFloat16) return forward<fp16>(*a);
  return kBadArgument;
}

int sofa_logprob_backward(const sofa_model::LogprobArgs* a) {
  using namespace sofa_model;
  if (!sound(a) || !a->dlogits) return kBadArgument;
  DeviceGuard guard(a->device);
  if (guard.status()) return guard.status();
  if (a->type == kFloat32) return backward<float>(*a);
  if (a->type == kBFloat16) return backward<bf16>(*a);
  if (a->type == kFloat16) return backward<fp16>(*a);
  return kBadArgument;
}

}  // extern "C"
