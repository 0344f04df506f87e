// Self-attention over grouped heads and its gradients, on the matrix cores.
//
//   S = c Q K^T + mask      P = softmax(S) = e^(S - lse)       O = P V
//   dV = P^T dO             dP = dO V^T       delta = rowsum(dO O)
//   dS = P (dP - delta)     dQ = c dS K       dK = c dS^T Q
//
// The scores are never stored: the forward pass runs over the keys with a
// running maximum and sum (in 32 bits, base 2) and keeps lse; the backward
// pass computes P again from it.  It is two kernels, one that owns rows of
// dQ and one that owns rows of dK and dV (over all heads that share them):
// 7 products in place of 5, but no atomics, so the same bits every time.
//
// Every product is v_mfma_f32_32x32x16_bf16.  For a wave's lane l, h = l / 32:
//   A: row l % 32, k = 8 h + 0..7       B: column l % 32, k = 8 h + 0..7
//   D: column l % 32, value i in row 8 (i / 4) + 4 h + i % 4
// The kernels compute S^T (forward, dQ) or S (dK, dV) such that the lane's
// column is the row it owns: its softmax statistics are one value per lane,
// and 8 consecutive values of D are a B operand of the next product as they
// are, if that product takes its k in the order
//   slot (h, j) -> 4 h + j (j < 4), 8 + 4 h + j - 4 (j >= 4)
// of each 16.  Its A operand is read from LDS with ds_read_b64_tr_b16, which
// gives a lane 4 rows of one column, in that same order.  P and dS are rounded
// to bf16 for it: 2^-8 relative at most, as in the results themselves; sums
// stay in 32 bits.  Only delta, which dP - delta almost cancels in short rows,
// takes more of o than its 8 bits: the forward pass keeps what the rounding
// took off as well (with o's own rounding dQ and dK of 32 tokens were 3.1e-3
// off, 1.9 times what the rounding of the results is).
// delta, though, is a difference that short rows almost cancel: it is taken
// of o in 16 bits, kept as o and what its rounding took off.

#include "model_ops.h"

namespace sofa_model {
namespace {

struct AttentionArgs {
  const bf16 *q, *k, *v;  // [batch][heads][tokens][dim] by strides, dim dense
  bf16* o;
  bf16* o_low;            // what rounding took off o, laid out like it; or null
  float* lse;             // [batch][heads][tokens], base 2; +inf: no keys
  const int* lengths;     // [batch] valid tokens, or null
  const bf16* dout;
  float* delta;           // [batch][heads][tokens]
  bf16 *dq, *dk, *dv;
  void* stream;
  int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3];  // batch, head,
  int64_t dout_stride[3], dq_stride[3], dk_stride[3], dv_stride[3];  // token
  float scale;
  int batch, heads, kv_heads, tokens, dim, causal, device;
};
static_assert(sizeof(AttentionArgs) == 328, "as the caller packs it");

typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kRows = kWaves * 32;  // rows a workgroup owns
constexpr int kTile = 64;           // rows of the other side at a time

// Where the 8 elements `chunk` of `row` of a tile are in LDS.  Rows are 256 or
// 128 bytes, so that the same chunk of all rows falls on the same banks; the
// exclusive or moves pairs of chunks such that 8 rows (a row read) as well as
// 4 rows by 2 chunks (a transposed read) fall on different ones.
template <int DP>
__device__ __forceinline__ int swizzle(int row) {
  return DP == 128 ? (row & 7) << 1 : ((row >> 1) & 3) << 1;
}
template <int DP>
__device__ __forceinline__ int lds_at(int row, int chunk) {
  return row * DP + ((chunk ^ swizzle<DP>(row)) << 3);
}

// One thread's share of a tile of kTile rows on its way to LDS.  Rows behind
// the last valid one repeat it, and chunks behind the last one repeat that:
// what is computed from them is multiplied by zeros or not stored, and has
// only to be finite.
template <int DP>
struct Staged {
  static constexpr int kChunks = DP / 8;
  static constexpr int kPasses = kTile * kChunks / kThreads;
  bf16x8 x[kPasses];

  __device__ __forceinline__ void load(const bf16* base, int64_t stride,
                                       int first, int rows, int dim) {
    const int chunk = min((int) threadIdx.x % kChunks, dim / 8 - 1);
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row =
          first + p * (kThreads / kChunks) + (int) threadIdx.x / kChunks;
      x[p] = *reinterpret_cast<const bf16x8*>(
          base + (int64_t) min(row, rows - 1) * stride + chunk * 8);
    }
  }
  __device__ __forceinline__ void store(bf16* tile) const {
    const int chunk = threadIdx.x % kChunks;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = p * (kThreads / kChunks) + threadIdx.x / kChunks;
      *reinterpret_cast<bf16x8*>(tile + lds_at<DP>(row, chunk)) = x[p];
    }
  }
};

// A operand: rows first..first+31 of a tile, elements 16 s..16 s + 15
template <int DP>
__device__ __forceinline__ bf16x8 row_operand(const bf16* tile, int first,
                                              int s) {
  const int lane = threadIdx.x % kWave;
  return *reinterpret_cast<const bf16x8*>(
      tile + lds_at<DP>(first + lane % 32, s * 2 + lane / 32));
}

// A operand: columns 32 block..32 block + 31 of rows first..first+15 of a tile,
// its k in the order that D gives a B operand
template <int DP>
__device__ __forceinline__ bf16x8 column_operand(const bf16* tile, int first,
                                                 int block) {
  typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
  const int lane = threadIdx.x % kWave;
  const int row = first + lane / 32 * 4 + lane % 16 / 4;
  const int chunk = block * 4 + lane % 32 / 16 * 2 + lane % 4 / 2;
  const int within = lane % 2 * 4;
  const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_shortx4*) (tile + lds_at<DP>(row, chunk) + within));
  const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_shortx4*) (tile + lds_at<DP>(row + 8, chunk) + within));
  union {
    shortx4 half[2];
    bf16x8 whole;
  } u = {{a, b}};
  return u.whole;
}

// B operand out of values 8 part..8 part + 7 of D
__device__ __forceinline__ bf16x8 rounded(const floatx16& d, int part) {
  bf16x8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (bf16) d[part * 8 + j];
  return r;
}

__device__ __forceinline__ floatx16 mfma(bf16x8 a, bf16x8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// A row's elements as B operands, straight from memory; zeros where there are
// none
template <int DP>
__device__ __forceinline__ void load_row(bf16x8 (&x)[DP / 16], const bf16* row,
                                         bool valid, int dim) {
  const int h = threadIdx.x % kWave / 32;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int at = s * 16 + h * 8;
    x[s] = valid && at < dim ? *reinterpret_cast<const bf16x8*>(row + at)
                             : bf16x8{};
  }
}

// The transposed result of a wave: the lane's row, in DP / 32 blocks of D;
// zeros in a row that is not valid, whatever was computed for it.  `low`, if
// there is one, takes what the rounding took off.
template <int DP>
__device__ __forceinline__ void store_row(bf16* row,
                                          const floatx16 (&acc)[DP / 32],
                                          float factor, bool valid, int dim,
                                          bf16* low = nullptr) {
  const int h = threadIdx.x % kWave / 32;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = b * 32 + i * 8 + h * 4;
      bf16x4 x, rest;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = valid ? acc[b][i * 4 + j] * factor : 0.f;
        x[j] = (bf16) y;
        rest[j] = (bf16) (y - (float) x[j]);
      }
      if (at < dim) {
        *reinterpret_cast<bf16x4*>(row + at) = x;
        if (low) *reinterpret_cast<bf16x4*>(low + at) = rest;
      }
    }
}

__device__ __forceinline__ float other_half(float x) {
  return __shfl_xor(x, 32);
}

// Which head and which block of rows a workgroup has.  Workgroups go to the 8
// XCDs in turn; the heads are dealt such that those which share keys stay on
// one XCD and its L2.  With a causal mask the blocks with most work go first.
__device__ __forceinline__ void whose(int heads, int blocks, bool last_first,
                                      int& head, int& block) {
  const int slot = blockIdx.x % heads;
  block = blockIdx.x / heads;
  if (last_first) block = blocks - 1 - block;
  head = heads % 8 == 0 ? slot % 8 * (heads / 8) + slot / 8 : slot;
}

__device__ __forceinline__ int valid_tokens(const AttentionArgs& a, int batch) {
  return a.lengths ? min(max(a.lengths[batch], 0), a.tokens) : a.tokens;
}

template <int DP, bool CAUSAL>
__global__ __launch_bounds__(kThreads, 2) void attention_forward_kernel(
    AttentionArgs a) {
  __shared__ __align__(16) bf16 k_tile[kTile * DP];
  __shared__ __align__(16) bf16 v_tile[kTile * DP];
  const int blocks = (a.tokens + kRows - 1) / kRows;
  int bh, block;
  whose(a.batch * a.heads, blocks, CAUSAL, bh, block);
  const int batch = bh / a.heads, head = bh % a.heads;
  const int kv_head = head / (a.heads / a.kv_heads);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int h = lane / 32;
  const int n = valid_tokens(a, batch);
  const int wave_row = block * kRows + wave * 32;
  const int row = wave_row + lane % 32;

  const bf16* k = a.k + batch * a.k_stride[0] + kv_head * a.k_stride[1];
  const bf16* v = a.v + batch * a.v_stride[0] + kv_head * a.v_stride[1];
  bf16x8 q[DP / 16];
  load_row<DP>(q,
               a.q + batch * a.q_stride[0] + head * a.q_stride[1] +
                   (int64_t) row * a.q_stride[2],
               row < n, a.dim);
  floatx16 acc[DP / 32] = {};
  float m = -INFINITY, l = 0.f;
  const float scale = a.scale * kLog2e;

  int end = block * kRows < n ? n : 0;
  if (CAUSAL) end = min(end, (block + 1) * kRows);
  for (int first = 0; first < end; first += kTile) {
    Staged<DP> ks, vs;
    ks.load(k, a.k_stride[2], first, n, a.dim);
    vs.load(v, a.v_stride[2], first, n, a.dim);
    __syncthreads();
    ks.store(k_tile);
    vs.store(v_tile);
    __syncthreads();
    if (CAUSAL && first > wave_row + 31) continue;

    floatx16 s[2] = {};
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        s[b] = mfma(row_operand<DP>(k_tile, b * 32, d), q[d], s[b]);
    if (first + kTile > n || (CAUSAL && first + kTile - 1 > wave_row)) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = first + b * 32 + i / 4 * 8 + h * 4 + i % 4;
          if (key >= n || (CAUSAL && key > row)) s[b][i] = -INFINITY;
        }
    }
    float most = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) most = fmaxf(most, s[i / 16][i % 16]);
    most = fmaxf(most, other_half(most));
    // the first tile holds key 0, which every row sees: m is finite after it
    const float next = fmaxf(m, most * scale);
    const float fade = exp2_fast(m - next);
    m = next;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float p = exp2_fast(s[i / 16][i % 16] * scale - m);
      s[i / 16][i % 16] = p;
      sum += p;
    }
    l = l * fade + sum;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) acc[b] *= fade;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const bf16x8 prob = rounded(s[p / 2], p % 2);
#pragma unroll
      for (int b = 0; b < DP / 32; ++b)
        acc[b] = mfma(column_operand<DP>(v_tile, p * 16, b), prob, acc[b]);
    }
  }

  if (row >= a.tokens) return;
  l += other_half(l);
  const bool valid = row < n;
  const int64_t o_at = batch * a.o_stride[0] + head * a.o_stride[1] +
                       (int64_t) row * a.o_stride[2];
  store_row<DP>(a.o + o_at, acc, 1.f / l, valid, a.dim,
                a.o_low ? a.o_low + o_at : nullptr);
  if (a.lse && h == 0)
    a.lse[(int64_t) bh * a.tokens + row] =
        valid ? m + log2_fast(l) : INFINITY;
}

// dQ, and delta for the other kernel
template <int DP, bool CAUSAL>
__global__ __launch_bounds__(kThreads, 2) void attention_dq_kernel(
    AttentionArgs a) {
  __shared__ __align__(16) bf16 k_tile[kTile * DP];
  __shared__ __align__(16) bf16 v_tile[kTile * DP];
  const int blocks = (a.tokens + kRows - 1) / kRows;
  int bh, block;
  whose(a.batch * a.heads, blocks, CAUSAL, bh, block);
  const int batch = bh / a.heads, head = bh % a.heads;
  const int kv_head = head / (a.heads / a.kv_heads);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int h = lane / 32;
  const int n = valid_tokens(a, batch);
  const int wave_row = block * kRows + wave * 32;
  const int row = wave_row + lane % 32;
  const bool valid = row < n;

  const bf16* k = a.k + batch * a.k_stride[0] + kv_head * a.k_stride[1];
  const bf16* v = a.v + batch * a.v_stride[0] + kv_head * a.v_stride[1];
  bf16x8 q[DP / 16], dout[DP / 16];
  float delta = 0.f;
  {
    bf16x8 o[DP / 16], o_low[DP / 16];
    load_row<DP>(q,
                 a.q + batch * a.q_stride[0] + head * a.q_stride[1] +
                     (int64_t) row * a.q_stride[2],
                 valid, a.dim);
    load_row<DP>(dout,
                 a.dout + batch * a.dout_stride[0] + head * a.dout_stride[1] +
                     (int64_t) row * a.dout_stride[2],
                 valid, a.dim);
    const int64_t o_at = batch * a.o_stride[0] + head * a.o_stride[1] +
                         (int64_t) row * a.o_stride[2];
    load_row<DP>(o, a.o + o_at, valid, a.dim);
    load_row<DP>(o_low, a.o_low + o_at, valid, a.dim);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        delta += (float) dout[s][j] * ((float) o[s][j] + (float) o_low[s][j]);
    delta += other_half(delta);
  }
  const int64_t at = (int64_t) bh * a.tokens + row;
  if (row < a.tokens && h == 0) a.delta[at] = delta;
  // +inf makes every probability of a row without keys 0
  const float lse = valid ? a.lse[at] : INFINITY;
  floatx16 acc[DP / 32] = {};
  const float scale = a.scale * kLog2e;

  int end = block * kRows < n ? n : 0;
  if (CAUSAL) end = min(end, (block + 1) * kRows);
  for (int first = 0; first < end; first += kTile) {
    Staged<DP> ks, vs;
    ks.load(k, a.k_stride[2], first, n, a.dim);
    vs.load(v, a.v_stride[2], first, n, a.dim);
    __syncthreads();
    ks.store(k_tile);
    vs.store(v_tile);
    __syncthreads();
    if (CAUSAL && first > wave_row + 31) continue;

    const bool masked = first + kTile > n ||
                        (CAUSAL && first + kTile - 1 > wave_row);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      floatx16 s = {}, dp = {};
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        s = mfma(row_operand<DP>(k_tile, b * 32, d), q[d], s);
        dp = mfma(row_operand<DP>(v_tile, b * 32, d), dout[d], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float p = exp2_fast(s[i] * scale - lse);
        if (masked) {
          const int key = first + b * 32 + i / 4 * 8 + h * 4 + i % 4;
          if (key >= n || (CAUSAL && key > row)) p = 0.f;
        }
        s[i] = p * (dp[i] - delta);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const bf16x8 ds = rounded(s, p);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)
          acc[c] =
              mfma(column_operand<DP>(k_tile, b * 32 + p * 16, c), ds, acc[c]);
      }
    }
  }
  if (row >= a.tokens) return;
  store_row<DP>(a.dq + batch * a.dq_stride[0] + head * a.dq_stride[1] +
                    (int64_t) row * a.dq_stride[2],
                acc, a.scale, valid, a.dim);
}

// dK and dV, summed over the heads that share them
template <int DP, bool CAUSAL>
__global__ __launch_bounds__(kThreads, 1) void attention_dkv_kernel(
    AttentionArgs a) {
  __shared__ __align__(16) bf16 q_tile[kTile * DP];
  __shared__ __align__(16) bf16 do_tile[kTile * DP];
  __shared__ __align__(16) float lse_tile[kTile], delta_tile[kTile];
  const int blocks = (a.tokens + kRows - 1) / kRows;
  int bh, block;
  whose(a.batch * a.kv_heads, blocks, false, bh, block);
  const int batch = bh / a.kv_heads, kv_head = bh % a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int h = lane / 32;
  const int n = valid_tokens(a, batch);
  const int wave_key = block * kRows + wave * 32;
  const int key = wave_key + lane % 32;
  const bool valid = key < n;

  bf16x8 k[DP / 16], v[DP / 16];
  load_row<DP>(k,
               a.k + batch * a.k_stride[0] + kv_head * a.k_stride[1] +
                   (int64_t) key * a.k_stride[2],
               valid, a.dim);
  load_row<DP>(v,
               a.v + batch * a.v_stride[0] + kv_head * a.v_stride[1] +
                   (int64_t) key * a.v_stride[2],
               valid, a.dim);
  floatx16 dk[DP / 32] = {}, dv[DP / 32] = {};
  const float scale = a.scale * kLog2e;

  const int end = block * kRows < n ? n : 0;
  const int start = CAUSAL ? block * kRows : 0;  // a multiple of kTile
  for (int g = 0; g < group; ++g) {
    const int head = kv_head * group + g;
    const bf16* q = a.q + batch * a.q_stride[0] + head * a.q_stride[1];
    const bf16* dout =
        a.dout + batch * a.dout_stride[0] + head * a.dout_stride[1];
    const int64_t stats = ((int64_t) batch * a.heads + head) * a.tokens;
    for (int first = start; first < end; first += kTile) {
      Staged<DP> qs, dos;
      qs.load(q, a.q_stride[2], first, n, a.dim);
      dos.load(dout, a.dout_stride[2], first, n, a.dim);
      float lse = INFINITY, delta = 0.f;
      if (threadIdx.x < kTile && first + (int) threadIdx.x < n) {
        lse = a.lse[stats + first + threadIdx.x];
        delta = a.delta[stats + first + threadIdx.x];
      }
      __syncthreads();
      qs.store(q_tile);
      dos.store(do_tile);
      if (threadIdx.x < kTile) {
        lse_tile[threadIdx.x] = lse;
        delta_tile[threadIdx.x] = delta;
      }
      __syncthreads();
      if (CAUSAL && first + kTile - 1 < wave_key) continue;

      const bool masked = CAUSAL && first < wave_key + 31;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        floatx16 s = {}, dp = {};
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          s = mfma(row_operand<DP>(q_tile, b * 32, d), k[d], s);
          dp = mfma(row_operand<DP>(do_tile, b * 32, d), v[d], dp);
        }
        floatx16 prob;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int line = b * 32 + i * 8 + h * 4;
          const floatx4 lses = *reinterpret_cast<floatx4*>(lse_tile + line);
          const floatx4 deltas = *reinterpret_cast<floatx4*>(delta_tile + line);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float p = exp2_fast(s[i * 4 + j] * scale - lses[j]);
            if (masked && key > first + line + j) p = 0.f;
            prob[i * 4 + j] = p;
            s[i * 4 + j] = p * (dp[i * 4 + j] - deltas[j]);
          }
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const bf16x8 probs = rounded(prob, p), ds = rounded(s, p);
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            const int line = b * 32 + p * 16;
            dv[c] = mfma(column_operand<DP>(do_tile, line, c), probs, dv[c]);
            dk[c] = mfma(column_operand<DP>(q_tile, line, c), ds, dk[c]);
          }
        }
      }
    }
  }
  if (key >= a.tokens) return;
  store_row<DP>(a.dk + batch * a.dk_stride[0] + kv_head * a.dk_stride[1] +
                    (int64_t) key * a.dk_stride[2],
                dk, a.scale, valid, a.dim);
  store_row<DP>(a.dv + batch * a.dv_stride[0] + kv_head * a.dv_stride[1] +
                    (int64_t) key * a.dv_stride[2],
                dv, 1.f, valid, a.dim);
}

template <int DP, bool CAUSAL>
int forward(const AttentionArgs& a) {
  const int64_t blocks = (a.tokens + kRows - 1) / kRows;
  hipLaunchKernelGGL((attention_forward_kernel<DP, CAUSAL>),
                     dim3((unsigned) (blocks * a.batch * a.heads)),
                     dim3(kThreads), 0, static_cast<hipStream_t>(a.stream), a);
  return (int) hipGetLastError();
}

template <int DP, bool CAUSAL>
int backward(const AttentionArgs& a) {
  const int64_t blocks = (a.tokens + kRows - 1) / kRows;
  hipLaunchKernelGGL((attention_dq_kernel<DP, CAUSAL>),
                     dim3((unsigned) (blocks * a.batch * a.heads)),
                     dim3(kThreads), 0, static_cast<hipStream_t>(a.stream), a);
  int status = (int) hipGetLastError();
  if (status) return status;
  hipLaunchKernelGGL((attention_dkv_kernel<DP, CAUSAL>),
                     dim3((unsigned) (blocks * a.batch * a.kv_heads)),
                     dim3(kThreads), 0, static_cast<hipStream_t>(a.stream), a);
  return (int) hipGetLastError();
}

bool sound(const AttentionArgs* a) {
  if (!a || a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 ||
      a->heads % a->kv_heads || a->tokens <= 0 || a->dim <= 0 || a->dim % 8 ||
      a->dim > 128 || !a->q || !a->k || !a->v || !a->o)
    return false;
  // the grid, and row numbers up to the end of a block
  return a->tokens <= (1 << 24) &&
         (int64_t) a->batch * a->heads * ((a->tokens + kRows - 1) / kRows) <=
             INT32_MAX;
}

}  // namespace
}  // namespace sofa_model

extern "C" {

int sofa_attention_forward(const sofa_model::AttentionArgs* a) {
  using namespace sofa_model;
  if (!sound(a)) return kBadArgument;
  DeviceGuard guard(a->device);
  if (guard.status()) return guard.status();
  if (a->dim <= 64)
    return a->causal ? forward<64, true>(*a) : forward<64, false>(*a);
  return a->causal ? forward<128, true>(*a) : forward<128, false>(*a);
}

int sofa_attention_backward(const sofa_model::AttentionArgs* a) {
  using namespace sofa_model;
  if (!sound(a) || !a->dout || !a->o_low || !a->lse || !a->delta || !a->dq || !a->dk ||
      !a->dv)
    return kBadArgument;
  DeviceGuard guard(a->device);
  if (guard.status()) return guard.status();
  if (a->dim <= 64)
    return a->causal ? backward<64, true>(*a) : backward<64, false>(*a);
  return a->causal ? backward<128, true>(*a) : backward<128, false>(*a);
}

}  // extern "C"
