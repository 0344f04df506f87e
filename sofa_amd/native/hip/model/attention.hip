// Self-attention over grouped heads and its gradients, on the matrix cores.
//
//   S = c Q K^T + mask      P = softmax(S) = e^(S - lse) = e^(c (Q K^T - L))
//   O = P V
//   dV = P^T dO             dP = dO V^T       delta = rowsum(dO O)
//   dS = P (dP - delta)     dQ = c dS K       dK = c dS^T Q
//
// The scores are never stored: the forward pass runs over the keys with a
// running maximum and sum (in 32 bits, base 2) and keeps L = lse / c, in units
// of the products: a row that is sure of one key has L equal to that product, bit
// by bit, however large it is, and the backward pass computes P = 1 again.  (lse
// itself, next to scores in the hundred thousands, is 2^-6 apart.)  The products
// are summed in the same order each time.  The backward pass is two kernels, one that owns rows of
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
// gives a lane 4 rows of one column, in that same order.
//
// Roundings: P and dS to bf16 for their products, 2^-8 relative at most, as in
// the results themselves; sums stay in 32 bits.  Only delta, which dP - delta
// almost cancels in short rows, takes more of O than its 8 bits: the forward
// pass keeps what the rounding took off as well (with O's own rounding dQ and
// dK of 32 tokens were 1.9 times as far off as their own rounding leaves them).
//
// Measured at 32 query and 8 key heads of 128, causal, in products' TFLOP/s
// (2, 3 and 4 products; a large library product reaches 1220):
//                  2 x 2048      2 x 4096       1 x 8192 tokens
//   forward, lse  100 us  690    312 us  880    568 us  970
//   dQ            124 us  830    416 us  990    740 us 1115
//   dK, dV        172 us  800    555 us  990   1035 us 1065
// What bounds them there is the issue of a wave's own instructions: products take
// 40 % of its cycles, exponentials and their surroundings as many, and two waves
// on a SIMD (256 registers each) fill each other's gaps only in part.  Where all
// workgroups are resident at once (up to about 2 x 2048 of these) it is the longest
// chain of tiles that one of them goes through.  Heads are padded to 64 or 128
// elements, and the padding is multiplied.

#include "model_ops.h"

namespace sofa_model {
namespace {

typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kRows = kWaves * 32;  // rows a workgroup owns
constexpr int kTile = 64;           // rows of the other side at a time
constexpr int kShort = 256;         // tokens that leave a compute unit room
constexpr int kFewKeys = 256;       // up to which P and dS have 16 bits

// Where the 8 elements `chunk` of `row` of a tile are in LDS.  A row is 256 or
// 128 bytes and the banks 256, so one chunk of all rows falls on the same banks;
// the exclusive or moves it such that what one cycle pair reads is on different
// ones: 16 rows of one chunk (a row operand), and 4 rows by 4 chunks (a column
// operand).  Its lower two bits tell rows 4 apart, the next those 1 apart.  (With
// pairs of chunks moved by 8 rows, 40 % of LDS cycles were conflicts.)
template <int DP>
__device__ __forceinline__ int swizzle(int row) {
  return DP == 128 ? (row & 3) << 2 | (row >> 2 & 3)
                   : (row >> 1 & 1) << 2 | (row >> 2 & 3);
}
template <int DP>
__device__ __forceinline__ int lds_at(int row, int chunk) {
  return row * DP + ((chunk ^ swizzle<DP>(row)) << 3);
}

// Starts a tile of ROWS rows on its way from memory to LDS, 16 bytes a lane
// and past the registers: a wave's part of LDS is filled in the order of its
// lanes, so each lane takes the chunk that belongs in its place.  `tile` is the
// tile's first row, the same for the whole workgroup; addresses are then a
// scalar base and one 32-bit offset.  Rows behind the last valid one repeat it,
// and chunks behind the last one repeat that: what is computed from them is
// multiplied by zeros or not stored, and has only to be finite.
template <int DP, int ROWS = kTile>
__device__ __forceinline__ void load_tile(const bf16* tile, int64_t stride,
                                          int rows, int dim, bf16* to) {
  typedef const __attribute__((address_space(1))) uint32_t* from_t;
  typedef __attribute__((address_space(3))) uint32_t* to_t;
  constexpr int kChunks = DP / 8;
  constexpr int kStep = kThreads / kChunks;  // rows a pass
  const uint32_t row = threadIdx.x / kChunks;
  const int chunk = threadIdx.x % kChunks ^ swizzle<DP>(row);
  const uint32_t at = min(chunk, dim / 8 - 1) * 8;
  const uint32_t step = (uint32_t) stride;  // up to kMaxTokenStride
  to += __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * kWave * 8;
#pragma unroll
  for (int p = 0; p < ROWS / kStep; ++p) {
    // swizzle() repeats after 16 rows, so that the chunk is the same each pass
    const bf16* from =
        rows >= ROWS
            ? tile + p * kStep * stride + (row * step + at)
            : tile + (min(row + p * kStep, (uint32_t) rows - 1) * step + at);
    __builtin_amdgcn_global_load_lds((from_t) from, (to_t) (to + p * kStep * DP),
                                     16, 0, 0);
  }
}

// All of the workgroup's tiles on their way are there.  Reads of LDS wait for
// this wave's own loads before that, so the next ones start where no more reads
// follow for some time, after the scores' products.  Staged in registers instead,
// for a whole tile's time, the forward pass took 8 % more.
__device__ __forceinline__ void arrived() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
}

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

// What that rounding took off
__device__ __forceinline__ bf16x8 rest_of(const floatx16& d, int part,
                                          bf16x8 rounded) {
  bf16x8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    r[j] = (bf16) (d[part * 8 + j] - (float) rounded[j]);
  return r;
}

__device__ __forceinline__ floatx16 mfma(bf16x8 a, bf16x8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// sum + the 8 values
__device__ __forceinline__ float add_all(bf16x8 x, float sum) {
  const bf16x2 one = {(bf16) 1.f, (bf16) 1.f};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[2 * j], x[2 * j + 1]}, one,
                                          sum, false);
  return sum;
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

// Orders this wave's accesses to LDS between its lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The 32 rows of a wave's result, which are its lanes' columns of D, to memory
// by way of LDS (`stage`: the wave's 32 DP elements), so that whole rows are
// written: a lane's own pieces are 8 bytes in a row of its own.  Rows that are
// not valid are zeros, whatever was computed for them; `rows` exist.  `rest`:
// what rounding took off in place of the result.
template <int DP>
__device__ __forceinline__ void store_rows(bf16* stage, bf16* to,
                                           int64_t stride, int rows, int dim,
                                           const floatx16 (&acc)[DP / 32],
                                           float factor, bool valid,
                                           bool rest = false) {
  constexpr int kChunks = DP / 8;
  const int lane = threadIdx.x % kWave, h = lane / 32;
  wave_sync();
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = valid ? acc[b][i * 4 + j] * factor : 0.f;
        x[j] = (bf16) y;
        if (rest) x[j] = (bf16) (y - (float) x[j]);
      }
      *reinterpret_cast<bf16x4*>(stage + lds_at<DP>(lane % 32, b * 4 + i) +
                                 h * 4) = x;
    }
  wave_sync();
#pragma unroll
  for (int p = 0; p < 32 * kChunks / kWave; ++p) {
    const int row = (p * kWave + lane) / kChunks, chunk = lane % kChunks;
    if (row < rows && chunk * 8 < dim)
      *reinterpret_cast<bf16x8*>(to + row * stride + chunk * 8) =
          *reinterpret_cast<const bf16x8*>(stage + lds_at<DP>(row, chunk));
  }
}

// The same in 32 bits, 32 columns at a time, rows `dim` apart
template <int DP>
__device__ __forceinline__ void store_rows(bf16* stage, float* to, int rows,
                                           int dim,
                                           const floatx16 (&acc)[DP / 32],
                                           bool valid) {
  float* buffer = reinterpret_cast<float*>(stage);
  const int lane = threadIdx.x % kWave, h = lane / 32;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
    wave_sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      floatx4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = valid ? acc[b][i * 4 + j] : 0.f;
      *reinterpret_cast<floatx4*>(
          buffer + lane % 32 * 32 + ((i * 2 + h) ^ (lane & 7)) * 4) = x;
    }
    wave_sync();
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int row = p * 8 + lane / 8, at = b * 32 + lane % 8 * 4;
      if (row < rows && at < dim)
        *reinterpret_cast<floatx4*>(to + row * dim + at) =
            *reinterpret_cast<const floatx4*>(
                buffer + row * 32 + (lane % 8 ^ (row & 7)) * 4);
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

// Short heads of long rows: four workgroups on a compute unit, at the cost of a
// register or three spilled (2 x 4096 tokens, 32/8 heads of 64, no mask: 337 us in
// place of 348 with three, 321 in place of 325 without lse); a few hundred tokens
// do not fill them, and lose 3 %.
// KEEP: with lse, whose own sum of the probabilities takes 4 % of the time.
template <int DP, bool CAUSAL, bool SHORT, bool KEEP>
__global__ __launch_bounds__(kThreads, DP > 64 ? 2 : SHORT ? 3 : 4)
void attention_forward_kernel(
    AttentionArgs a) {
  __shared__ __align__(16) bf16 k_tiles[2][kTile * DP];
  __shared__ __align__(16) bf16 v_tiles[2][kTile * DP];
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
  // l sums what 16 bits leave of the probabilities, since it divides their
  // product: the weights are 1 together then. (Summed before they are rounded, a
  // row with one large probability is off by all of its rounding, and dP - delta,
  // almost 0 there, by more than itself.) lse takes their sum before they are
  // rounded: what the backward pass computes from it is not rounded yet.
  float m = -INFINITY, l = 0.f, l_exact = 0.f;
  float largest = -INFINITY;  // KEEP: of the products
  const float scale = a.scale * kLog2e;

  int end = block * kRows < n ? n : 0;
  if (CAUSAL) end = min(end, (block + 1) * kRows);
  auto load = [&](int first, int buffer) {
    if (first >= end) return;
    load_tile<DP>(k + first * a.k_stride[2], a.k_stride[2], n - first, a.dim,
                  k_tiles[buffer]);
    load_tile<DP>(v + first * a.v_stride[2], a.v_stride[2], n - first, a.dim,
                  v_tiles[buffer]);
  };
  auto tile = [&]<bool MASKED>(int first, int buffer) {
    const bf16 *k_tile = k_tiles[buffer], *v_tile = v_tiles[buffer];
    floatx16 s[2] = {};
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        s[b] = mfma(row_operand<DP>(k_tile, b * 32, d), q[d], s[b]);
    load(first + kTile, buffer ^ 1);
    if (MASKED) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int key = first + i / 4 * 8 + h * 4 + i % 4;
        if (key >= n || (CAUSAL && key > row)) s[i / 16][i % 16] = -INFINITY;
      }
    }
    float most = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) most = fmaxf(most, s[i / 16][i % 16]);
    most = fmaxf(most, other_half(most));
    if (KEEP) largest = fmaxf(largest, most);
    // m follows the maximum in steps of 2^8 or more: the probabilities are
    // relative to it anyway, and most tiles need no new factor for the sums.
    // The first tile holds key 0, which every row sees: m is finite after it.
    if (__any(most * scale > m + 8.f)) {
      const float next = fmaxf(m, most * scale);
      const float fade = exp2_fast(m - next);
      m = next;
      l *= fade;
      if (KEEP) l_exact *= fade;
#pragma unroll
      for (int b = 0; b < DP / 32; ++b) acc[b] *= fade;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float p = exp2_fast(fmaf(s[i / 16][i % 16], scale, -m));
      if (KEEP) l_exact += p;
      s[i / 16][i % 16] = p;
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const bf16x8 prob = rounded(s[p / 2], p % 2);
      l = add_all(prob, l);
#pragma unroll
      for (int b = 0; b < DP / 32; ++b)
        acc[b] = mfma(column_operand<DP>(v_tile, p * 16, b), prob, acc[b]);
    }
  };
  // tiles that every row sees whole, then the others
  const int whole = (CAUSAL ? min(block * kRows, n) : n) / kTile * kTile;
  int first = 0, buffer = 0;
  load(0, 0);
  for (; first < min(whole, end); first += kTile, buffer ^= 1) {
    arrived();
    tile.template operator()<false>(first, buffer);
  }
  for (; first < end; first += kTile, buffer ^= 1) {
    arrived();
    if (CAUSAL && first > wave_row + 31)
      load(first + kTile, buffer ^ 1);
    else
      tile.template operator()<true>(first, buffer);
  }

  l += other_half(l);
  if (KEEP) l_exact += other_half(l_exact);
  const bool valid = row < n;
  if (KEEP && row < a.tokens && h == 0)
    a.lse[(int64_t) bh * a.tokens + row] =
        // m is the rounding of a product's multiple, or lags behind: what the sum
        // is relative to, less that
        valid ? largest + (log2_fast(l_exact) - fmaf(largest, scale, -m)) / scale
              : INFINITY;
  __syncthreads();  // the tiles are not read any more
  bf16* stage = k_tiles[0] + wave * 32 * DP;
  const int64_t o_at = batch * a.o_stride[0] + head * a.o_stride[1] +
                       (int64_t) wave_row * a.o_stride[2];
  store_rows<DP>(stage, a.o + o_at, a.o_stride[2], a.tokens - wave_row, a.dim,
                 acc, 1.f / l, valid);
  if (a.o_low)
    store_rows<DP>(stage, a.o_low + o_at, a.o_stride[2], a.tokens - wave_row,
                   a.dim, acc, 1.f / l, valid, true);
}

// dQ, and delta for the other kernel.
//
// EXACT, and for rows that see up to kFewKeys keys: dS, and P for dV, are taken
// with 16 bits, as their rounding and what that took off.  In long rows their
// rounding is one of many and leaves the gradients 1.4 times as far off as their
// own rounding does; in short ones it was up to 1.8 times.  The rule is one of the
// keys that a workgroup's rows see, so that a sequence is as exact in whatever
// batch, and the first rows of a long one as a short one.  The
// products that this adds are not what takes the time there.
template <int DP, bool CAUSAL, bool EXACT>
__global__ __launch_bounds__(kThreads, DP > 64 ? 2 : 3)
void attention_dq_kernel(
    AttentionArgs a) {
  __shared__ __align__(16) bf16 k_tiles[2][kTile * DP];
  __shared__ __align__(16) bf16 v_tiles[2][kTile * DP];
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
  // +inf makes every probability of a row without keys 0; and with one key alone
  // dS is 0, not what roundings leave of dP - delta
  const bool sees = valid && !(n == 1 || (CAUSAL && row == 0));
  const float scale = a.scale * kLog2e;
  const float start = sees ? a.lse[at] : 0.f;
  const float lse = sees ? start * scale : INFINITY;
  // what that product's rounding took off is a factor of the whole row
  const float factor = a.scale * (sees ? exp2_fast(-fmaf(start, scale, -lse)) : 1.f);
  floatx16 acc[DP / 32] = {};

  int end = block * kRows < n ? n : 0;
  if (CAUSAL) end = min(end, (block + 1) * kRows);
  auto load = [&](int first, int buffer) {
    if (first >= end) return;
    load_tile<DP>(k + first * a.k_stride[2], a.k_stride[2], n - first, a.dim,
                  k_tiles[buffer]);
    load_tile<DP>(v + first * a.v_stride[2], a.v_stride[2], n - first, a.dim,
                  v_tiles[buffer]);
  };
  // 32 kBlocks keys at a time: short heads gain more from a third workgroup on
  // the compute unit (168 registers) than from two independent chains
  constexpr int kBlocks = DP <= 64 ? 1 : 2;
  auto tile = [&]<bool MASKED, bool FEW>(int first, int buffer) {
    const bf16 *k_tile = k_tiles[buffer], *v_tile = v_tiles[buffer];
#pragma unroll
    for (int part = 0; part < 2 / kBlocks; ++part) {
      floatx16 s[kBlocks] = {}, dp[kBlocks] = {};
      const int line = part * kBlocks * 32;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          s[b] = mfma(row_operand<DP>(k_tile, line + b * 32, d), q[d], s[b]);
          dp[b] =
              mfma(row_operand<DP>(v_tile, line + b * 32, d), dout[d], dp[b]);
        }
      if (part == 2 / kBlocks - 1) load(first + kTile, buffer ^ 1);
#pragma unroll
      for (int i = 0; i < 16 * kBlocks; ++i) {
        float p = exp2_fast(fmaf(s[i / 16][i % 16], scale, -lse));
        if (MASKED) {
          const int key = first + line + i / 4 * 8 + h * 4 + i % 4;
          if (key >= n || (CAUSAL && key > row)) p = 0.f;
        }
        s[i / 16][i % 16] = p * (dp[i / 16][i % 16] - delta);
      }
#pragma unroll
      for (int p = 0; p < 2 * kBlocks; ++p) {
        const bf16x8 ds = rounded(s[p / 2], p % 2);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          const bf16x8 keys = column_operand<DP>(k_tile, line + p * 16, c);
          acc[c] = mfma(keys, ds, acc[c]);
          if (FEW) acc[c] = mfma(keys, rest_of(s[p / 2], p % 2, ds), acc[c]);
        }
      }
    }
  };
  // tiles that every row sees whole, then the others
  const int whole = (CAUSAL ? min(block * kRows, n) : n) / kTile * kTile;
  auto all = [&]<bool FEW>() {
    int first = 0, buffer = 0;
    load(0, 0);
    for (; first < min(whole, end); first += kTile, buffer ^= 1) {
      arrived();
      tile.template operator()<false, FEW>(first, buffer);
    }
    for (; first < end; first += kTile, buffer ^= 1) {
      arrived();
      if (CAUSAL && first > wave_row + 31)
        load(first + kTile, buffer ^ 1);
      else
        tile.template operator()<true, FEW>(first, buffer);
    }
  };
  if (EXACT || end <= kFewKeys)
    all.template operator()<true>();
  else
    all.template operator()<false>();
  __syncthreads();  // the tiles are not read any more
  store_rows<DP>(k_tiles[0] + wave * 32 * DP,
                 a.dq + batch * a.dq_stride[0] + head * a.dq_stride[1] +
                     (int64_t) wave_row * a.dq_stride[2],
                 a.dq_stride[2], a.tokens - wave_row, a.dim, acc, factor,
                 valid);
}

// dK and dV, summed over the heads that share them.  A workgroup takes its
// share, one of key_parts, of the tiles of these heads' rows.
//
// What bounds it is that a wave's products wait for LDS and for its own
// exponentials, so two workgroups have to share a compute unit.  The results
// take 128 of the 256 registers that leaves a wave with DP = 128, K 32 more; V
// is in LDS then and tiles have 32 rows.  With V in registers too and one
// workgroup (of 64 rows a tile) the same 2 x 4096 tokens, 32/8 heads, took 1.26
// ms in place of 1.04, without a mask.
//
// P and dS of rows that see up to kFewKeys keys have 16 bits, as in dQ.  SHORT: all
// of them, next to the products of what rounding leaves.  Otherwise the tiles of
// such rows are gone over once more for the products of the rest: in the loop
// over all tiles a second body, or a branch, takes 9 to 30 % (registers).  Those of
// longer rows have one rounding each for heads of up to 32 too, where dQ has 16
// bits: it would take 129 us in place of 86 at 2 x 2048 tokens, 32 heads of 16.
template <int DP, bool CAUSAL, bool SHORT>
__global__ __launch_bounds__(kThreads, 2) void
attention_dkv_kernel(AttentionArgs a) {
  constexpr bool kKeepV = DP <= 64;
  constexpr int kLines = kKeepV ? 64 : 32;  // rows of a tile
  constexpr int kBlocks = kLines / 32;
  __shared__ __align__(16) bf16 v_rows[kKeepV ? 8 : kRows * DP];
  __shared__ __align__(16) bf16 tiles_of[2][2][kLines * DP];
  bf16(*q_tiles)[kLines * DP] = tiles_of[0];
  bf16(*do_tiles)[kLines * DP] = tiles_of[1];
  // lse, and -delta, which the products of a row start from
  __shared__ __align__(16) float lse_tiles[2][kLines];
  __shared__ __align__(16) float delta_tiles[2][kLines];
  const int blocks = (a.tokens + kRows - 1) / kRows;
  int bh, block;
  whose(a.batch * a.kv_heads, blocks * a.key_parts, false, bh, block);
  const int part = block % a.key_parts;
  block /= a.key_parts;
  const int batch = bh / a.kv_heads, kv_head = bh % a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int h = lane / 32;
  const int n = valid_tokens(a, batch);
  const int wave_key = block * kRows + wave * 32;
  const int key = wave_key + lane % 32;
  const bool valid = key < n;

  bf16x8 k[DP / 16], v[kKeepV ? DP / 16 : 1];
  load_row<DP>(k,
               a.k + batch * a.k_stride[0] + kv_head * a.k_stride[1] +
                   (int64_t) key * a.k_stride[2],
               valid, a.dim);
  {
    bf16x8 row[DP / 16];
    load_row<DP>(row,
                 a.v + batch * a.v_stride[0] + kv_head * a.v_stride[1] +
                     (int64_t) key * a.v_stride[2],
                 valid, a.dim);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      if constexpr (kKeepV)
        v[d] = row[d];
      else  // read by this wave only, in order
        *reinterpret_cast<bf16x8*>(
            v_rows + lds_at<DP>(wave * 32 + lane % 32, d * 2 + h)) = row[d];
    }
  }
  floatx16 dk[DP / 32] = {}, dv[DP / 32] = {};
  const float scale = a.scale * kLog2e;

  // the tiles of one head after those of the other; in each from the last
  // rows to the first, so that workgroups of other keys, which start at other
  // rows where the mask is causal, read the same tiles at the same time
  const int start = CAUSAL ? block * kRows : 0;  // a multiple of kLines
  const int tiles = block * kRows < n ? (n - start + kLines - 1) / kLines : 0;
  const int masked = CAUSAL ? min(tiles, kRows / kLines) : 0;  // the last ones
  int step = (int) ((int64_t) tiles * group * part / a.key_parts);
  const int stop = (int) ((int64_t) tiles * group * (part + 1) / a.key_parts);
  float lse = 0.f, delta = 0.f;
  auto load = [&](int step, int buffer) {
    if (step >= stop) return;
    const int head = kv_head * group + step / tiles;
    const int first = start + (tiles - 1 - step % tiles) * kLines;
    load_tile<DP, kLines>(a.q + batch * a.q_stride[0] +
                              head * a.q_stride[1] + first * a.q_stride[2],
                          a.q_stride[2], n - first, a.dim, q_tiles[buffer]);
    load_tile<DP, kLines>(
        a.dout + batch * a.dout_stride[0] + head * a.dout_stride[1] +
            first * a.dout_stride[2],
        a.dout_stride[2], n - first, a.dim, do_tiles[buffer]);
    // +inf makes every probability of a row that is not there 0
    lse = INFINITY;
    delta = 0.f;
    if (threadIdx.x < kLines && first + (int) threadIdx.x < n) {
      const int64_t at = ((int64_t) batch * a.heads + head) * a.tokens + first +
                         threadIdx.x;
      lse = a.lse[at];
      delta = a.delta[at];
    }
  };
  auto store = [&](int buffer) {
    if (threadIdx.x < kLines) {
      lse_tiles[buffer][threadIdx.x] = lse;
      delta_tiles[buffer][threadIdx.x] = -delta;
    }
  };
  // REST: the products of what rounding takes off P and dS; `next` comes after it
  auto tile = [&]<bool MASKED, bool REST>(int step, int next, int buffer) {
    const bf16 *q_tile = q_tiles[buffer], *do_tile = do_tiles[buffer];
    floatx16 s[kBlocks] = {}, dp[kBlocks];
#pragma unroll
    for (int i = 0; i < 4 * kBlocks; ++i) {
      const floatx4 y =
          *reinterpret_cast<const floatx4*>(delta_tiles[buffer] + i * 8 + h * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) dp[i / 4][i % 4 * 4 + j] = y[j];
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        s[b] = mfma(row_operand<DP>(q_tile, b * 32, d), k[d], s[b]);
        if constexpr (kKeepV)
          dp[b] = mfma(row_operand<DP>(do_tile, b * 32, d), v[d], dp[b]);
        else
          dp[b] = mfma(row_operand<DP>(do_tile, b * 32, d),
                       row_operand<DP>(v_rows, wave * 32, d), dp[b]);
      }
    load(next, buffer ^ 1);
    const int first = start + (tiles - 1 - step % tiles) * kLines;
#pragma unroll
    for (int i = 0; i < 4 * kBlocks; ++i) {
      const int line = i * 8 + h * 4;
      const floatx4 x =
          *reinterpret_cast<const floatx4*>(lse_tiles[buffer] + line);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = i % 4 * 4 + j;
        float p = exp2_fast((s[i / 4][at] - x[j]) * scale);
        if (MASKED && key > first + line + j) p = 0.f;
        s[i / 4][at] = p;
        dp[i / 4][at] *= p;
      }
    }
    // row 0 sees key 0 alone: dS is 0, not what roundings leave of dP - delta
    if (MASKED && first == 0 && h == 0) dp[0][0] = 0.f;
#pragma unroll
    for (int p = 0; p < 2 * kBlocks; ++p) {
      bf16x8 probs = rounded(s[p / 2], p % 2);
      bf16x8 ds = rounded(dp[p / 2], p % 2);
      if (REST) {
        probs = rest_of(s[p / 2], p % 2, probs);
        ds = rest_of(dp[p / 2], p % 2, ds);
      }
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        const bf16x8 douts = column_operand<DP>(do_tile, p * 16, c);
        dv[c] = mfma(douts, probs, dv[c]);
        if (SHORT) dv[c] = mfma(douts, rest_of(s[p / 2], p % 2, probs), dv[c]);
        const bf16x8 rows = column_operand<DP>(q_tile, p * 16, c);
        dk[c] = mfma(rows, ds, dk[c]);
        if (SHORT) dk[c] = mfma(rows, rest_of(dp[p / 2], p % 2, ds), dk[c]);
      }
    }
  };
  int buffer = 0;
  const int begin = step;
  load(step, 0);
  store(0);
  while (step < stop) {
    // tiles whose rows all see every key, then those of the mask's edge
    int until = min(stop, step - step % tiles + tiles - masked);
    for (; step < until; ++step, buffer ^= 1) {
      arrived();
      tile.template operator()<false, false>(step, step + 1, buffer);
      store(buffer ^ 1);
    }
    if (!CAUSAL) continue;
    until = min(stop, step - step % tiles + tiles);
    if (step % tiles < tiles - masked) until = step;
    for (; step < until; ++step, buffer ^= 1) {
      arrived();
      const int first = start + (tiles - 1 - step % tiles) * kLines;
      if (first + kLines - 1 < wave_key)
        load(step + 1, buffer ^ 1);
      else
        tile.template operator()<true, false>(step, step + 1, buffer);
      store(buffer ^ 1);
    }
  }
  // the last tiles of each head, whose rows see few keys
  const int few = n <= kFewKeys ? tiles
                  : CAUSAL      ? min(tiles, max(0, kFewKeys - start) / kLines)
                                : 0;
  if (!SHORT && few && begin < stop) {
    auto from = [&](int step) {  // the first of these that is not before `step`
      return step + max(0, tiles - few - step % tiles);
    };
    step = from(begin);
    __syncthreads();  // the tiles are not read any more
    load(step, buffer);
    store(buffer);
    for (; step < stop; step = from(step + 1), buffer ^= 1) {
      arrived();
      tile.template operator()<CAUSAL, true>(step, from(step + 1), buffer);
      store(buffer ^ 1);
    }
  }

  __syncthreads();  // the tiles are not read any more
  bf16* stage = tiles_of[0][0] + wave * 32 * DP;
  const int rows = a.tokens - wave_key;
  const bool has_dk = valid && n > 1;  // dS is 0 for one key alone
  if (a.key_parts > 1) {
    const int64_t size = (int64_t) a.batch * a.kv_heads * a.tokens * a.dim;
    float* out = a.partial + part * 2 * size +
                 ((int64_t) bh * a.tokens + wave_key) * a.dim;
    store_rows<DP>(stage, out, rows, a.dim, dk, has_dk);
    store_rows<DP>(stage, out + size, rows, a.dim, dv, valid);
    return;
  }
  store_rows<DP>(stage,
                 a.dk + batch * a.dk_stride[0] + kv_head * a.dk_stride[1] +
                     (int64_t) wave_key * a.dk_stride[2],
                 a.dk_stride[2], rows, a.dim, dk, a.scale, has_dk);
  store_rows<DP>(stage,
                 a.dv + batch * a.dv_stride[0] + kv_head * a.dv_stride[1] +
                     (int64_t) wave_key * a.dv_stride[2],
                 a.dv_stride[2], rows, a.dim, dv, 1.f, valid);
}

// dK and dV as the sum of their parts, in order; 8 elements a thread
__global__ __launch_bounds__(kThreads) void attention_join_kernel(
    AttentionArgs a) {
  const int64_t size = (int64_t) a.batch * a.kv_heads * a.tokens * a.dim;
  const int64_t at = ((int64_t) blockIdx.x * kThreads + threadIdx.x) * 8;
  if (at >= 2 * size) return;
  const bool is_v = at >= size;
  float sum[8] = {};
  for (int part = 0; part < a.key_parts; ++part) {
    float x[8];
    load8(a.partial + part * 2 * size + at, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] += x[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[j] *= is_v ? 1.f : a.scale;
  const int64_t row = (is_v ? at - size : at) / a.dim;
  const int64_t token = row % a.tokens, head = row / a.tokens % a.kv_heads;
  const int64_t batch = row / a.tokens / a.kv_heads;
  const int64_t* stride = is_v ? a.dv_stride : a.dk_stride;
  store8((is_v ? a.dv : a.dk) + batch * stride[0] + head * stride[1] +
             token * stride[2] + at % a.dim,
         sum);
}

template <int DP, bool CAUSAL, bool SHORT, bool KEEP>
int forward(const AttentionArgs& a) {
  const int64_t blocks = (a.tokens + kRows - 1) / kRows;
  hipLaunchKernelGGL((attention_forward_kernel<DP, CAUSAL, SHORT, KEEP>),
                     dim3((unsigned) (blocks * a.batch * a.heads)),
                     dim3(kThreads), 0, static_cast<hipStream_t>(a.stream), a);
  return (int) hipGetLastError();
}

template <int DP, bool CAUSAL, bool KEEP>
int forward(const AttentionArgs& a) {
  return DP <= 64 && a.tokens <= kShort ? forward<DP, CAUSAL, DP <= 64, KEEP>(a)
                                        : forward<DP, CAUSAL, false, KEEP>(a);
}

template <int DP>
int forward(const AttentionArgs& a) {
  if (a.lse) return a.causal ? forward<DP, true, true>(a) : forward<DP, false, true>(a);
  return a.causal ? forward<DP, true, false>(a) : forward<DP, false, false>(a);
}

template <int DP, bool CAUSAL, bool EXACT>
int dq(const AttentionArgs& a) {
  const int64_t blocks = (a.tokens + kRows - 1) / kRows;
  hipLaunchKernelGGL((attention_dq_kernel<DP, CAUSAL, EXACT>),
                     dim3((unsigned) (blocks * a.batch * a.heads)),
                     dim3(kThreads), 0, static_cast<hipStream_t>(a.stream), a);
  return (int) hipGetLastError();
}

template <int DP, bool CAUSAL, bool SHORT>
int dkv(const AttentionArgs& a) {
  const int64_t blocks = (a.tokens + kRows - 1) / kRows;
  hipLaunchKernelGGL((attention_dkv_kernel<DP, CAUSAL, SHORT>),
                     dim3((unsigned) (blocks * a.batch * a.kv_heads *
                                      a.key_parts)),
                     dim3(kThreads), 0, static_cast<hipStream_t>(a.stream), a);
  return (int) hipGetLastError();
}

template <int DP, bool CAUSAL>
int backward(const AttentionArgs& a) {
  // dQ of short heads with 16 bits everywhere, where it was 1.5 times as far off as
  // its own rounding leaves it (1.44 from 64 elements on): 79 us in place of 64 at
  // 2 x 2048 tokens, 32 heads of 16
  int status = DP <= 64 && a.dim <= 32 ? dq<DP, CAUSAL, DP <= 64>(a)
                                       : dq<DP, CAUSAL, false>(a);
  if (status) return status;
  status = a.tokens <= kFewKeys ? dkv<DP, CAUSAL, true>(a) : dkv<DP, CAUSAL, false>(a);
  if (status || a.key_parts == 1) return status;
  const int64_t threads =
      (int64_t) a.batch * a.kv_heads * a.tokens * (a.dim / 8) * 2;
  hipLaunchKernelGGL(attention_join_kernel,
                     dim3((unsigned) ((threads + kThreads - 1) / kThreads)),
                     dim3(kThreads), 0, static_cast<hipStream_t>(a.stream), a);
  return (int) hipGetLastError();
}

bool sound(const AttentionArgs* a) {
  if (!a || a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 ||
      a->heads % a->kv_heads || a->tokens <= 0 || a->dim <= 0 || a->dim % 8 ||
      a->dim > kMaxHeadDim || !a->q || !a->k || !a->v || !a->o)
    return false;
  for (const int64_t* stride : {a->q_stride, a->k_stride, a->v_stride})
    if (stride[2] < 0 || stride[2] > kMaxTokenStride) return false;
  // row numbers up to the end of a block, and a launch's 2^32 threads
  return a->tokens <= kMaxTokens &&
         (int64_t) a->batch * a->heads * ((a->tokens + kRows - 1) / kRows) <=
             kMaxBlocks;
}

}  // namespace
}  // namespace sofa_model

extern "C" {

int sofa_attention_forward(const sofa_model::AttentionArgs* a) {
  using namespace sofa_model;
  if (!sound(a)) return kBadArgument;
  DeviceGuard guard(a->device);
  if (guard.status()) return guard.status();
  return a->dim <= 64 ? forward<64>(*a) : forward<128>(*a);
}

int sofa_attention_backward(const sofa_model::AttentionArgs* a) {
  using namespace sofa_model;
  if (!sound(a) || !a->dout || !a->o_low || !a->lse || !a->delta || !a->dq || !a->dk ||
      !a->dv || a->key_parts < 1 || a->key_parts > kMaxKeyParts ||
      (a->key_parts > 1 && !a->partial) || a->dout_stride[2] < 0 ||
      a->dout_stride[2] > kMaxTokenStride ||
      (int64_t) a->batch * a->kv_heads * a->key_parts *
              ((a->tokens + kRows - 1) / kRows) > kMaxBlocks)
    return kBadArgument;
  DeviceGuard guard(a->device);
  if (guard.status()) return guard.status();
  if (a->dim <= 64)
    return a->causal ? backward<64, true>(*a) : backward<64, false>(*a);
  return a->causal ? backward<128, true>(*a) : backward<128, false>(*a);
}

}  // extern "C"
