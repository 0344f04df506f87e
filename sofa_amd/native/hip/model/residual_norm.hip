// Residual norm and its gradients, one pass over each row.
//
//   h = branch, or norm(branch) post       norm(z) = z / sqrt(mean z^2 + eps)
//   r = x + scale gate h                   y = norm(r) weight
//
// and, with u = dy weight, n = norm(r), s = 1 / sqrt(mean r^2 + eps):
//
//   d  = dr + s (u - n mean(u n))          dx = d          dweight = sum dy n
//   dh = scale gate d                      dgate = sum scale d h
//   dbranch = dh, or through the branch's norm as above; dpost = sum dh norm(branch)
//
// Every value is read and written once; what a row needs twice stays in
// registers.  A row belongs to a team of one wave (short rows) or one
// workgroup, 8 VPT elements a thread, so the statistics take one reduction
// each.  Sums over rows (dweight, dpost, dgate) stay in registers over the
// team's rows, are joined in LDS, go to one partial row per workgroup and are
// added in a fixed order by a second kernel: no atomics, the same bits every
// time.

#include "model_ops.h"

namespace sofa_model {
namespace {

// Sums of N <= 2 values over a team, in every thread of it.  `parity` alternates
// between calls, so that one barrier is enough: a buffer is written again
// only after the barrier of the call between.
template <int TEAM, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float* smem,
                                         int& parity) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = wave_sum(v[k]);
  if constexpr (TEAM > kWave) {
    constexpr int kWaves = TEAM / kWave;
    float* buf = smem + parity * kWaves * 2;
    parity ^= 1;
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) buf[wave * 2 + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += buf[w * 2 + k];
      v[k] = s;
    }
  }
}

template <int TEAM>
constexpr int kBlock = TEAM > 256 ? TEAM : 256;

template <typename X, typename B, typename Y, int TEAM, int VPT>
__global__ __launch_bounds__(kBlock<TEAM>) void norm_forward_kernel(
    NormArgs a) {
  constexpr int kTeams = kBlock<TEAM> / TEAM;
  __shared__ float smem[TEAM > kWave ? 2 * 2 * TEAM / kWave : 1];
  const int lane = threadIdx.x % TEAM;
  const int64_t team = (int64_t) blockIdx.x * kTeams + threadIdx.x / TEAM;
  const int64_t teams = (int64_t) gridDim.x * kTeams;
  const float inv_dim = 1.f / (float) a.dim;
  int parity = 0;

  float weight[VPT][8], post[VPT][8];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int at = (v * TEAM + lane) * 8;
    load8_any(a.weight, a.weight_type, at, weight[v], a.dim - at);
    if (a.post) load8_any(a.post, a.post_type, at, post[v], a.dim - at);
  }

  for (int64_t row = team; row < a.rows; row += teams) {
    const X* x = static_cast<const X*>(a.x) + row * a.dim;
    float r[VPT][8];
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int at = (v * TEAM + lane) * 8;
      load8(x + at, r[v], a.dim - at);
    }
    if (a.branch) {
      const B* branch = static_cast<const B*>(a.branch) + row * a.dim;
      float h[VPT][8];
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int at = (v * TEAM + lane) * 8;
        load8(branch + at, h[v], a.dim - at);
      }
      if (a.post) {
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[0] += h[v][j] * h[v][j];
        team_sum<TEAM>(sum, smem, parity);
        const float s = rsqrtf(sum[0] * inv_dim + a.eps);
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
          for (int j = 0; j < 8; ++j) h[v][j] *= s * post[v][j];
        sum[0] = 0.f;
      }
      const int64_t gate_row = a.gate ? row / a.group_rows * a.dim : 0;
      X* out = static_cast<X*>(a.r) + row * a.dim;
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int at = (v * TEAM + lane) * 8;
        if (a.gate) {
          float gate[8];
          load8_any(a.gate, a.gate_type, gate_row + at, gate, a.dim - at);
#pragma unroll
          for (int j = 0; j < 8; ++j) h[v][j] *= gate[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) r[v][j] += a.scale * h[v][j];
        store8(out + at, r[v], a.dim - at);
      }
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[0] += r[v][j] * r[v][j];
    team_sum<TEAM>(sum, smem, parity);
    const float s = rsqrtf(sum[0] * inv_dim + a.eps);
    Y* y = static_cast<Y*>(a.y) + row * a.dim;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int at = (v * TEAM + lane) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) r[v][j] *= s * weight[v][j];
      store8(y + at, r[v], a.dim - at);
    }
  }
}

// A workgroup takes consecutive rows of one gate's group, so that the gate and
// its gradient stay in registers too; its teams take them in turn.
// EXTRA: the branch has a norm or a gate; without them their registers
// (5 of 8 vectors) are not held.  x is r where that is held in 32 bits (or there
// is no branch); a 16-bit r has lost what the gradients of the weights need,
// so x is x then and r is summed up again.
template <typename X, typename B, typename Y, int TEAM, int VPT, bool EXTRA>
__global__ __launch_bounds__(kBlock<TEAM>) void norm_backward_kernel(
    NormArgs a) {
  constexpr int kTeams = kBlock<TEAM> / TEAM;
  __shared__ float smem[TEAM > kWave ? 2 * 2 * TEAM / kWave : 1];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const int64_t group = blockIdx.x / a.group_blocks;
  const int64_t part = blockIdx.x % a.group_blocks;
  const int64_t first =
      group * a.group_rows + a.group_rows * part / a.group_blocks;
  const int64_t last =
      group * a.group_rows + a.group_rows * (part + 1) / a.group_blocks;
  const float inv_dim = 1.f / (float) a.dim;
  int parity = 0;

  float weight[VPT][8], post[VPT][8], gate[VPT][8];
  float dweight[VPT][8] = {}, dpost[VPT][8] = {}, dgate[VPT][8] = {};
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int at = (v * TEAM + lane) * 8;
    load8_any(a.weight, a.weight_type, at, weight[v], a.dim - at);
    if constexpr (EXTRA) {
      if (a.post)
        load8_any(a.post, a.post_type, at, post[v], a.dim - at);
      if (a.gate)
        load8_any(a.gate, a.gate_type, group * a.dim + at, gate[v], a.dim - at);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!a.post) post[v][j] = 1.f;
        gate[v][j] = a.gate ? gate[v][j] * a.scale : a.scale;
      }
    }
  }

  for (int64_t row = first + team; row < last; row += kTeams) {
    const X* x = static_cast<const X*>(a.x) + row * a.dim;
    const Y* dy = static_cast<const Y*>(a.dy) + row * a.dim;
    const X* dr = static_cast<const X*>(a.dr) + row * a.dim;
    const B* branch = static_cast<const B*>(a.branch) + row * a.dim;
    X* dx = static_cast<X*>(a.dx) + row * a.dim;
    B* dbranch = static_cast<B*>(a.dbranch) + row * a.dim;
    float d[VPT][8], z[VPT][8], h[VPT][8], in[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int at = (v * TEAM + lane) * 8;
      load8(x + at, z[v], a.dim - at);
      load8(dy + at, d[v], a.dy ? a.dim - at : 0);
      load8(dr + at, in[v], a.dr ? a.dim - at : 0);
      if constexpr (EXTRA) load8(branch + at, h[v], a.dim - at);
    }
    // without a norm of the branch: its unit is h, and no mean to take off
    float sh = 1.f, ch = 0.f;
    if constexpr (EXTRA) {
      if (a.post) {
        float sums[1] = {0.f};
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
          for (int j = 0; j < 8; ++j) sums[0] += h[v][j] * h[v][j];
        team_sum<TEAM>(sums, smem, parity);
        sh = rsqrtf(sums[0] * inv_dim + a.eps);
      }
    }
    if constexpr (sizeof(X) == 2) {
      if (a.branch) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
          const int at = (v * TEAM + lane) * 8;
          if constexpr (EXTRA) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              z[v][j] += gate[v][j] * (sh * post[v][j]) * h[v][j];
          } else {
            float hs[8];
            load8(branch + at, hs, a.dim - at);
#pragma unroll
            for (int j = 0; j < 8; ++j) z[v][j] += a.scale * hs[j];
          }
        }
      }
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[0] += z[v][j] * z[v][j];
        sum[1] += d[v][j] * weight[v][j] * z[v][j];
      }
    team_sum<TEAM>(sum, smem, parity);
    const float s = rsqrtf(sum[0] * inv_dim + a.eps);
    // in this order: s^3 leaves 32 bits for rows of 1e13 and more, or 1e-13
    const float c = s * sum[1] * inv_dim * s * s;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int at = (v * TEAM + lane) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dweight[v][j] += d[v][j] * z[v][j] * s;
        d[v][j] = in[v][j] + (s * weight[v][j] * d[v][j] - c * z[v][j]);
      }
      store8(dx + at, d[v], a.dim - at);
    }
    if constexpr (!EXTRA) {
      if (!a.dbranch) continue;
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int at = (v * TEAM + lane) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) d[v][j] *= a.scale;
        store8(dbranch + at, d[v], a.dim - at);
      }
    } else {
      if (a.post) {
        float sums[1] = {0.f};
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            sums[0] += d[v][j] * gate[v][j] * post[v][j] * h[v][j];
        team_sum<TEAM>(sums, smem, parity);
        ch = sh * sums[0] * inv_dim * sh * sh;
      }
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int at = (v * TEAM + lane) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float unit = h[v][j] * sh, dh = d[v][j] * gate[v][j];
          dpost[v][j] += dh * unit;
          dgate[v][j] += d[v][j] * unit * post[v][j];
          d[v][j] = sh * post[v][j] * dh - ch * h[v][j];
        }
        if (a.dbranch) store8(dbranch + at, d[v], a.dim - at);
      }
    }
  }

  // the workgroup's sums: its teams' in order
  float* out = a.partial + (int64_t) blockIdx.x * a.dim;
  const int64_t sum_size = (int64_t) gridDim.x * a.dim;
  auto put = [&](float (&sums)[VPT][8]) {
    if constexpr (kTeams > 1) {
      __shared__ float joined[kTeams > 1 ? (kTeams - 1) * VPT * 8 * TEAM : 1];
      __syncthreads();
      if (team) {
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            joined[(((team - 1) * VPT + v) * 8 + j) * TEAM + lane] = sums[v][j];
      }
      __syncthreads();
      if (team == 0) {
#pragma unroll
        for (int t = 0; t < kTeams - 1; ++t)
#pragma unroll
          for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              sums[v][j] += joined[((t * VPT + v) * 8 + j) * TEAM + lane];
      }
    }
    if (team == 0) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int at = (v * TEAM + lane) * 8;
        store8(out + at, sums[v], a.dim - at);
      }
    }
    out += sum_size;
  };
  if (a.dweight) put(dweight);
  if constexpr (EXTRA) {
    if (a.dpost) put(dpost);
    if (a.dgate) {
#pragma unroll
      for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) dgate[v][j] *= a.scale;
      put(dgate);
    }
  }
}

// Adds the partial rows: dweight and dpost over all workgroups, dgate over
// those of its group.  blockIdx.x counts the output rows in that order.
constexpr int kSumColumns = 32, kSumRows = 32;

__global__ __launch_bounds__(kSumColumns* kSumRows) void norm_sum_kernel(
    NormArgs a) {
  __shared__ float smem[kSumRows][kSumColumns + 1];
  const int column = threadIdx.x % kSumColumns, line = threadIdx.x / kSumColumns;
  const int at = blockIdx.y * kSumColumns + column;
  const int64_t rows = a.rows / a.group_rows * a.group_blocks;
  const float* in = a.partial;
  int64_t which = blockIdx.x, first = 0, count = rows;
  void* out = nullptr;
  int type = kFloat32;
  if (a.dweight && which-- == 0) {
    out = a.dweight;
    type = a.weight_type;
  }
  if (!out && a.dweight) in += rows * a.dim;
  if (!out && a.dpost && which-- == 0) {
    out = a.dpost;
    type = a.post_type;
  }
  if (!out && a.dpost) in += rows * a.dim;
  int64_t row = 0;
  if (!out) {  // `which` is the gate's row now
    out = a.dgate;
    type = a.gate_type;
    row = which;
    first = which * a.group_blocks;
    count = a.group_blocks;
  }
  float s = 0.f;
  if (at < a.dim)
    for (int64_t t = line; t < count; t += kSumRows)
      s += in[(first + t) * a.dim + at];
  smem[line][column] = s;
  __syncthreads();
  if (line == 0 && at < a.dim) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < kSumRows; ++k) total += smem[k][column];
    store_any(out, type, row * a.dim + at, total);
  }
}

// Calls f.template operator()<X, B, Y, TEAM, VPT>() for the types and the row
// length: a wave up to 1024 elements, since a reduction within it needs no
// barrier, then as many threads as hold the row at 8 elements each.
template <typename X, typename B, typename Y, typename F>
int by_dim(int dim, F f) {
  if (dim <= 512) return f.template operator()<X, B, Y, 64, 1>();
  if (dim <= 1024) return f.template operator()<X, B, Y, 64, 2>();
  if (dim <= 2048) return f.template operator()<X, B, Y, 256, 1>();
  if (dim <= 4096) return f.template operator()<X, B, Y, 512, 1>();
  if (dim <= 8192) return f.template operator()<X, B, Y, 1024, 1>();
  if (dim <= 16384) return f.template operator()<X, B, Y, 1024, 2>();
  return kBadArgument;
}

template <typename F>
int by_types(const NormArgs& a, F f) {
  const int key = a.x_type * 100 + a.branch_type * 10 + a.y_type;
  switch (key) {
    case kFloat32 * 100 + kFloat32 * 10 + kFloat32:
      return by_dim<float, float, float>(a.dim, f);
    case kFloat32 * 100 + kBFloat16 * 10 + kFloat32:
      return by_dim<float, bf16, float>(a.dim, f);
    case kFloat32 * 100 + kBFloat16 * 10 + kBFloat16:
      return by_dim<float, bf16, bf16>(a.dim, f);
    case kFloat32 * 100 + kFloat16 * 10 + kFloat32:
      return by_dim<float, fp16, float>(a.dim, f);
    case kFloat32 * 100 + kFloat16 * 10 + kFloat16:
      return by_dim<float, fp16, fp16>(a.dim, f);
    case kBFloat16 * 100 + kBFloat16 * 10 + kBFloat16:
      return by_dim<bf16, bf16, bf16>(a.dim, f);
    case kFloat16 * 100 + kFloat16 * 10 + kFloat16:
      return by_dim<fp16, fp16, fp16>(a.dim, f);
  }
  return kBadArgument;
}

constexpr int kCus = 256;

struct Forward {
  const NormArgs& a;
  template <typename X, typename B, typename Y, int TEAM, int VPT>
  int operator()() const {
    constexpr int kTeams = kBlock<TEAM> / TEAM;
    int64_t blocks = (a.rows + kTeams - 1) / kTeams;
    if (blocks > kCus * 8) blocks = kCus * 8;
    hipLaunchKernelGGL((norm_forward_kernel<X, B, Y, TEAM, VPT>),
                       dim3((unsigned) blocks), dim3(kBlock<TEAM>), 0,
                       static_cast<hipStream_t>(a.stream), a);
    return (int) hipGetLastError();
  }
};

struct Backward {
  const NormArgs& a;
  template <typename X, typename B, typename Y, int TEAM, int VPT>
  int operator()() const {
    const int64_t blocks = a.rows / a.group_rows * a.group_blocks;
    const dim3 grid((unsigned) blocks), block(kBlock<TEAM>);
    const hipStream_t stream = static_cast<hipStream_t>(a.stream);
    if (a.post || a.gate)
      hipLaunchKernelGGL((norm_backward_kernel<X, B, Y, TEAM, VPT, true>), grid,
                         block, 0, stream, a);
    else
      hipLaunchKernelGGL((norm_backward_kernel<X, B, Y, TEAM, VPT, false>),
                         grid, block, 0, stream, a);
    return (int) hipGetLastError();
  }
};

bool sound(const NormArgs* a) {
  return a && a->rows > 0 && a->rows <= INT32_MAX && a->dim > 0 &&
         a->dim <= kMaxNormDim &&
         a->group_rows > 0 && a->rows % a->group_rows == 0 && a->x &&
         a->weight && (a->branch || !(a->post || a->gate));
}

}  // namespace
}  // namespace sofa_model

extern "C" {

int sofa_norm_forward(const sofa_model::NormArgs* a) {
  using namespace sofa_model;
  if (!sound(a) || !a->y || (a->branch && !a->r)) return kBadArgument;
  DeviceGuard guard(a->device);
  if (guard.status()) return guard.status();
  return by_types(*a, Forward{*a});
}

int sofa_norm_backward(const sofa_model::NormArgs* a) {
  using namespace sofa_model;
  if (!sound(a) || !a->dx || !(a->dr || a->dy) || a->group_blocks < 1 ||
      a->rows / a->group_rows > kMaxGates ||
      a->rows / a->group_rows * a->group_blocks > kMaxBlocks / 4)
    return kBadArgument;
  if ((a->dweight || a->dpost || a->dgate) && !a->partial) return kBadArgument;
  if ((a->dpost && !a->post) || (a->dgate && !a->gate)) return kBadArgument;
  DeviceGuard guard(a->device);
  if (guard.status()) return guard.status();
  int status = by_types(*a, Backward{*a});
  if (status) return status;
  const int64_t outputs = (a->dweight ? 1 : 0) + (a->dpost ? 1 : 0) +
                          (a->dgate ? a->rows / a->group_rows : 0);
  if (outputs == 0) return 0;
  hipLaunchKernelGGL(norm_sum_kernel,
                     dim3((unsigned) outputs,
                          (a->dim + kSumColumns - 1) / kSumColumns),
                     dim3(kSumColumns * kSumRows), 0,
                     static_cast<hipStream_t>(a->stream), *a);
  return (int) hipGetLastError();
}

}  // extern "C"
