// What the model kernels' C entries take: the one description of it for the
// kernels and for their callers. Strides and sizes are in elements, pointers are
// to device memory, and an entry only launches: nothing it is given is kept, and
// nothing is allocated. An entry returns 0, a hipError_t, or kBadArgument.

#pragma once

#include <cstdint>

namespace sofa_model {

#ifdef __HIPCC__
using bf16 = __bf16;
#else
struct bf16;  // the host only passes them on
#endif

// element type codes
enum Type : int { kFloat32 = 0, kBFloat16 = 1, kFloat16 = 2 };

constexpr int kBadArgument = -1;

constexpr int kMaxBlocks = (1 << 24) - 1;  // of 256 threads, in one dimension
constexpr int kMaxHeadDim = 128;
constexpr int kMaxTokens = 1 << 24;
constexpr int64_t kMaxTokenStride = 1 << 24;
constexpr int kMaxKeyParts = 8;
constexpr int kMaxTop = 32;
constexpr int kMaxVocab = 1 << 30;
constexpr int kMaxVocabParts = 64;
constexpr int kMaxNormDim = 16384;
constexpr int kMaxGates = 1 << 21;

struct AttentionArgs {
  const bf16 *q, *k, *v;  // [batch][heads][tokens][dim] by strides, dim dense
  bf16* o;
  bf16* o_low;            // what rounding took off o, laid out like it; or null
  float* lse;             // [batch][heads][tokens], over scale; +inf: no keys
  const int* lengths;     // [batch] valid tokens, or null
  const bf16* dout;
  float* delta;           // [batch][heads][tokens]
  bf16 *dq, *dk, *dv;
  float* partial;         // [key_parts][2][batch][kv_heads][tokens][dim], or null
  void* stream;
  int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3];  // batch, head,
  int64_t dout_stride[3], dq_stride[3], dk_stride[3], dv_stride[3];  // token
  float scale;
  int batch, heads, kv_heads, tokens, dim, causal, key_parts, device;
};

struct LogprobArgs {
  const void* logits;
  const int64_t* tokens;
  float *logprob, *entropy;
  float* norm;         // [rows][2]: the largest logit, log of the sum relative to it
  int64_t* top_ids;    // [rows][top], or null
  float* top_logprobs;
  // when parts > 1: (m, s, a) and the top candidates of each part of a row
  float* part_sums;    // [rows][parts][3]
  uint64_t* part_top;  // [rows][parts][top]
  const float *dlogprob, *dentropy;  // either may be null
  void* dlogits;                     // [rows][vocab]
  void* stream;
  int64_t rows, inner;        // row i is at (i / inner) outer_stride
  int64_t outer_stride, inner_stride;  //  + (i % inner) inner_stride elements
  int64_t grad_outer_stride, grad_inner_stride;    // of dlogprob
  int64_t grad2_outer_stride, grad2_inner_stride;  // of dentropy
  int64_t token_outer_stride, token_inner_stride;
  int64_t ignore_index;
  int vocab, top, parts, part_size;  // part_size: a multiple of kStep
  int type, device;
};

struct NormArgs {
  const void *x, *branch, *weight, *post, *gate;  // branch, post, gate: or null
  void *r, *y;                                    // r: null without a branch
  const void *dr, *dy;                            // either may be null
  void *dx, *dbranch;                             // dbranch: or null
  float* partial;  // [sums][workgroups][dim]: dweight, then dpost, then dgate
  void *dweight, *dpost, *dgate;                  // each or null
  void* stream;
  int64_t rows, group_rows;  // rows, and rows that share one gate
  float eps, scale;
  int dim, x_type, branch_type, y_type, weight_type, post_type, gate_type;
  int group_blocks;          // backward: workgroups that share a gate's rows
  int device;
};

}  // namespace sofa_model

extern "C" {
int sofa_attention_forward(const sofa_model::AttentionArgs* a);
int sofa_attention_backward(const sofa_model::AttentionArgs* a);
int sofa_logprob_forward(const sofa_model::LogprobArgs* a);
int sofa_logprob_backward(const sofa_model::LogprobArgs* a);
int sofa_norm_forward(const sofa_model::NormArgs* a);
int sofa_norm_backward(const sofa_model::NormArgs* a);
}
