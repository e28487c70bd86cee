// Operators whose weights are picked per row of activations: a mixture-of-experts router and the experts of a few tokens, and
// low-rank adapters of many requests.  Parameter blocks are plain data that the C entries (row_ops.hip) have checked.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace tts {

// 16-bit types are told apart by `bf16` where one of them is all there can be
enum ElemKind { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 2, ELEM_I8 = 3, ELEM_I32 = 4 };
enum Activation { ACT_SILU = 0, ACT_GELU_TANH = 1, ACT_RELU = 2 };

constexpr int ROUTE_MAX_EXPERTS = 1024, ROUTE_MAX_TOP = 64;

struct RouteParams {
  const void *logits;   // [tokens, experts]
  const float *bias;    // [experts] or null
  int *ids;             // [tokens, top]
  float *weights;       // [tokens, top]
  int64_t tokens, ld, ld_ids, ld_weights;
  int experts, top;
  int elem;             // of the logits: f32, f16 or bf16
  int sigmoid, renormalize;
  float scale;
};
hipError_t launch_route(const RouteParams &p, hipStream_t s);

constexpr int EXPERTS_MAX_SLOTS = 4096;

// One of the two products: rows of activations against the matrix of their slot's expert.  Element (k, n) of expert e is at
// w + e * w_expert + k * w_k + n * w_n; one of w_k and w_n is 1.
struct ExpertMatrix {
  const void *w;
  const float *scale;   // int8: [experts, outputs], else null
  int64_t w_expert, w_k, w_n, scale_expert;
};

struct ExpertsParams {
  const void *x;        // [tokens, hidden]
  const int *ids;       // [tokens, top]
  const float *weights; // [tokens, top]
  void *out;            // [tokens, outputs]
  ExpertMatrix up, down;
  int64_t ld_x, ld_ids, ld_weights, ld_out;
  int64_t tokens, hidden, inner, outputs;
  int top, experts;
  int bf16, int8, gated, activation;
  void *workspace;
};
size_t experts_workspace_bytes(const ExpertsParams &p);
bool experts_fit_a_grid(const ExpertsParams &p);  // (a launch of 2^32 lanes and more starts only their remainder)
hipError_t launch_experts(const ExpertsParams &p, hipStream_t s);

constexpr int LORA_MAX_RANK = 1024;

struct LoraParams {
  const void *base;     // [tokens, outputs]
  const void *x;        // [tokens, inputs]
  const void *a;        // [adapters, rank, inputs]
  const void *b;        // [adapters, outputs, rank]
  const int *ids;       // [tokens]
  const float *scales;  // [adapters] or null
  void *out;            // [tokens, outputs]
  int64_t ld_base, ld_x, ld_out, stride_ids;
  int64_t a_adapter, a_rank, b_adapter, b_col;
  int64_t tokens, inputs, outputs;
  int rank, adapters, bf16;
  void *workspace;
};
size_t lora_workspace_bytes(const LoraParams &p);
hipError_t launch_lora(const LoraParams &p, hipStream_t s);

}  // namespace tts
