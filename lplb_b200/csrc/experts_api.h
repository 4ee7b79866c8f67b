// Host-side launch interface of the operators around a layer's experts in 16 and 32 bits: the router's choice, rows sorted
// by expert and back.  Plain C++, as ops_api.h.  The reference has no operators of this kind.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "ops_api.h"

namespace lplb {
namespace ops {

// ---- the router's choice ------------------------------------------------------------------------
constexpr int kGateMaxExperts = 1024, kGateMaxTopk = 32;
struct Gate {
  const void* logits;     // [tokens, experts], row stride ld
  float* weights;         // [tokens, topk]
  int64_t* idx;           // [tokens, topk]; -1 where fewer than topk experts can be chosen
  const float* dweights;  // backward: [tokens, topk]
  void* dlogits;          // backward: [tokens, experts] of the logits' type
  int64_t ld, tokens;
  int experts, topk, sigmoid, renormalize;
  float scale;
  Type type;
};
cudaError_t launch_gate(const Gate& g, cudaStream_t stream);
cudaError_t launch_gate_backward(const Gate& g, cudaStream_t stream);

// ---- rows sorted by expert ----------------------------------------------------------------------
constexpr int kOrderMaxExperts = 1024, kOrderMaxTopk = 1024;
struct Order {
  const void* idx;  // [pairs] int64 or int32; outside [0, experts): no expert
  int* counts;      // [experts]
  int* place;       // [pairs] the pair's row, or -1
  int* source;      // [pairs] the row's pair, or -1 behind the last
  int64_t pairs;
  int experts, is64;
};
cudaError_t launch_order(const Order& o, int device, cudaStream_t stream);

// rows[place[t, k]] = x[t]; rows without a pair are zero.  Rows are bytes here.
struct TakeRows {
  const void* x;       // [tokens, row_bytes], row stride ld_bytes
  const int* place;    // [tokens, topk]
  const int* source;   // [tokens * topk]
  void* rows;          // [tokens * topk, row_bytes]
  int64_t ld_bytes, row_bytes, tokens;
  int topk;
};
cudaError_t launch_take_rows(const TakeRows& t, int n_sms, cudaStream_t stream);

// out[t] = sum over k of weights[t, k] * rows[place[t, k]] (weights null: ones), in 32 bits, in the order of k
struct CombineRows {
  const void* rows;      // [tokens * topk, cols], row stride ld
  const int* place;      // [tokens, topk]
  const int* source;     // backward: [tokens * topk]
  const float* weights;  // [tokens, topk], or null
  void* out;             // [tokens, cols] of the rows' type
  const void* dout;      // backward: [tokens, cols], row stride dout_ld
  void* drows;           // backward: [tokens * topk, cols], or null
  float* dweights;       // backward: [tokens, topk], or null
  int64_t ld, dout_ld, tokens;
  int cols, topk;
  Type type;
};
cudaError_t launch_combine_rows(const CombineRows& c, int n_sms, cudaStream_t stream);
cudaError_t launch_combine_rows_backward(const CombineRows& c, int n_sms, cudaStream_t stream);

}  // namespace ops
}  // namespace lplb
