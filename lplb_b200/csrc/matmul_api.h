// Host-side launch interface of the product with an epilogue, and of its gradients.  Plain C++, as ops_api.h.  The reference has
// no operators of this kind.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "ops_api.h"

namespace lplb {
namespace ops {

enum Activation : int { kNoActivation = 0, kRelu = 1, kGelu = 2, kSilu = 3, kSwiglu = 4 };
constexpr int kMatmulMaxGroups = 1024;
constexpr int kGateBlock = 128;  // kSwiglu: gate columns in front of their up columns

// z = a @ b^T + bias,   out = act(z) + residual.  With `rows`, matrix e of b (and row e of the bias) belongs to rows[e] rows of a,
// which follow those of matrix e - 1; rows of a behind the last group have no product: their out is the residual, or zero.
struct Matmul {
  const void* a;         // [m, k] bf16 or f16, row stride a_ld
  const void* b;         // [groups, n, k] of a's type
  const int* rows;       // [groups] on the device, or null: one matrix, all rows
  const void* bias;      // [groups, n] of bias_type, or null
  const void* residual;  // [m, cols] of out_type, row stride residual_ld, or null
  void* out;             // [m, cols] of out_type, row stride out_ld; cols is n, with kSwiglu n / 2
  float* pre;            // [m, n], row stride pre_ld: z, or null
  int64_t m, n, k, a_ld, residual_ld, out_ld, pre_ld;
  int groups;
  Activation activation;
  Type type, out_type, bias_type;
};
cudaError_t launch_matmul(const Matmul& p, int device, cudaStream_t stream);

// dz of float16 operands, whose type has no more than five bits of an exponent, is stored in parts of a power of two: of a row for da, of a
// column (and group) for db, so that its largest finite magnitude there is at least 2^14 and below 2^15.  `most` is that magnitude
// before, as a float's bits; 0 has the factor of the smallest.  Null: dz as it is.

// da = dz @ b: [m, k] of the type, row stride da_ld; rows behind the last group are zero
struct MatmulInput {
  const void* dz;  // [m, n], row stride dz_ld
  const uint32_t* most;  // [m], or null
  const void* b;   // [groups, n, k]
  const int* rows;
  void* da;
  int64_t m, n, k, dz_ld, da_ld;
  int groups;
  Type type;
};
cudaError_t launch_matmul_input(const MatmulInput& p, int device, cudaStream_t stream);

// db[e] = dz_e^T @ a_e over the rows of group e: [groups, n, k] of the type; there is a row at least
struct MatmulWeight {
  const void* dz;  // [m, n], row stride dz_ld
  const uint32_t* most;  // [groups, n], or null
  const void* a;   // [m, k], row stride a_ld
  const int* rows;
  void* db;
  void* copies;    // with rows: matmul_weight_copies() bytes on a 16-byte boundary, of this call alone
  int64_t m, n, k, dz_ld, a_ld;
  int groups;
  Type type;
};
int64_t matmul_weight_copies(const MatmulWeight& p);
cudaError_t launch_matmul_weight(const MatmulWeight& p, int device, cudaStream_t stream);

// dz = dout * act'(pre), and the bias's gradient, the sum of dz over the rows of a group
struct MatmulPre {
  const void* dout;  // [m, cols] of out_type, row stride dout_ld
  const float* pre;  // [m, n], row stride pre_ld; null without an activation
  const int* rows;
  void* dz;          // [m, n] of `type`, row stride dz_ld, or null: not wanted
  void* dz_weight;   // with `column_most`: dz by columns for db, as dz
  uint32_t* row_most;     // [m], taken and used here, or null: dz is not stored in parts
  uint32_t* column_most;  // [groups, n], the same
  void* dbias;       // [groups, n] of bias_type, or null
  float* parts;      // matmul_pre_parts(): sums of a part of a group's rows
  int64_t m, n, dout_ld, pre_ld, dz_ld;
  int groups;
  Activation activation;
  Type type, out_type, bias_type;
};
// Floats that `parts` needs, and the number of parts that a group's rows are summed in.
cudaError_t matmul_pre_parts(const MatmulPre& p, int device, int64_t* floats, int* splits);
cudaError_t launch_matmul_pre(const MatmulPre& p, int device, cudaStream_t stream);

}  // namespace ops
}  // namespace lplb
