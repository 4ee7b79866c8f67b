// Host-side launch interface of the 8-bit serving operators.  Plain C++ so that the CUDA
// translation units need no torch headers.  The reference has no operators of this kind.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace lplb {
namespace ops {

enum class Type : int { kF32 = 0, kBf16 = 1, kF16 = 2 };

// ---- rows in 8 bits -------------------------------------------------------------------------
constexpr int kMaxRowLength = 16384;

struct RowFp8 {
  const void* x;         // [rows, cols], row stride x_ld elements
  const void* residual;  // the same, or null
  const void* weight;    // [cols] of the type `weight_type`, or null: no norm, only the conversion
  void* sum;             // [rows, cols] of x's type: x + residual; null without a residual
  void* normed;          // [rows, cols] of x's type: the normed rows, or null
  uint8_t* q;            // [rows, cols] e4m3
  uint8_t* scale;        // [rows, ceil(cols / 128)] e8m0
  int64_t x_ld, residual_ld;
  int64_t rows;
  int cols;
  float eps;
  Type type, weight_type;
};
cudaError_t launch_row_fp8(const RowFp8& a, int n_sms, cudaStream_t stream);

// w: [matrices, rows, cols] contiguous -> e4m3, with one scale per 128 x 128:
// [matrices, ceil(rows / 128), ceil(cols / 128)]
cudaError_t launch_weight_fp8(const void* w, Type type, int64_t matrices, int64_t rows, int64_t cols, uint8_t* q, uint8_t* scale,
                              cudaStream_t stream);

// ---- block-scaled product -------------------------------------------------------------------
// out[m, n] = sum over k of a[m, k] * b[n, k], both e4m3, a with a scale per row and 128, b with one per 128 x 128.
// With `rows`, matrix e belongs to rows[e] rows of a, which follow those of matrix e - 1; rows behind the last group are
// neither read nor written.
constexpr int kMaxGroups = 128;
constexpr int kMaxRows = INT32_MAX - 255;  // of a, and of all matrices of b: no tile ends behind 2^31
struct Product {
  const void* a;           // [m, k], row stride a_ld
  const void* b;           // [groups, n, k]
  const uint8_t* a_scale;  // [m, ceil(k / 128)], row stride a_scale_ld
  const uint8_t* b_scale;  // [groups, ceil(n / 128), ceil(k / 128)]
  const int* rows;         // [groups] on the device, or null: one matrix, all rows
  void* out;               // [m, n], row stride out_ld, bf16 or float32
  int* status;             // takes the call's first error; null: the device's word does
  int64_t m, n, k, a_ld, a_scale_ld, out_ld;
  int groups, out_f32;
};
cudaError_t launch_matmul_fp8(const Product& p, int device, cudaStream_t stream);

// ---- MoE layer for a few tokens ---------------------------------------------------------------
constexpr int kMoeFewMaxTokens = 64, kMoeFewMaxTopk = 32, kMoeFewMaxExperts = 512, kMoeFewMaxHidden = 16384, kMoeFewMaxInter = 65536;

// What the first kernel tells the second, in a workspace of the call.  A row is a token's choice of an expert; the
// rows of a slot (an expert that was chosen) follow those of the slot before, in the tokens' order.
struct MoeFewPlan {
  int* slots;         // number of slots
  int* ticket;        // shares taken
  int2* slot;         // [slots] expert, first row << 8 | rows
  uint8_t* token;     // [tokens * topk + 4] the rows' tokens; 0 behind the last row
  int2* pair;         // [tokens * topk] row << 10 | slot, or -1; bits of the weight
  int* ready;         // [slots] finished tiles of `act`
  int* tile_parts;    // [slots * inter / 128] parts summed so far
  int* products;      // products with down made so far, or pieces of them
};
struct MoeFew {
  const void* x;             // [tokens, hidden] bf16 (row stride x_ld) or e4m3 (with x_scale)
  const uint8_t* x_scale;    // [tokens, hidden / 128], row stride x_scale_ld; null: x is bf16
  const void* idx;           // [tokens, topk]
  const float* weight;       // [tokens, topk]
  const void* w13;           // [experts, 2 * inter, hidden] bf16 or e4m3, in blocks of 128 gate and 128 up rows
  const void* w2;            // [experts, hidden, inter]
  const uint8_t* w13_scale;  // null: bf16 weights
  const uint8_t* w2_scale;
  void* out;                 // [tokens, hidden] bf16
  void* workspace;           // moe_few_workspace() bytes, 256-byte aligned
  int* status;               // takes the call's first error; null: the device's word does
  int64_t x_ld, x_scale_ld;
  int idx_is64, tokens, topk, experts, hidden, inter;
};
cudaError_t moe_few_workspace(const MoeFew& m, int device, size_t* bytes);
cudaError_t launch_moe_few(const MoeFew& m, int device, cudaStream_t stream);

// First error that a kernel of these operators has seen on the current device (0: none).  It stays until it is cleared; reading
// waits for the device.
enum OpsErr : int { kOpsTimeout = 21 };  // a wait inside a kernel gave up, its results are not valid
cudaError_t read_ops_error(int* code, bool clear);
// How long a wait inside a kernel lasts at most, of launches from now on (all devices).
constexpr unsigned long long kDefaultWaitBudgetNs = 2000000000ull;
unsigned long long wait_budget_ns();
void set_wait_budget_ns(unsigned long long ns);
// Where the kernels put it.
constexpr int kMaxDevices = 64;
cudaError_t ops_error_word(int device, int** word);
// Multiprocessors of a device, asked for once.
cudaError_t multiprocessors(int device, int* count);

}  // namespace ops
}  // namespace lplb
