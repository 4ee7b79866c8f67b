// The error word of the 8-bit serving operators, one per device.
#include <atomic>

#include "ops_api.h"

namespace lplb {
namespace ops {

// Part of the module, so that it is there (and zero) without an allocation, inside a stream capture too.
static __device__ int g_ops_error = 0;

cudaError_t ops_error_word(int device, int** word) {
  static std::atomic<int*> known[kMaxDevices];
  if (device < 0 || device >= kMaxDevices) return cudaErrorInvalidDevice;
  *word = known[device].load(std::memory_order_relaxed);
  if (*word != nullptr) return cudaSuccess;
  void* p = nullptr;
  const cudaError_t err = cudaGetSymbolAddress(&p, g_ops_error);
  if (err != cudaSuccess) return err;
  *word = static_cast<int*>(p);
  known[device].store(*word, std::memory_order_relaxed);
  return cudaSuccess;
}

cudaError_t multiprocessors(int device, int* count) {
  static std::atomic<int> known[kMaxDevices];
  if (device < 0 || device >= kMaxDevices) return cudaErrorInvalidDevice;
  *count = known[device].load(std::memory_order_relaxed);
  if (*count) return cudaSuccess;
  cudaError_t err = cudaDeviceGetAttribute(count, cudaDevAttrMultiProcessorCount, device);
  if (err == cudaSuccess) known[device].store(*count, std::memory_order_relaxed);
  return err;
}

static std::atomic<unsigned long long> g_wait_budget_ns{kDefaultWaitBudgetNs};
unsigned long long wait_budget_ns() { return g_wait_budget_ns.load(std::memory_order_relaxed); }
void set_wait_budget_ns(unsigned long long ns) { g_wait_budget_ns.store(ns, std::memory_order_relaxed); }

cudaError_t read_ops_error(int* code, bool clear) {
  cudaError_t err = cudaDeviceSynchronize();
  if (err == cudaSuccess) err = cudaMemcpyFromSymbol(code, g_ops_error, sizeof(int));
  const int zero = 0;
  if (err == cudaSuccess && clear) err = cudaMemcpyToSymbol(g_ops_error, &zero, sizeof(int));
  return err;
}

}  // namespace ops
}  // namespace lplb
