// Launcher of the block-scaled matrix product.
#include "ops_api.h"

#include <atomic>

#include "matmul_fp8.cuh"
#include "moe_gemm.cuh"
#include "tensor_map.h"

namespace lplb {
namespace ops {

namespace {

// Half of an SM's shared memory: the next kernel's CTAs can set themselves up beside these
// (64 rows x 4096 x 7168 10.3 -> 9.8 us; a third of it is too little, 10.8 us).
constexpr uint32_t kRingBytes = 96 * 1024;
constexpr int kFewSmem = 512 * kSmemPerColumn;  // at most

cudaError_t rows_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld};
  const cuuint32_t box[2] = {(cuuint32_t)kKBytes, box_rows};
  return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, 2, dims, strides, box) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename Kernel>
cudaLaunchConfig_t cluster_config(cudaLaunchAttribute (&attrs)[2], int ctas, int split, uint32_t smem, cudaStream_t stream, Kernel) {
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = split;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(kFewThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attrs;
  config.numAttrs = 2;
  return config;
}

// Clusters of `split` CTAs that the device holds at once, one CTA per SM (GPCs of odd sizes leave SMs over).
template <typename Kernel>
cudaError_t resident_clusters(int device, int split, Kernel kernel, int* clusters) {
  static std::atomic<int> known[kMaxDevices][kMaxSplit + 1];
  if (device < 0 || device >= kMaxDevices) return cudaErrorInvalidDevice;
  *clusters = known[device][split].load(std::memory_order_relaxed);
  if (*clusters > 0) return cudaSuccess;
  cudaLaunchAttribute attrs[2]{};
  cudaLaunchConfig_t config = cluster_config(attrs, split, split, kFewSmem, nullptr, kernel);
  config.numAttrs = 1;
  const cudaError_t err = cudaOccupancyMaxActiveClusters(clusters, kernel, &config);
  if (err == cudaSuccess) known[device][split].store(*clusters, std::memory_order_relaxed);
  return err;
}

template <typename Out>
cudaError_t launch_few(const Product& p, int device, cudaStream_t stream) {
  auto kernel = few_rows_kernel<Out>;
  static std::atomic<bool> prepared[kMaxDevices];
  if (device < 0 || device >= kMaxDevices) return cudaErrorInvalidDevice;
  cudaError_t err = cudaSuccess;
  if (!prepared[device].load(std::memory_order_relaxed)) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
    if (err != cudaSuccess) return err;
    prepared[device].store(true, std::memory_order_relaxed);
  }
  FewArgs a{};
  a.error = p.status;
  if (a.error == nullptr && (err = ops_error_word(device, &a.error)) != cudaSuccess) return err;
  a.budget_ns = wait_budget_ns();
  a.a_scale = p.a_scale;
  a.b_scale = p.b_scale;
  a.out = p.out;
  a.a_scale_ld = p.a_scale_ld;
  a.out_ld = p.out_ld;
  a.m = (int)p.m;
  a.n = (int)p.n;
  a.k_blocks = (int)((p.k + kKBytes - 1) / kKBytes);
  a.scale_words = a.k_blocks % 4 == 0 && a.a_scale_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(a.a_scale) & 3) == 0 &&
                  (reinterpret_cast<uintptr_t>(a.b_scale) & 3) == 0;
  a.tiles = (a.n + kTileRows - 1) / kTileRows;
  // How many CTAs share a tile's k blocks, and in how many parts the rows of A go: the least time by this measure, in units
  // of a k block of 128 weight rows (0.3 us): 6 for a round's beginning, the blocks with their rows, the rows' way out, 4
  // for a join.  176 x 105 x 528 took 10 us on one CTA.
  const int least_groups = (a.m + kFewMaxRows - 1) / kFewMaxRows;
  int split = 1, groups = 1;
  float least = 1e30f;
  for (int s = 1; s <= kMaxSplit && s <= a.k_blocks; ++s) {
    int fit = 0;
    if ((err = resident_clusters(device, s, kernel, &fit)) != cudaSuccess) return err;
    if (fit < 1) continue;
    for (int g = least_groups; g <= (a.m + 15) / 16 && g < least_groups + 16; ++g) {
      const int cols = ((a.m + g - 1) / g + 15) / 16 * 16;
      const int rounds = (a.tiles * ((a.m + cols - 1) / cols) + fit - 1) / fit, blocks = (a.k_blocks + s - 1) / s;
      const float cost = rounds * (blocks * (1.f + cols / 256.f) + 6 + cols / 16.f) + (s > 1 ? 4 : 0);
      if (cost < least) least = cost, split = s, groups = (a.m + cols - 1) / cols, a.cols = cols;
    }
  }
  if (a.cols == 0) return cudaErrorInvalidConfiguration;
  const uint32_t stage = kWeightStage + a.cols * kKBytes;
  a.stages = (int)(kRingBytes / stage);
  if (a.stages > kMaxRingStages) a.stages = kMaxRingStages;
  const int most = (a.k_blocks + split - 1) / split;
  if (a.stages > most) a.stages = most;
  CUtensorMap map_b, map_a;
  if ((err = rows_map(&map_b, p.b, p.n, p.k, p.k, kTileRows)) != cudaSuccess) return err;
  if ((err = rows_map(&map_a, p.a, p.m, p.k, p.a_ld, a.cols)) != cudaSuccess) return err;
  cudaLaunchAttribute attrs[2]{};
  const cudaLaunchConfig_t config = cluster_config(attrs, a.tiles * groups * split, split, FewLayout(a.cols, a.stages).request, stream, kernel);
  return cudaLaunchKernelEx(&config, kernel, map_b, map_a, a);
}

// Many rows, or the rows of many matrices: the grouped GEMM of CTA pairs.
template <int EPI>
cudaError_t launch_many(const Product& p, int device, cudaStream_t stream) {
  auto kernel = moe::grouped_gemm_kernel<EPI, false, true>;
  static std::atomic<bool> prepared[kMaxDevices];
  int n_sm = 0;
  cudaError_t err = multiprocessors(device, &n_sm);
  if (err != cudaSuccess) return err;
  if (!prepared[device].load(std::memory_order_relaxed)) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)moe::kGemmSmemFp8);
    if (err != cudaSuccess) return err;
    prepared[device].store(true, std::memory_order_relaxed);
  }
  moe::GemmArgs a{};
  a.status = p.status;
  if (a.status == nullptr && (err = ops_error_word(device, &a.status)) != cudaSuccess) return err;
  a.rows = p.rows;
  a.n_experts = p.rows ? p.groups : 1;
  a.w_rows = (int)p.n;
  a.w_blocks = (int)((p.n + 127) / 128);
  a.n_tiles_w = (int)((p.n + moe::kBM - 1) / moe::kBM);
  a.k_blocks = (int)((p.k + kKBytes - 1) / kKBytes);
  a.n_ranks = 1;
  a.timeout_ns = wait_budget_ns();
  a.w_scale = p.b_scale;
  a.row_scale = p.a_scale;
  a.row_scale_ld = p.a_scale_ld;
  a.scale_words = a.k_blocks % 4 == 0 && p.a_scale_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(p.a_scale) & 3) == 0 &&
                  (reinterpret_cast<uintptr_t>(p.b_scale) & 3) == 0;
  a.out = p.out;
  a.out_stride = p.out_ld;
  a.n_rows = (int)p.m;
  a.wide_rows = p.n % 8 == 0 && p.out_ld % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  // One group: tiles of equal height, so high that the fewest rounds over the CTA pairs come out (a tile costs its
  // steps and about one more).  Several groups: their rows are only known on the device.
  constexpr int kMostSteps = moe::kBNFp8 / moe::kStepN;
  a.tile_steps = kMostSteps;
  if (!p.rows) {
    const int64_t steps = (p.m + moe::kStepN - 1) / moe::kStepN;
    int64_t least = INT64_MAX;
    for (int s = kMostSteps; s >= 2; --s) {
      const int64_t tiles = (steps + s - 1) / s, high = (steps + tiles - 1) / tiles;
      const int64_t cost = (tiles * a.n_tiles_w + n_sm / 2 - 1) / (n_sm / 2) * (high + 1);
      if (cost < least) least = cost, a.tile_steps = (int)high;
    }
  }
  CUtensorMap map_w;
  moe::RowMaps rows;
  if ((err = rows_map(&map_w, p.b, (uint64_t)a.n_experts * p.n, p.k, p.k, moe::kCtaM)) != cudaSuccess) return err;
  for (int b = 0; b < moe::kRowBoxes; ++b)
    if ((err = rows_map(&rows.box[b], p.a, p.m, p.k, p.a_ld, moe::kBN / 2 >> b)) != cudaSuccess) return err;
  return launch_after(kernel, dim3(n_sm & ~1), dim3(moe::kGemmThreadsFp8), moe::kGemmSmemFp8, stream, map_w, rows, a);
}

cudaError_t launch_rows_many(const Product& p, int device, cudaStream_t stream) {
  return p.out_f32 ? launch_many<moe::kStoreF32>(p, device, stream) : launch_many<moe::kStore>(p, device, stream);
}

}  // namespace

cudaError_t launch_matmul_fp8(const Product& p, int device, cudaStream_t stream) {
  if (p.m < 0 || p.n < 1 || p.k < 1 || p.k % 16 || p.groups < 1 || p.groups > kMaxGroups || p.m > kMaxRows || p.groups * p.n > kMaxRows)
    return cudaErrorInvalidValue;
  if (p.m == 0) return cudaSuccess;
  if (p.rows != nullptr) return launch_rows_many(p, device, stream);
  // More than 256 rows go to the CTA pairs, but for small products, whose tiles of 128 x 256 find an SM each and whose k is
  // short, up to 12 k blocks of a tile per SM.  One CTA per tile starts sooner and splits k; the pairs read less from the
  // L2.  In us, this kernel and the pairs: 400 x 1000 x 4096 (3.5 blocks per SM) 9.0, 11.7; 600 x 4096 x 1024 (5.2) 7.7,
  // 9.9; 2000 x 1000 x 2048 (6.9) 8.1, 10.6; 3916 x 353 x 5568 (14) 22.2, 17.1; 1024 x 2048 x 7168 (24) 28.7, 19.7; 1500 x
  // 4096 x 512 (192 tiles) 12.7, 12.0.
  if (p.m > kFewMaxRows) {
    int n_sm = 0;
    if (cudaError_t err = multiprocessors(device, &n_sm)) return err;
    const int64_t tiles = (p.n + kTileRows - 1) / kTileRows * ((p.m + kFewMaxRows - 1) / kFewMaxRows);
    if (tiles > n_sm || tiles * ((p.k + kKBytes - 1) / kKBytes) > 12 * n_sm) return launch_rows_many(p, device, stream);
  }
  return p.out_f32 ? launch_few<float>(p, device, stream) : launch_few<__nv_bfloat16>(p, device, stream);
}

}  // namespace ops
}  // namespace lplb
