// Rows of many pools copied in one launch: pages of a paged cache (forks take a copy of the page that their prompt ends in, compaction moves whole pages)
// and slots of recurrent state.
//
// What bounds it: memory, every copied byte read and written once; for a fork of one prompt the launch.  Torch takes an indexed read and an indexed
// write per pool, each with index tensors to build.  Here the pairs and the pools' addresses travel as kernel parameters: nothing is
// allocated and nothing is copied to the device, and a captured call keeps its pairs.  us on the device, 28 layers of 8 x 128 keys and values in bf16: 7 parts of pages 4.3, 240 parts
// (16 prompts into 16 each; 17 MB read, 198 written) 46, 249 whole pages 137 = 6.3 TB/s, a plain copy's rate.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include <algorithm>

#include "common.cuh"
#include "host.h"

namespace tk {

namespace cc {
constexpr int POOLS = 128, THREADS = 256, UNROLL = 4;
}

// Offsets count vectors of the launch's width.
template <int PAIRS>
struct CacheCopy {
  char* pool[cc::POOLS];
  uint32_t unit[cc::POOLS];       // vectors of a token (of a whole row where pairs copy whole rows)
  uint32_t row_units;             // tokens of a row
  int src[PAIRS], dst[PAIRS];
  int units[PAIRS];               // tokens to copy
};

template <typename V, int PAIRS>
__global__ void __launch_bounds__(cc::THREADS) cache_copy_kernel(const __grid_constant__ CacheCopy<PAIRS> p) {
  using namespace cc;
  const int pair = blockIdx.x;
  const size_t unit = p.unit[blockIdx.y], row = unit * p.row_units, total = unit * p.units[pair];
  const V* src = reinterpret_cast<const V*>(p.pool[blockIdx.y]) + row * p.src[pair];
  V* dst = reinterpret_cast<V*>(p.pool[blockIdx.y]) + row * p.dst[pair];
  for (size_t i = threadIdx.x; i < total; i += THREADS * UNROLL) {
    V v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * THREADS < total) v[u] = src[i + u * THREADS];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * THREADS < total) dst[i + u * THREADS] = v[u];
  }
}

template <int PAIRS>
static void launch_copies(const std::vector<char*>& base, const std::vector<int64_t>& bytes, int64_t row_units, const std::vector<int64_t>& src, const std::vector<int64_t>& dst,
                          const std::vector<int64_t>& units, int vector, cudaStream_t stream) {
  for (size_t p0 = 0; p0 < base.size(); p0 += cc::POOLS)
    for (size_t i0 = 0; i0 < src.size(); i0 += PAIRS) {
      CacheCopy<PAIRS> p;
      const int pools = static_cast<int>(std::min<size_t>(cc::POOLS, base.size() - p0)), pairs = static_cast<int>(std::min<size_t>(PAIRS, src.size() - i0));
      for (int i = 0; i < pools; ++i) {
        p.pool[i] = base[p0 + i];
        p.unit[i] = static_cast<uint32_t>(bytes[p0 + i] / vector);
      }
      for (int i = 0; i < pairs; ++i) {
        p.src[i] = static_cast<int>(src[i0 + i]);
        p.dst[i] = static_cast<int>(dst[i0 + i]);
        p.units[i] = static_cast<int>(units[i0 + i]);
      }
      p.row_units = static_cast<uint32_t>(row_units);
      const dim3 grid(pairs, pools);
      switch (vector) {
        case 16: cache_copy_kernel<uint4, PAIRS><<<grid, cc::THREADS, 0, stream>>>(p); break;
        case 4: cache_copy_kernel<uint32_t, PAIRS><<<grid, cc::THREADS, 0, stream>>>(p); break;
        default: cache_copy_kernel<uint8_t, PAIRS><<<grid, cc::THREADS, 0, stream>>>(p);
      }
      count_launch();
      TK_CUDA_CHECK(cudaGetLastError());
    }
}

// pools [N, ...] contiguous; row dst[i] of each becomes row src[i], or its first tokens[i] entries along the second dimension.  Rows that are written are
// neither read nor written by another pair: the pairs then have no order.
void cache_copy(const std::vector<torch::Tensor>& pools, const std::vector<int64_t>& src, const std::vector<int64_t>& dst, const std::vector<int64_t>& tokens) {
  TORCH_CHECK(!pools.empty(), "cache_copy: no pools");
  TORCH_CHECK(src.size() == dst.size() && (tokens.empty() || tokens.size() == src.size()), "cache_copy: one destination (and number of tokens) per source");
  const auto& first = pools[0];
  TORCH_CHECK(first.dim() >= 1, "cache_copy: pools [rows, ...]");
  const int64_t rows = first.size(0), row_units = tokens.empty() ? 1 : (first.dim() >= 2 ? first.size(1) : 0);
  TORCH_CHECK(rows < (int64_t(1) << 31) && row_units < (int64_t(1) << 31), "cache_copy: too many rows");
  int vector = 16;
  std::vector<char*> base;
  std::vector<int64_t> bytes;
  for (const auto& t : pools) {
    TORCH_CHECK(t.is_cuda() && t.device() == first.device() && t.is_contiguous() && t.dim() >= 1 && t.size(0) == rows, "cache_copy: contiguous pools of one device and one number of rows");
    TORCH_CHECK(tokens.empty() || (t.dim() >= 2 && t.size(1) == row_units), "cache_copy: pools of one page size");
    const int64_t per = rows * row_units > 0 ? t.numel() / (rows * row_units) * static_cast<int64_t>(t.element_size()) : 0;
    if (per == 0) continue;
    TORCH_CHECK(per < (int64_t(1) << 31), "cache_copy: rows beyond 2 GiB");
    while (vector > 1 && (per % vector != 0 || reinterpret_cast<uintptr_t>(t.data_ptr()) % vector != 0)) vector = vector == 16 ? 4 : 1;
    base.push_back(reinterpret_cast<char*>(t.data_ptr()));
    bytes.push_back(per);
  }
  std::vector<int64_t> s, d, n, read(src), written(dst);
  for (size_t i = 0; i < src.size(); ++i) {
    const int64_t k = tokens.empty() ? 1 : tokens[i];
    TORCH_CHECK(src[i] >= 0 && src[i] < rows && dst[i] >= 0 && dst[i] < rows, "cache_copy: rows ", src[i], " -> ", dst[i], " of ", rows);
    TORCH_CHECK(k >= 0 && k <= row_units, "cache_copy: ", k, " tokens of a row of ", row_units);
    if (k == 0) continue;
    s.push_back(src[i]); d.push_back(dst[i]); n.push_back(k);
  }
  std::sort(read.begin(), read.end());
  std::sort(written.begin(), written.end());
  for (size_t i = 0, j = 0; i < written.size(); ++i) {
    TORCH_CHECK(i == 0 || written[i] != written[i - 1], "cache_copy: row ", written[i], " is written twice");
    while (j < read.size() && read[j] < written[i]) ++j;
    TORCH_CHECK(j == read.size() || read[j] != written[i], "cache_copy: row ", written[i], " is read and written");
  }
  if (base.empty() || s.empty()) return;
  c10::cuda::CUDAGuard guard(first.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  // parameters of a few pairs are 2 KB, of many 26 KB
  if (s.size() <= 64) launch_copies<64>(base, bytes, row_units, s, d, n, vector, stream);
  else launch_copies<2048>(base, bytes, row_units, s, d, n, vector, stream);
}

}  // namespace tk
