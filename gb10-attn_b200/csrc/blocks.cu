// blocks.cu -- page operations of the KV pool: copies of pages for every
// layer in one launch (pa_copy_blocks) and the rewrite of block tables after
// pages have moved (pa_remap_block_tables).  A fork copies the part-filled last
// page of the parent for each child; a compaction moves the pages at the top
// of a pool into free ones below.
#include <algorithm>

#include "common.cuh"

namespace pa {
namespace blocks {

constexpr int kMaxLayers = 64;  // layers per launch; more are split on the host
constexpr int kThreads = 256;
constexpr int kUnroll = 4;      // accesses in flight per thread

struct Params {
  char* k_layers[kMaxLayers];
  char* v_layers[kMaxLayers];
  const int32_t* src;
  const int32_t* dst;
  const int32_t* rows;  // null: whole pages
  int64_t n;            // pairs
  int64_t row_bytes, page_bytes, BS, NB;
  int64_t tensors;      // 2 x layers
  int64_t chunks;       // work units per page
  int32_t* dev_status;
};

// One work unit = kThreads x kUnroll accesses of V bytes of one (pair,
// tensor): a page of one layer's K or V is contiguous, so its first `rows`
// token rows are too.  HBM-bound, a read and a write of the bytes: a compaction
// that moves 694 MB takes 112 us (6.2 TB/s, 95 % of a copy's rate), the part-filled
// last pages of 250 forks (157 MB) 24.5 us (98 %), those of seven 3.1 us (latency).
template <typename V>
__global__ void __launch_bounds__(kThreads) copy_blocks_kernel(const __grid_constant__ Params p) {
  constexpr int64_t kUnit = (int64_t)kThreads * kUnroll * sizeof(V);
  const int64_t units = p.n * p.tensors * p.chunks;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t c = u % p.chunks;
    const int64_t pt = u / p.chunks;
    const int64_t i = pt % p.n;
    const int64_t t = pt / p.n;
    const int64_t from = p.src[i], to = p.dst[i];
    if (from < 0 || from >= p.NB || to < 0 || to >= p.NB) {
      if (threadIdx.x == 0) report(p.dev_status, PA_DEVERR_BLOCK_ID);
      continue;
    }
    if (from == to) continue;
    int64_t bytes = p.page_bytes;
    if (p.rows) bytes = min(max((int64_t)p.rows[i], (int64_t)0), p.BS) * p.row_bytes;
    char* pool = (t & 1) ? p.v_layers[t >> 1] : p.k_layers[t >> 1];
    const char* a = pool + from * p.page_bytes + c * kUnit;
    char* b = pool + to * p.page_bytes + c * kUnit;
    const int64_t left = bytes - c * kUnit;
    V x[kUnroll];
#pragma unroll
    for (int e = 0; e < kUnroll; ++e) {
      const int64_t o = (int64_t)(e * kThreads + threadIdx.x) * sizeof(V);
      if (o < left) x[e] = *reinterpret_cast<const V*>(a + o);
    }
#pragma unroll
    for (int e = 0; e < kUnroll; ++e) {
      const int64_t o = (int64_t)(e * kThreads + threadIdx.x) * sizeof(V);
      if (o < left) *reinterpret_cast<V*>(b + o) = x[e];
    }
  }
}

__global__ void __launch_bounds__(kThreads) remap_kernel(int32_t* out, const int32_t* tables,
                                                         const int32_t* map, int64_t n, int64_t NB) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const int32_t b = tables[i];
    out[i] = b >= 0 && b < NB ? map[b] : b;
  }
}

template <typename V>
static int launch(Params& p, int sms, cudaStream_t s) {
  constexpr int64_t kUnit = (int64_t)kThreads * kUnroll * sizeof(V);
  p.chunks = (p.page_bytes + kUnit - 1) / kUnit;
  const int64_t units = p.n * p.tensors * p.chunks;
  copy_blocks_kernel<V><<<(unsigned)std::min<int64_t>(units, (int64_t)sms * 16), kThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError());
}

}  // namespace blocks
}  // namespace pa

extern "C" int pa_copy_blocks(void* const* k_layers, void* const* v_layers, int pool_dtype,
                              const int32_t* src_blocks, const int32_t* dst_blocks,
                              const int32_t* num_rows, int64_t num_pairs, int64_t num_layers,
                              int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                              int64_t num_blocks, int32_t* dev_status, void* stream) {
  using namespace pa;
  using blocks::kMaxLayers;
  if (num_pairs < 0 || num_layers < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      num_blocks < 0)
    return PA_ERR_INVALID_ARGUMENT;
  const int es = dtype_size(pool_dtype);
  if (es == 0) return PA_ERR_DTYPE;
  if (num_pairs == 0 || num_layers == 0) return PA_OK;
  if (!k_layers || !v_layers || !src_blocks || !dst_blocks) return PA_ERR_INVALID_ARGUMENT;
  for (int64_t l = 0; l < num_layers; ++l)
    if (!k_layers[l] || !v_layers[l]) return PA_ERR_INVALID_ARGUMENT;
  int sms = 0;
  if (device_sm_count(&sms) != PA_OK) return PA_ERR_NO_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  for (int64_t l0 = 0; l0 < num_layers; l0 += kMaxLayers) {
    const int64_t nl = std::min<int64_t>(kMaxLayers, num_layers - l0);
    blocks::Params p = {};
    p.src = src_blocks;
    p.dst = dst_blocks;
    p.rows = num_rows;
    p.n = num_pairs;
    p.row_bytes = num_kv_heads * head_dim * es;
    p.page_bytes = block_size * p.row_bytes;
    p.BS = block_size;
    p.NB = num_blocks;
    p.tensors = 2 * nl;
    p.dev_status = dev_status;
    bool wide = p.row_bytes % 16 == 0;
    for (int64_t l = 0; l < nl; ++l) {
      p.k_layers[l] = static_cast<char*>(k_layers[l0 + l]);
      p.v_layers[l] = static_cast<char*>(v_layers[l0 + l]);
      wide = wide && aligned16(p.k_layers[l]) && aligned16(p.v_layers[l]);
    }
    // rows that are no multiple of 16 bytes, or bases off that boundary: by bytes
    const int st = wide ? blocks::launch<uint4>(p, sms, s) : blocks::launch<uint8_t>(p, sms, s);
    if (st) return st;
  }
  return PA_OK;
}

extern "C" int pa_remap_block_tables(int32_t* out, const int32_t* block_tables,
                                     const int32_t* block_map, int64_t num_entries,
                                     int64_t num_blocks, void* stream) {
  using namespace pa;
  if (num_entries < 0 || num_blocks < 0) return PA_ERR_INVALID_ARGUMENT;
  if (num_entries == 0) return PA_OK;
  if (!out || !block_tables || (!block_map && num_blocks)) return PA_ERR_INVALID_ARGUMENT;
  int sms = 0;
  if (device_sm_count(&sms) != PA_OK) return PA_ERR_NO_DEVICE;
  const int64_t ctas = std::min<int64_t>((num_entries + blocks::kThreads - 1) / blocks::kThreads, (int64_t)sms * 8);
  blocks::remap_kernel<<<(unsigned)ctas, blocks::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      out, block_tables, block_map, num_entries, num_blocks);
  return cuda_status(cudaGetLastError());
}
