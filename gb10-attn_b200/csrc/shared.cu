// shared.cu -- decode attention of sequences that share a prefix
// (pa_paged_attention_shared).
//
// All members of a group have the same first P tokens in the same pages.  The
// softmax sum of a row splits at P:
//   out = (A_p + A_s) / (l_p + l_s),  A = sum_j e^{s_j - m} V_j, l = sum_j e^{s_j - m}
// over the keys before and from P on, with one reference m, so the prefix can
// be done for all members at once: their query heads of one KV head are the
// rows of products, and each K/V element of the prefix is read once for 16 rows
// (by warps) or 256 (in tensor memory) instead of once for a sequence's.
//
// Two launches, the second a programmatic dependent of the first: the attention
// and the merge of its partials.  Every CTA of the first makes the same plan in
// shared memory (the groups' usable prefixes, running counts of the work) and
// takes an equal run of one kind of work; only for many sequences the plan is a
// launch of its own.
#include <algorithm>
#include <atomic>
#include <mutex>
#include <vector>

#include "shared.cuh"

namespace pa {
namespace shared {

// The plan as a launch of its own, for more sequences or groups than kPlanMax
// and for counts past 32 bits.
__global__ void __launch_bounds__(1024) plan_kernel(const __grid_constant__ Params p) {
  pdl_trigger();
  make_plan<long long>(p, plan_at(p, 0), p.plan + p.scratch_off, true);
}

// All of the work by warps: pools that the tensor-memory part does not load.
// Bound by the reads of a prefix for every 16 rows, out of the L2 mostly, and by
// instruction latency.  128 sequences on 8k: 32 / 8 heads of 128 in pages of 8 166 us
// (59 with the tensor memory, on pages of 16), 16 / 2 heads of 256 344, 32 / 8 of 32 66;
// 64 on 2k, 12 / 12 heads of 64 in pages of 8, 22.
template <int D> struct Cfg {
  static constexpr int STAGES = 4;
  static constexpr int RING = STAGES * (int)stage_bytes(D);
  // warps per CTA (one CTA per SM): what 224 KB of rings hold, 16 at most
  static constexpr int WARPS = 224 * 1024 / RING < 16 ? 224 * 1024 / RING : 16;
  static constexpr int SMEM = WARPS * RING;
  static_assert(plan_scratch(kPlanMax, kPlanMax) <= SMEM, "the plan's scratch is in the rings");
};

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::WARPS * 32, 1) warps_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5;
  pdl_trigger();
  const Plan plan = take_plan(p, smem);
  // consecutive workers sit on different SMs
  const int64_t worker = (int64_t)warp * gridDim.x + blockIdx.x;
  warp_work<T, D, Cfg<D>::STAGES>(p, plan, load_plan(plan.totals), smem_u32(smem) + warp * Cfg<D>::RING, worker,
                                  worker);
}

// ---------------------------------------------------------------------------
// merge: W warps per output row, each a run of its pieces, all in a fixed order.
// Bound by latency with few rows (eight warps then take a row: one sequence of
// 20k tokens 46 us with one warp, 23 with eight), by its loads with many.
// ---------------------------------------------------------------------------

template <typename T, int D, int W>
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ Params p) {
  constexpr int E = D / 32;
  __shared__ float part[W > 1 ? W : 1][W > 1 ? D : 1];
  __shared__ float2 part_ml[W > 1 ? W : 1];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
  if (row >= p.B * p.H) return;
  const Pieces at = load_plan(p.pieces + row);
  const int32_t own_rows = min(p.G, ROWS), n_pre = at.n_pre, n_own = at.n_own;
  const int all = n_pre + n_own, first = W > 1 ? all * warp / W : 0;
  const int n = W > 1 ? all * (warp + 1) / W - first : all;
  auto piece = [&](int c) -> int64_t {
    c += first;
    return c < n_pre ? at.pre0 + (int64_t)c * at.pre_step : at.own0 + (int64_t)(c - n_pre) * own_rows;
  };
  // 32 pieces at a time, lane c with the maximum and sum of piece c; then their
  // O, several in flight
  constexpr int V = D >= 128 ? 4 : D / 32;  // elements per load
  float acc[E] = {}, L = 0.f, M = -INFINITY;
  constexpr int K = D == 256 ? 4 : 8;
  float x[K][E];
  auto fetch = [&](int c) {  // O of K pieces from c on (past the last the last again)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float* src = p.part_o + piece(min(c + k, n - 1)) * D + lane * V;
#pragma unroll
      for (int i = 0; i < E / V; ++i) {
        if constexpr (V == 4) {
          const float4 f = *reinterpret_cast<const float4*>(src + i * 128);
          x[k][4 * i] = f.x, x[k][4 * i + 1] = f.y, x[k][4 * i + 2] = f.z, x[k][4 * i + 3] = f.w;
        } else if constexpr (V == 2) {
          const float2 f = *reinterpret_cast<const float2*>(src);
          x[k][0] = f.x, x[k][1] = f.y;
        } else {
          x[k][0] = *src;
        }
      }
    }
  };
  for (int c0 = 0; c0 < n; c0 += 32) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (c0 + lane < n) ml = p.part_ml[piece(c0 + lane)];
    fetch(c0);
    const bool none = ml.x == -INFINITY && ml.y == 0.f;  // without keys, or only scores of -inf: O not used
    float top = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float Mn = fmaxf(M, top), base = Mn == -INFINITY ? 0.f : Mn;
    const float alpha = fast_exp2(M - base), w = fast_exp2(ml.x - base);
    M = Mn;
    float l = none ? 0.f : w * ml.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    L = fmaf(L, alpha, l);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= alpha;
    const uint32_t used = __ballot_sync(0xffffffffu, !none);
    const int cnt = min(32, n - c0);
    for (int c = 0; c < cnt; c += K) {
      if (c) fetch(c0 + c);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float wc = __shfl_sync(0xffffffffu, w, min(c + k, 31));
        const bool in = c + k < cnt && (used >> (c + k) & 1);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(in ? wc : 0.f, in ? x[k][e] : 0.f, acc[e]);
      }
    }
  }
  if constexpr (W > 1) {
    static_assert(W == 8, "the CTA's warps");
    if (lane == 0) part_ml[warp] = make_float2(M, L);
#pragma unroll
    for (int e = 0; e < E; ++e) part[warp][(e / V * 32 + lane) * V + e % V] = acc[e];
    __syncthreads();
    if (warp) return;
    M = lane < W ? part_ml[lane].x : -INFINITY;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    M = __shfl_sync(0xffffffffu, M, 0);
    const float base = M == -INFINITY ? 0.f : M;
    L = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float2 ml = part_ml[w];
      const float f = fast_exp2(ml.x - base);
      L = fmaf(f, ml.y, L);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(f, part[w][(e / V * 32 + lane) * V + e % V], acc[e]);
    }
  }
  // no key, or only scores of -inf: L = 0, so out is NaN and lse -inf
  const float inv = 1.f / L;
  T* out = static_cast<T*>(p.out) + row * D + lane * V;
#pragma unroll
  for (int i = 0; i < E / V; ++i) {
    struct alignas(2 * V) {
      T x[V];
    } v;
#pragma unroll
    for (int e = 0; e < V; ++e) v.x[e] = T(acc[i * V + e] * inv);
    *reinterpret_cast<decltype(v)*>(out + i * 128) = v;
  }
  if (p.lse && lane == 0) p.lse[row] = (M + log2f(L)) * kLn2;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Rows of a group from which its prefix may go to the tensor memory.  Over 66
// batches (listed beside kTcMinTiles) 17 takes 1.02 times as long and 65 1.01 times in the
// mean: 17 up to 1.19 times (one group of 32 rows on 128 tokens 13.6 us, 16.1), 65
// 0.82 times where many groups of 64 rows share 64 tokens (128 groups 164 us, 134),
// 1.4 to 1.6 times where 4 or 8 groups of 48 or 64 rows share 8k (8 of 48: 84, 126).
constexpr int kTcRows = 33;

constexpr int64_t kAlign = 256;  // of the workspace's parts

static std::atomic<int> g_waits{1};  // pa_set_shared_waits

struct Layout {
  bool tc, planned;
  int64_t warps, plan_bytes, group_off, seq_off, scratch_off, own_row0, tc_row0;
  size_t pieces, ml, o, total;
};

static int warps_per_cta(int64_t D) {
  return D == 32 ? Cfg<32>::WARPS : D == 64 ? Cfg<64>::WARPS : D == 128 ? Cfg<128>::WARPS : Cfg<256>::WARPS;
}

// Slots for partials: unit + worker < units + workers, for prefixes with ROWS
// rows each, for sequences' own units with min(G, ROWS), for the tensor
// memory's with TC_ROWS.  `tc`: whether this launch has that part (a size query,
// which does not know the pool, assumes the larger).  Offsets are multiples of 256
// from the workspace's first address that is one (partials are stored 32 bytes at
// a time); `total` has room for the bytes before it.
static int layout(int64_t B, int64_t NG, int64_t H, int64_t HKV, int64_t D, int sms, bool tc, int64_t max_ctx,
                  Layout* y) {
  const int64_t G = H / HKV;
  y->tc = tc && NG && B * G >= kTcRows && (D == 64 || D == 128);
  y->warps = (int64_t)sms * (y->tc ? kTcWarps : warps_per_cta(D));
  const int64_t most = (int64_t)sms * std::max(kTcWarps, warps_per_cta(D));
  const int64_t pre_units = NG ? HKV * (B * G / ROWS + NG) : 0, own_units = B * HKV * ((G + ROWS - 1) / ROWS);
  y->own_row0 = NG ? (pre_units + most) * ROWS : 0;
  y->tc_row0 = y->own_row0 + (own_units + most) * std::min<int64_t>(G, ROWS);
  int64_t rows = y->tc_row0;
  if (y->tc) rows += (HKV * (B * G / TC_ROWS + std::min<int64_t>(NG, B * G / kTcRows)) + sms) * TC_ROWS;
  if (rows >= (int64_t(1) << 31) || B * H >= (int64_t(1) << 31)) return PA_ERR_TOO_LARGE;
  auto up = [](int64_t x) { return (x + kAlign - 1) & ~(kAlign - 1); };
  // tiles of every unit if all had the longest context
  const double most_tiles = (double)(pre_units + own_units) * ((double)max_ctx / KT + 1 + kTcUnitCost);
  y->planned = B > kPlanMax || NG > kPlanMax || most_tiles >= 2147483647.0;
  y->group_off = kAlign;
  y->seq_off = y->group_off + up(NG * (int64_t)sizeof(Group));
  y->scratch_off = y->seq_off + up(B * (int64_t)sizeof(Seq));
  y->plan_bytes = y->scratch_off + (y->planned ? up(plan_scratch(B, NG)) : 0);
  y->pieces = (size_t)(y->plan_bytes * (y->planned ? 1 : sms));
  y->ml = y->pieces + (size_t)up(B * H * (int64_t)sizeof(Pieces));
  y->o = y->ml + (size_t)up(rows * (int64_t)sizeof(float2));
  y->total = y->o + (size_t)up(rows * D * (int64_t)sizeof(float)) + kAlign - 16;
  return PA_OK;
}

template <typename T, int D>
static int launch_typed(const Params& p, int sms, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (p.planned) {
    plan_kernel<<<1, 1024, 0, s>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_status(e);
  }
  if (p.tc_rows) {
    const int st = launch_tc(p, DTypeId<T>::value, D, s);
    if (st) return st;
  } else {
    using C = Cfg<D>;
    auto kern = warps_kernel<T, D>;
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_status(e);
    {
      std::lock_guard<std::mutex> lk(mu);
      if (std::find(done.begin(), done.end(), dev) == done.end()) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return cuda_status(e);
        done.push_back(dev);
      }
    }
    e = launch(kern, sms, C::WARPS * 32, C::SMEM, s, p, p.planned);
    if (e != cudaSuccess) return cuda_status(e);
  }
  // Eight warps a row while one CTA each fits the GPU at once (few rows have
  // many pieces: with one warp, a sequence of 20k alone took 46 us, 30 of them
  // here), else one
  if (p.B * p.H <= 8 * sms) return cuda_status(launch(merge_kernel<T, D, 8>, p.B * p.H, 256, 0, s, p, true));
  return cuda_status(launch(merge_kernel<T, D, 1>, (p.B * p.H + 7) / 8, 256, 0, s, p, true));
}

template <typename T>
static int launch_dtype(const Params& p, int64_t D, int sms, cudaStream_t s) {
  switch (D) {
    case 32: return launch_typed<T, 32>(p, sms, s);
    case 64: return launch_typed<T, 64>(p, sms, s);
    case 128: return launch_typed<T, 128>(p, sms, s);
    default: return launch_typed<T, 256>(p, sms, s);
  }
}

static int check(int64_t B, int64_t NG, int64_t H, int64_t HKV, int64_t D, int dtype) {
  if (B < 0 || NG < 0 || H <= 0 || HKV <= 0 || D <= 0) return PA_ERR_INVALID_ARGUMENT;
  if (H % HKV) return PA_ERR_NUM_HEADS;
  if (D != 32 && D != 64 && D != 128 && D != 256) return PA_ERR_HEAD_DIM;
  if (dtype != PA_DTYPE_F16 && dtype != PA_DTYPE_BF16) return PA_ERR_DTYPE;
  if (B > 0x7fffffff || NG > 0x7fffffff || H > 0x7fffffff) return PA_ERR_TOO_LARGE;
  return PA_OK;
}

}  // namespace shared
}  // namespace pa

extern "C" int pa_set_shared_waits(int waits) { return pa::shared::g_waits.exchange(waits != 0); }

extern "C" int pa_shared_workspace_size(int64_t num_seqs, int64_t num_groups, int64_t num_heads,
                                        int64_t num_kv_heads, int64_t head_dim, int kv_dtype,
                                        size_t* bytes) {
  using namespace pa;
  if (!bytes) return PA_ERR_INVALID_ARGUMENT;
  int st = shared::check(num_seqs, num_groups, num_heads, num_kv_heads, head_dim, kv_dtype);
  if (st) return st;
  *bytes = 0;
  if (num_seqs == 0) return PA_OK;
  int sms = 0;
  if (device_sm_count(&sms) != PA_OK) return PA_ERR_NO_DEVICE;
  shared::Layout y;
  // for either place of the plan
  st = shared::layout(num_seqs, num_groups, num_heads, num_kv_heads, head_dim, sms, true, 0, &y);
  if (st) return st;
  *bytes = y.total;
  st = shared::layout(num_seqs, num_groups, num_heads, num_kv_heads, head_dim, sms, true, int64_t(1) << 62, &y);
  if (st) return st;
  *bytes = std::max(*bytes, y.total);
  return PA_OK;
}

extern "C" int pa_paged_attention_shared(
    void* out, float* lse, const void* q, int io_dtype, const void* k_cache, const void* v_cache,
    int kv_dtype, const int32_t* block_tables, const int32_t* context_lens,
    const int32_t* group_starts, const int32_t* prefix_lens, int64_t num_seqs, int64_t num_groups,
    int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
    int64_t num_blocks, int64_t max_blocks, double scale, void* workspace, size_t workspace_bytes,
    int32_t* dev_status, void* stream) {
  using namespace pa;
  int st = shared::check(num_seqs, num_groups, num_heads, num_kv_heads, head_dim, kv_dtype);
  if (st) return st;
  if (io_dtype != kv_dtype) return PA_ERR_DTYPE;
  if (block_size <= 0 || num_blocks < 0 || max_blocks < 0) return PA_ERR_INVALID_ARGUMENT;
  if (num_seqs == 0) return PA_OK;
  if (num_blocks == 0) return PA_ERR_INVALID_ARGUMENT;
  if (!out || !q || !k_cache || !v_cache || !block_tables || !context_lens ||
      (num_groups && (!group_starts || !prefix_lens)))
    return PA_ERR_INVALID_ARGUMENT;
  if (!aligned16(out) || !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache)) return PA_ERR_ALIGNMENT;
  // pool rows of head_dim elements are numbered in 32 bits (a larger pool
  // does not fit the GPU), page numbers too
  if (block_size > 0x7fffffff || num_blocks > 0x7fffffff ||
      num_blocks * block_size > 0xffffffffll / num_kv_heads)
    return PA_ERR_TOO_LARGE;
  int sms = 0;
  if (device_sm_count(&sms) != PA_OK) return PA_ERR_NO_DEVICE;
  shared::Layout y;
  st = shared::layout(num_seqs, num_groups, num_heads, num_kv_heads, head_dim, sms,
                      shared::tc_takes(head_dim, block_size, num_blocks), block_size * max_blocks, &y);
  if (st) return st;
  if (!workspace || workspace_bytes < y.total) return PA_ERR_WORKSPACE;
  if (!aligned16(workspace)) return PA_ERR_ALIGNMENT;
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + shared::kAlign - 1) &
                                     ~(uintptr_t)(shared::kAlign - 1));
  shared::Params p = {};
  p.out = out;
  p.lse = lse;
  p.q = q;
  p.k = k_cache;
  p.v = v_cache;
  p.block_tables = block_tables;
  p.context_lens = context_lens;
  p.group_starts = group_starts;
  p.prefix_lens = prefix_lens;
  p.B = num_seqs;
  p.NG = num_groups;
  p.H = num_heads;
  p.HKV = num_kv_heads;
  p.BS = block_size;
  p.NB = num_blocks;
  p.MB = max_blocks;
  p.qscale = (float)(scale * 1.4426950408889634);
  p.G = (int32_t)(num_heads / num_kv_heads);
  p.bs_shift = -1;
  if ((block_size & (block_size - 1)) == 0)
    for (p.bs_shift = 0; (int64_t(1) << p.bs_shift) < block_size; ++p.bs_shift) {}
  p.plan = ws;
  p.plan_bytes = y.plan_bytes;
  p.group_off = y.group_off;
  p.seq_off = y.seq_off;
  p.scratch_off = y.scratch_off;
  p.planned = y.planned;
  p.warps = (int32_t)y.warps;
  p.own_row0 = y.own_row0;
  p.tc_row0 = y.tc_row0;
  p.tc_rows = y.tc ? shared::kTcRows : 0;
  p.tc_ctas = sms;
  p.waits = shared::g_waits.load(std::memory_order_relaxed);
  p.pieces = reinterpret_cast<shared::Pieces*>(ws + y.pieces);
  p.part_ml = reinterpret_cast<float2*>(ws + y.ml);
  p.part_o = reinterpret_cast<float*>(ws + y.o);
  p.dev_status = dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv_dtype == PA_DTYPE_BF16 ? shared::launch_dtype<__nv_bfloat16>(p, head_dim, sms, s)
                                   : shared::launch_dtype<__half>(p, head_dim, sms, s);
}
