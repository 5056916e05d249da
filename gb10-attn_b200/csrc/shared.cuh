// shared.cuh -- what the launches of the shared-prefix decode have in common:
// how its work is counted, cut and numbered (shared.cu has the plan, the warp
// kernel and the merge, shared_tc.cu the tensor-memory kernel).
#pragma once

#include "common.cuh"

namespace pa {
namespace shared {

constexpr int KT = 16;    // keys per tile
constexpr int ROWS = 16;  // query rows per item (the M of one mma)

// tensor-memory kernel: keys per tile, rows per unit (two chains of 128; a unit
// of at most 128 rows gives both chains the same rows and every other tile)
constexpr int TC_KT = 128;
constexpr int TC_ROWS = 256;

// The work, counted in tiles of KT keys: first the groups' prefixes, then the
// sequences' own tokens.  A unit is one (group or sequence, KV head, tile of
// rows); its tiles are consecutive, and the units of a group or sequence too,
// in the order (KV head, tile of rows).  The `warps` workers of a launch take
// equal consecutive runs of the total, worker w the tiles
// [w T / W, (w + 1) T / W), so a unit is cut where a worker's run ends.  A piece
// is the overlap of unit u and worker w; u + w grows strictly from piece to
// piece, so it numbers the pieces' slots for partials, with no table of them.
//   Groups with many rows are the tensor-memory kernel's (shared_tc.cu), with
// tiles, units and workers of its own, numbered the same way.
struct alignas(16) Group {
  long long tile0[2];           // first tile: of the warps' work, of the tensor-memory kernel's
  int32_t b0, n, table, prefix; // members b0 .. b0 + n - 1; table row that serves; tokens shared
  int32_t unit0[2], tc, pad;    // first unit; whether the tensor-memory kernel does it
};
struct alignas(16) Seq {
  long long tile0[1];
  int32_t from, ctx, group, pad;  // own tokens from .. ctx - 1; its group or -1
};
struct alignas(16) Totals {
  int64_t prefix_tiles, tiles, workers;  // the warps' work
  int64_t tc_tiles, tc_workers;          // the tensor-memory kernel's
};

struct Params {
  void* out;
  float* lse;  // [B, H]
  const void *q, *k, *v;
  const int32_t *block_tables, *context_lens, *group_starts, *prefix_lens;
  int64_t B, NG, H, HKV, BS, NB, MB;
  float qscale;     // scale * log2(e)
  int32_t G;        // query heads per KV head
  int32_t warps;    // warps of the attention launch
  int32_t bs_shift; // log2(BS) if BS is a power of two, else -1
  // workspace
  Totals* totals;
  Group* groups;
  Seq* seqs;
  float2* part_ml;  // (running max in log2 units, sum)
  float* part_o;
  int64_t own_row0; // first partial row of the sequences' own units
  int64_t tc_row0;  // and of the tensor-memory kernel's units
  int32_t tc_rows;  // rows from which a group is the tensor-memory kernel's (0: none is)
  int32_t tc_ctas;
  int32_t* dev_status;
};

__host__ __device__ __forceinline__ int32_t cdiv(int32_t a, int32_t b) { return (a + b - 1) / b; }

// Worker w's first tile, and the worker of tile x, for T tiles over W workers.
__device__ __forceinline__ int64_t first_tile(int64_t w, int64_t T, int64_t W) { return w * T / W; }
__device__ __forceinline__ int64_t worker_of(int64_t x, int64_t T, int64_t W) { return ((x + 1) * W - 1) / T; }

// One of the structs above, past the L1: the launch after next reads the plan
// without having waited for it itself.
template <typename E> __device__ __forceinline__ E load_plan(const E* e) {
  static_assert(sizeof(E) % 16 == 0, "");
  union {
    int4 w[sizeof(E) / 16];
    E e;
  } u;
#pragma unroll
  for (int i = 0; i < (int)sizeof(E) / 16; ++i) u.w[i] = __ldcg(reinterpret_cast<const int4*>(e) + i);
  return u.e;
}

// The last of n entries (their tile0[I] rising from at most x) with
// tile0[I] <= x.  All lanes probe at once: two steps for 1024 entries.
template <int I, typename E>
__device__ __forceinline__ int32_t find(const E* e, int32_t n, int64_t x, int lane) {
  int32_t lo = 0, len = n;  // the answer is in [lo, lo + len)
  while (len > 1) {
    const int32_t step = (len + 31) / 32, at = lo + lane * step;
    const uint32_t m = __ballot_sync(0xffffffffu, lane * step < len && __ldcg(&e[at].tile0[I]) <= x);
    const int32_t k = 31 - __clz(m);
    len = min(step, len - k * step);
    lo += k * step;
  }
  return lo;
}

template <typename K, typename A>
inline cudaError_t launch_pdl(K kern, dim3 grid, dim3 block, size_t smem, cudaStream_t s, const A& p) {
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

// One tensor-memory launch on the plan in p (shared_tc.cu).
bool tc_takes(int64_t D, int64_t BS, int64_t NB);
int launch_tc(const Params& p, int dtype, int64_t D, cudaStream_t s);

}  // namespace shared
}  // namespace pa
