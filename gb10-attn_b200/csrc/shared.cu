// shared.cu -- decode attention of sequences that share a prefix
// (pa_paged_attention_shared).
//
// All members of a group have the same first P tokens in the same pages.  The
// softmax sum of a row splits at P:
//   out = (A_p + A_s) / (l_p + l_s),  A = sum_j e^{s_j - m} V_j, l = sum_j e^{s_j - m}
// over the keys before and from P on, with one reference m, so the prefix can
// be done for all members at once: their query heads of one KV head are the
// rows of one product, and each K/V element of the prefix is read once a group
// instead of once a sequence.
//
// Launches, chained with programmatic dependent launch: a plan (one CTA: the
// groups' usable prefixes and running counts of the work), the prefixes of
// groups with many rows on the tensor cores (shared_tc.cu), all other prefixes
// and the sequences' own tokens (every warp takes an equal run of the work),
// and the merge of the partials.
#include <algorithm>
#include <mutex>
#include <vector>

#include "shared.cuh"

namespace pa {
namespace shared {

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------

constexpr int kPlanThreads = 1024;
constexpr int kMinTiles = 2;    // tiles per worker when there are few
constexpr int kMinTcTiles = 1;  // of the tensor-memory kernel's

// Exclusive scan of (a, b) over the block on top of the running totals `base`.
struct Pair {
  int64_t a, b;
};
__device__ __forceinline__ Pair block_scan(Pair x, Pair* warp_sums, Pair& base) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto warp_scan = [&](Pair s) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, s.a, o), b = __shfl_up_sync(0xffffffffu, s.b, o);
      if (lane >= o) s.a += a, s.b += b;
    }
    return s;
  };
  const Pair s = warp_scan(x);
  __syncthreads();
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) warp_sums[lane] = warp_scan(warp_sums[lane]);
  __syncthreads();
  const Pair before = warp ? warp_sums[warp - 1] : Pair{0, 0};
  const Pair r = {base.a + before.a + s.a - x.a, base.b + before.b + s.b - x.b};
  base.a += warp_sums[31].a;
  base.b += warp_sums[31].b;
  return r;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ Params p) {
  __shared__ Pair sums[32];
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t B = (int32_t)p.B, NG = (int32_t)p.NG, HKV = (int32_t)p.HKV, G = p.G;
  const int32_t max_ctx = (int32_t)min(p.MB * p.BS, (int64_t)0x7fffff00);
  const int32_t own_y = cdiv(G, ROWS);
  auto context = [&](int32_t b) {
    const int32_t c = p.context_lens[b];
    if (c > max_ctx) report(p.dev_status, PA_DEVERR_CONTEXT);
    return min(max(c, 0), max_ctx);
  };
  // group bounds that are not 0 <= s_0 <= s_1 <= ... <= B: no sharing at all
  int bad = 0;
  for (int32_t g = tid; g < NG; g += kPlanThreads) {
    const int32_t a = p.group_starts[g], b = p.group_starts[g + 1];
    bad |= a < 0 || b < a || b > B;
  }
  bad = __syncthreads_or(bad);
  if (bad && tid == 0) report(p.dev_status, PA_DEVERR_GROUP);
  const int32_t groups = bad ? 0 : NG;
  for (int32_t b = tid; b < B; b += kPlanThreads) p.seqs[b].group = -1;
  __syncthreads();
  // a group's usable prefix: no longer than any member that has tokens; the
  // first such member's table row serves it.  One member alone shares nothing.
  for (int32_t g = warp; g < groups; g += kPlanThreads / 32) {
    const int32_t a = p.group_starts[g], e = p.group_starts[g + 1];
    int32_t least = 0x7fffffff, first = 0x7fffffff, live = 0;
    for (int32_t b = a + lane; b < e; b += 32) {
      const int32_t c = context(b);
      if (c > 0) least = min(least, c), first = min(first, b), ++live;
      p.seqs[b].group = g;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    first = __reduce_min_sync(0xffffffffu, first);
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) {
      Group& gp = p.groups[g];
      gp.b0 = a;
      gp.n = e - a;
      gp.table = first;
      gp.prefix = live > 1 ? max(0, min(p.prefix_lens[g], least)) : 0;
      gp.tc = p.tc_rows && gp.n * G >= p.tc_rows;
    }
  }
  __syncthreads();
  Pair base = {0, 0}, tc_base = {0, 0};  // tiles and units so far
  for (int32_t g0 = 0; g0 < groups; g0 += kPlanThreads) {
    const int32_t g = g0 + tid;
    Pair x = {0, 0}, y = {0, 0};
    if (g < groups) {
      const Group& gp = p.groups[g];
      if (gp.tc) {
        y.b = (int64_t)HKV * cdiv(gp.n * G, TC_ROWS);
        y.a = y.b * cdiv(gp.prefix, TC_KT);
      } else {
        x.b = (int64_t)HKV * cdiv(gp.n * G, ROWS);
        x.a = x.b * cdiv(gp.prefix, KT);
      }
    }
    const Pair at = block_scan(x, sums, base);
    const Pair tc_at = p.tc_rows ? block_scan(y, sums, tc_base) : Pair{0, 0};
    if (g < groups) {
      Group& gp = p.groups[g];
      gp.tile0[0] = at.a;
      gp.tile0[1] = tc_at.a;
      gp.unit0[0] = (int32_t)at.b;
      gp.unit0[1] = (int32_t)tc_at.b;
    }
  }
  const int64_t prefix_tiles = base.a;
  for (int32_t b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int32_t b = b0 + tid;
    Pair x = {0, 0};
    int32_t ctx = 0, from = 0;
    if (b < B) {
      const int32_t g = p.seqs[b].group;
      ctx = context(b);
      if (g >= 0) from = min(p.groups[g].prefix, ctx);
      x.a = (int64_t)HKV * own_y * cdiv(ctx - from, KT);
    }
    const Pair at = block_scan(x, sums, base);
    if (b < B) {
      p.seqs[b].tile0[0] = at.a;
      p.seqs[b].from = from;
      p.seqs[b].ctx = ctx;
    }
  }
  if (tid == 0)
    *p.totals = Totals{prefix_tiles, base.a,
                       min((int64_t)p.warps, max((base.a + kMinTiles - 1) / kMinTiles, (int64_t)1)), tc_base.a,
                       min((int64_t)p.tc_ctas, max((tc_base.a + kMinTcTiles - 1) / kMinTcTiles, (int64_t)1))};
}

// ---------------------------------------------------------------------------
// attention: one warp per worker
// ---------------------------------------------------------------------------

// What a warp computes at a time: rows r0 .. r0 + nrows - 1 of a unit (row r:
// sequence b0 + r / G, head kvh * G + r % G) against keys t0 .. t1 - 1 of table
// row `table`; partials from row prow on.
struct Item {
  int32_t table, b0, r0, nrows, kvh, t0, t1, prow;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// c[16 x 8] += a[16 x 16] b[16 x 8], fp32 sums
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half*) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16*) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16*) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half*) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int D> struct Cfg {
  static constexpr int STAGES = 4;
  static constexpr int STAGE = 2 * KT * D * 2;  // K tile, V tile
  static constexpr int WARP = STAGES * STAGE;
  // warps per CTA (one CTA per SM): what 224 KB of stages hold, 16 at most
  static constexpr int WARPS = 224 * 1024 / WARP < 16 ? 224 * 1024 / WARP : 16;
  static constexpr int SMEM = WARPS * WARP;
};

// A warp streams its item's K and V rows through a ring of its own (16-byte
// asynchronous copies, so any page size and any first token serve), with the
// keys of a tile as the N of S = Q K^T and the K of P V; the running maximum
// and sum, the products' sums and O stay in fp32 registers.  P is rounded to
// the pool's type for the second product (its error, 2^-9 or 2^-12 of a weight
// at most and averaged over the keys, is at the level of the output's own
// rounding); the sum l is of the unrounded weights.
template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::WARPS * 32, 1) attention_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D>;
  constexpr int NST = C::STAGES, CH = D / 8;  // 16-byte chunks per row
  extern __shared__ __align__(128) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // (with a tensor-memory launch before this one, the plan is complete when
  // this grid starts: that launch waits for it before it lets this one go)
  if (!p.tc_rows) pdl_wait();
  pdl_trigger();
  const uint32_t ring = smem_u32(smem) + warp * C::WARP;
  const Totals tot = load_plan(p.totals);
  // rows of a tile sit `D * 2` bytes apart with their 16-byte chunks permuted
  // by the row, so the eight rows of a matrix load fall on different banks
  auto chunk_at = [](int row, int c) -> uint32_t {
    return (uint32_t)(row * (D * 2) + ((c ^ (CH >= 8 ? (row & 7) : ((row >> 1) & 3))) << 4));
  };
  // consecutive workers sit on different SMs
  const int64_t worker = warp * gridDim.x + blockIdx.x;
  const int32_t HKV = (int32_t)p.HKV, own_y = cdiv(p.G, ROWS);
  int64_t x = 0, end = 0;
  if (worker < tot.workers) {
    x = first_tile(worker, tot.tiles, tot.workers);
    end = first_tile(worker + 1, tot.tiles, tot.workers);
  }
  int32_t at = -1;  // the group or sequence of tile x; of which is `x < prefix_tiles`
  bool in_prefix = x < tot.prefix_tiles;
  if (x < end)
    at = in_prefix ? find<0>(p.groups, (int32_t)p.NG, x, lane) : find<0>(p.seqs, (int32_t)p.B, x, lane);
  while (x < end) {
    if (in_prefix && x >= tot.prefix_tiles) in_prefix = false, at = 0;
    Item im;
    int64_t left;  // tiles of the unit from x on
    if (in_prefix) {
      const Group gp = load_plan(p.groups + at);
      const int32_t rows = gp.n * p.G, ry = cdiv(rows, ROWS), nt = cdiv(gp.prefix, KT);
      const int64_t done = x - gp.tile0[0];
      if (gp.tc || done >= (int64_t)HKV * ry * nt) { ++at; continue; }
      const int32_t u = (int32_t)(done / nt), j = (int32_t)(done - (int64_t)u * nt);
      left = min((int64_t)(nt - j), end - x);
      im.table = gp.table;
      im.b0 = gp.b0;
      im.kvh = u / ry;
      im.r0 = (u - im.kvh * ry) * ROWS;
      im.nrows = min(ROWS, rows - im.r0);
      im.t0 = j * KT;
      im.t1 = min(gp.prefix, im.t0 + (int32_t)left * KT);
      im.prow = (int32_t)((gp.unit0[0] + u + worker) * ROWS);
    } else {
      const Seq sp = load_plan(p.seqs + at);
      const int32_t nt = cdiv(sp.ctx - sp.from, KT);
      const int64_t done = x - sp.tile0[0];
      if (done >= (int64_t)HKV * own_y * nt) { ++at; continue; }
      const int32_t u = (int32_t)(done / nt), j = (int32_t)(done - (int64_t)u * nt);
      left = min((int64_t)(nt - j), end - x);
      im.table = im.b0 = at;
      im.kvh = u / own_y;
      im.r0 = (u - im.kvh * own_y) * ROWS;
      im.nrows = min(ROWS, p.G - im.r0);
      im.t0 = sp.from + j * KT;
      im.t1 = min(sp.ctx, im.t0 + (int32_t)left * KT);
      im.prow = (int32_t)(p.own_row0 + ((int64_t)at * HKV * own_y + u + worker) * min(p.G, ROWS));
    }
    x += left;
    const int32_t* table = p.block_tables + (int64_t)im.table * p.MB;
    const int n_tiles = (im.t1 - im.t0 + KT - 1) / KT;

    // pool row (in rows of D elements) of token t0 + 16 j + lane, lanes 0-15
    auto row_of = [&](int j) -> uint32_t {
      const int32_t t = im.t0 + j * KT + lane;
      if (lane >= KT || t >= im.t1) return 0xffffffffu;
      const int32_t page = p.bs_shift >= 0 ? t >> p.bs_shift : t / (int32_t)p.BS;
      int32_t blk = __ldg(table + page);
      if (blk < 0 || blk >= p.NB) {
        report(p.dev_status, PA_DEVERR_BLOCK_ID);
        blk = 0;
      }
      return (uint32_t)(((int64_t)blk * p.BS + (t - page * (int32_t)p.BS)) * p.HKV + im.kvh);
    };
    // rows past the item's last key are zeros: their scores are masked, and
    // no weight of zero meets a NaN of an unwritten row
    auto load = [&](int j, uint32_t row) {
      if (j < n_tiles) {
        const uint32_t st = ring + (j % NST) * C::STAGE;
#pragma unroll
        for (int i = 0; i < KT * CH / 32; ++i) {
          const int idx = i * 32 + lane, r = idx / CH, c = idx % CH;
          const uint32_t pr = __shfl_sync(0xffffffffu, row, r);
          const int bytes = pr == 0xffffffffu ? 0 : 16;
          const int64_t off = bytes ? ((int64_t)pr * CH + c) * 16 : 0;
          cp_async16(st + chunk_at(r, c), static_cast<const char*>(p.k) + off, bytes);
          cp_async16(st + KT * D * 2 + chunk_at(r, c), static_cast<const char*>(p.v) + off, bytes);
        }
      }
      cp_async_commit();
    };

    uint32_t rows_next = row_of(0);
#pragma unroll
    for (int j = 0; j < NST - 1; ++j) {
      const uint32_t rows = rows_next;
      rows_next = row_of(j + 1);
      load(j, rows);
    }

    // Q: lane holds rows lane / 4 and lane / 4 + 8 of the A operand
    uint32_t qa[D / 16][4];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = im.r0 + (lane >> 2) + 8 * hf;
      const bool in = (lane >> 2) + 8 * hf < im.nrows;
      const T* src = static_cast<const T*>(p.q) +
                     ((int64_t)(im.b0 + r / p.G) * p.H + im.kvh * p.G + r % p.G) * D + 2 * (lane & 3);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qa[kk][hf] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16)) : 0u;
        qa[kk][hf + 2] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16 + 8)) : 0u;
      }
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int mi = lane >> 3, mr = lane & 7;  // matrix and row this lane addresses

    for (int j = 0; j < n_tiles; ++j) {
      const uint32_t rows = rows_next;
      rows_next = row_of(j + NST);
      cp_async_wait<NST - 2>();
      __syncwarp();
      load(j + NST - 1, rows);  // into the stage of tile j - 1, which every lane has left
      const uint32_t ks = ring + (j % NST) * C::STAGE, vs = ks + KT * D * 2;
      float s[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t b[4];
        ldsm4(b, ks + chunk_at(mr + 8 * (mi >> 1), 2 * kk + (mi & 1)));
        mma(s[0], qa[kk], b[0], b[1], (T*)nullptr);
        mma(s[1], qa[kk], b[2], b[3], (T*)nullptr);
      }
      const int valid = im.t1 - im.t0 - j * KT;
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in = 8 * n + 2 * (lane & 3) + (e & 1) < valid;
          s[n][e] = in ? s[n][e] * p.qscale : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
        }
      float alpha[2], base[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
        mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
        const float mn = fmaxf(m[hf], mx[hf]);
        base[hf] = mn == -INFINITY ? 0.f : mn;  // only -inf scores so far
        alpha[hf] = fast_exp2(m[hf] - base[hf]);
        m[hf] = mn;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= alpha[0];
          o[i][1] *= alpha[0];
          o[i][2] *= alpha[1];
          o[i][3] *= alpha[1];
        }
        l[0] *= alpha[0];
        l[1] *= alpha[1];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = fast_exp2(s[n][e] - base[e >> 1]);
          l[e >> 1] += s[n][e];
        }
      const uint32_t pa[4] = {pack2(s[0][0], s[0][1], (T*)nullptr), pack2(s[0][2], s[0][3], (T*)nullptr),
                              pack2(s[1][0], s[1][1], (T*)nullptr), pack2(s[1][2], s[1][3], (T*)nullptr)};
#pragma unroll
      for (int dd = 0; dd < D / 16; ++dd) {
        uint32_t b[4];
        ldsm4t(b, vs + chunk_at(mr + 8 * (mi & 1), 2 * dd + (mi >> 1)));
        mma(o[2 * dd], pa, b[0], b[1], (T*)nullptr);
        mma(o[2 * dd + 1], pa, b[2], b[3], (T*)nullptr);
      }
      __syncwarp();
    }
    cp_async_wait<0>();
    __syncwarp();

#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
      const int r = (lane >> 2) + 8 * hf;
      if (r < im.nrows) {
        const int64_t row = im.prow + r;
        if ((lane & 3) == 0) p.part_ml[row] = make_float2(m[hf], l[hf]);
        float* dst = p.part_o + row * D + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[i][2 * hf], o[i][2 * hf + 1]);
      }
    }
  }
  // the merge waits for this grid alone, so this grid ends after the one before
  if (p.tc_rows) pdl_wait();
}

// ---------------------------------------------------------------------------
// merge: one warp per output row, pieces in a fixed order
// ---------------------------------------------------------------------------

template <typename T, int D>
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ Params p) {
  constexpr int E = D / 32;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= p.B * p.H) return;
  const int64_t b = row / p.H;
  const int32_t h = (int32_t)(row % p.H), kv = h / p.G, g = h % p.G;
  const int32_t own_y = cdiv(p.G, ROWS), own_rows = min(p.G, ROWS);
  const Totals tot = load_plan(p.totals);
  const Seq sp = load_plan(p.seqs + b);
  // this row's pieces: first of its prefix unit, pre_step rows apart, then of its own
  int64_t pre0 = 0, own0 = 0;
  int32_t n_pre = 0, n_own = 0, pre_step = 0;
  if (sp.group >= 0 && sp.from > 0) {
    const Group gp = load_plan(p.groups + sp.group);
    const int32_t rows = gp.n * p.G, r = ((int32_t)b - gp.b0) * p.G + g;
    const int32_t R = gp.tc ? TC_ROWS : ROWS, ry = cdiv(rows, R), nt = cdiv(gp.prefix, gp.tc ? TC_KT : KT);
    const int64_t tiles = gp.tc ? tot.tc_tiles : tot.tiles, workers = gp.tc ? tot.tc_workers : tot.workers;
    const int32_t u = kv * ry + r / R;
    const int64_t a = gp.tile0[gp.tc] + (int64_t)u * nt;
    const int64_t w0 = worker_of(a, tiles, workers);
    n_pre = (int32_t)(worker_of(a + nt - 1, tiles, workers) - w0) + 1;
    pre0 = (gp.tc ? p.tc_row0 : 0) + (gp.unit0[gp.tc] + u + w0) * R + r % R;
    pre_step = R;
    // a unit of at most 128 rows: a piece from each chain
    if (gp.tc && rows - r / R * R <= R / 2) pre_step = R / 2, n_pre *= 2;
  }
  if (sp.ctx > sp.from) {
    const int32_t nt = cdiv(sp.ctx - sp.from, KT), u = kv * own_y + g / ROWS;
    const int64_t a = sp.tile0[0] + (int64_t)u * nt;
    const int64_t w0 = worker_of(a, tot.tiles, tot.workers);
    n_own = (int32_t)(worker_of(a + nt - 1, tot.tiles, tot.workers) - w0) + 1;
    own0 = p.own_row0 + (b * p.HKV * own_y + u + w0) * own_rows + g % ROWS;
  }
  const int n = n_pre + n_own;
  auto piece = [&](int c) -> int64_t {
    return c < n_pre ? pre0 + (int64_t)c * pre_step : own0 + (int64_t)(c - n_pre) * own_rows;
  };
  float M = -INFINITY;
  for (int c = lane; c < n; c += 32) M = fmaxf(M, p.part_ml[piece(c)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float acc[E] = {}, L = 0.f;
#pragma unroll 4
  for (int c = 0; c < n; ++c) {
    const int64_t at = piece(c);
    const float2 ml = p.part_ml[at];
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // a piece without keys, or only scores of -inf
    const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
    L = fmaf(w, ml.y, L);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(w, p.part_o[at * D + e * 32 + lane], acc[e]);
  }
  // no key, or only scores of -inf: L = 0, so out is NaN and lse -inf
  const float inv = 1.f / L;
  T* out = static_cast<T*>(p.out) + row * D;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e * 32 + lane] = T(acc[e] * inv);
  if (p.lse && lane == 0) p.lse[row] = (M + log2f(L)) * kLn2;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Rows of a group from which the tensor-memory kernel takes its prefix.
constexpr int kTcRows = 64;

struct Layout {
  int64_t own_row0, tc_row0;
  size_t groups, seqs, ml, o, total;
};

static int warps_per_cta(int64_t D) {
  return D == 32 ? Cfg<32>::WARPS : D == 64 ? Cfg<64>::WARPS : D == 128 ? Cfg<128>::WARPS : Cfg<256>::WARPS;
}

// Slots for partials: unit + worker < units + workers, for prefixes with ROWS
// rows each, for sequences' own units with min(G, ROWS), for the
// tensor-memory kernel's with TC_ROWS.
static int layout(int64_t B, int64_t NG, int64_t H, int64_t HKV, int64_t D, int sms, Layout* y) {
  const int64_t G = H / HKV, warps = (int64_t)sms * warps_per_cta(D);
  const int64_t pre_units = NG ? HKV * (B * G / ROWS + NG) : 0, own_units = B * HKV * ((G + ROWS - 1) / ROWS);
  y->own_row0 = NG ? (pre_units + warps) * ROWS : 0;
  y->tc_row0 = y->own_row0 + (own_units + warps) * std::min<int64_t>(G, ROWS);
  int64_t rows = y->tc_row0;
  if (NG && B * G >= kTcRows && (D == 64 || D == 128))
    rows += (HKV * (B * G / TC_ROWS + std::min<int64_t>(NG, B * G / kTcRows)) + sms) * TC_ROWS;
  if (rows >= (int64_t(1) << 31)) return PA_ERR_TOO_LARGE;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  y->groups = 256;
  y->seqs = y->groups + up((size_t)NG * sizeof(Group));
  y->ml = y->seqs + up((size_t)B * sizeof(Seq));
  y->o = y->ml + up((size_t)rows * sizeof(float2));
  y->total = y->o + up((size_t)rows * D * sizeof(float));
  return PA_OK;
}

template <typename T, int D>
static int launch_typed(Params& p, int sms, cudaStream_t s) {
  using C = Cfg<D>;
  auto kern = attention_kernel<T, D>;
  static std::mutex mu;
  static std::vector<int> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
      if (e != cudaSuccess) return cuda_status(e);
      done.push_back(dev);
    }
  }
  p.warps = sms * C::WARPS;
  p.tc_ctas = sms;
  plan_kernel<<<1, kPlanThreads, 0, s>>>(p);
  e = cudaGetLastError();
  if (e == cudaSuccess && p.tc_rows) {
    const int st = launch_tc(p, DTypeId<T>::value, D, s);
    if (st) return st;
  }
  if (e == cudaSuccess) e = launch_pdl(kern, dim3((unsigned)sms), dim3(C::WARPS * 32), C::SMEM, s, p);
  if (e == cudaSuccess)
    e = launch_pdl(merge_kernel<T, D>, dim3((unsigned)((p.B * p.H + 7) / 8)), dim3(256), 0, s, p);
  return cuda_status(e);
}

template <typename T>
static int launch_dtype(Params& p, int64_t D, int sms, cudaStream_t s) {
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
  st = shared::layout(num_seqs, num_groups, num_heads, num_kv_heads, head_dim, sms, &y);
  if (st) return st;
  *bytes = y.total;
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
  st = shared::layout(num_seqs, num_groups, num_heads, num_kv_heads, head_dim, sms, &y);
  if (st) return st;
  if (!workspace || workspace_bytes < y.total) return PA_ERR_WORKSPACE;
  if (!aligned16(workspace)) return PA_ERR_ALIGNMENT;
  char* ws = static_cast<char*>(workspace);
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
  p.totals = reinterpret_cast<shared::Totals*>(ws);
  p.groups = reinterpret_cast<shared::Group*>(ws + y.groups);
  p.seqs = reinterpret_cast<shared::Seq*>(ws + y.seqs);
  p.own_row0 = y.own_row0;
  p.tc_row0 = y.tc_row0;
  if (num_groups && num_seqs * p.G >= shared::kTcRows && shared::tc_takes(head_dim, block_size, num_blocks))
    p.tc_rows = shared::kTcRows;
  p.part_ml = reinterpret_cast<float2*>(ws + y.ml);
  p.part_o = reinterpret_cast<float*>(ws + y.o);
  p.dev_status = dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv_dtype == PA_DTYPE_BF16 ? shared::launch_dtype<__nv_bfloat16>(p, head_dim, sms, s)
                                   : shared::launch_dtype<__half>(p, head_dim, sms, s);
}
