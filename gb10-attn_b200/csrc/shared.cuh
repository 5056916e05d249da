// shared.cuh -- what the launches of the shared-prefix decode have in common:
// how its work is counted, cut and numbered, the plan, and a warp's part of the
// work (shared.cu has the launch for pools that the tensor-memory part cannot
// load, the merge and the entry points, shared_tc.cu the launch that has both).
#pragma once

#include "common.cuh"

namespace pa {
namespace shared {

constexpr int KT = 16;    // keys per tile
constexpr int ROWS = 16;  // query rows per item (the M of one mma)

// tensor-memory part: keys per tile, rows per unit (two chains of 128; a unit
// of at most 128 rows gives both chains the same rows and every other tile)
constexpr int TC_KT = 64;
constexpr int TC_ROWS = 256;

// The work, counted in tiles of KT keys: first the groups' prefixes, then the
// sequences' own tokens.  A unit is one (group or sequence, KV head, tile of
// rows); its tiles are consecutive, and the units of a group or sequence too,
// in the order (KV head, tile of rows).  The `warps` workers of a launch take
// equal consecutive runs of the total, worker w the tiles
// [w T / W, (w + 1) T / W), so a unit is cut where a worker's run ends.  A piece
// is the overlap of unit u and worker w; u + w grows strictly from piece to
// piece, so it numbers the pieces' slots for partials, with no table of them.
//   A unit counts as a few tiles more than it has, before its first: what taking
// it up costs (its queries, the partials of the one before), so that workers
// that meet a unit's start have less to read.  A piece of these alone is empty.
//   The prefixes of groups with many rows are done in tensor memory
// (shared_tc.cu), with tiles, units and workers (CTAs) of their own, numbered
// the same way.  Some CTAs do these then and the others' warps the rest.
struct alignas(16) Group {
  long long tile0[2];           // first tile: of the warps' work, of the tensor memory's
  int32_t b0, n, table, prefix; // members b0 .. b0 + n - 1; table row that serves; tokens shared
  int32_t unit0[2], tc, pad;    // first unit; whether it is done in tensor memory
};
struct alignas(16) Seq {
  long long tile0[1];             // counted from the end of the prefixes
  int32_t from, ctx, group, pad;  // own tokens from .. ctx - 1; its group or -1
};
struct alignas(16) Totals {
  int64_t prefix_tiles, tiles, workers;  // the warps' work
  int64_t tc_tiles, tc_workers;          // the tensor memory's
  int64_t own_cta0, pad;                 // first CTA whose warps take work
};

// Where the partials of an output row are: n_pre pieces of its prefix unit,
// pre_step rows apart, and n_own of its own.
struct alignas(16) Pieces {
  int64_t pre0, own0;
  int32_t n_pre, n_own, pre_step, pad;
};

struct Params {
  void* out;
  float* lse;  // [B, H]
  const void *q, *k, *v;
  const int32_t *block_tables, *context_lens, *group_starts, *prefix_lens;
  int64_t B, NG, H, HKV, BS, NB, MB;
  float qscale;     // scale * log2(e)
  int32_t G;        // query heads per KV head
  int32_t warps;    // warps of the attention launch that take work
  int32_t bs_shift; // log2(BS) if BS is a power of two, else -1
  // workspace
  char* plan;           // the plan (Plan below); every CTA that makes its own has one
  int64_t plan_bytes;   // bytes of one
  int64_t group_off, seq_off, scratch_off;  // its groups, sequences, scratch (made by plan_kernel only)
  int32_t planned;      // a launch of its own makes the plan
  Pieces* pieces;       // [B, H]
  float2* part_ml;  // (running max in log2 units, sum)
  float* part_o;
  int64_t own_row0; // first partial row of the sequences' own units
  int64_t tc_row0;  // and of the tensor memory's units
  int32_t tc_rows;  // rows from which a group's prefix goes to the tensor memory (0: none does)
  int32_t tc_ctas;
  int32_t waits;        // 0: the tensor memory's softmax gives up at its first tile (pa_set_shared_waits)
  int32_t* dev_status;
};

__host__ __device__ __forceinline__ int32_t cdiv(int32_t a, int32_t b) { return (a + b - 1) / b; }

// Worker w's first tile, and the worker of tile x, for T tiles over W workers
// (in 32 bits where that holds the products: the division is several times
// shorter, and stands in the way of a call's first loads).
__device__ __forceinline__ int64_t first_tile(int64_t w, int64_t T, int64_t W) {
  if ((w | W) < 0x10000 && T < 0x10000) return (uint32_t)w * (uint32_t)T / (uint32_t)W;
  return w * T / W;
}
__device__ __forceinline__ int64_t worker_of(int64_t x, int64_t T, int64_t W) {
  if (T < 0x10000 && W < 0x10000) return ((uint32_t)(x + 1) * (uint32_t)W - 1) / (uint32_t)T;
  return ((x + 1) * W - 1) / T;
}

// One of the structs above, in 16-byte loads.
template <typename E> __device__ __forceinline__ E load_plan(const E* e) {
  static_assert(sizeof(E) % 16 == 0, "");
  union {
    int4 w[sizeof(E) / 16];
    E e;
  } u;
#pragma unroll
  for (int i = 0; i < (int)sizeof(E) / 16; ++i) u.w[i] = reinterpret_cast<const int4*>(e)[i];
  return u.e;
}

// The last of n entries (their tile0[I] rising from at most x) with
// tile0[I] <= x.  All lanes probe at once: two steps for 1024 entries.
template <int I, typename E>
__device__ __forceinline__ int32_t find(const E* e, int32_t n, int64_t x, int lane) {
  int32_t lo = 0, len = n;  // the answer is in [lo, lo + len)
  while (len > 1) {
    const int32_t step = (len + 31) / 32, at = lo + lane * step;
    const uint32_t m = __ballot_sync(0xffffffffu, lane * step < len && e[at].tile0[I] <= x);
    const int32_t k = 31 - __clz(m);
    len = min(step, len - k * step);
    lo += k * step;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------

struct Plan {
  Totals* totals;
  Group* groups;
  Seq* seqs;
};
__device__ __forceinline__ Plan plan_at(const Params& p, int64_t copy) {
  char* base = p.plan + copy * p.plan_bytes;
  return {reinterpret_cast<Totals*>(base), reinterpret_cast<Group*>(base + p.group_off),
          reinterpret_cast<Seq*>(base + p.seq_off)};
}

// Sequences and groups up to which every CTA makes the plan itself, in shared
// memory, if its counts fit 32 bits: one launch less, which small calls notice.
constexpr int kPlanMax = 1024;
constexpr int64_t kScanBytes = 2 * 32 * 40 + 16;  // the scans' sums, two counters
__host__ __device__ constexpr int64_t plan_scratch(int64_t B, int64_t NG) {
  return kScanBytes + (2 * B + 3 * (NG + 1)) * 4;
}

// 16-key tiles per warp when there are few: 2, 3, 4 give 12.8, 13.3, 14.3 us for
// four samples of 512 tokens, 29.9, 23.7, 22.0 for one sequence of 20k (its
// pieces are more to merge).
constexpr int kMinTiles = 3;
// 64-key tiles per CTA below which the warps do all.  Over 66 batches (2 to 1024
// sequences of 8 to 512 rows a group, prefixes of 16 to 32768, head_dim 64 and 128) 2 and 4
// take as long as 6 in the mean (2: 0.85 times for 64 on 2k with 32 / 8 heads, 1.06 at
// most), 9 1.04 and 14 1.04 times: up to 2.2 times for 64 on 8k, which has 7 tiles a CTA
// (41 us, 90), 0.85 times for 16 groups on 16 tokens.
constexpr int kTcMinTiles = 6;
// Tiles that a unit costs beside its own (swept: 1, 2, 4 of 16 keys and 2, 5, 8,
// 14 of 64 keys give 76-82 us for 128 sequences on 8k, 56-60 for seven prompts,
// each best at another; these are within 3 % of the best of both).
constexpr int kUnitCost = 2;
constexpr int kTcUnitCost = 6;

// What a warps' tile and a tensor-memory tile of one chain's rows cost an SM,
// in percent of a tensor-memory tile of both chains (0.15 and 1.2 us).  Swept: 11,
// 12, 13 with 75 to 85 give 260, 268, 245 us for 256 sequences on 32k (too few
// CTAs for the own tokens are dear there), 63, 63, 65 for 128 on 8k, 50 for seven
// prompts with any of them.  Swept with head_dim 128 and four query heads a KV head;
// others take the same.
constexpr double kTileCost = 13, kTcSmallCost = 85;

// Tiles that a unit of `keys` keys counts as.
__host__ __device__ __forceinline__ int32_t unit_tiles(int32_t keys) { return keys ? cdiv(keys, KT) + kUnitCost : 0; }
__host__ __device__ __forceinline__ int32_t tc_unit_tiles(int32_t keys) {
  return keys ? cdiv(keys, TC_KT) + kTcUnitCost : 0;
}

// Exclusive scan of N counts over the block on top of the running totals
// `base`; warp_sums: one entry a warp, not in use by an earlier scan any more.
// I: 32 bits where the host knows that the counts fit.
template <typename I, int N> struct Sums {
  I v[N];
};
template <typename I, int N>
__device__ __forceinline__ Sums<I, N> block_scan(const Sums<I, N>& x, Sums<I, N>* warp_sums, Sums<I, N>& base) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  auto warp_scan = [&](Sums<I, N> s) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const I y = __shfl_up_sync(0xffffffffu, s.v[i], o);
        if (lane >= o) s.v[i] += y;
      }
    return s;
  };
  const Sums<I, N> s = warp_scan(x);
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  const Sums<I, N> all = warp_scan(lane < warps ? warp_sums[lane] : Sums<I, N>{});
  Sums<I, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const I before = __shfl_sync(0xffffffffu, all.v[i], max(warp - 1, 0));
    r.v[i] = base.v[i] + (warp ? before : 0) + s.v[i] - x.v[i];
    base.v[i] += __shfl_sync(0xffffffffu, all.v[i], 31);
  }
  return r;
}

// One CTA makes the plan; `scratch`: plan_scratch() bytes, in shared memory or
// its own part of the workspace.  Ends with a barrier.  3 to 4 us of loads, scans
// and barriers, for 4 sequences as for 256.
template <typename I>
__device__ __forceinline__ void make_plan(const Params& p, const Plan& out, void* scratch, bool tell) {
  using S = Sums<I, 5>;
  auto sums = static_cast<S(*)[32]>(scratch);
  // the tensor memory's tiles if it takes what it may, and those of them in
  // units of one chain's rows
  auto tc_work = reinterpret_cast<unsigned long long*>(static_cast<char*>(scratch) + 2 * 32 * 40);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const int32_t B = (int32_t)p.B, NG = (int32_t)p.NG, HKV = (int32_t)p.HKV, G = p.G;
  const int32_t max_ctx = (int32_t)min(p.MB * p.BS, (int64_t)0x7fffff00);
  int32_t *ctx = reinterpret_cast<int32_t*>(static_cast<char*>(scratch) + kScanBytes), *grp = ctx + B, *gs = grp + B, *pre = gs + NG + 1, *lead = pre + NG + 1;
  if (tid == 0) tc_work[0] = tc_work[1] = 0;
  int far = 0;
  for (int32_t b = tid; b < B; b += threads) {
    const int32_t c = p.context_lens[b];
    far |= c > max_ctx;
    ctx[b] = min(max(c, 0), max_ctx);
    grp[b] = -1;
  }
  for (int32_t g = tid; g < NG; g += threads) pre[g] = p.prefix_lens[g];
  for (int32_t g = tid; g <= NG && NG; g += threads) gs[g] = p.group_starts[g];
  if (far && tell) report(p.dev_status, PA_DEVERR_CONTEXT);
  __syncthreads();
  // group bounds that are not 0 <= s_0 <= s_1 <= ... <= B: no sharing at all
  int bad = 0;
  for (int32_t g = tid; g < NG; g += threads) bad |= gs[g] < 0 || gs[g + 1] < gs[g] || gs[g + 1] > B;
  bad = __syncthreads_or(bad);
  if (bad && tid == 0 && tell) report(p.dev_status, PA_DEVERR_GROUP);
  const int32_t groups = bad ? 0 : NG;
  // a group's usable prefix: no longer than any member that has tokens; the
  // first such member's table row serves it.  One member alone shares nothing.
  for (int32_t g = warp; g < groups; g += threads / 32) {
    const int32_t a = gs[g], e = gs[g + 1];
    int32_t least = 0x7fffffff, first = 0x7fffffff, live = 0;
    for (int32_t b = a + lane; b < e; b += 32) {
      const int32_t c = ctx[b];
      if (c > 0) least = min(least, c), first = min(first, b), ++live;
      grp[b] = g;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    first = __reduce_min_sync(0xffffffffu, first);
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) {
      const int32_t prefix = live > 1 ? max(0, min(pre[g], least)) : 0;
      pre[g] = prefix;
      lead[g] = first;
      const int32_t rows = (e - a) * G;
      if (p.tc_rows && rows >= p.tc_rows) {
        const unsigned long long n = (unsigned long long)HKV * tc_unit_tiles(prefix);
        atomicAdd(&tc_work[0], n * cdiv(rows, TC_ROWS));
        if ((rows - 1) % TC_ROWS < TC_ROWS / 2) atomicAdd(&tc_work[1], n);
      }
    }
  }
  __syncthreads();
  const bool use_tc = p.tc_rows && tc_work[0] >= (unsigned long long)kTcMinTiles * p.tc_ctas;
  // running counts: the groups' tiles and units (the warps', the tensor
  // memory's), the sequences' tiles
  S base = {};
  for (int32_t i0 = 0, k = 0; i0 < max(B, groups); i0 += threads, k ^= 1) {
    const int32_t i = i0 + tid;
    S x = {};
    int32_t n = 0, prefix = 0, tc = 0, from = 0, g = -1;
    if (i < groups) {
      n = gs[i + 1] - gs[i];
      prefix = pre[i];
      tc = use_tc && n * G >= p.tc_rows;
      const I units = (I)HKV * cdiv(n * G, tc ? TC_ROWS : ROWS);
      x = tc ? S{{0, units * tc_unit_tiles(prefix), 0, units, 0}} : S{{units * unit_tiles(prefix), 0, units, 0, 0}};
    }
    if (i < B) {
      g = grp[i];
      if (g >= 0) from = min(pre[g], ctx[i]);
      x.v[4] = (I)HKV * cdiv(G, ROWS) * unit_tiles(ctx[i] - from);
    }
    const S at = block_scan(x, sums[k], base);
    if (i < groups)
      out.groups[i] = Group{{at.v[0], at.v[1]}, gs[i], n, lead[i], prefix, {(int32_t)at.v[2], (int32_t)at.v[3]}, tc, 0};
    if (i < B) out.seqs[i] = Seq{{at.v[4]}, from, ctx[i], g, 0};
  }
  if (tid == 0) {
    const int64_t tiles = (int64_t)base.v[0] + base.v[4], tc_tiles = base.v[1];
    // The CTAs that take the warps' work: with tensor-memory work beside it as
    // many as their part of the cost, so that both end together.  (All CTAs for
    // one and then for the other leave HBM idle first and the tensor cores next:
    // 256 sequences on 32k 260 us, so 245, 128 on 8k 74 and 64, seven prompts 57 and
    // 51.)
    int64_t own0 = 0, own_ctas = p.tc_ctas, tc_ctas = p.tc_ctas;
    if (tc_tiles && tiles && tc_ctas > 1) {
      const double own = (double)kTileCost * (double)tiles;
      const double tc = 100. * (double)tc_work[0] - (100. - kTcSmallCost) * (double)tc_work[1];
      own_ctas = min(max((int64_t)(own / (own + tc) * p.tc_ctas + 0.5), (int64_t)1), tc_ctas - 1);
      tc_ctas -= own_ctas;
      own0 = tc_ctas;
    }
    const int64_t warps = min((int64_t)p.warps / p.tc_ctas * own_ctas, max((tiles + kMinTiles - 1) / kMinTiles, (int64_t)1));
    *out.totals = Totals{base.v[0], tiles, warps, tc_tiles, min(tc_ctas, max(tc_tiles, (int64_t)1)), own0, 0};
  }
  __syncthreads();
}

// The plan that this CTA works by.
__device__ __forceinline__ Plan take_plan(const Params& p, void* smem_scratch) {
  if (p.planned) {
    pdl_wait();
    return plan_at(p, 0);
  }
  const Plan plan = plan_at(p, blockIdx.x);
  make_plan<int32_t>(p, plan, smem_scratch, blockIdx.x == 0);
  return plan;
}

// ---------------------------------------------------------------------------
// a warp's work: its run of 16-key tiles
// ---------------------------------------------------------------------------

// What a warp computes at a time: rows r0 .. r0 + nrows - 1 of a unit (row r:
// sequence b0 + r / G, head kvh * G + r % G) against keys t0 .. t1 - 1 of table
// row `table`; partials from row prow on.
struct Item {
  int32_t table, b0, r0, nrows, kvh, t0, t1;
  int64_t prow;
};

// The items of a worker's run, in order.
struct Run {
  const Group* groups;
  const Seq* seqs;
  int64_t left, worker, slot;    // tiles left; partial row of the entry's unit 0
  int32_t at, u, j, nt, units;   // entry (a group, or a sequence if !pre), unit and tile in it
  int32_t table, b0, rows, from, to, unit_y;
  bool pre;

  __device__ __forceinline__ Run(const Params& p, const Plan& plan, const Totals& tot, int64_t w, int lane)
      : groups(plan.groups), seqs(plan.seqs), left(0), worker(w) {
    at = u = j = units = 0;
    pre = false;
    if (w >= tot.workers) return;
    int64_t x = first_tile(w, tot.tiles, tot.workers);
    left = first_tile(w + 1, tot.tiles, tot.workers) - x;
    if (left == 0) return;
    pre = x < tot.prefix_tiles;
    if (!pre) x -= tot.prefix_tiles;
    at = pre ? find<0>(groups, (int32_t)p.NG, x, lane) : find<0>(seqs, (int32_t)p.B, x, lane);
    const int64_t done = x - entry(p);
    u = (int32_t)(done / nt);
    j = (int32_t)(done - (int64_t)u * nt);
  }
  // Takes up entry `at`; its first tile.
  __device__ __forceinline__ int64_t entry(const Params& p) {
    int64_t tile0;
    if (pre) {
      const Group gp = load_plan(groups + at);
      tile0 = gp.tile0[0];
      table = gp.table;
      b0 = gp.b0;
      rows = gp.n * p.G;
      from = 0;
      to = gp.tc ? 0 : gp.prefix;
      slot = (int64_t)gp.unit0[0] * ROWS;
    } else {
      const Seq sp = load_plan(seqs + at);
      tile0 = sp.tile0[0];
      table = b0 = at;
      rows = p.G;
      from = sp.from;
      to = sp.ctx;
      slot = p.own_row0 + (int64_t)at * p.HKV * cdiv(p.G, ROWS) * min(p.G, ROWS);
    }
    nt = unit_tiles(to - from);
    unit_y = cdiv(rows, ROWS);
    units = nt ? (int32_t)p.HKV * unit_y : 0;
    return tile0;
  }
  __device__ __forceinline__ bool next(const Params& p, Item& im) {
    if (left == 0) return false;
    while (u == units) {  // (an entry with tiles follows, since some are left)
      if (++at == p.NG && pre) pre = false, at = 0;
      entry(p);
      u = 0;
    }
    const int32_t n = (int32_t)min((int64_t)(nt - j), left);
    im.table = table;
    im.b0 = b0;
    im.kvh = u / unit_y;
    im.r0 = (u - im.kvh * unit_y) * ROWS;
    im.nrows = min(ROWS, rows - im.r0);
    im.t0 = from + max(j - kUnitCost, 0) * KT;
    im.t1 = min(to, from + max(j + n - kUnitCost, 0) * KT);
    im.prow = slot + (u + worker) * (pre ? ROWS : min(p.G, ROWS));
    left -= n;
    j += n;
    if (j == nt) j = 0, ++u;
    return true;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
               "l"(policy)
               : "memory");
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

// One stage of a warp's ring: the K rows of a tile, then its V rows.
__host__ __device__ constexpr uint32_t stage_bytes(int D) { return 2 * KT * D * 2; }

// The pieces of output row `row`.
__device__ __forceinline__ Pieces locate(const Params& p, const Plan& plan, const Totals& tot, int64_t row) {
  const int64_t b = row / p.H;
  const int32_t h = (int32_t)(row % p.H), kv = h / p.G, g = h % p.G;
  const int32_t own_y = cdiv(p.G, ROWS), own_rows = min(p.G, ROWS);
  const Seq sp = load_plan(plan.seqs + b);
  int64_t pre0 = 0, own0 = 0;
  int32_t n_pre = 0, n_own = 0, pre_step = 0;
  if (sp.group >= 0 && sp.from > 0) {
    const Group gp = load_plan(plan.groups + sp.group);
    const int32_t rows = gp.n * p.G, r = ((int32_t)b - gp.b0) * p.G + g;
    const int32_t R = gp.tc ? TC_ROWS : ROWS, ry = cdiv(rows, R);
    const int32_t nt = gp.tc ? tc_unit_tiles(gp.prefix) : unit_tiles(gp.prefix);
    const int64_t tiles = gp.tc ? tot.tc_tiles : tot.tiles, workers = gp.tc ? tot.tc_workers : tot.workers;
    const int32_t u = kv * ry + r / R;
    const int64_t a = (gp.tc ? gp.tile0[1] : gp.tile0[0]) + (int64_t)u * nt;
    const int64_t w0 = worker_of(a, tiles, workers);
    n_pre = (int32_t)(worker_of(a + nt - 1, tiles, workers) - w0) + 1;
    pre0 = (gp.tc ? p.tc_row0 : 0) + ((gp.tc ? gp.unit0[1] : gp.unit0[0]) + u + w0) * R + r % R;
    pre_step = R;
    // a unit of at most 128 rows: a piece from each chain
    if (gp.tc && rows - r / R * R <= R / 2) pre_step = R / 2, n_pre *= 2;
  }
  if (sp.ctx > sp.from) {
    const int32_t nt = unit_tiles(sp.ctx - sp.from), u = kv * own_y + g / ROWS;
    const int64_t a = tot.prefix_tiles + sp.tile0[0] + (int64_t)u * nt;
    const int64_t w0 = worker_of(a, tot.tiles, tot.workers);
    n_own = (int32_t)(worker_of(a + nt - 1, tot.tiles, tot.workers) - w0) + 1;
    own0 = p.own_row0 + (b * p.HKV * own_y + u + w0) * own_rows + g % ROWS;
  }
  return {pre0, own0, n_pre, n_own, pre_step, 0};
}

// A worker's share of the rows, for the merge.  Every worker of the launch calls
// it, with work or without.
__device__ __forceinline__ void locate_rows(const Params& p, const Plan& plan, const Totals& tot, int64_t worker) {
  for (int64_t r = worker * 32 + (threadIdx.x & 31); r < p.B * p.H; r += (int64_t)p.warps * 32)
    p.pieces[r] = locate(p, plan, tot, r);
}

// A warp streams its items through a ring of its own: for each the rows of Q,
// then tile after tile the rows of K and V (16-byte asynchronous copies, so any
// page size and any first token serve).  The copies run NST - 1 stages ahead
// across items, and the block ids one stage further, so no item waits for its
// first bytes: with a few tiles an item that wait was most of the time.
//   The keys of a tile are the N of S = Q K^T and the K of P V; the running
// maximum and sum, the products' sums and O stay in fp32 registers.  P is rounded
// to the pool's type for the second product (by 2^-9 or 2^-12 of a weight at most
// and averaged over the keys: at the level of the output's own rounding; in fp16 a
// weight below 2^-14 of the piece's largest by up to 2^-25 of that, which
// reaches the output's own rounding when some 2^13 keys weigh that little beside
// one); the sum l is of the unrounded weights.
//   HBM-bound on long runs on all SMs: 256 sequences' own 671 MB of 8 KV heads of 128
// in 105 us (6.4 TB/s).  On fewer of them bound by the latency of its instructions,
// 0.15 us a tile and SM, and some four such an item where units have a tile or two:
// 181 sequences of 32 / 32 heads, 85 MB in all, take 57 us.
template <typename T, int D, int NST>
__device__ __forceinline__ void warp_work(const Params& p, const Plan& plan, const Totals& tot, uint32_t ring,
                                          int64_t worker, int64_t index) {
  constexpr int CH = D / 8;  // 16-byte chunks per row
  constexpr uint32_t STAGE = stage_bytes(D), NONE = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  // rows of a tile sit `D * 2` bytes apart with their 16-byte chunks permuted
  // by the row, so the eight rows of a matrix load fall on different banks
  auto chunk_at = [](int row, int c) -> uint32_t {
    return (uint32_t)(row * (D * 2) + ((c ^ (CH >= 8 ? (row & 7) : ((row >> 1) & 3))) << 4));
  };

  // ---- the copies' side: what goes into the next stage
  Run ahead(p, plan, tot, worker, lane);
  Run run = ahead;
  Item ld = {};
  int32_t ld_j = 0, ld_n = 0;   // stage of item ld (0: Q), its stages
  uint32_t row = NONE;          // the coming stage: the row of this lane (of D elements; lanes 0-15)
  int kind = 0;                 // and what it is: 0 nothing, 1 Q, 2 a tile
  int32_t ids = 0, page0 = 0;   // block ids of pages page0 + lane of item ld
  auto page_of = [&](int32_t t) { return p.bs_shift >= 0 ? t >> p.bs_shift : t / (int32_t)p.BS; };
  auto load_ids = [&](int32_t t) {
    page0 = page_of(t);
    ids = page0 + lane <= page_of(ld.t1 - 1) ? __ldg(p.block_tables + (int64_t)ld.table * p.MB + page0 + lane) : 0;
  };
  auto plan_stage = [&] {
    if (ld_j == ld_n) {
      kind = 0;
      if (!ahead.next(p, ld)) return;
      ld_j = 0;
      ld_n = 1 + cdiv(ld.t1 - ld.t0, KT);
    }
    row = NONE;
    if (ld_j == 0) {
      kind = 1;
      if (ld_n > 1) load_ids(ld.t0);  // needed a stage later
      const int32_t r = ld.r0 + lane;
      if (lane < ld.nrows) row = (uint32_t)((ld.b0 + r / p.G) * (int32_t)p.H + ld.kvh * p.G + r % p.G);
    } else {
      kind = 2;
      const int32_t t0 = ld.t0 + (ld_j - 1) * KT, t = t0 + lane, page = page_of(t);
      if (page_of(min(t0 + KT, ld.t1) - 1) >= page0 + 32) load_ids(t0);
      int32_t blk = __shfl_sync(0xffffffffu, ids, page - page0);
      if (lane < KT && t < ld.t1) {
        if (blk < 0 || blk >= p.NB) {
          report(p.dev_status, PA_DEVERR_BLOCK_ID);
          blk = 0;
        }
        row = (uint32_t)(((int64_t)blk * p.BS + (t - page * (int32_t)p.BS)) * p.HKV + ld.kvh);
      }
    }
    ++ld_j;
  };
  // Rows of no key or query are zeros: their scores are masked, and no weight
  // of zero meets a NaN of an unwritten row.
  // Most are read once: all leave the L2 first, which keeps prefixes that several
  // units read (128 sequences on 8k 64 -> 61 us, 100 of 24 / 8 heads on 4k 55 -> 52,
  // 14 on 15k 27 -> 25.5; 256 on 32k 238 -> 246).
  uint64_t once;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
  auto fill = [&](uint32_t st, int kind, uint32_t row) {
    if (kind) {
      const char* a = static_cast<const char*>(kind == 1 ? p.q : p.k);
#pragma unroll
      for (int i = 0; i < KT * CH / 32; ++i) {
        const int idx = i * 32 + lane, r = idx / CH, c = idx % CH;
        const uint32_t pr = __shfl_sync(0xffffffffu, row, r);
        const int bytes = pr == NONE ? 0 : 16;
        const int64_t off = bytes ? ((int64_t)pr * CH + c) * 16 : 0;
        cp_async16(ring + st + chunk_at(r, c), a + off, bytes, once);
        if (kind == 2)
          cp_async16(ring + st + KT * D * 2 + chunk_at(r, c), static_cast<const char*>(p.v) + off, bytes, once);
      }
    }
    cp_async_commit();
  };
  uint32_t st_ld = 0, st = 0;  // stage to fill, stage to read
  auto step = [](uint32_t& s) { s = s + STAGE == NST * STAGE ? 0 : s + STAGE; };
  plan_stage();
#pragma unroll 1
  for (int i = 0; i < NST - 1; ++i) {
    const uint32_t r = row;
    const int k = kind;
    plan_stage();
    fill(st_ld, k, r);
    step(st_ld);
  }
  // The stage at `st` is there, and the one before it, which every lane has
  // left, is being filled.
  auto arrive = [&] {
    const uint32_t r = row;
    const int k = kind;
    plan_stage();
    cp_async_wait<NST - 2>();
    __syncwarp();
    fill(st_ld, k, r);
    step(st_ld);
  };

  // While the first bytes are on their way
  locate_rows(p, plan, tot, index);

  // ---- the products' side
  const int mi = lane >> 3, mr = lane & 7;  // matrix and row that this lane addresses
  Item im;
  while (run.next(p, im)) {
    arrive();
    uint32_t qa[D / 16][4];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) ldsm4(qa[kk], ring + st + chunk_at(mr + 8 * (mi & 1), 2 * kk + (mi >> 1)));
    step(st);
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int valid = im.t1 - im.t0; valid > 0; valid -= KT) {
      arrive();
      const uint32_t ks = ring + st, vs = ks + KT * D * 2;
      float s[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t b[4];
        ldsm4(b, ks + chunk_at(mr + 8 * (mi >> 1), 2 * kk + (mi & 1)));
        mma(s[0], qa[kk], b[0], b[1], (T*)nullptr);
        mma(s[1], qa[kk], b[2], b[3], (T*)nullptr);
      }
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
      step(st);
    }

#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
      const int r = (lane >> 2) + 8 * hf;
      if (r < im.nrows) {
        const int64_t out = im.prow + r;
        if ((lane & 3) == 0) p.part_ml[out] = make_float2(m[hf], l[hf]);
        float* dst = p.part_o + out * D + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[i][2 * hf], o[i][2 * hf + 1]);
      }
    }
  }
  cp_async_wait<0>();
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// `after`: as a programmatic dependent of the launch before it.
template <typename K, typename A>
inline cudaError_t launch(K kern, int64_t grid, int block, size_t smem, cudaStream_t s, const A& p, bool after) {
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

// The attention launch with the tensor-memory part (shared_tc.cu): which pools
// it can load, how many of a CTA's warps take 16-key tiles, the launch.
bool tc_takes(int64_t D, int64_t BS, int64_t NB);
constexpr int kTcWarps = 8;
int launch_tc(const Params& p, int dtype, int64_t D, cudaStream_t s);

}  // namespace shared
}  // namespace pa
