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
// Three launches, chained with programmatic dependent launch: a plan (one
// CTA: the groups' usable prefixes, and the work cut into items of nearly
// equal length), the attention itself (one warp per item), and the merge of
// the items' partials.
#include <algorithm>
#include <mutex>
#include <vector>

#include "common.cuh"

namespace pa {
namespace shared {

constexpr int KT = 16;    // keys per tile
constexpr int ROWS = 16;  // query rows per item (the M of one mma)

// What a warp computes: rows r0 .. r0 + nrows - 1 of a unit (row r: sequence
// b0 + r / G, head kvh * G + r % G) against keys t0 .. t1 - 1 of table row
// `table`; partials go to rows prow .. prow + nrows - 1.
struct Item {
  int32_t table, b0, r0, nrows, kvh, t0, t1, prow;
};

// Where a sequence's partials are: piece c of its prefix for KV head kv at row
// pre_row + (kv * n_pre + c) * pre_rows + g, of its own tokens at
// own_row + (kv * n_own + c) * G + g.
struct SeqPlan {
  int32_t n_pre, pre_row, pre_rows, n_own, own_row, ctx, pad[2];
};

struct GroupPlan {
  int32_t b0, n, table, prefix;
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
  int32_t* n_items;
  GroupPlan* groups;
  SeqPlan* seqs;
  Item* items;
  float2* part_ml;  // (running max in log2 units, sum)
  float* part_o;
  int32_t* dev_status;
};

__device__ __forceinline__ int32_t cdiv(int32_t a, int32_t b) { return (a + b - 1) / b; }

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------

constexpr int kPlanThreads = 1024;

// Exclusive scan of (a, b) over the block, with running totals in `base`.
__device__ __forceinline__ int2 block_scan(int2 x, int2* warp_sums, int2& base) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) s.x += a, s.y += b;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int2 w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, w.x, o), b = __shfl_up_sync(0xffffffffu, w.y, o);
      if (lane >= o) w.x += a, w.y += b;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const int2 before = warp ? warp_sums[warp - 1] : make_int2(0, 0);
  const int2 r = make_int2(base.x + before.x + s.x - x.x, base.y + before.y + s.y - x.y);
  base.x += warp_sums[31].x;
  base.y += warp_sums[31].y;
  return r;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ Params p) {
  __shared__ int2 sums[32];
  __shared__ int32_t bad_groups;
  __shared__ unsigned long long total_tiles;
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t B = (int32_t)p.B, NG = (int32_t)p.NG, HKV = (int32_t)p.HKV, G = p.G;
  const int32_t max_ctx = (int32_t)min(p.MB * p.BS, (int64_t)0x7fffff00);
  const int32_t own_tiles_y = cdiv(G, ROWS);
  if (tid == 0) bad_groups = 0, total_tiles = 0;
  __syncthreads();
  // group bounds that are not 0 <= s_0 <= s_1 <= ... <= B: no sharing at all
  for (int32_t g = tid; g < NG; g += kPlanThreads) {
    const int32_t a = p.group_starts[g], b = p.group_starts[g + 1];
    if (a < 0 || b < a || b > B) bad_groups = 1;
  }
  __syncthreads();
  if (bad_groups && tid == 0) report(p.dev_status, PA_DEVERR_GROUP);
  auto context = [&](int32_t b) {
    const int32_t c = p.context_lens[b];
    if (c > max_ctx) report(p.dev_status, PA_DEVERR_CONTEXT);
    return min(max(c, 0), max_ctx);
  };
  // a group's usable prefix: no longer than any member that has tokens; the
  // first such member's table row serves it.  One member alone shares nothing.
  const int32_t groups = bad_groups ? 0 : NG;
  unsigned long long tiles = 0;
  for (int32_t g = warp; g < groups; g += kPlanThreads / 32) {
    const int32_t a = p.group_starts[g], e = p.group_starts[g + 1];
    int32_t least = 0x7fffffff, first = 0x7fffffff, live = 0;
    for (int32_t b = a + lane; b < e; b += 32) {
      const int32_t c = context(b);
      if (c > 0) least = min(least, c), first = min(first, b), ++live;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    first = __reduce_min_sync(0xffffffffu, first);
    live = __reduce_add_sync(0xffffffffu, live);
    const int32_t prefix = live > 1 ? max(0, min(p.prefix_lens[g], least)) : 0;
    if (lane == 0) {
      p.groups[g] = GroupPlan{a, e - a, first, prefix};
      tiles += (unsigned long long)HKV * cdiv((e - a) * G, ROWS) * cdiv(prefix, KT);
    }
  }
  __syncthreads();
  // the group of sequence b (largest g with group_starts[g] <= b), -1: none
  auto group_of = [&](int32_t b) -> int32_t {
    if (groups == 0 || b < p.group_starts[0] || b >= p.group_starts[groups]) return -1;
    int32_t lo = 0, hi = groups;
    while (hi - lo > 1) {
      const int32_t m = (lo + hi) >> 1;
      if (p.group_starts[m] <= b) lo = m;
      else hi = m;
    }
    return lo;
  };
  for (int32_t b = tid; b < B; b += kPlanThreads) {
    const int32_t g = group_of(b), ctx = context(b);
    const int32_t from = g >= 0 ? min(p.groups[g].prefix, ctx) : 0;
    tiles += (unsigned long long)HKV * own_tiles_y * cdiv(ctx - from, KT);
  }
  atomicAdd(&total_tiles, tiles);
  __syncthreads();
  // tiles per item: the whole work over the warps of the launch
  const int32_t C = (int32_t)max((total_tiles + p.warps - 1) / p.warps, 1ull);

  int2 base = make_int2(0, 0);  // (items, partial rows) so far
  for (int32_t g0 = 0; g0 < groups; g0 += kPlanThreads) {
    const int32_t g = g0 + tid;
    GroupPlan gp = {0, 0, 0, 0};
    if (g < groups) gp = p.groups[g];
    const int32_t nt = cdiv(gp.prefix, KT), n = cdiv(nt, C), rows = gp.n * G, ry = cdiv(rows, ROWS);
    const int2 at = block_scan(make_int2(n * HKV * ry, n * HKV * rows), sums, base);
    if (n > 0) {
      int32_t i = at.x;
      for (int32_t kv = 0; kv < HKV; ++kv)
        for (int32_t c = 0; c < n; ++c)
          for (int32_t y = 0; y < ry; ++y)
            p.items[i++] = Item{gp.table, gp.b0, y * ROWS, min(ROWS, rows - y * ROWS), kv,
                                (int32_t)((int64_t)nt * c / n) * KT,
                                min(gp.prefix, (int32_t)((int64_t)nt * (c + 1) / n) * KT),
                                at.y + (kv * n + c) * rows + y * ROWS};
    }
    if (g < groups)
      for (int32_t m = 0; m < gp.n; ++m) {
        SeqPlan& sp = p.seqs[gp.b0 + m];
        sp.n_pre = n;
        sp.pre_row = at.y + m * G;
        sp.pre_rows = rows;
      }
  }
  __syncthreads();
  for (int32_t b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int32_t b = b0 + tid;
    int32_t g = -1, ctx = 0, from = 0;
    if (b < B) {
      g = group_of(b);
      ctx = context(b);
      from = g >= 0 ? min(p.groups[g].prefix, ctx) : 0;
    }
    const int32_t nt = cdiv(ctx - from, KT), n = cdiv(nt, C);
    const int2 at = block_scan(make_int2(n * HKV * own_tiles_y, n * HKV * G), sums, base);
    if (b < B) {
      SeqPlan& sp = p.seqs[b];
      if (g < 0 || ctx == 0) sp.n_pre = 0;
      sp.n_own = n;
      sp.own_row = at.y;
      sp.ctx = ctx;
      int32_t i = at.x;
      for (int32_t kv = 0; kv < HKV; ++kv)
        for (int32_t c = 0; c < n; ++c)
          for (int32_t y = 0; y < own_tiles_y; ++y)
            p.items[i++] = Item{b, b, y * ROWS, min(ROWS, G - y * ROWS), kv,
                                from + (int32_t)((int64_t)nt * c / n) * KT,
                                min(ctx, from + (int32_t)((int64_t)nt * (c + 1) / n) * KT),
                                at.y + (kv * n + c) * G + y * ROWS};
    }
  }
  if (tid == 0) *p.n_items = base.x;
}

// ---------------------------------------------------------------------------
// attention: one warp per item
// ---------------------------------------------------------------------------

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
  pdl_wait();
  pdl_trigger();
  const uint32_t ring = smem_u32(smem) + warp * C::WARP;
  const int32_t n_items = *p.n_items;
  // rows of a tile sit `D * 2` bytes apart with their 16-byte chunks permuted
  // by the row, so the eight rows of a matrix load fall on different banks
  auto chunk_at = [](int row, int c) -> uint32_t {
    return (uint32_t)(row * (D * 2) + ((c ^ (CH >= 8 ? (row & 7) : ((row >> 1) & 3))) << 4));
  };
  // consecutive items go to different SMs
  for (int32_t it = warp * gridDim.x + blockIdx.x; it < n_items; it += p.warps) {
    const int4 w0 = reinterpret_cast<const int4*>(p.items + it)[0];
    const int4 w1 = reinterpret_cast<const int4*>(p.items + it)[1];
    const Item im = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    const int n_tiles = (im.t1 - im.t0 + KT - 1) / KT;
    const int32_t* table = p.block_tables + (int64_t)im.table * p.MB;

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
  const SeqPlan sp = p.seqs[b];
  const int n = sp.n_pre + sp.n_own;
  auto piece = [&](int c) -> int64_t {
    return c < sp.n_pre ? (int64_t)sp.pre_row + (int64_t)(kv * sp.n_pre + c) * sp.pre_rows + g
                        : (int64_t)sp.own_row + (int64_t)(kv * sp.n_own + c - sp.n_pre) * p.G + g;
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

struct Layout {
  size_t groups, seqs, items, ml, o, total;
};

static int warps_per_cta(int64_t D) {
  return D == 32 ? Cfg<32>::WARPS : D == 64 ? Cfg<64>::WARPS : D == 128 ? Cfg<128>::WARPS : Cfg<256>::WARPS;
}

// Items: a unit (rows x KV head) of x tiles makes ceil(x / C) of them with
// C >= sum x / warps, so at most warps + units in all; an item has at most
// ROWS rows, so the partial rows are at most ROWS x warps + the units' rows.
static int layout(int64_t B, int64_t NG, int64_t H, int64_t HKV, int64_t D, int sms, Layout* y) {
  const int64_t G = H / HKV, warps = (int64_t)sms * warps_per_cta(D);
  const int64_t units = HKV * ((B * G + ROWS - 1) / ROWS + NG + B * ((G + ROWS - 1) / ROWS));
  const int64_t items = warps + units, rows = ROWS * warps + 2 * B * H;
  if (items >= (int64_t(1) << 31) || rows >= (int64_t(1) << 31)) return PA_ERR_TOO_LARGE;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  y->groups = 256;
  y->seqs = y->groups + up((size_t)NG * sizeof(GroupPlan));
  y->items = y->seqs + up((size_t)B * sizeof(SeqPlan));
  y->ml = y->items + up((size_t)items * sizeof(Item));
  y->o = y->ml + up((size_t)rows * sizeof(float2));
  y->total = y->o + up((size_t)rows * D * sizeof(float));
  return PA_OK;
}

template <typename K>
static cudaError_t launch_pdl(K kern, dim3 grid, dim3 block, size_t smem, cudaStream_t s, const Params& p) {
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
  plan_kernel<<<1, kPlanThreads, 0, s>>>(p);
  e = cudaGetLastError();
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
  p.n_items = reinterpret_cast<int32_t*>(ws);
  p.groups = reinterpret_cast<shared::GroupPlan*>(ws + y.groups);
  p.seqs = reinterpret_cast<shared::SeqPlan*>(ws + y.seqs);
  p.items = reinterpret_cast<shared::Item*>(ws + y.items);
  p.part_ml = reinterpret_cast<float2*>(ws + y.ml);
  p.part_o = reinterpret_cast<float*>(ws + y.o);
  p.dev_status = dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv_dtype == PA_DTYPE_BF16 ? shared::launch_dtype<__nv_bfloat16>(p, head_dim, sms, s)
                                   : shared::launch_dtype<__half>(p, head_dim, sms, s);
}
