// shared_tc.cu -- the attention launch of the shared-prefix decode for pools
// that tiled TMA can load (whole 16-row groups inside a page, head_dim 64 or
// 128): first the prefixes shared by many query rows, on the sm_100a tensor
// cores with S, P and O in tensor memory, then the rest, a warp at a time
// (shared.cuh).
//
// A CTA (one per SM) takes its run of 128-key tiles and walks the units that it
// crosses: the members' query heads of one KV head are the rows of S = Q K^T and
// O = P V.  Two softmax warpgroups run two chains: rows 0-127 and 128-255 of a
// unit, or, in a unit of at most 128 rows, the same rows on every other tile,
// so that one chain's exponentials overlap the other's products.
// Thread = row = TMEM lane: it reads its 128 scores, keeps the row's reference
// maximum and sum in fp32 and writes P over S.  Two warps feed K and V by tiled
// TMA, 16 rows at a time through the pages; one thread issues the MMAs.
//   Precision: one 16-bit product each for S (Q and K as they are, products
// exact, fp32 sums) and P V (P rounded to 16 bits, as the output will be; the
// sum l is of the unrounded weights).  The scale is applied to S in fp32.
//   Every wait is bounded; on a timeout the CTA reports PA_DEVERR_TIMEOUT, stops
// issuing work and still frees its tensor memory.
#include <algorithm>
#include <mutex>
#include <vector>

#include "prefill_tc.cuh"
#include "shared.cuh"

namespace pa {
namespace shared {

using prefill::sw128_offset;
using prefill::v_group_sanitised;
using prefill::warp_wait;
using prefill::warp_wait_rx;

constexpr int kMmaWarp = 8, kKWarp = 9, kVWarp = 10;
constexpr int kTcThreads = 384;
// 384 threads launched at 168 registers (64512): the softmax warpgroups take
// 224, the rest keep 56: 256 x 224 + 128 x 56 = 64512.
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kTcThreads * 168, "register split");

template <int D> struct TcCfg {
  static constexpr int NH = D / 64;                    // 128-byte column halves of a row
  static constexpr uint32_t TILE = 128 * D * 2;        // Q of a chain, K or V of a tile
  static constexpr int NK = D == 128 ? 3 : 6, NV = D == 128 ? 2 : 6;
  static constexpr uint32_t OFF_K = 2 * TILE, OFF_V = OFF_K + NK * TILE, OFF_BAR = OFF_V + NV * TILE;
  static constexpr uint32_t N_BARS = 2 * NK + 2 * NV + 2 * 4;
  static constexpr uint32_t SMEM = OFF_BAR + N_BARS * 8 + 16 + 1024;  // + alignment slack
  // afterwards the warps' rings, in the same bytes
  static constexpr int STAGES = (int)(OFF_BAR / kTcWarps / stage_bytes(D));
  static constexpr uint32_t RING = STAGES * stage_bytes(D);
  static_assert(plan_scratch(kPlanMax, kPlanMax) <= OFF_BAR, "the plan's scratch comes before all");
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
  // tensor memory columns: S (and P) of the chains, O of the chains
  static constexpr uint32_t COL_S = 0, COL_O = 256;
};

struct TcParams {
  CUtensorMap tmap_k, tmap_v;  // 3-D [D, HKV, NB * BS] views, box {64, 1, 16}
  Params p;
};

// A unit's part of a CTA's run: rows r0 .. r0 + rows - 1 of the group (at most
// 256), KV head kvh, tiles j0 .. j0 + n - 1 (n may be 0), keys below `prefix`.
struct TcItem {
  int32_t table, b0, r0, rows, kvh, j0, n, prefix;
  int64_t prow;  // first partial row
};

// The items of a CTA's run in order; every role walks them alike.
struct Walk {
  int64_t x, end;
  int32_t at;
  const Group* groups;
  __device__ __forceinline__ Walk(const Params& p, const Plan& plan, const Totals& tot, int64_t worker, int lane) {
    groups = plan.groups;
    x = end = 0;
    at = 0;
    if (worker < tot.tc_workers) {
      x = first_tile(worker, tot.tc_tiles, tot.tc_workers);
      end = first_tile(worker + 1, tot.tc_tiles, tot.tc_workers);
    }
    if (x < end) at = find<1>(groups, (int32_t)p.NG, x, lane);
  }
  __device__ __forceinline__ bool next(const Params& p, int64_t worker, TcItem& im) {
    while (x < end) {
      const Group gp = load_plan(groups + at);
      const int32_t rows = gp.n * p.G, ry = cdiv(rows, TC_ROWS), nt = tc_unit_tiles(gp.prefix);
      const int64_t done = x - gp.tile0[1];
      if (!gp.tc || done >= (int64_t)p.HKV * ry * nt) {
        ++at;
        continue;
      }
      const int32_t u = (int32_t)(done / nt);
      const int32_t j = (int32_t)(done - (int64_t)u * nt), n = (int32_t)min((int64_t)(nt - j), end - x);
      im.j0 = max(j - kTcUnitCost, 0);
      im.n = max(j + n - kTcUnitCost, 0) - im.j0;
      im.table = gp.table;
      im.b0 = gp.b0;
      im.kvh = u / ry;
      im.r0 = (u - im.kvh * ry) * TC_ROWS;
      im.rows = min(TC_ROWS, rows - im.r0);
      im.prefix = gp.prefix;
      im.prow = p.tc_row0 + (gp.unit0[1] + u + worker) * TC_ROWS;
      x += n;
      return true;
    }
    return false;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1) shared_tc_kernel(const __grid_constant__ TcParams tp) {
  using C = TcCfg<D>;
  constexpr int NK = C::NK, NV = C::NV;
  const Params& p = tp.p;
  extern __shared__ unsigned char smem_raw[];
  // 1024-byte alignment for the 128-byte-swizzle atoms
  unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // [NK] K tile landed
  uint64_t* k_empty = k_full + NK;   // [NK] every S of it done
  uint64_t* v_full = k_empty + NK;   // [NV]
  uint64_t* v_empty = v_full + NV;   // [NV]
  uint64_t* s_full = v_empty + NV;   // [2] a chain's S in tensor memory
  uint64_t* p_full = s_full + 2;     // [2] its P written
  uint64_t* o_ready = p_full + 2;    // [2] its P V done
  uint64_t* q_ready = o_ready + 2;   // [2] its Q in shared memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_ready + 2);
  int32_t* abort_s = reinterpret_cast<int32_t*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_trigger();
  const Plan plan = take_plan(p, smem);
  // the scratch in shared memory, written and read as usual, is the TMA's next
  tc::fence_proxy_async_smem();
  if (threadIdx.x == 0) {
    for (int s = 0; s < NK; ++s) mbar_init(&k_full[s], 1), mbar_init(&k_empty[s], 1);
    for (int s = 0; s < NV; ++s) mbar_init(&v_full[s], 1), mbar_init(&v_empty[s], 1);
    for (int c = 0; c < 2; ++c) {
      mbar_init(&s_full[c], 1);
      mbar_init(&p_full[c], 4);  // one arrival per warp of the chain
      mbar_init(&o_ready[c], 1);
      mbar_init(&q_ready[c], 4);
    }
    *abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const Totals tot = load_plan(plan.totals);
  const int64_t worker = blockIdx.x;
  Walk walk(p, plan, tot, worker, lane);
  TcItem im;

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int c = warp >> 2, r = (warp & 3) * 32 + lane;  // chain, row of the chain = TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t scol = C::COL_S + 128 * c, ocol = C::COL_O + 128 * c;
    // S is scaled by |qscale|; a negative scale is in Q's sign bits
    const float qs = fabsf(p.qscale);
    const uint32_t flip = p.qscale < 0.f ? 0x80008000u : 0u;
    uint32_t uses = 0;  // tiles of this chain so far: the phase of its barriers
    bool ok = true;
    while (ok && walk.next(p, worker, im)) {
      const bool by_keys = im.rows <= 128;
      const int row = by_keys ? r : 128 * c + r;  // of the unit
      const int tiles = by_keys ? (im.n - c + 1) / 2 : im.n;
      if (im.n > 0) {
        unsigned char* qd = smem + c * C::TILE;
        const int rr = im.r0 + row;
        const bool in = row < im.rows;
        const uint4* src = reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.q) +
            ((int64_t)(im.b0 + rr / p.G) * p.H + (int64_t)im.kvh * p.G + rr % p.G) * D);
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          uint4 u = in ? __ldg(src + k) : make_uint4(0, 0, 0, 0);
          u.x ^= flip, u.y ^= flip, u.z ^= flip, u.w ^= flip;
          *reinterpret_cast<uint4*>(qd + sw128_offset(r, 8 * k, 128)) = u;
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_ready[c]);
      }
      float m_ref = -INFINITY, l = 0.f;
      for (int i = 0; i < tiles && ok; ++i, ++uses) {
        if (!warp_wait_rx(&s_full[c], uses & 1, abort_s)) { ok = false; break; }
        tc::fence_after_sync();
        const int j = im.j0 + (by_keys ? 2 * i + c : i);
        const int lim = im.prefix - j * TC_KT;  // keys of the tile below the prefix's end
        uint32_t u[128];
#pragma unroll
        for (int k = 0; k < 4; ++k) tc::tmem_ld32(lane_base + scol + 32 * k, *reinterpret_cast<uint32_t(*)[32]>(u + 32 * k));
        tc::tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 4; ++k) tc::reg_fence(*reinterpret_cast<uint32_t(*)[32]>(u + 32 * k));
        if (lim < TC_KT) {
#pragma unroll
          for (int k = 0; k < 128; ++k)
            if (k >= lim) u[k] = __float_as_uint(-INFINITY);
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 128; ++k) m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(u[k]));
        const float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * qs;
        // The reference only moves when the row's maximum grows by more than
        // 2^8; then O and l are rescaled (by 1 in rows that keep theirs)
        const bool need = mt > m_ref + 8.f;
        const float factor = need ? fast_exp2(m_ref - mt) : 1.f;  // 0 on a row's first tile
        const bool rescale = __any_sync(0xffffffffu, need) && i > 0;
        if (need) {
          l *= factor;
          m_ref = mt;
        }
        const float neg = m_ref == -INFINITY ? 0.f : -m_ref;
        const float2 neg2 = make_float2(neg, neg), qs2 = make_float2(qs, qs);
        float2 ls = make_float2(0.f, 0.f);
        // P = exp2(s - m_ref), keys 2k and 2k + 1 in column k
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = fma2(make_float2(__uint_as_float(u[32 * k + 2 * e]), __uint_as_float(u[32 * k + 2 * e + 1])), qs2, neg2);
            const float2 y = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            ls = add2(ls, y);
            w[e] = pack2(y.x, y.y, (T*)nullptr);
          }
          tc::tmem_st16(lane_base + scol + 16 * k, w);
        }
        l += ls.x + ls.y;
        if (rescale) {
          // (the chain's previous P V must have finished)
          if (!warp_wait_rx(&o_ready[c], (uses - 1) & 1, abort_s)) { ok = false; break; }
          tc::fence_after_sync();
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            uint32_t o[32];
            tc::tmem_ld32(lane_base + ocol + 32 * k, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tc::tmem_st32(lane_base + ocol + 32 * k, o);
          }
        }
        tc::tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[c]);
      }
      // the piece's partials: (m_ref, l) and O as they are
      if (ok && tiles > 0 && !warp_wait_rx(&o_ready[c], (uses - 1) & 1, abort_s)) ok = false;
      if (!ok) break;
      if (tiles > 0) tc::fence_after_sync();
      const int64_t out = im.prow + (by_keys ? 128 * c + r : row);
      const bool in = row < im.rows;
      if (in) p.part_ml[out] = make_float2(m_ref, l);
      if (tiles > 0) {
        float* dst = p.part_o + out * D;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          uint32_t o[32];
          tc::tmem_ld32(lane_base + ocol + 32 * k, o);
          tc::tmem_wait_ld();
          if (in) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(dst + 32 * k + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        // these reads come before the next unit's first P V, which follows P's arrival
        tc::fence_before_sync();
      }
    }
    if (!ok && lane == 0) report(p.dev_status, PA_DEVERR_TIMEOUT);
    // Both chains done: every product has been taken, and the shared memory is
    // free for the rings of the warps' own work
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (*reinterpret_cast<volatile int32_t*>(abort_s) == 0)
      warp_work<T, D, C::STAGES>(p, plan, tot, smem_u32(smem) + warp * C::RING, (int64_t)warp * gridDim.x + blockIdx.x);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kMmaWarp) {
      // ------------------------------------------------------------ MMA issuer
      constexpr uint32_t idesc_s = tc::idesc_f16(prefill::Fmt<T>::id, 128, TC_KT, false);
      constexpr uint32_t idesc_o = tc::idesc_f16(prefill::Fmt<T>::id, 128, D, true);
      uint32_t k0 = 0, items = 0;       // tiles, items so far
      uint32_t uses0 = 0, uses1 = 0;    // tiles of the chains so far
      bool ok = true;
      while (walk.next(p, worker, im)) {
        if (lane != 0 || !ok || im.n == 0) continue;  // (the other lanes only walk along)
        const bool by_keys = im.rows <= 128;
        // element e: chain e & 1 on tile e (by keys) or e / 2
        const int E = by_keys ? im.n : 2 * im.n;
        auto tile_of = [&](int e) -> uint32_t { return k0 + (by_keys ? e : e >> 1); };
        auto issue_s = [&](int e) -> bool {
          const int c = e & 1;
          const uint32_t t = tile_of(e), st = t % NK;
          if (e < 2 && !mbar_wait(&q_ready[c], items & 1, abort_s)) return false;
          if (!mbar_wait(&k_full[st], (t / NK) & 1, abort_s)) return false;
          tc::fence_after_sync();
          const uint32_t qb = smem_u32(smem) + c * C::TILE, kb = smem_u32(smem) + C::OFF_K + st * C::TILE;
          const uint32_t dcol = tmem + C::COL_S + 128 * c;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk >> 2) * (128 * 128) + (kk & 3) * 32;
            tc::mma_ss(dcol, tc::smem_desc_sw128(qb + off, 16, 1024), tc::smem_desc_sw128(kb + off, 16, 1024), idesc_s,
                       kk != 0);
          }
          tc::mma_commit(&s_full[c]);
          if (by_keys || c) tc::mma_commit(&k_empty[st]);
          return true;
        };
        ok = issue_s(0);
        if (ok && E > 1) ok = issue_s(1);
        for (int e = 0; e < E && ok; ++e) {
          const int c = e & 1;
          const uint32_t t = tile_of(e), st = t % NV, uses = c ? uses1 : uses0;
          if (!mbar_wait(&v_full[st], (t / NV) & 1, abort_s) || !mbar_wait(&p_full[c], uses & 1, abort_s)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t vb = smem_u32(smem) + C::OFF_V + st * C::TILE;
          const uint32_t pcol = tmem + C::COL_S + 128 * c, dcol = tmem + C::COL_O + 128 * c;
#pragma unroll
          for (int kk = 0; kk < TC_KT / 16; ++kk)  // 16 keys: 8 columns of pairs
            tc::mma_ts(dcol, pcol + kk * 8, tc::smem_desc_sw128(vb + kk * 16 * 128, 128 * 128, 1024), idesc_o,
                       (e > 1 || kk > 0) ? 1u : 0u);
          if (by_keys || c) tc::mma_commit(&v_empty[st]);
          tc::mma_commit(&o_ready[c]);
          if (c) ++uses1;
          else ++uses0;
          if (e + 2 < E) ok = issue_s(e + 2);
        }
        if (!ok) report(p.dev_status, PA_DEVERR_TIMEOUT);
        k0 += im.n;
        ++items;
      }
    } else if (warp == kKWarp || warp == kVWarp) {
      // ---------------------------------------------------- K and V producers
      // Lane l < 8 NH loads one 16-row group x 64-column half of a tile; its
      // block id is fetched a tile ahead.
      const bool is_v = warp == kVWarp;
      const int n_st = is_v ? NV : NK;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      unsigned char* base = smem + (is_v ? C::OFF_V : C::OFF_K);
      const CUtensorMap* map = is_v ? &tp.tmap_v : &tp.tmap_k;
      constexpr int NBOX = 8 * C::NH;
      const int g16 = lane / C::NH, hf = lane % C::NH;
      const int32_t BS = (int32_t)p.BS;
      uint32_t n = 0;
      bool ok = true;
      while (ok && walk.next(p, worker, im)) {
        if (im.n == 0) continue;
        const int32_t* table = p.block_tables + (int64_t)im.table * p.MB;
        auto row_of = [&](int j) -> int32_t {  // pool row of this lane's group of tile j
          const int32_t t = j * TC_KT + g16 * 16;
          if (lane >= NBOX || t >= im.prefix) return 0;
          const int32_t page = p.bs_shift >= 0 ? t >> p.bs_shift : t / BS;
          int32_t blk = __ldg(table + page);
          if (blk < 0 || blk >= p.NB) {
            report(p.dev_status, PA_DEVERR_BLOCK_ID);
            blk = 0;
          }
          return blk * BS + (t - page * BS);
        };
        int32_t next_row = row_of(im.j0);
        for (int i = 0; i < im.n && ok; ++i, ++n) {
          const int j = im.j0 + i;
          const int32_t row = next_row;
          if (i + 1 < im.n) next_row = row_of(j + 1);
          const uint32_t st = n % n_st;
          if (!warp_wait(&empty[st], ((n / n_st) & 1) ^ 1, abort_s)) { ok = false; break; }
          unsigned char* dst = base + st * C::TILE + hf * (128 * 128) + g16 * 16 * 128;
          // a V group that reaches past the prefix is written by its lane, its
          // rows past the end as zeros; a K group there loads any row (its
          // scores are masked)
          const int valid = im.prefix - (j * TC_KT + g16 * 16);
          const bool manual = is_v && lane < NBOX && valid < 16;
          if (manual) {
            v_group_sanitised(dst, static_cast<const char*>(p.v), row, valid, p.HKV, im.kvh, hf, D);
            tc::fence_proxy_async_smem();
          }
          const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, lane < NBOX && !manual));
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(&full[st], boxes * 16u * 128u);
          __syncwarp();
          if (lane < NBOX && !manual) tc::tma_load_3d(dst, map, hf * 64, im.kvh, row, &full[st]);
        }
      }
      if (!ok) {
        if (lane == 0) report(p.dev_status, PA_DEVERR_TIMEOUT);
        // copies still in flight land before the CTA gives up its memory
        for (uint32_t i = n > (uint32_t)n_st ? n - n_st : 0; i < n; ++i)
          (void)mbar_wait(&full[i % n_st], (i / n_st) & 1);
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// True when the tensor-memory kernel can load these pools: whole 16-row groups
// inside a page, row coordinates in 32 bits.
bool tc_takes(int64_t D, int64_t BS, int64_t NB) {
  return (D == 64 || D == 128) && BS % 16 == 0 && NB > 0 && NB * BS <= 0x7fffffff;
}

template <typename T, int D>
static int launch_tc_typed(const TcParams& tp, cudaStream_t s) {
  using C = TcCfg<D>;
  auto kern = shared_tc_kernel<T, D>;
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
  return cuda_status(launch(kern, tp.p.tc_ctas, kTcThreads, C::SMEM, s, tp, tp.p.planned));
}

int launch_tc(const Params& p, int dtype, int64_t D, cudaStream_t s) {
  TcParams tp;
  tp.p = p;
  int st = prefill::make_map(&tp.tmap_k, p.k, dtype, D, p.HKV, p.NB * p.BS);
  if (st) return st;
  st = prefill::make_map(&tp.tmap_v, p.v, dtype, D, p.HKV, p.NB * p.BS);
  if (st) return st;
  if (dtype == PA_DTYPE_BF16)
    return D == 128 ? launch_tc_typed<__nv_bfloat16, 128>(tp, s) : launch_tc_typed<__nv_bfloat16, 64>(tp, s);
  return D == 128 ? launch_tc_typed<__half, 128>(tp, s) : launch_tc_typed<__half, 64>(tp, s);
}

}  // namespace shared
}  // namespace pa
