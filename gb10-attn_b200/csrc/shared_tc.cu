// shared_tc.cu -- the attention launch of the shared-prefix decode for pools
// that tiled TMA can load (whole 16-row groups inside a page, head_dim 64 or
// 128): first the prefixes shared by many query rows, on the sm_100a tensor
// cores with S, P and O in tensor memory; beside it, in CTAs of their own, the
// rest, a warp at a time (shared.cuh).
//
// A CTA of the first kind takes its run of 64-key tiles and walks the units that it
// crosses: the members' query heads of one KV head are the rows of S = Q K^T and
// O = P V.  Two softmax warpgroups run two chains: rows 0-127 and 128-255 of a
// unit, or, in a unit of at most 128 rows, the same rows on every other tile,
// so that one chain's exponentials overlap the other's products.
// Thread = row = TMEM lane: it reads its 64 scores of a tile, keeps the row's
// reference maximum and sum in fp32 and writes P over S.  Two warps feed K and V
// by tiled TMA, 16 rows at a time through the pages; one thread per chain issues
// its MMAs.
//   Bound by the softmax warps and the MMAs together (1.2 us a tile of 256 rows: on
// all SMs 1.05 PFLOP/s of S and P V, 63 % of the bf16 burst rate, 76 % of the
// sustained one), while the CTAs with the sequences' own tokens are bound by
// instruction latency (0.15 us a 16-key tile).  256 sequences of 32 / 8 heads of 128
// behind 32768 tokens, with 256 to 1024 of their own: 275 to 297 us in steady calls,
// by how far the power cap lowers the clock (246 from a cool start), some 88 CTAs
// with the prefix and 60 with the rest.
//   Tiles of 64 keys, not 128: two S of each chain then fit the tensor memory
// beside both O, and S of the next tile is computed while a chain works on this
// one (an MMA of N = 64 takes 48 cycles, of N = 128 64, but the pipe waits less).
//   Precision: one 16-bit product each for S (Q and K as they are, products
// exact, fp32 sums) and P V (P rounded to 16 bits, as the output will be, in fp16
// by up to 2^-25 where it is below 2^-14; the sum l is of the unrounded weights).
// The scale is applied to S in fp32.
//   Every wait is bounded; on a timeout the CTA reports PA_DEVERR_TIMEOUT to
// callers that give a status word (the torch operators give none), stops issuing
// work, makes NaN of the rows in its run, lets its copies and products end and
// frees its tensor memory.
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

constexpr int kMmaWarp = 8, kKWarp = 10, kVWarp = 11;  // (an issuer per chain: 8 and 9)
constexpr int kTcThreads = 384;
// 384 threads launched at 168 registers (64512).  After the tensor-memory part
// (at once in a CTA that has none of it) the issuing and loading warps give theirs
// up and the warps' own work takes 240: 256 x 240 + 128 x 24 = 64512.
constexpr int kWorkRegs = 240, kDoneRegs = 24;
static_assert(256 * kWorkRegs + 128 * kDoneRegs <= kTcThreads * 168, "register split");

// A warp's bounded wait on a barrier that hands tensor-memory data on, usually
// passed at once.
__device__ __forceinline__ bool wait_tmem(uint64_t* bar, uint32_t parity, int32_t* abort_flag) {
  if (__all_sync(0xffffffffu, mbar_try_wait_rx(bar, parity, 0u))) return true;
  return warp_wait_rx(bar, parity, abort_flag);
}

template <int D> struct TcCfg {
  static constexpr int NH = D / 64;                    // 128-byte column halves of a row
  static constexpr uint32_t QTILE = 128 * D * 2;       // Q of a chain
  static constexpr uint32_t TILE = TC_KT * D * 2;      // K or V of a tile
  static constexpr int NK = D == 128 ? 5 : 12, NV = NK;
  static constexpr uint32_t OFF_K = 2 * QTILE, OFF_V = OFF_K + NK * TILE, OFF_BAR = OFF_V + NV * TILE;
  static constexpr uint32_t N_BARS = 2 * NK + 2 * NV + 16;
  static constexpr uint32_t SMEM = OFF_BAR + N_BARS * 8 + 16 + 1024;  // + alignment slack
  // afterwards the warps' rings, in the same bytes
  static constexpr int STAGES = (int)(OFF_BAR / kTcWarps / stage_bytes(D));
  static constexpr uint32_t RING = STAGES * stage_bytes(D);
  static_assert(plan_scratch(kPlanMax, kPlanMax) <= OFF_BAR, "the plan's scratch comes before all");
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
  // tensor memory columns: two S (and P) per chain, O of the chains
  static constexpr uint32_t COL_S = 0, COL_O = 256;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 32 bytes, a whole sector.
__device__ __forceinline__ void store32(float* dst, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// One lane of the warp, in a form that the compiler knows for a single thread's:
// its branch keeps the operands of the MMAs in uniform registers (32 cycles to
// issue one; 47 behind a test of the lane's number).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;}" : "=r"(p));
  return p != 0;
}

struct TcParams {
  CUtensorMap tmap_k, tmap_v;  // 3-D [D, HKV, NB * BS] views, box {64, 1, 16}
  Params p;
};

// Two 16-bit elements times zero: NaN for infinities and NaN, else zero.
__device__ __forceinline__ uint32_t times_zero(uint32_t w, __half*) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(0.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t times_zero(uint32_t w, __nv_bfloat16*) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w), __float2bfloat162_rn(0.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}

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

// What the softmax warps of a CTA that gave up do instead of their own work (a
// CTA that had prefixes has none: own_cta0).  Every piece of its run becomes NaN,
// done or not, and with it the output rows that have one; the merge's addresses
// have to hold.  (Out of line: among the softmax warps' code it took registers
// from the tiles; 128 sequences on 8k take 3 % longer with that and 1.5 % so than
// without it, 60 us.)
__device__ __noinline__ void give_up(const Params& p, int64_t index) {
  const Plan plan = plan_at(p, p.planned ? 0 : blockIdx.x);
  const Totals tot = load_plan(plan.totals);
  locate_rows(p, plan, tot, index);
  const float nan = __int_as_float(0x7fc00000);
  const int t = threadIdx.x;  // 128 x chain + row of the chain
  Walk walk(p, plan, tot, blockIdx.x, t & 31);
  TcItem im;
  while (walk.next(p, blockIdx.x, im))
    if ((im.rows <= 128 ? t & 127 : t) < im.rows) p.part_ml[im.prow + t] = make_float2(nan, nan);
}

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
  uint64_t* s_full = v_empty + NV;   // [2][2] S of a chain in tensor memory
  uint64_t* p_full = s_full + 4;     // [2][2] its P written
  uint64_t* o_ready = p_full + 4;    // [2] a chain's P V done
  uint64_t* o_last = o_ready + 2;    // [2] its last P V of an item done
  uint64_t* q_ready = o_last + 2;    // [2] its Q in shared memory
  uint64_t* drained = q_ready + 2;   // [2] every product of a chain done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
  int32_t* abort_s = reinterpret_cast<int32_t*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_trigger();
  const Plan plan = take_plan(p, smem);
  // the scratch in shared memory, written and read as usual, is the TMA's next
  tc::fence_proxy_async_smem();
  if (threadIdx.x == 0) {
    for (int s = 0; s < NK; ++s) mbar_init(&k_full[s], 1), mbar_init(&k_empty[s], 2);
    for (int s = 0; s < NV; ++s) mbar_init(&v_full[s], 1), mbar_init(&v_empty[s], 2);
    for (int c = 0; c < 4; ++c) mbar_init(&s_full[c], 1), mbar_init(&p_full[c], 4);  // one arrival per warp
    for (int c = 0; c < 2; ++c) {
      mbar_init(&o_ready[c], 1);
      mbar_init(&o_last[c], 1);
      mbar_init(&q_ready[c], 4);
      mbar_init(&drained[c], 1);
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
  TcItem im = {};

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax
    const int c = warp >> 2, r = (warp & 3) * 32 + lane;  // chain, row of the chain = TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ocol = C::COL_O + 128 * c;
    // S is scaled by |qscale|; a negative scale is in Q's sign bits, one of zero in
    // Q too (masked keys are at -inf before the scale, and -inf * 0 is NaN)
    const bool zero = p.qscale == 0.f;
    const float qs = zero ? 1.f : fabsf(p.qscale);
    const uint32_t flip = p.qscale < 0.f ? 0x80008000u : 0u;
    auto signed_q = [&](uint32_t w) { return zero ? times_zero(w, (T*)nullptr) : w ^ flip; };
    uint32_t uses = 0, done = 0;  // tiles, items with tiles of this chain: the phases of its barriers
    // Q of this thread's row of an item (zeros for none: written in any case, so
    // that it takes no registers while the tiles are worked on)
    uint4 qr[D / 8];
    auto load_q = [&](const TcItem& it, bool there) {
      const int row = it.rows <= 128 ? r : 128 * c + r, rr = it.r0 + row;
      const uint4* src = reinterpret_cast<const uint4*>(
          static_cast<const T*>(p.q) + ((int64_t)(it.b0 + rr / p.G) * p.H + (int64_t)it.kvh * p.G + rr % p.G) * D);
#pragma unroll
      for (int k = 0; k < D / 8; ++k) qr[k] = there && row < it.rows ? __ldg(src + k) : make_uint4(0, 0, 0, 0);
    };
    bool more = walk.next(p, worker, im);
    bool ok = p.waits || !more;  // (a test lets it give up at its first tile)
    load_q(im, more);
    while (more) {
      const bool by_keys = im.rows <= 128;
      const int row = by_keys ? r : 128 * c + r;  // of the unit
      const int tiles = by_keys ? (im.n - c + 1) / 2 : im.n;
      // (Q is handed over only with a tile: an item that has none for this chain,
      // one of a single tile by keys, ends without a wait on its issuer, who may not
      // fall behind by the two phases that a parity cannot tell apart)
      if (tiles > 0) {
        unsigned char* qd = smem + c * C::QTILE;
#pragma unroll
        for (int k = 0; k < D / 8; ++k)
          *reinterpret_cast<uint4*>(qd + sw128_offset(r, 8 * k, 128)) =
              make_uint4(signed_q(qr[k].x), signed_q(qr[k].y), signed_q(qr[k].z), signed_q(qr[k].w));
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_ready[c]);
      }
      float m_ref = -INFINITY, l = 0.f;
      for (int i = 0; i < tiles && ok; ++i, ++uses) {
        const uint32_t b = uses & 1, scol = lane_base + C::COL_S + 128 * c + 64 * b;
        if (!wait_tmem(&s_full[2 * c + b], (uses >> 1) & 1, abort_s)) { ok = false; break; }
        tc::fence_after_sync();
        uint32_t u[64];
#pragma unroll
        for (int k = 0; k < 2; ++k) tc::tmem_ld32(scol + 32 * k, *reinterpret_cast<uint32_t(*)[32]>(u + 32 * k));
        tc::tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 2; ++k) tc::reg_fence(*reinterpret_cast<uint32_t(*)[32]>(u + 32 * k));
        // keys of this tile below the prefix's end
        const int lim = im.prefix - (im.j0 + (by_keys ? 2 * i + c : i)) * TC_KT;
        if (lim < TC_KT) {
#pragma unroll
          for (int k = 0; k < 64; ++k)
            if (k >= lim) u[k] = __float_as_uint(-INFINITY);
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 64; k += 2)
          m4[k / 2 & 3] = max3(m4[k / 2 & 3], __uint_as_float(u[k]), __uint_as_float(u[k + 1]));
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
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 x = fma2(make_float2(__uint_as_float(u[2 * e]), __uint_as_float(u[2 * e + 1])), qs2, neg2);
          const float2 y = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          ls = add2(ls, y);
          w[e] = pack2(y.x, y.y, (T*)nullptr);
        }
        tc::tmem_st32(scol, w);
        l += ls.x + ls.y;
        if (rescale) {
          // the chain's P V before this one must have finished (the one before
          // that has: this S was issued after it)
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
        if (lane == 0) mbar_arrive(&p_full[2 * c + b]);
      }
      // the piece's partials: (m_ref, l) and O as they are
      // (the next item's Q comes meanwhile)
      const TcItem cur = im;
      more = ok && walk.next(p, worker, im);
      load_q(im, more);
      if (ok && tiles > 0 && !warp_wait_rx(&o_last[c], done++ & 1, abort_s)) ok = false;
      if (!ok) break;
      if (tiles > 0) tc::fence_after_sync();
      const int64_t out = cur.prow + (by_keys ? 128 * c + r : row);
      const bool in = row < cur.rows;
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
            for (int e = 0; e < 32; e += 8) store32(dst + 32 * k + e, o + e);
          }
        }
        // these reads come before the next unit's first P V, which follows P's arrival
        tc::fence_before_sync();
      }
    }
    if (!ok) {
      tc::tmem_wait_st();
      if (lane == 0) {
        atomicExch(abort_s, 1);
        report(p.dev_status, PA_DEVERR_TIMEOUT);
      }
    }
    // Both chains done: every product has been taken, and the shared memory is
    // free for the rings of the warps' own work
    asm volatile("bar.sync 1, 256;" ::: "memory");
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWorkRegs));
    const int64_t index = (int64_t)warp * gridDim.x + blockIdx.x;
    const int64_t own = blockIdx.x < tot.own_cta0 ? tot.workers
                                                  : warp * (gridDim.x - tot.own_cta0) + blockIdx.x - tot.own_cta0;
    if (*reinterpret_cast<volatile int32_t*>(abort_s) == 0)
      warp_work<T, D, C::STAGES>(p, plan, tot, smem_u32(smem) + warp * C::RING, own, index);
    else
      give_up(p, index);
  } else {
    if (warp == kMmaWarp || warp == kMmaWarp + 1) {
      // ------------------------------------ MMA issuer of chain `warp - kMmaWarp`
      // A chain has two S, so that the next is there while the softmax works on
      // this one: per tile P V, then S of the tile after next, which takes the
      // place of P and waits for that P V to be done (products of different
      // accumulators are not ordered by themselves).  Every tile is taken up
      // and given back by both chains, so both follow its barriers' phases;
      // with by_keys a chain passes over the other's tiles.
      constexpr uint32_t idesc_s = tc::idesc_f16(prefill::Fmt<T>::id, 128, TC_KT, false);
      constexpr uint32_t idesc_o = tc::idesc_f16(prefill::Fmt<T>::id, 128, D, true);
      const int c = warp - kMmaWarp;
      const uint64_t qd = tc::smem_desc_sw128(smem_u32(smem) + c * C::QTILE, 16, 1024);
      const uint64_t kd = tc::smem_desc_sw128(smem_u32(smem) + C::OFF_K, 16, 1024);
      const uint64_t vd = tc::smem_desc_sw128(smem_u32(smem) + C::OFF_V, TC_KT * 128, 1024);
      const uint32_t scol = tmem + C::COL_S + 128 * c, ocol = tmem + C::COL_O + 128 * c;
      uint32_t kn = 0, kp = 0, vn = 0, vp = 0;  // stage and phase of the coming K and V tile
      uint32_t items = 0, ns = 0, np = 0;       // items with tiles, S and P V of this chain
      bool ok = true;
      const bool issues = elect_one();
      if (issues) while (walk.next(p, worker, im)) {
        if (!ok || im.n == 0) continue;
        const bool by_keys = im.rows <= 128;
        auto own = [&](int t) { return !by_keys || (t & 1) == c; };
        int ts = 0, tv = 0, first = 1;  // tiles of the item whose S (P V) have been issued or passed over
        // S of the chain's next tile, if there is one
        auto start = [&](bool wait_pv) {
          while (ts < im.n) {
            if (!mbar_wait(&k_full[kn], kp, abort_s)) return false;
            const bool mine = own(ts++);
            if (mine) {
              if (wait_pv && !mbar_wait(&o_ready[c], (np - 1) & 1, abort_s)) return false;
              tc::fence_after_sync();
              const uint64_t b = kd + (uint64_t)(kn * (C::TILE >> 4));
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                tc::mma_ss(scol + 64 * (ns & 1), qd + (((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4),
                           b + (((kk >> 2) * (TC_KT * 128) + (kk & 3) * 32) >> 4), idesc_s, kk != 0);
              tc::mma_commit(&s_full[2 * c + (ns & 1)]);
              tc::mma_commit(&k_empty[kn]);
              ++ns;
            } else {
              mbar_arrive(&k_empty[kn]);
            }
            if (++kn == NK) kn = 0, kp ^= 1;
            if (mine) break;
          }
          return true;
        };
        const bool any = !by_keys || im.n > c;
        ok = (!any || mbar_wait(&q_ready[c], items & 1, abort_s)) && start(false) && start(false);
        while (tv < im.n && ok) {
          if (!mbar_wait(&v_full[vn], vp, abort_s)) { ok = false; break; }
          const bool mine = own(tv++);
          if (mine) {
            if (!mbar_wait(&p_full[2 * c + (np & 1)], (np >> 1) & 1, abort_s)) { ok = false; break; }
            tc::fence_after_sync();
            const uint64_t b = vd + (uint64_t)(vn * (C::TILE >> 4));
#pragma unroll
            for (int kk = 0; kk < TC_KT / 16; ++kk)  // 16 keys: 8 columns of pairs
              tc::mma_ts(ocol, scol + 64 * (np & 1) + kk * 8, b + (uint64_t)(kk * 128), idesc_o, kk > 0 || !first);
            first = 0;
            ++np;
            tc::mma_commit(&o_ready[c]);
            if (tv + (by_keys ? 1 : 0) >= im.n) tc::mma_commit(&o_last[c]);
            tc::mma_commit(&v_empty[vn]);
          } else {
            mbar_arrive(&v_empty[vn]);
          }
          if (++vn == NV) vn = 0, vp ^= 1;
          if (mine) ok = start(true);
        }
        if (!ok) report(p.dev_status, PA_DEVERR_TIMEOUT);
        items += any;
      }
      if (issues && ns) {  // the CTA may not end before its products, taken or not
        tc::mma_commit(&drained[c]);
        (void)mbar_wait(&drained[c], 0);
      }
    } else if (warp == kKWarp || warp == kVWarp) {
      // ---------------------------------------------------- K and V producers
      // Lane l < 4 NH loads one 16-row group x 64-column half of a tile; its
      // block id is fetched a tile ahead.
      const bool is_v = warp == kVWarp;
      const int n_st = is_v ? NV : NK;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      unsigned char* base = smem + (is_v ? C::OFF_V : C::OFF_K);
      const CUtensorMap* map = is_v ? &tp.tmap_v : &tp.tmap_k;
      constexpr int NBOX = TC_KT / 16 * C::NH;
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
          unsigned char* dst = base + st * C::TILE + hf * (TC_KT * 128) + g16 * 16 * 128;
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
      if (!ok && lane == 0) report(p.dev_status, PA_DEVERR_TIMEOUT);
      // copies still in flight land before the CTA may end, taken or not: lane
      // l waits for the last tile of stage l
      if (lane < n_st && (uint32_t)lane < n) {
        const uint32_t last = n - 1 - (n - 1 - lane) % n_st;
        (void)mbar_wait(&full[lane], (last / n_st) & 1);
      }
    }
    __syncwarp();
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDoneRegs));
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
