// qk_append.cu -- what lies between a layer's q / k / v projection and its
// attention, in one launch (pa_qk_norm_rope_append): RMS norm of every query
// and key head, rotation by the token's position, q to the output, k and v to
// the token's row of the paged pool.
//
// Per head x of D elements: r = 1 / sqrt(mean(x^2) + eps), y = x r w, then the
// first R elements turn in pairs (a, b) -> (a cos - b sin, b cos + a sin) with
// the angles of the token's position.  All of it in fp32; one rounding, to the
// output's type.
#include <algorithm>

#include "common.cuh"

namespace pa {
namespace qkappend {

struct Params {
  const char *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;  // element strides
  const char *q_weight, *k_weight;                      // [D], null: no norm
  int32_t w_f32;                                        // weights are fp32, else of the source type
  float eps;
  const float* cos_sin;  // [max_pos, R]: cos of the R / 2 angles, then sin
  int64_t max_pos;
  int32_t R, interleaved;
  const int32_t *positions, *seq_ids, *tables;
  int64_t T, H, HKV, MB, n_seqs, BS, NB;
  char *q_out, *k_cache, *v_cache;
  const float *k_scale, *v_scale;  // FP8 pools: [HKV], null = 1
  int32_t lph_shift;  // log2(head_dim / 8)
  int32_t bs_shift;   // log2(BS) if BS is a power of two, else -1
  int32_t* dev_status;
};

template <typename S> __device__ __forceinline__ float to_f32(S x) { return (float)x; }
template <typename P> __device__ __forceinline__ P from_f32(float x) { return (P)x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
// round to nearest even, saturating to the largest finite e4m3 (+-448)
template <> __device__ __forceinline__ __nv_fp8_e4m3 from_f32<__nv_fp8_e4m3>(float x) {
  __nv_fp8_e4m3 r;
  r.__x = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  return r;
}

// Where token t's K and V rows go: the pool row, or -1 for none (padding, or a
// place outside the table or pool, which is reported if `tell`).
__device__ __forceinline__ int64_t pool_row(const Params& p, int64_t t, int64_t pos, bool tell) {
  if (pos < 0) return -1;
  if (pos >= p.max_pos) {
    if (tell) report(p.dev_status, PA_DEVERR_CONTEXT);
    return -1;
  }
  const int64_t seq = p.seq_ids ? p.seq_ids[t] : t;
  const int64_t page = p.bs_shift >= 0 ? pos >> p.bs_shift : pos / p.BS;
  if (seq < 0 || seq >= p.n_seqs || page >= p.MB) {
    if (tell) report(p.dev_status, PA_DEVERR_CONTEXT);
    return -1;
  }
  const int64_t blk = p.tables[seq * p.MB + page];
  if (blk < 0 || blk >= p.NB) {
    if (tell) report(p.dev_status, PA_DEVERR_BLOCK_ID);
    return -1;
  }
  return blk * p.BS + (pos - page * p.BS);
}

// One element of a turned pair: x cos + other sin (sin negated for the first
// of the pair).  Pinned, as is the order of the sums of squares (a lane's four
// pairs of elements, then a tree over the lanes), so that every variant gives
// the same bits.
__device__ __forceinline__ float turned(float x, float other, float c, float s) {
  return fmaf(other, s, __fmul_rn(x, c));
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 pa, pb, pd;\n\tmov.b64 pa, {%2, %3};\n\tmov.b64 pb, {%4, %5};\n\t"
      "mul.rn.f32x2 pd, pa, pb;\n\tmov.b64 {%0, %1}, pd;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// A lane's eight elements of a head are two runs of four, from a and from b on:
// for pairs (i, i + R / 2) the two halves' same places, so that a pair never
// leaves its lane; otherwise neighbouring runs.
struct Place {
  int a, b;
  bool turns;
};
__device__ __forceinline__ Place place(const Params& p, int sub) {
  const bool turns = sub * 8 < p.R;
  if (turns && !p.interleaved) return {4 * sub, p.R / 2 + 4 * sub, true};
  return {8 * sub, 8 * sub + 4, turns};
}

// Four elements of a source row as loaded, and stores of four elements.
template <typename S> struct Raw4;
template <> struct Raw4<float> { using T = uint4; };
template <> struct Raw4<__half> { using T = uint2; };
template <> struct Raw4<__nv_bfloat16> { using T = uint2; };

template <typename S> __device__ __forceinline__ void unpack4(const typename Raw4<S>::T& u, float2* f) {
  if constexpr (sizeof(S) == 4) {
    f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  } else if constexpr (DTypeId<S>::value == PA_DTYPE_BF16) {  // the high half of an fp32
    f[0] = make_float2(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u));
    f[1] = make_float2(__uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
  } else {
    f[0] = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    f[1] = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  }
}
template <typename P> __device__ __forceinline__ void store4(P* dst, const float2* f) {
  if constexpr (DTypeId<P>::value == PA_DTYPE_BF16) {
    __nv_bfloat162 v[2] = {__float22bfloat162_rn(f[0]), __float22bfloat162_rn(f[1])};
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
  } else if constexpr (DTypeId<P>::value == PA_DTYPE_F16) {
    __half2 v[2] = {__float22half2_rn(f[0]), __float22half2_rn(f[1])};
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
  } else {
    struct alignas(sizeof(P) >= 4 ? 16 : 4 * sizeof(P)) Four {
      P x[4];
    };
    const Four v = {{from_f32<P>(f[0].x), from_f32<P>(f[0].y), from_f32<P>(f[1].x), from_f32<P>(f[1].y)}};
    *reinterpret_cast<Four*>(dst) = v;
  }
}

constexpr int kThreads = 64;
constexpr int kBatch = 4;  // heads in flight per thread

// HBM-bound: a token's q, k and v are read once and written once.  One CTA per
// token, or three (q, k, v) while that leaves SMs idle: the loads of the three
// follow one another otherwise, and a few tokens take that long.  D / 8 lanes
// hold a head, eight elements each, so the CTA works on 512 / D heads at a time
// and has four times as many in flight.  A thread keeps its place in the head:
// the cosines and sines of its four pairs and its eight weights are loaded once
// for all of its heads.
//   4 x 4096 tokens of 3 x 32 heads of 128 in bf16 (808 MB): 138 us, 5.9 TB/s, 89 %
// of a copy's rate.  CTAs of 32, 64, 128 and 256 threads: 152, 140, 148 and 195
// us; six heads in flight instead of four: 146.
//   TOKENS 2: a warp per token, for tokens whose query heads (H D <= 1024) fill
// no more than the four heads that a warp's lanes have in flight; twice the
// tokens are under way then (17873 tokens of 8 + 2 heads of 128 in bf16: 40 us
// with 1, 29 with 2).
//   Other types at 4 x 4096 tokens of 3 x 32 heads of 128, source -> pool: fp32 -> bf16 211 us
// (97 % of a copy's rate), fp32 -> fp32 251 (98 %), bf16 -> fp32 175 (94 %), bf16 ->
// fp64 291 (85 %); bf16 -> e4m3 186 (55 %) and fp32 -> e4m3 223 (83 %), bound by the
// divisions and conversions.
template <typename S, typename P, int TOKENS>
__global__ void __launch_bounds__(kThreads) qk_append_kernel(const __grid_constant__ Params p) {
  using R4 = typename Raw4<S>::T;
  constexpr int kTeam = kThreads / TOKENS;  // threads of a token
  const int tid = threadIdx.x % kTeam;
  const int lph = 1 << p.lph_shift;  // lanes per head, D / 8
  const int sub = tid & (lph - 1), grp = tid >> p.lph_shift;
  const int groups = kTeam >> p.lph_shift;
  const int warp_grp = (tid & ~31) >> p.lph_shift;  // the warp's first group
  const int D = lph * 8, H = (int)p.H, HKV = (int)p.HKV;
  const int64_t t = (int64_t)blockIdx.x * TOKENS + threadIdx.x / kTeam;
  if (TOKENS > 1 && t >= p.T) return;
  const Place at = place(p, sub);
  const int64_t pos = p.positions[t];
  S* const q_out = reinterpret_cast<S*>(p.q_out) + t * H * D;

  const int part = gridDim.y == 1 ? -1 : blockIdx.y;  // 0: q, 1: k, 2: v, -1: all

  if (pos < 0 || pos >= p.max_pos) {  // a padding token's q is zero, one past the table's is NaN
    if (part > 0) return;
    if (pos >= 0 && tid == 0) report(p.dev_status, PA_DEVERR_CONTEXT);
    const float x = pos < 0 ? 0.f : __int_as_float(0x7fc00000);
    const float2 y[2] = {make_float2(x, x), make_float2(x, x)};
    for (int e = tid * 4; e < H * D; e += kTeam * 4) store4<S>(q_out + e, y);
    return;
  }
  const int64_t row = part == 0 ? -1 : pool_row(p, t, pos, tid == 0);

  float2 c[2] = {}, s[2] = {};
  if (at.turns) {
    const float* cs = p.cos_sin + pos * p.R + 4 * sub;
    const float4 x = *reinterpret_cast<const float4*>(cs), y = *reinterpret_cast<const float4*>(cs + p.R / 2);
    c[0] = make_float2(x.x, x.y), c[1] = make_float2(x.z, x.w);
    s[0] = make_float2(y.x, y.y), s[1] = make_float2(y.z, y.w);
  }

  // Every head of x[n heads]: norm, turn, `put`.
  auto each = [&](const char* base, int64_t head_stride, int n, const char* w, bool turn, auto put) {
    const S* src = reinterpret_cast<const S*>(base);
    float2 g[4];
    if (w) {
      if (p.w_f32) {
        unpack4<float>(*reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(w) + at.a), g);
        unpack4<float>(*reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(w) + at.b), g + 2);
      } else {
        unpack4<S>(*reinterpret_cast<const R4*>(reinterpret_cast<const S*>(w) + at.a), g);
        unpack4<S>(*reinterpret_cast<const R4*>(reinterpret_cast<const S*>(w) + at.b), g + 2);
      }
    }
    for (int h0 = 0; h0 + warp_grp < n; h0 += kBatch * groups) {
      R4 raw[kBatch][2];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int h = h0 + i * groups + grp;
        raw[i][0] = raw[i][1] = R4{};
        if (h < n) {
          raw[i][0] = __ldcs(reinterpret_cast<const R4*>(src + h * head_stride + at.a));
          raw[i][1] = __ldcs(reinterpret_cast<const R4*>(src + h * head_stride + at.b));
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int h = h0 + i * groups + grp;
        if (h0 + i * groups + warp_grp >= n) break;  // the whole warp leaves
        float2 y[4];
        unpack4<S>(raw[i][0], y);
        unpack4<S>(raw[i][1], y + 2);
        if (w) {
          float2 q2 = mul2(y[0], y[0]);
#pragma unroll
          for (int e = 1; e < 4; ++e) q2 = fma2(y[e], y[e], q2);
          float sum = q2.x + q2.y;
          for (int o = lph >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float r = rsqrtf(sum * (1.f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = mul2(mul2(y[e], make_float2(r, r)), g[e]);
        }
        if (turn && at.turns) {
          if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float cc = e & 1 ? c[e >> 1].y : c[e >> 1].x, ss = e & 1 ? s[e >> 1].y : s[e >> 1].x;
              y[e] = make_float2(turned(y[e].x, y[e].y, cc, -ss), turned(y[e].y, y[e].x, cc, ss));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 a = y[e], b = y[e + 2];
              y[e] = fma2(b, make_float2(-s[e].x, -s[e].y), mul2(a, c[e]));
              y[e + 2] = fma2(a, s[e], mul2(b, c[e]));
            }
          }
        }
        if (h < n) put(h, y);
      }
    }
  };
  auto to_pool = [&](char* cache, const float* scale) {
    P* dst = reinterpret_cast<P*>(cache) + row * HKV * D;
    return [=](int h, float2 (&y)[4]) {
      if constexpr (sizeof(P) == 1) {
        const float qs = scale ? scale[h] : 1.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = make_float2(__fdiv_rn(y[e].x, qs), __fdiv_rn(y[e].y, qs));
      }
      store4<P>(dst + h * D + at.a, y);
      store4<P>(dst + h * D + at.b, y + 2);
    };
  };
  if (row >= 0) {
    if (part != 1) each(p.v + t * p.v_tok * sizeof(S), p.v_head, HKV, nullptr, false, to_pool(p.v_cache, p.v_scale));
    if (part != 2) each(p.k + t * p.k_tok * sizeof(S), p.k_head, HKV, p.k_weight, true, to_pool(p.k_cache, p.k_scale));
  }
  if (part <= 0) each(p.q + t * p.q_tok * sizeof(S), p.q_head, H, p.q_weight, true, [&](int h, float2 (&y)[4]) {
    store4<S>(q_out + h * D + at.a, y);
    store4<S>(q_out + h * D + at.b, y + 2);
  });
}

// Any alignment and strides, and rotated parts that are no multiple of eight:
// one warp per (token, head), D / 8 lanes with eight elements each, one access
// an element, a pair's other element by a second load.  Bound by the number of its
// accesses: 4 x 4096 tokens of 3 x 32 heads of 128, one element off a 16-byte boundary, 1032 us in
// bf16 (12 % of a copy's rate), 939 from fp32; 256 tokens of 32 / 8 heads 12 us.
template <typename S, typename P>
__global__ void __launch_bounds__(kThreads) qk_append_any_kernel(const __grid_constant__ Params p) {
  const int lane = threadIdx.x & 31, lph = 1 << p.lph_shift, D = 8 * lph;
  const int64_t heads = p.H + 2 * p.HKV;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (unit >= p.T * heads) return;
  const int64_t t = unit / heads, hh = unit % heads;
  const int kind = hh < p.H ? 0 : (hh < p.H + p.HKV ? 1 : 2);  // q, k, v
  const int64_t h = kind == 0 ? hh : (kind == 1 ? hh - p.H : hh - p.H - p.HKV);
  const int64_t pos = p.positions[t];
  const bool known = pos >= 0 && pos < p.max_pos, mine = lane < lph;
  const int64_t row = kind ? pool_row(p, t, pos, lane == 0) : 0;
  if (row < 0) return;
  Place at = place(p, lane);
  if (p.R % 8) at = {8 * lane, 8 * lane + 4, false};
  auto element = [&](int i) { return i < 4 ? at.a + i : at.b + i - 4; };
  S* q_out = reinterpret_cast<S*>(p.q_out) + (t * p.H + h) * D;
  if (!known) {  // a padding token's q is zero, one past the table's is NaN
    if (pos >= 0 && lane == 0) report(p.dev_status, PA_DEVERR_CONTEXT);
    for (int i = 0; i < 8 && mine; ++i) q_out[element(i)] = from_f32<S>(pos < 0 ? 0.f : __int_as_float(0x7fc00000));
    return;
  }
  const S* src = kind == 0   ? reinterpret_cast<const S*>(p.q) + t * p.q_tok + h * p.q_head
                 : kind == 1 ? reinterpret_cast<const S*>(p.k) + t * p.k_tok + h * p.k_head
                             : reinterpret_cast<const S*>(p.v) + t * p.v_tok + h * p.v_head;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = mine ? to_f32<S>(src[element(i)]) : 0.f;
  if (kind != 2) {
    const char* w = kind == 0 ? p.q_weight : p.k_weight;
    float r = 1.f;
    if (w) {
      float even = __fmul_rn(y[0], y[0]), odd = __fmul_rn(y[1], y[1]);
#pragma unroll
      for (int i = 2; i < 8; i += 2) even = fmaf(y[i], y[i], even), odd = fmaf(y[i + 1], y[i + 1], odd);
      float sum = even + odd;
      for (int o = lph >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      r = rsqrtf(sum * (1.f / D) + p.eps);
    }
    auto normed = [&](float x, int e) -> float {
      if (!w) return x;
      const float g = p.w_f32 ? reinterpret_cast<const float*>(w)[e] : to_f32<S>(reinterpret_cast<const S*>(w)[e]);
      return __fmul_rn(__fmul_rn(x, r), g);
    };
    const int half = p.R / 2;
    const float* cs = p.cos_sin + pos * p.R;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = element(i);
      if (!mine) break;
      y[i] = normed(y[i], e);
      if (e < p.R) {
        // the pair's other element, and whether this is its first
        const bool first = p.interleaved ? (e & 1) == 0 : e < half;
        const int other = p.interleaved ? e ^ 1 : (first ? e + half : e - half);
        const int a = p.interleaved ? e >> 1 : (first ? e : e - half);
        const float s = cs[half + a];
        y[i] = turned(y[i], normed(to_f32<S>(src[other]), other), cs[a], first ? -s : s);
      }
    }
  }
  if (!mine) return;
  if (kind == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q_out[element(i)] = from_f32<S>(y[i]);
  } else {
    P* out = reinterpret_cast<P*>(kind == 1 ? p.k_cache : p.v_cache) + (row * p.HKV + h) * D;
    const float* sc = kind == 1 ? p.k_scale : p.v_scale;
    const float qs = sizeof(P) == 1 && sc ? sc[h] : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) out[element(i)] = from_f32<P>(sizeof(P) == 1 ? __fdiv_rn(y[i], qs) : y[i]);
  }
}

template <typename S, typename P>
static int launch_typed(const Params& p, cudaStream_t s) {
  const int64_t D = int64_t(8) << p.lph_shift, heads = p.H + 2 * p.HKV;
  auto strides = [](int64_t tok, int64_t head) { return (tok * sizeof(S)) % 16 == 0 && (head * sizeof(S)) % 16 == 0; };
  const bool wide = aligned16(p.q) && aligned16(p.k) && aligned16(p.v) && strides(p.q_tok, p.q_head) &&
                    strides(p.k_tok, p.k_head) && strides(p.v_tok, p.v_head) && aligned16(p.q_out) &&
                    aligned16(p.k_cache) && aligned16(p.v_cache) && aligned16(p.q_weight) &&
                    aligned16(p.k_weight) && aligned16(p.cos_sin) && p.R % 8 == 0;
  if (wide && p.T <= 0x7fffffff && p.H * D <= 0x7fffffff) {
    int sms = 0;
    if (device_sm_count(&sms) != PA_OK) return PA_ERR_NO_DEVICE;
    if (p.T <= 4 * sms)
      qk_append_kernel<S, P, 1><<<dim3((unsigned)p.T, 3), kThreads, 0, s>>>(p);
    else if (p.H * D <= 1024)
      qk_append_kernel<S, P, 2><<<(unsigned)((p.T + 1) / 2), kThreads, 0, s>>>(p);
    else
      qk_append_kernel<S, P, 1><<<(unsigned)p.T, kThreads, 0, s>>>(p);
  } else {
    const int64_t ctas = (p.T * heads + kThreads / 32 - 1) / (kThreads / 32);
    if (ctas > 0x7fffffff) return PA_ERR_TOO_LARGE;
    qk_append_any_kernel<S, P><<<(unsigned)ctas, kThreads, 0, s>>>(p);
  }
  return cuda_status(cudaGetLastError());
}

template <typename S>
static int launch_src(const Params& p, int pool_dtype, cudaStream_t s) {
  switch (pool_dtype) {
    case PA_DTYPE_F16: return launch_typed<S, __half>(p, s);
    case PA_DTYPE_BF16: return launch_typed<S, __nv_bfloat16>(p, s);
    case PA_DTYPE_F32: return launch_typed<S, float>(p, s);
    case PA_DTYPE_F64: return launch_typed<S, double>(p, s);
    default: return launch_typed<S, __nv_fp8_e4m3>(p, s);
  }
}

}  // namespace qkappend
}  // namespace pa

extern "C" int pa_qk_norm_rope_append(
    void* q_out, const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
    int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
    int64_t v_head_stride, int io_dtype, const void* q_weight, const void* k_weight,
    int weight_dtype, double eps, const float* cos_sin, int64_t max_positions, int64_t rot_dim,
    int interleaved, const int32_t* positions, const int32_t* seq_ids, int64_t num_tokens,
    void* k_cache, void* v_cache, int kv_dtype, const float* k_scale, const float* v_scale,
    const int32_t* block_tables, int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t block_size, int64_t num_blocks, int64_t max_blocks,
    int32_t* dev_status, void* stream) {
  using namespace pa;
  if (num_tokens < 0 || num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      block_size <= 0 || num_blocks < 0 || max_blocks < 0 || max_positions < 0 || rot_dim < 0 ||
      rot_dim > head_dim || (rot_dim & 1))
    return PA_ERR_INVALID_ARGUMENT;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256) return PA_ERR_HEAD_DIM;
  if (io_dtype != PA_DTYPE_F32 && io_dtype != PA_DTYPE_F16 && io_dtype != PA_DTYPE_BF16) return PA_ERR_DTYPE;
  if (dtype_size(kv_dtype) == 0) return PA_ERR_DTYPE;
  if ((q_weight || k_weight) && weight_dtype != PA_DTYPE_F32 && weight_dtype != io_dtype) return PA_ERR_DTYPE;
  if (!seq_ids && num_tokens > num_seqs) return PA_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return PA_OK;
  if (!q_out || !q || !k || !v || !positions || !k_cache || !v_cache || !block_tables || (!cos_sin && rot_dim))
    return PA_ERR_INVALID_ARGUMENT;
  int sms = 0;
  if (device_sm_count(&sms) != PA_OK) return PA_ERR_NO_DEVICE;
  qkappend::Params p = {};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.q_tok = q_token_stride;
  p.q_head = q_head_stride;
  p.k_tok = k_token_stride;
  p.k_head = k_head_stride;
  p.v_tok = v_token_stride;
  p.v_head = v_head_stride;
  p.q_weight = static_cast<const char*>(q_weight);
  p.k_weight = static_cast<const char*>(k_weight);
  p.w_f32 = weight_dtype == PA_DTYPE_F32;
  p.eps = (float)eps;
  p.cos_sin = cos_sin;
  p.max_pos = max_positions;
  p.R = (int32_t)rot_dim;
  p.interleaved = interleaved;
  p.positions = positions;
  p.seq_ids = seq_ids;
  p.tables = block_tables;
  p.T = num_tokens;
  p.H = num_heads;
  p.HKV = num_kv_heads;
  p.MB = max_blocks;
  p.n_seqs = num_seqs;
  p.BS = block_size;
  p.NB = num_blocks;
  p.q_out = static_cast<char*>(q_out);
  p.k_cache = static_cast<char*>(k_cache);
  p.v_cache = static_cast<char*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  for (p.lph_shift = 2; (int64_t(8) << p.lph_shift) < head_dim; ++p.lph_shift) {}
  p.bs_shift = -1;
  if ((block_size & (block_size - 1)) == 0)
    for (p.bs_shift = 0; (int64_t(1) << p.bs_shift) < block_size; ++p.bs_shift) {}
  p.dev_status = dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (io_dtype) {
    case PA_DTYPE_F32: return qkappend::launch_src<float>(p, kv_dtype, s);
    case PA_DTYPE_F16: return qkappend::launch_src<__half>(p, kv_dtype, s);
    default: return qkappend::launch_src<__nv_bfloat16>(p, kv_dtype, s);
  }
}
