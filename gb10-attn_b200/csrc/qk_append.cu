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

// One warp per (token, head) of the H + 2 HKV heads; lane holds elements
// lane + 32 i.
template <typename S, typename P, int D>
__global__ void __launch_bounds__(256) qk_append_kernel(const __grid_constant__ Params p) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t heads = p.H + 2 * p.HKV;
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= p.T * heads) return;
  const int64_t t = unit / heads, hh = unit % heads;
  const int kind = hh < p.H ? 0 : (hh < p.H + p.HKV ? 1 : 2);  // q, k, v
  const int64_t h = kind == 0 ? hh : (kind == 1 ? hh - p.H : hh - p.H - p.HKV);
  const int64_t pos = p.positions[t];
  const bool known = pos >= 0 && pos < p.max_pos;

  // the row of the pool
  char* row = nullptr;
  if (kind != 0) {
    if (pos < 0) return;
    if (!known) {
      if (lane == 0) report(p.dev_status, PA_DEVERR_CONTEXT);
      return;
    }
    const int64_t seq = p.seq_ids ? p.seq_ids[t] : t;
    const int64_t page = pos / p.BS;
    if (seq < 0 || seq >= p.n_seqs || page >= p.MB) {
      if (lane == 0) report(p.dev_status, PA_DEVERR_CONTEXT);
      return;
    }
    const int64_t blk = p.tables[seq * p.MB + page];
    if (blk < 0 || blk >= p.NB) {
      if (lane == 0) report(p.dev_status, PA_DEVERR_BLOCK_ID);
      return;
    }
    row = (kind == 1 ? p.k_cache : p.v_cache) +
          ((blk * p.BS + (pos - page * p.BS)) * p.HKV + h) * D * (int64_t)sizeof(P);
  } else if (!known) {
    // a padding token's q is zero, one past the table's is NaN
    if (pos >= 0 && lane == 0) report(p.dev_status, PA_DEVERR_CONTEXT);
    S* out = reinterpret_cast<S*>(p.q_out) + (t * p.H + h) * D;
    for (int i = 0; i < N; ++i) out[lane + 32 * i] = from_f32<S>(pos < 0 ? 0.f : __int_as_float(0x7fc00000));
    return;
  }

  const S* src = kind == 0   ? reinterpret_cast<const S*>(p.q) + t * p.q_tok + h * p.q_head
                 : kind == 1 ? reinterpret_cast<const S*>(p.k) + t * p.k_tok + h * p.k_head
                             : reinterpret_cast<const S*>(p.v) + t * p.v_tok + h * p.v_head;
  float y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = to_f32<S>(src[lane + 32 * i]);
  if (kind != 2) {
    const char* w = kind == 0 ? p.q_weight : p.k_weight;
    float r = 1.f;
    if (w) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) sum = fmaf(y[i], y[i], sum);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      r = rsqrtf(sum * (1.f / D) + p.eps);
    }
    auto weight = [&](int e) -> float {
      if (!w) return 1.f;
      return p.w_f32 ? reinterpret_cast<const float*>(w)[e] : to_f32<S>(reinterpret_cast<const S*>(w)[e]);
    };
    const int half = p.R / 2;
    const float* cs = p.cos_sin + pos * p.R;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = lane + 32 * i;
      const float x = y[i] * r * weight(e);
      if (e < p.R) {
        // the pair's other element, and whether this is its first
        const bool first = p.interleaved ? (e & 1) == 0 : e < half;
        const int other = p.interleaved ? e ^ 1 : (first ? e + half : e - half);
        const int a = p.interleaved ? e >> 1 : (first ? e : e - half);
        const float xo = to_f32<S>(src[other]) * r * weight(other);
        const float c = cs[a], s = cs[half + a];
        y[i] = first ? x * c - xo * s : x * c + xo * s;
      } else {
        y[i] = x;
      }
    }
  }
  if (kind == 0) {
    S* out = reinterpret_cast<S*>(p.q_out) + (t * p.H + h) * D;
#pragma unroll
    for (int i = 0; i < N; ++i) out[lane + 32 * i] = from_f32<S>(y[i]);
  } else {
    P* out = reinterpret_cast<P*>(row);
    const float* sc = kind == 1 ? p.k_scale : p.v_scale;
    const float qs = sizeof(P) == 1 && sc ? sc[h] : 1.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      out[lane + 32 * i] = from_f32<P>(sizeof(P) == 1 ? __fdiv_rn(y[i], qs) : y[i]);
  }
}

template <typename S, typename P>
static int launch_typed(const Params& p, int64_t D, cudaStream_t s) {
  const int64_t ctas = (p.T * (p.H + 2 * p.HKV) + 7) / 8;
  if (ctas > (int64_t(1) << 31) - 1) return PA_ERR_TOO_LARGE;
  switch (D) {
    case 32: qk_append_kernel<S, P, 32><<<(unsigned)ctas, 256, 0, s>>>(p); break;
    case 64: qk_append_kernel<S, P, 64><<<(unsigned)ctas, 256, 0, s>>>(p); break;
    case 128: qk_append_kernel<S, P, 128><<<(unsigned)ctas, 256, 0, s>>>(p); break;
    default: qk_append_kernel<S, P, 256><<<(unsigned)ctas, 256, 0, s>>>(p); break;
  }
  return cuda_status(cudaGetLastError());
}

template <typename S>
static int launch_src(const Params& p, int pool_dtype, int64_t D, cudaStream_t s) {
  switch (pool_dtype) {
    case PA_DTYPE_F16: return launch_typed<S, __half>(p, D, s);
    case PA_DTYPE_BF16: return launch_typed<S, __nv_bfloat16>(p, D, s);
    case PA_DTYPE_F32: return launch_typed<S, float>(p, D, s);
    case PA_DTYPE_F64: return launch_typed<S, double>(p, D, s);
    default: return launch_typed<S, __nv_fp8_e4m3>(p, D, s);
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
  p.dev_status = dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (io_dtype) {
    case PA_DTYPE_F32: return qkappend::launch_src<float>(p, kv_dtype, head_dim, s);
    case PA_DTYPE_F16: return qkappend::launch_src<__half>(p, kv_dtype, head_dim, s);
    default: return qkappend::launch_src<__nv_bfloat16>(p, kv_dtype, head_dim, s);
  }
}
