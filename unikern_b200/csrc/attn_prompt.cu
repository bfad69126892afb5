// attn_prompt.cu -- attention over packed prompts, causal or full, with grouped
// heads: O[i][h] = sum_j w_j V[j][g], w = softmax_j(scale * Q[i][h] . K[j][g])
// over the keys row i sees, in one pass with the softmax's running maximum and
// sum (scores carry scale * log2 e, so every exponential is a power of two).
#include "kv_cache.cuh"

namespace uk {
__device__ unsigned int g_attn_prompt_fault = 0;
}  // namespace uk

namespace {

constexpr int WARPS = 4;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Args {
  const uint16_t *q, *k, *v;
  uint16_t* o;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  float* lse;
  const int32_t *cu_q, *cu_k;
  int n_seq, heads_q, heads_kv, group, dim, causal;
  int64_t total_q, total_k;
  float scale2;
};

__device__ __forceinline__ float4 row4(const uint16_t* row, int lane, int dim) {
  if (lane * 4 >= dim) return make_float4(0.f, 0.f, 0.f, 0.f);
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(row) + lane);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  return make_float4(x.x, x.y, y.x, y.y);
}

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// One warp per (query row, head), a lane four of the row's values.
__global__ void __launch_bounds__(WARPS * 32) k_attn_prompt_rows(Args a) {
  const int64_t w = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t t = w / a.heads_q;
  const int h = (int)(w - t * a.heads_q), g = h / a.group;
  if (t >= a.total_q) return;
  const int b = uk_find_seq(a.cu_q, a.n_seq, t);
  if (b < 0) return;
  const int64_t q1 = clamp64(__ldg(a.cu_q + b + 1), 0, a.total_q);
  const int64_t k0 = clamp64(__ldg(a.cu_k + b), 0, a.total_k), k1 = clamp64(__ldg(a.cu_k + b + 1), k0, a.total_k);
  const int64_t end = a.causal ? k1 - (q1 - 1 - t) : k1;  // one past the last key this row sees
  const float4 q = row4(a.q + t * a.q_token + h * a.q_head, lane, a.dim);
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t j = k0; j < end; ++j) {
    const float4 k = row4(a.k + j * a.k_token + g * a.k_head, lane, a.dim);
    const float4 v = row4(a.v + j * a.v_token + g * a.v_head, lane, a.dim);
    const float s = uk_warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * a.scale2;
    const float m2 = fmaxf(m, s);
    const float f = m2 == -INFINITY ? 1.f : exp2f(m - m2), e = m2 == -INFINITY ? 0.f : exp2f(s - m2);
    m = m2;
    l = l * f + e;
    o = make_float4(o.x * f + e * v.x, o.y * f + e * v.y, o.z * f + e * v.z, o.w * f + e * v.w);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane * 4 < a.dim) {
    const __half2 x = __floats2half2_rn(o.x * inv, o.y * inv), y = __floats2half2_rn(o.z * inv, o.w * inv);
    reinterpret_cast<uint2*>(a.o + t * a.o_token + h * a.o_head)[lane] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
  if (a.lse != nullptr && lane == 0) a.lse[t * a.heads_q + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

}  // namespace

namespace uk {
unsigned attn_prompt_fault_take() {
  unsigned v = 0;
  const unsigned zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_prompt_fault, sizeof(v)) != cudaSuccess) return 0xFFFFFFFFu;
  cudaMemcpyToSymbol(g_attn_prompt_fault, &zero, sizeof(zero));
  return v;
}
}  // namespace uk

extern "C" int uk_cuda_attn_prompt_f16(const uint16_t* Q, int64_t q_token_stride, int64_t q_head_stride,
                                       const uint16_t* K, int64_t k_token_stride, int64_t k_head_stride,
                                       const uint16_t* V, int64_t v_token_stride, int64_t v_head_stride,
                                       const int32_t* cu_q, const int32_t* cu_k, int n_seq, int64_t total_q,
                                       int64_t total_k, int heads_q, int heads_kv, int dim, float scale, int causal,
                                       uint16_t* O, int64_t o_token_stride, int64_t o_head_stride, float* LSE,
                                       void* stream) {
  if (n_seq < 0 || total_q < 0 || total_k < 0 || total_q > 0x7fffffff || total_k > 0x7fffffff)
    return uk::fail(UK_EINVAL, "attn_prompt: n_seq %d, total_q %lld, total_k %lld", n_seq, (long long)total_q,
                    (long long)total_k);
  if (heads_kv < 1 || heads_q < 1 || heads_q > 65535 || heads_q % heads_kv != 0)
    return uk::fail(UK_EINVAL, "attn_prompt: %d query heads do not divide over %d key heads", heads_q, heads_kv);
  if (dim < 8 || dim > 128 || dim % 8 != 0)
    return uk::fail(UK_EINVAL, "attn_prompt: dim %d must be a multiple of 8 from 8 to 128", dim);
  if (!(scale - scale == 0.f)) return uk::fail(UK_EINVAL, "attn_prompt: the scale is not finite");
  if (total_q == 0 || n_seq == 0) return UK_OK;
  if (int rc = uk::check_rows("attn_prompt", "Q", Q, total_q, heads_q, q_token_stride, q_head_stride, dim)) return rc;
  if (int rc = uk::check_rows("attn_prompt", "O", O, total_q, heads_q, o_token_stride, o_head_stride, dim)) return rc;
  if (total_k > 0) {
    if (int rc = uk::check_rows("attn_prompt", "K", K, total_k, heads_kv, k_token_stride, k_head_stride, dim)) return rc;
    if (int rc = uk::check_rows("attn_prompt", "V", V, total_k, heads_kv, v_token_stride, v_head_stride, dim)) return rc;
  }
  if (int rc = uk::check_device_ptr(cu_q, "cu_q")) return rc;
  if (int rc = uk::check_device_ptr(cu_k, "cu_k")) return rc;
  if (LSE != nullptr)
    if (int rc = uk::check_device_ptr(LSE, "LSE")) return rc;
  Args a{Q, K, V, O, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
         o_token_stride, o_head_stride, LSE, cu_q, cu_k, n_seq, heads_q, heads_kv, heads_q / heads_kv, dim, causal,
         total_q, total_k, scale * LOG2E};
  const int64_t blocks = (total_q * heads_q + WARPS - 1) / WARPS;
  if (blocks > 0x7fffffff) return uk::fail(UK_EINVAL, "attn_prompt: total_q * heads_q exceeds the grid");
  k_attn_prompt_rows<<<(unsigned)blocks, WARPS * 32, 0, (cudaStream_t)stream>>>(a);
  return uk::check_launch("attn_prompt");
}
