// attn_decode.cu -- attention of one new token per sequence over a paged cache:
//   O[b][h] = sum_p w_p V[p][g],  w = softmax(scale * Q[b][h] . K[p][g]),
// p < seq_lens[b], g = h / (query heads per key head), in one pass over the
// cache with the running maximum m and sum l of the softmax:
//   m' = max(m, s),  l' = l 2^(m - m') + 2^(s - m'),  o' = o 2^(m - m') + 2^(s - m') v
// (scores s carry scale * log2 e, so every exponential is a power of two).
#include "kv_cache.cuh"

namespace uk {
__device__ unsigned int g_attn_decode_fault = 0;
}  // namespace uk

namespace {

constexpr int WARPS = 4;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Args {
  const uint16_t* q;
  int64_t q_seq, q_head;
  uint16_t* o;
  int64_t o_seq, o_head;
  float* lse;
  const int32_t* lens;
  int n_seq, heads_q, group;
  float scale2;  // scale * log2 e
};

// four values of a cache row as floats
__device__ __forceinline__ float4 row4(const UkKvView& c, const uint8_t* row, const uint8_t* e, int lane) {
  if (lane * 4 >= c.dim) return make_float4(0.f, 0.f, 0.f, 0.f);
  uint2 h;
  float s = 1.f;
  if (c.kind == UK_KV_F16) {
    h = __ldg(reinterpret_cast<const uint2*>(row) + lane);
  } else {
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(row) + lane);
    h = make_uint2(uk_e4m3x2_to_half2(w), uk_e4m3x2_to_half2(w >> 16));
    s = uk_exp_scale(__ldg(e));
  }
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&h.x)), b = __half22float2(*reinterpret_cast<__half2*>(&h.y));
  return make_float4(a.x * s, a.y * s, b.x * s, b.y * s);
}

// One CTA per (sequence, query head); each warp takes every fourth position,
// a lane four of the row's values.
__global__ void __launch_bounds__(WARPS * 32) k_attn_decode(Args a, UkKvView c) {
  __shared__ float sm[WARPS], sl[WARPS];
  __shared__ float4 so[WARPS][32];
  const int b = blockIdx.x / a.heads_q, h = blockIdx.x % a.heads_q, g = h / a.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t room = (int64_t)c.max_pages * c.page_size;
  int len = max(__ldg(a.lens + b), 0);
  if (len > room) {
    if (threadIdx.x == 0) atomicOr(&uk::g_attn_decode_fault, UK_FAULT_PAGE);
    len = (int)room;
  }
  float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
  if (lane * 4 < c.dim) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(a.q + b * a.q_seq + h * a.q_head) + lane);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    q = make_float4(x.x, x.y, y.x, y.y);
  }
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = warp; p < len; p += WARPS) {
    int off;
    const int page = uk_kv_page(c, b, p, &off);
    if (page < 0) {
      if (lane == 0) atomicOr(&uk::g_attn_decode_fault, UK_FAULT_PAGE);
      continue;
    }
    const int64_t at = uk_kv_row(c, page, off, g), ea = uk_kv_exp(c, page, off, g);
    const float4 k = row4(c, c.k + at, c.k_exp + ea, lane), v = row4(c, c.v + at, c.v_exp + ea, lane);
    const float s = uk_warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * a.scale2;
    const float m2 = fmaxf(m, s);
    const float f = m2 == -INFINITY ? 1.f : exp2f(m - m2), e = m2 == -INFINITY ? 0.f : exp2f(s - m2);
    m = m2;
    l = l * f + e;
    o = make_float4(o.x * f + e * v.x, o.y * f + e * v.y, o.z * f + e * v.z, o.w * f + e * v.w);
  }
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  so[warp][lane] = o;
  __syncthreads();
  if (warp != 0) return;
  m = -INFINITY;
  for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sm[w]);
  l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = 0; w < WARPS; ++w) {
    const float f = sm[w] == -INFINITY ? (sl[w] != 0.f ? 1.f : 0.f) : exp2f(sm[w] - m);
    const float4 x = so[w][lane];
    l += sl[w] * f;
    o = make_float4(o.x + x.x * f, o.y + x.y * f, o.z + x.z * f, o.w + x.w * f);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane * 4 < c.dim) {
    const __half2 x = __floats2half2_rn(o.x * inv, o.y * inv), y = __floats2half2_rn(o.z * inv, o.w * inv);
    reinterpret_cast<uint2*>(a.o + b * a.o_seq + h * a.o_head)[lane] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
  if (a.lse != nullptr && lane == 0) a.lse[(int64_t)b * a.heads_q + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

}  // namespace

namespace uk {
unsigned attn_decode_fault_take() {
  unsigned v = 0;
  const unsigned zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_decode_fault, sizeof(v)) != cudaSuccess) return 0xFFFFFFFFu;
  cudaMemcpyToSymbol(g_attn_decode_fault, &zero, sizeof(zero));
  return v;
}
}  // namespace uk

extern "C" size_t uk_cuda_attn_decode_workspace_size(int heads_q, int heads_kv, int dim) {
  if (heads_q <= 0 || heads_kv <= 0 || dim <= 0) return 0;
  return 16;
}

extern "C" int uk_cuda_attn_decode_f16(const uint16_t* Q, int64_t q_seq_stride, int64_t q_head_stride,
                                       const uk_kv_cache* cache, const int32_t* block_table, int64_t table_stride,
                                       int max_pages, const int32_t* seq_lens, int n_seq, int heads_q, float scale,
                                       uint16_t* O, int64_t o_seq_stride, int64_t o_head_stride, float* LSE,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  if (n_seq < 0 || heads_q < 1) return uk::fail(UK_EINVAL, "attn_decode: n_seq %d, heads_q %d", n_seq, heads_q);
  if (!(scale - scale == 0.f)) return uk::fail(UK_EINVAL, "attn_decode: the scale is not finite");
  UkKvView c;
  if (int rc = uk::kv_view(cache, block_table, table_stride, n_seq, max_pages, "attn_decode", &c)) return rc;
  if (heads_q % cache->heads != 0)
    return uk::fail(UK_EINVAL, "attn_decode: %d query heads do not divide over %d key heads", heads_q, cache->heads);
  if (n_seq == 0) return UK_OK;
  if ((int64_t)n_seq * heads_q > 0x7fffffff) return uk::fail(UK_EINVAL, "attn_decode: n_seq * heads_q exceeds the grid");
  if (int rc = uk::check_rows("attn_decode", "Q", Q, n_seq, heads_q, q_seq_stride, q_head_stride, 0)) return rc;
  if (int rc = uk::check_rows("attn_decode", "O", O, n_seq, heads_q, o_seq_stride, o_head_stride, cache->dim)) return rc;
  if (int rc = uk::check_device_ptr(seq_lens, "seq_lens")) return rc;
  if (LSE != nullptr)
    if (int rc = uk::check_device_ptr(LSE, "LSE")) return rc;
  if (int rc = uk::check_device_ptr(workspace, "workspace")) return rc;
  const size_t need = uk_cuda_attn_decode_workspace_size(heads_q, cache->heads, cache->dim);
  if (workspace_bytes < need || !uk::aligned16(workspace))
    return uk::fail(UK_EINVAL, "attn_decode: workspace of %zu bytes, %zu wanted, 16-byte aligned", workspace_bytes, need);
  Args a{Q, q_seq_stride, q_head_stride, O, o_seq_stride, o_head_stride, LSE, seq_lens, n_seq, heads_q,
         heads_q / cache->heads, scale * LOG2E};
  k_attn_decode<<<(unsigned)(n_seq * heads_q), WARPS * 32, 0, (cudaStream_t)stream>>>(a, c);
  return uk::check_launch("attn_decode");
}
