// kv_cache.cu -- the paged key-value cache: appending packed rows (with their
// quantisation to e4m3) and gathering them back.
//
// A row is one head's `dim` (<= 128) values of one token; a group of 4, 8 or 16
// lanes takes it, 16 bytes of binary16 per lane.  The quantisation is
//   e = smallest integer >= -15 with max |x| <= 448 * 2^e,
//   code = e4m3(x * 2^-e)  (round to nearest even),
// which is bit arithmetic on the maximum: with max |x| = 1.f * 2^E and
// 448 = 1.75 * 2^8, e = E - 8 + (1.f > 1.75).  Scaling by a power of two is
// exact, so the only rounding is the one to e4m3.
#include "kv_cache.cuh"

namespace uk {
__device__ unsigned int g_kv_fault = 0;
}  // namespace uk

namespace {

constexpr int THREADS = 256;
constexpr float VALUE_MAX = 61440.f;  // 240 * 2^8

struct Rows {  // packed rows [total][heads][dim], strides in elements
  uint16_t* k;
  uint16_t* v;
  int64_t k_token, k_head, v_token, v_head;
  int64_t total;
};

// position in the cache of packed row t: sequence, page and offset.  False
// when the row has none (padding, below position 0, or no page: *absent).
__device__ __forceinline__ bool locate(const UkKvView& c, const int32_t* cu, const int32_t* lens, int n_seq, int64_t t,
                                       int* page, int* off, bool* mine) {
  const int b = uk_find_seq(cu, n_seq, t);
  *mine = b >= 0;
  if (b < 0) return false;
  const int64_t pos = max(__ldg(lens + b), 0) - ((int64_t)__ldg(cu + b + 1) - t);
  if (pos < 0) return false;
  *page = pos <= 0x7fffffff ? uk_kv_page(c, b, (int)pos, off) : -1;
  if (*page < 0) atomicOr(&uk::g_kv_fault, UK_FAULT_PAGE);
  return *page >= 0;
}

template <int GL>
__global__ void __launch_bounds__(THREADS) k_kv_append(Rows in, UkKvView c, const int32_t* __restrict__ cu,
                                                       const int32_t* __restrict__ lens, int n_seq) {
  const int64_t row = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / GL;
  const int l = threadIdx.x % GL;
  const int64_t t = row / (2 * c.heads);
  const int r = (int)(row - t * (2 * c.heads));
  const bool is_v = r >= c.heads;
  const int h = is_v ? r - c.heads : r;
  int page = 0, off = 0;
  bool mine = false;
  const bool ok = t < in.total && locate(c, cu, lens, n_seq, t, &page, &off, &mine);
  const bool act = ok && l * 8 < c.dim;
  uint4 x = make_uint4(0, 0, 0, 0);
  if (act) {
    const uint16_t* p = is_v ? in.v + t * in.v_token + h * in.v_head : in.k + t * in.k_token + h * in.k_head;
    x = __ldg(reinterpret_cast<const uint4*>(p) + l);
  }
  uint8_t* dst = (is_v ? c.v : c.k) + uk_kv_row(c, page, off, h);
  if (c.kind == UK_KV_F16) {
    if (act) reinterpret_cast<uint4*>(dst)[l] = x;
    return;
  }
  float f[8];
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t2 = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t2.x;
    f[2 * i + 1] = t2.y;
    top = fmaxf(top, fmaxf(fabsf(t2.x), fabsf(t2.y)));
  }
#pragma unroll
  for (int o = GL / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  top = fminf(top, VALUE_MAX);
  // exponent of the scale, biased by 127: carry into the exponent field when
  // the significand is above 1.75
  const int e = max((int)((__float_as_uint(top) + 0x1FFFFFu) >> 23) - 8, 127 - 15);
  const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
  if (!act) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // a NaN fails both comparisons and stays
    f[i] = f[i] > VALUE_MAX ? VALUE_MAX : f[i] < -VALUE_MAX ? -VALUE_MAX : f[i];
    f[i] *= inv;
  }
  uint2 codes;
  codes.x = uk_float2_to_e4m3x2(f[0], f[1]) | uk_float2_to_e4m3x2(f[2], f[3]) << 16;
  codes.y = uk_float2_to_e4m3x2(f[4], f[5]) | uk_float2_to_e4m3x2(f[6], f[7]) << 16;
  reinterpret_cast<uint2*>(dst)[l] = codes;
  if (l == 0) (is_v ? c.v_exp : c.k_exp)[uk_kv_exp(c, page, off, h)] = (uint8_t)e;
}

template <int GL>
__global__ void __launch_bounds__(THREADS) k_kv_gather(Rows out, UkKvView c, const int32_t* __restrict__ cu,
                                                       const int32_t* __restrict__ lens, int n_seq) {
  const int64_t row = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / GL;
  const int l = threadIdx.x % GL;
  const int64_t t = row / (2 * c.heads);
  const int r = (int)(row - t * (2 * c.heads));
  const bool is_v = r >= c.heads;
  const int h = is_v ? r - c.heads : r;
  int page = 0, off = 0;
  bool mine = false;
  if (t >= out.total || l * 8 >= c.dim) return;
  const bool ok = locate(c, cu, lens, n_seq, t, &page, &off, &mine);
  if (!mine) return;
  uint4 x = make_uint4(0, 0, 0, 0);
  if (ok) {
    const uint8_t* src = (is_v ? c.v : c.k) + uk_kv_row(c, page, off, h);
    if (c.kind == UK_KV_F16) {
      x = reinterpret_cast<const uint4*>(src)[l];
    } else {
      const uint2 codes = reinterpret_cast<const uint2*>(src)[l];
      const float s = uk_exp_scale((is_v ? c.v_exp : c.k_exp)[uk_kv_exp(c, page, off, h)]);
      const uint32_t w[4] = {codes.x, codes.x >> 16, codes.y, codes.y >> 16};
      uint32_t y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t h2 = uk_e4m3x2_to_half2(w[i]);
        float2 t2 = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        const __half2 o2 = __floats2half2_rn(t2.x * s, t2.y * s);
        y[i] = *reinterpret_cast<const uint32_t*>(&o2);
      }
      x = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
  uint16_t* p = is_v ? out.v + t * out.v_token + h * out.v_head : out.k + t * out.k_token + h * out.k_head;
  reinterpret_cast<uint4*>(p)[l] = x;
}


int lanes_for(int dim) { return dim <= 32 ? 4 : dim <= 64 ? 8 : 16; }

}  // namespace

namespace uk {

int check_rows(const char* what, const char* name, const void* p, int64_t tokens, int heads, int64_t token_stride,
               int64_t head_stride, int64_t least) {
  if (int rc = check_device_ptr(p, name)) return rc;
  if (!aligned16(p)) return fail(UK_EINVAL, "%s: %s is not 16-byte aligned", what, name);
  if ((tokens > 1 && (token_stride < least || token_stride % 8 != 0)) ||
      (heads > 1 && (head_stride < least || head_stride % 8 != 0)))
    return fail(UK_EINVAL, "%s: strides of %s (%lld per token, %lld per head) must be multiples of 8, at least %lld",
                what, name, (long long)token_stride, (long long)head_stride, (long long)least);
  return UK_OK;
}

int kv_view(const uk_kv_cache* c, const int32_t* table, int64_t table_stride, int n_seq, int max_pages,
            const char* what, UkKvView* out) {
  if (c == nullptr) return fail(UK_EINVAL, "%s: the cache is NULL", what);
  if (c->kind != UK_KV_F16 && c->kind != UK_KV_E4M3) return fail(UK_EINVAL, "%s: unknown cache kind %d", what, c->kind);
  const int es = c->kind == UK_KV_F16 ? 2 : 1, step = 16 / es;
  if (c->dim < 8 || c->dim > 128 || c->dim % step != 0)
    return fail(UK_EINVAL, "%s: dim %d must be a multiple of %d from %d to 128", what, c->dim, step, step);
  if (c->heads < 1 || c->heads > 65535 || c->page_size < 1 || c->pages < 0 || c->pages > 0x7fffffff)
    return fail(UK_EINVAL, "%s: heads %d, page_size %d, pages %lld", what, c->heads, c->page_size,
                (long long)c->pages);
  if (max_pages < 0 || (n_seq > 1 && table_stride < max_pages))
    return fail(UK_EINVAL, "%s: max_pages %d, table_stride %lld", what, max_pages, (long long)table_stride);
  // kernels look some tiles ahead of the last position in 32 bits
  if ((int64_t)max_pages * c->page_size > 0x7ffff000)
    return fail(UK_EINVAL, "%s: max_pages * page_size = %lld positions do not fit 31 bits", what,
                (long long)max_pages * c->page_size);
  if ((c->pages > 1 && (c->page_stride < c->dim || c->page_stride % step != 0)) ||
      (c->page_size > 1 && (c->token_stride < c->dim || c->token_stride % step != 0)) ||
      (c->heads > 1 && (c->head_stride < c->dim || c->head_stride % step != 0)))
    return fail(UK_EINVAL, "%s: cache strides %lld / %lld / %lld must be multiples of %d, at least dim", what,
                (long long)c->page_stride, (long long)c->token_stride, (long long)c->head_stride, step);
  if (c->pages > 0) {
    if (int rc = check_device_ptr(c->k, "cache k")) return rc;
    if (int rc = check_device_ptr(c->v, "cache v")) return rc;
    if (!aligned16(c->k) || !aligned16(c->v)) return fail(UK_EINVAL, "%s: the pools must be 16-byte aligned", what);
    if (c->kind == UK_KV_E4M3) {
      if (int rc = check_device_ptr(c->k_exp, "cache k_exp")) return rc;
      if (int rc = check_device_ptr(c->v_exp, "cache v_exp")) return rc;
    }
  }
  if (max_pages > 0)
    if (int rc = check_device_ptr(table, "block_table")) return rc;
  *out = UkKvView{(uint8_t*)c->k, (uint8_t*)c->v, c->k_exp, c->v_exp, c->page_stride * es, c->token_stride * es,
                  c->head_stride * es, c->pages, c->page_size, c->heads, c->dim, c->kind,
                  UkFastDiv::make((uint32_t)c->page_size), table, table_stride, max_pages};
  return UK_OK;
}

unsigned kv_fault_take() {
  unsigned v = 0;
  const unsigned zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_kv_fault, sizeof(v)) != cudaSuccess) return 0xFFFFFFFFu;
  cudaMemcpyToSymbol(g_kv_fault, &zero, sizeof(zero));
  return v;
}

}  // namespace uk

namespace {

// checks shared by append and gather; *blocks = 0 when there is nothing to do
int prepare(const char* what, Rows* rows, const uk_kv_cache* cache, const int32_t* table, int64_t table_stride,
            int max_pages, const int32_t* cu, const int32_t* lens, int n_seq, int64_t least, UkKvView* view,
            int64_t* blocks) {
  *blocks = 0;
  if (rows->total < 0 || n_seq < 0) return uk::fail(UK_EINVAL, "%s: negative total or n_seq", what);
  if (rows->total > 0x7fffffff) return uk::fail(UK_EINVAL, "%s: total %lld exceeds 31 bits", what, (long long)rows->total);
  if (int rc = uk::kv_view(cache, table, table_stride, n_seq, max_pages, what, view)) return rc;
  if (rows->total == 0 || n_seq == 0) return UK_OK;
  if (int rc = uk::check_rows(what, "K", rows->k, rows->total, cache->heads, rows->k_token, rows->k_head, least)) return rc;
  if (int rc = uk::check_rows(what, "V", rows->v, rows->total, cache->heads, rows->v_token, rows->v_head, least)) return rc;
  if (int rc = uk::check_device_ptr(cu, "cu_seqlens")) return rc;
  if (int rc = uk::check_device_ptr(lens, "seq_lens")) return rc;
  const int per = THREADS / lanes_for(cache->dim);
  *blocks = (rows->total * 2 * cache->heads + per - 1) / per;
  if (*blocks > 0x7fffffff) return uk::fail(UK_EINVAL, "%s: %lld rows exceed the grid", what, (long long)rows->total);
  return UK_OK;
}

}  // namespace

extern "C" int uk_cuda_kv_append_f16(const uint16_t* K, int64_t k_token_stride, int64_t k_head_stride,
                                     const uint16_t* V, int64_t v_token_stride, int64_t v_head_stride, int64_t total,
                                     const uk_kv_cache* cache, const int32_t* block_table, int64_t table_stride,
                                     int max_pages, const int32_t* cu_new, const int32_t* seq_lens, int n_seq,
                                     void* stream) {
  Rows rows{(uint16_t*)K, (uint16_t*)V, k_token_stride, k_head_stride, v_token_stride, v_head_stride, total};
  UkKvView view;
  int64_t blocks;
  if (int rc = prepare("kv_append", &rows, cache, block_table, table_stride, max_pages, cu_new, seq_lens, n_seq, 0,
                       &view, &blocks))
    return rc;
  if (blocks == 0) return UK_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (lanes_for(cache->dim)) {
    case 4: k_kv_append<4><<<(unsigned)blocks, THREADS, 0, st>>>(rows, view, cu_new, seq_lens, n_seq); break;
    case 8: k_kv_append<8><<<(unsigned)blocks, THREADS, 0, st>>>(rows, view, cu_new, seq_lens, n_seq); break;
    default: k_kv_append<16><<<(unsigned)blocks, THREADS, 0, st>>>(rows, view, cu_new, seq_lens, n_seq); break;
  }
  return uk::check_launch("kv_append");
}

extern "C" int uk_cuda_kv_gather_f16(const uk_kv_cache* cache, const int32_t* block_table, int64_t table_stride,
                                     int max_pages, const int32_t* cu_out, const int32_t* seq_lens, int n_seq,
                                     uint16_t* K, int64_t k_token_stride, int64_t k_head_stride, uint16_t* V,
                                     int64_t v_token_stride, int64_t v_head_stride, int64_t total, void* stream) {
  Rows rows{K, V, k_token_stride, k_head_stride, v_token_stride, v_head_stride, total};
  UkKvView view;
  int64_t blocks;
  if (int rc = prepare("kv_gather", &rows, cache, block_table, table_stride, max_pages, cu_out, seq_lens, n_seq,
                       cache != nullptr ? cache->dim : 0, &view, &blocks))
    return rc;
  if (blocks == 0) return UK_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (lanes_for(cache->dim)) {
    case 4: k_kv_gather<4><<<(unsigned)blocks, THREADS, 0, st>>>(rows, view, cu_out, seq_lens, n_seq); break;
    case 8: k_kv_gather<8><<<(unsigned)blocks, THREADS, 0, st>>>(rows, view, cu_out, seq_lens, n_seq); break;
    default: k_kv_gather<16><<<(unsigned)blocks, THREADS, 0, st>>>(rows, view, cu_out, seq_lens, n_seq); break;
  }
  return uk::check_launch("kv_gather");
}
