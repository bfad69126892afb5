// kv_cache.cu -- the paged key-value cache: appending packed rows (with their
// quantisation to e4m3) and gathering them back.
//
// A block takes a run of 1 to 16 packed rows (tokens) with all their heads of
// keys and values.  One thread per token finds its sequence (binary search),
// page and offset, once; then groups of 2, 4 or 8 lanes take a head's row each,
// 16 values (32 bytes of binary16) a lane.  Bound
// by HBM: every row is read once and written once.  (One lookup per head's row
// and one row per lane group, as first written: 147 us for 4 x 16384 e4m3
// positions of 8 heads of 128.)
//
// The quantisation is
//   e = smallest integer >= -15 with max |x| <= 448 * 2^e,
//   code = e4m3(x * 2^-e)  (round to nearest even),
// which is bit arithmetic on the maximum: with max |x| = 1.f * 2^E and
// 448 = 1.75 * 2^8, e = E - 8 + (1.f > 1.75).  Scaling by a power of two is
// exact, so the only rounding is the one to e4m3.  Exponent bytes of
// neighbouring tokens are neighbours in memory: they are gathered in shared
// memory and written together.
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

constexpr int MAX_TOK = 16;   // tokens per block
constexpr int MAX_EXP = 2048; // exponent bytes staged per block
// Rows in flight per lane group, measured on one B200: the append runs its
// quantisation best with one (7000 tokens of 8 heads of 128 into e4m3 11.4 us,
// two 14.2, four 14.3), the gather, which only copies, with two and short
// blocks (4 x 16384 positions out of e4m3: 8 tokens a block 71.9 us, 16 72.6,
// 4 86.0; four rows 75.9, one 78.0).
constexpr int APPEND_ROWS = 1, GATHER_ROWS = 2, GATHER_TOK = 8;

struct Where {  // of a token: byte offset of head 0's row and index of its exponent
  int64_t row, exp;
};
constexpr int64_t ABSENT = -1, NOBODY = -2;  // no such position or page; no sequence's row

// The places of the block's tokens t0 .. t0 + tok - 1, by its first threads.  The
// bounds and lengths of up to MAX_SEQ sequences come into shared memory in one
// go and are searched there; more are searched where they lie.  (Searching in
// global memory, each step waiting for the last, cost a few microseconds of
// every call: a decode step's 32 rows.)
constexpr int MAX_SEQ = 1023;
struct Bounds {
  int32_t cu[MAX_SEQ + 1], lens[MAX_SEQ + 1];
};
__device__ __forceinline__ void locate(const UkKvView& c, const int32_t* cu, const int32_t* lens, int n_seq, int64_t t0,
                                       int tok, int64_t total, Bounds& s, Where* where) {
  const bool near = n_seq <= MAX_SEQ;
  if (near) {
    for (int i = threadIdx.x; i <= n_seq; i += THREADS) {
      s.cu[i] = __ldg(cu + i);
      if (i < n_seq) s.lens[i] = __ldg(lens + i);
    }
    __syncthreads();
  }
  if ((int)threadIdx.x < tok) {
    const int64_t t = t0 + threadIdx.x;
    Where w{NOBODY, 0};
    int b = -1;
    int64_t pos = -1;
    if (t < total) {
      b = near ? uk_find_seq<false>(s.cu, n_seq, t) : uk_find_seq<true>(cu, n_seq, t);
      if (b >= 0) pos = max(near ? s.lens[b] : __ldg(lens + b), 0) - ((near ? s.cu[b + 1] : __ldg(cu + b + 1)) - t);
    }
    if (b >= 0) w.row = ABSENT;
    if (pos >= 0) {
      int off;
      const int page = pos <= 0x7fffffff ? uk_kv_page(c, b, (int)pos, &off) : -1;
      if (page >= 0) {
        w.row = uk_kv_row(c, page, off, 0);
        w.exp = uk_kv_exp(c, page, off, 0);
      } else {
        atomicOr(&uk::g_kv_fault, UK_FAULT_PAGE);
      }
    }
    where[threadIdx.x] = w;
  }
  __syncthreads();
}

// 16 values of a binary16 row, the second 8 only where the row has them
struct Half16 {
  uint4 lo, hi;
};
__device__ __forceinline__ uint4 ldg16(const void* p, bool on) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (on)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}

// what a lane group works on: row i of the block's tokens x {k, v} x heads
struct Row {
  int tok, head;
  bool is_v;
};
__device__ __forceinline__ Row row_of(int i, int heads, const UkFastDiv& per_token) {
  Row r;
  r.tok = (int)per_token.div((uint32_t)i);
  const int x = i - r.tok * 2 * heads;
  r.is_v = x >= heads;
  r.head = r.is_v ? x - heads : x;
  return r;
}

__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// the larger of each half (a NaN loses)
__device__ __forceinline__ uint32_t max_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// each half within +- most (a NaN stays)
__device__ __forceinline__ uint32_t clamp_half2(uint32_t a, uint32_t most) {
  uint32_t r;
  asm("{\n\t.reg .b32 n, t;\n\tneg.f16x2 n, %2;\n\tmin.NaN.f16x2 t, %1, %2;\n\tmax.NaN.f16x2 %0, t, n;\n\t}"
      : "=r"(r)
      : "r"(a), "r"(most));
  return r;
}

template <int GL, bool kQuantise>
__global__ void __launch_bounds__(THREADS) k_kv_append(Rows in, UkKvView c, const int32_t* __restrict__ cu,
                                                       const int32_t* __restrict__ lens, int n_seq, int tok,
                                                       UkFastDiv per_token) {
  __shared__ Where where[MAX_TOK];
  __shared__ Bounds bounds;
  __shared__ uint8_t exps[kQuantise ? MAX_EXP : 1];
  const int64_t t0 = (int64_t)blockIdx.x * tok;
  locate(c, cu, lens, n_seq, t0, tok, in.total, bounds, where);
  const int l = threadIdx.x % GL, rows = tok * 2 * c.heads;
  const bool lo_on = l * 16 < c.dim, hi_on = l * 16 + 8 < c.dim;
  const bool stage = kQuantise && rows <= MAX_EXP;
  for (int base = 0; base < rows; base += THREADS / GL * APPEND_ROWS) {
    Half16 x[APPEND_ROWS];
    Row r[APPEND_ROWS];
    bool on[APPEND_ROWS];
#pragma unroll
    for (int u = 0; u < APPEND_ROWS; ++u) {
      const int i = base + u * (THREADS / GL) + threadIdx.x / GL;
      r[u] = row_of(i, c.heads, per_token);
      on[u] = i < rows && where[r[u].tok].row >= 0;
      const int64_t t = t0 + r[u].tok;
      const uint16_t* p = (r[u].is_v ? in.v + t * in.v_token + r[u].head * in.v_head
                                     : in.k + t * in.k_token + r[u].head * in.k_head) + l * 16;
      x[u].lo = ldg16(p, on[u] && lo_on);
      x[u].hi = ldg16(p + 8, on[u] && hi_on);
    }
#pragma unroll
    for (int u = 0; u < APPEND_ROWS; ++u) {
      const Where w = on[u] ? where[r[u].tok] : Where{0, 0};
      uint8_t* dst = (r[u].is_v ? c.v : c.k) + w.row + r[u].head * c.head_bytes;
      if (!kQuantise) {
        if (on[u] && lo_on) reinterpret_cast<uint4*>(dst)[2 * l] = x[u].lo;
        if (on[u] && hi_on) reinterpret_cast<uint4*>(dst)[2 * l + 1] = x[u].hi;
        continue;
      }
      const uint32_t h[8] = {x[u].lo.x, x[u].lo.y, x[u].lo.z, x[u].lo.w, x[u].hi.x, x[u].hi.y, x[u].hi.z, x[u].hi.w};
      uint32_t m2 = 0;  // the maxima of the even and the odd values
#pragma unroll
      for (int k = 0; k < 8; ++k) m2 = max_half2(m2, h[k] & 0x7fff7fffu);
#pragma unroll
      for (int o = GL / 2; o > 0; o >>= 1) m2 = max_half2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
      const float2 m = halves(m2);
      const float top = fminf(fmaxf(m.x, m.y), VALUE_MAX);
      // exponent of the scale, biased by 127: carry into the exponent field
      // when the significand is above 1.75
      const int e = max((int)((__float_as_uint(top) + 0x1FFFFFu) >> 23) - 8, 127 - 15);
      // a power of two times a half is exact down to 2^-14, and from 2^-10 on
      // down an e4m3 code is zero
      const uint32_t inv = uk_half2_of(__uint_as_float((uint32_t)(254 - e) << 23));
      uint32_t y[8], codes[4];
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = uk_mul_half2(h[k], inv);
      if (e == 127 + 8) {  // only here a value can be above 240 * 2^e; a NaN stays
        const uint32_t most = uk_half2_of(240.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = clamp_half2(y[k], most);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) codes[k] = uk_half2_to_e4m3x2(y[2 * k]) | uk_half2_to_e4m3x2(y[2 * k + 1]) << 16;
      if (on[u] && lo_on) reinterpret_cast<uint4*>(dst)[l] = make_uint4(codes[0], codes[1], codes[2], codes[3]);
      if (on[u] && l == 0) {
        if (stage) exps[(r[u].is_v * c.heads + r[u].head) * tok + r[u].tok] = (uint8_t)e;
        else (r[u].is_v ? c.v_exp : c.k_exp)[w.exp + (int64_t)r[u].head * c.page_size] = (uint8_t)e;
      }
    }
  }
  if (!stage) return;
  __syncthreads();
  for (int i = threadIdx.x; i < rows; i += THREADS) {
    const int x = i / tok, y = i % tok;  // tokens of one head side by side
    const Where w = where[y];
    if (w.row < 0) continue;
    if (x >= c.heads) c.v_exp[w.exp + (int64_t)(x - c.heads) * c.page_size] = exps[i];
    else c.k_exp[w.exp + (int64_t)x * c.page_size] = exps[i];
  }
}

// kWide: rows of whole lanes on 32-byte boundaries, stored by one instruction a
// lane (4 x 16384 positions out of e4m3: 67.9 us, by two 71.7).
__device__ __forceinline__ void st32(void* p, const Half16& x) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(x.lo.x), "r"(x.lo.y),
               "r"(x.lo.z), "r"(x.lo.w), "r"(x.hi.x), "r"(x.hi.y), "r"(x.hi.z), "r"(x.hi.w)
               : "memory");
}

template <int GL, bool kQuantise, bool kWide>
__global__ void __launch_bounds__(THREADS) k_kv_gather(Rows out, UkKvView c, const int32_t* __restrict__ cu,
                                                       const int32_t* __restrict__ lens, int n_seq, int tok,
                                                       UkFastDiv per_token) {
  __shared__ Where where[MAX_TOK];
  __shared__ Bounds bounds;
  const int64_t t0 = (int64_t)blockIdx.x * tok;
  locate(c, cu, lens, n_seq, t0, tok, out.total, bounds, where);
  const int l = threadIdx.x % GL, rows = tok * 2 * c.heads;
  const bool lo_on = l * 16 < c.dim, hi_on = l * 16 + 8 < c.dim;
  for (int base = 0; base < rows; base += THREADS / GL * GATHER_ROWS) {
    Half16 x[GATHER_ROWS];
    uint32_t e[GATHER_ROWS];
    Row r[GATHER_ROWS];
    bool mine[GATHER_ROWS];
#pragma unroll
    for (int u = 0; u < GATHER_ROWS; ++u) {
      const int i = base + u * (THREADS / GL) + threadIdx.x / GL;
      r[u] = row_of(i, c.heads, per_token);
      const Where w = i < rows ? where[r[u].tok] : Where{NOBODY, 0};
      mine[u] = w.row != NOBODY;
      const bool on = w.row >= 0;
      const uint8_t* src = (r[u].is_v ? c.v : c.k) + w.row + r[u].head * c.head_bytes;
      if (kQuantise) {
        x[u].lo = ldg16(src + l * 16, on && lo_on);
        e[u] = on ? __ldg((r[u].is_v ? c.v_exp : c.k_exp) + w.exp + (int64_t)r[u].head * c.page_size) : 127u;
      } else {
        x[u].lo = ldg16(src + l * 32, on && lo_on);
        x[u].hi = ldg16(src + l * 32 + 16, on && hi_on);
      }
    }
#pragma unroll
    for (int u = 0; u < GATHER_ROWS; ++u) {
      if (kQuantise) {
        const uint32_t codes[4] = {x[u].lo.x, x[u].lo.y, x[u].lo.z, x[u].lo.w};
        const uint32_t s = uk_half2_of(uk_exp_scale(e[u]));
        uint32_t y[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uk_e4m3x4_to_half2(codes[k], &y[2 * k], &y[2 * k + 1]);
          y[2 * k] = uk_mul_half2(y[2 * k], s);
          y[2 * k + 1] = uk_mul_half2(y[2 * k + 1], s);
        }
        x[u].lo = make_uint4(y[0], y[1], y[2], y[3]);
        x[u].hi = make_uint4(y[4], y[5], y[6], y[7]);
      }
      const int64_t t = t0 + r[u].tok;
      uint16_t* p = (r[u].is_v ? out.v + t * out.v_token + r[u].head * out.v_head
                               : out.k + t * out.k_token + r[u].head * out.k_head) + l * 16;
      if (kWide) {
        if (mine[u] && lo_on) st32(p, x[u]);
      } else {
        if (mine[u] && lo_on) *reinterpret_cast<uint4*>(p) = x[u].lo;
        if (mine[u] && hi_on) *reinterpret_cast<uint4*>(p + 8) = x[u].hi;
      }
    }
  }
}

int lanes_for(int dim) { return dim <= 32 ? 2 : dim <= 64 ? 4 : 8; }

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
            int most, int* tok, int64_t* blocks) {
  *blocks = 0;
  if (rows->total < 0 || n_seq < 0) return uk::fail(UK_EINVAL, "%s: negative total or n_seq", what);
  if (rows->total > 0x7fffffff || n_seq > uk::MAX_SEQS)
    return uk::fail(UK_EINVAL, "%s: total %lld (at most 2^31 - 1) or n_seq %d (at most 2^24)", what,
                    (long long)rows->total, n_seq);
  if (int rc = uk::kv_view(cache, table, table_stride, n_seq, max_pages, what, view)) return rc;
  if (rows->total == 0 || n_seq == 0) return UK_OK;
  const int heads = cache->heads;
  if (int rc = uk::check_rows(what, "K", rows->k, rows->total, heads, rows->k_token, rows->k_head, least)) return rc;
  if (int rc = uk::check_rows(what, "V", rows->v, rows->total, heads, rows->v_token, rows->v_head, least)) return rc;
  if (int rc = uk::check_device_ptr(cu, "cu_seqlens")) return rc;
  if (int rc = uk::check_device_ptr(lens, "seq_lens")) return rc;
  // as many tokens to a block as still give every SM four blocks
  *tok = most;
  while (*tok > 1 && rows->total / *tok < (int64_t)uk::sm_count() * 4) *tok /= 2;
  *blocks = (rows->total + *tok - 1) / *tok;
  return UK_OK;
}

template <bool kQuantise>
void launch_append(const Rows& rows, const UkKvView& v, const int32_t* cu, const int32_t* lens, int n_seq, int tok,
                   unsigned blocks, cudaStream_t st) {
  const UkFastDiv d = UkFastDiv::make(2u * v.heads);
  switch (lanes_for(v.dim)) {
    case 2: k_kv_append<2, kQuantise><<<blocks, THREADS, 0, st>>>(rows, v, cu, lens, n_seq, tok, d); break;
    case 4: k_kv_append<4, kQuantise><<<blocks, THREADS, 0, st>>>(rows, v, cu, lens, n_seq, tok, d); break;
    default: k_kv_append<8, kQuantise><<<blocks, THREADS, 0, st>>>(rows, v, cu, lens, n_seq, tok, d); break;
  }
}

template <bool kQuantise, bool kWide>
void launch_gather(const Rows& rows, const UkKvView& v, const int32_t* cu, const int32_t* lens, int n_seq, int tok,
                   unsigned blocks, cudaStream_t st) {
  const UkFastDiv d = UkFastDiv::make(2u * v.heads);
  switch (lanes_for(v.dim)) {
    case 2: k_kv_gather<2, kQuantise, kWide><<<blocks, THREADS, 0, st>>>(rows, v, cu, lens, n_seq, tok, d); break;
    case 4: k_kv_gather<4, kQuantise, kWide><<<blocks, THREADS, 0, st>>>(rows, v, cu, lens, n_seq, tok, d); break;
    default: k_kv_gather<8, kQuantise, kWide><<<blocks, THREADS, 0, st>>>(rows, v, cu, lens, n_seq, tok, d); break;
  }
}

// whole lanes of 16 values on 32-byte boundaries
bool wide_rows(const Rows& r, const UkKvView& v) {
  auto bad = [&](const uint16_t* p, int64_t token, int64_t head) {
    return reinterpret_cast<uintptr_t>(p) % 32 != 0 || (r.total > 1 && token % 16 != 0) ||
           (v.heads > 1 && head % 16 != 0);
  };
  return v.dim % 16 == 0 && !bad(r.k, r.k_token, r.k_head) && !bad(r.v, r.v_token, r.v_head);
}

}  // namespace

extern "C" int uk_cuda_kv_append_f16(const uint16_t* K, int64_t k_token_stride, int64_t k_head_stride,
                                     const uint16_t* V, int64_t v_token_stride, int64_t v_head_stride, int64_t total,
                                     const uk_kv_cache* cache, const int32_t* block_table, int64_t table_stride,
                                     int max_pages, const int32_t* cu_new, const int32_t* seq_lens, int n_seq,
                                     void* stream) {
  Rows rows{(uint16_t*)K, (uint16_t*)V, k_token_stride, k_head_stride, v_token_stride, v_head_stride, total};
  UkKvView view;
  int tok;
  int64_t blocks;
  if (int rc = prepare("kv_append", &rows, cache, block_table, table_stride, max_pages, cu_new, seq_lens, n_seq, 0,
                       &view, MAX_TOK, &tok, &blocks))
    return rc;
  if (blocks == 0) return UK_OK;
  if (cache->kind == UK_KV_E4M3)
    launch_append<true>(rows, view, cu_new, seq_lens, n_seq, tok, (unsigned)blocks, (cudaStream_t)stream);
  else
    launch_append<false>(rows, view, cu_new, seq_lens, n_seq, tok, (unsigned)blocks, (cudaStream_t)stream);
  return uk::check_launch("kv_append");
}

extern "C" int uk_cuda_kv_gather_f16(const uk_kv_cache* cache, const int32_t* block_table, int64_t table_stride,
                                     int max_pages, const int32_t* cu_out, const int32_t* seq_lens, int n_seq,
                                     uint16_t* K, int64_t k_token_stride, int64_t k_head_stride, uint16_t* V,
                                     int64_t v_token_stride, int64_t v_head_stride, int64_t total, void* stream) {
  Rows rows{K, V, k_token_stride, k_head_stride, v_token_stride, v_head_stride, total};
  UkKvView view;
  int tok;
  int64_t blocks;
  if (int rc = prepare("kv_gather", &rows, cache, block_table, table_stride, max_pages, cu_out, seq_lens, n_seq,
                       cache != nullptr ? cache->dim : 0, &view, GATHER_TOK, &tok, &blocks))
    return rc;
  if (blocks == 0) return UK_OK;
  const bool wide = wide_rows(rows, view);
  auto launch = cache->kind == UK_KV_E4M3 ? (wide ? launch_gather<true, true> : launch_gather<true, false>)
                                          : (wide ? launch_gather<false, true> : launch_gather<false, false>);
  launch(rows, view, cu_out, seq_lens, n_seq, tok, (unsigned)blocks, (cudaStream_t)stream);
  return uk::check_launch("kv_gather");
}
