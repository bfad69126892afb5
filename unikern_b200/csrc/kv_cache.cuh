// kv_cache.cuh -- the paged key-value cache as the kernels see it, shared by the
// operators that write it, read it back and attend over it.
//
// A cache is two pools of pages (keys and values) with the same strides.  A
// sequence owns the pages its row of the block table names, in order: position
// p lies in page table[b][p / page_size] at offset p % page_size.  A row is a
// head's `dim` values of one position, contiguous.  kind e4m3 holds a row as
// 8-bit codes c and one exponent byte e, value = c * 2^(e - 127): a power of
// two costs an 8-bit float no precision (only the lowest octave of its range),
// and makes every held value exactly a binary16 one.
//
// Nothing read from the block table or the length arrays is trusted: a page id
// outside the pool, or a position outside the table, is never dereferenced; it
// counts as absent and sets UK_FAULT_PAGE in the fault word.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "sm100_ptx.cuh"
#include "uk_common.cuh"

// division of 31-bit numbers by an invariant one: multiply by the rounded-up
// reciprocal 2^(32 + s) / d and shift (Granlund and Montgomery); exact for
// n < 2^31 with s = ceil(log2 d) - 1.
struct UkFastDiv {
  uint32_t d, mul, shift;
  __host__ static UkFastDiv make(uint32_t d) {
    UkFastDiv f{d, 0, 0};
    if (d > 1) {
      uint32_t s = 0;
      while ((1ull << (s + 1)) < d) ++s;  // s = ceil(log2 d) - 1
      f.mul = (uint32_t)(((1ull << (32 + s)) + d - 1) / d);
      f.shift = s;
    }
    return f;
  }
  __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
#ifdef __CUDA_ARCH__
    return d == 1 ? n : __umulhi(n, mul) >> shift;
#else
    return d == 1 ? n : (uint32_t)(((uint64_t)n * mul) >> 32) >> shift;
#endif
  }
};

struct UkKvView {
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_exp;  // [pages][heads][page_size], e4m3 only
  uint8_t* v_exp;
  int64_t page_bytes, token_bytes, head_bytes;  // strides
  int64_t pages;
  int page_size, heads, dim, kind;
  UkFastDiv div;
  const int32_t* table;  // [n_seq][table_stride]
  int64_t table_stride;
  int max_pages;  // entries of a table row that may be read
};

// page and offset of position p of sequence b; -1 when absent
__device__ __forceinline__ int uk_kv_page(const UkKvView& c, int b, int p, int* off) {
  const int i = (int)c.div.div((uint32_t)p);
  *off = p - i * c.page_size;
  if (i >= c.max_pages) return -1;
  const int page = __ldg(c.table + (int64_t)b * c.table_stride + i);
  return (unsigned)page < (uint64_t)c.pages ? page : -1;
}

__device__ __forceinline__ int64_t uk_kv_row(const UkKvView& c, int page, int off, int head) {
  return (int64_t)page * c.page_bytes + (int64_t)off * c.token_bytes + (int64_t)head * c.head_bytes;
}

__device__ __forceinline__ int64_t uk_kv_exp(const UkKvView& c, int page, int off, int head) {
  return ((int64_t)page * c.heads + head) * c.page_size + off;
}

// the sequence of a packed row t: cu[b] <= t < cu[b + 1] for a non-decreasing
// cu[0..n].  -1 when t lies before the first or behind the last sequence.
template <bool kGlobal>
__device__ __forceinline__ int uk_find_seq(const int32_t* cu, int n, int64_t t) {
  auto at = [&](int i) { return kGlobal ? __ldg(cu + i) : cu[i]; };
  if (t < at(0) || t >= at(n)) return -1;
  int lo = 0, hi = n;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at(mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// two e4m3 codes (low byte first) as two halves, exactly; NaN stays NaN
__device__ __forceinline__ uint32_t uk_e4m3x2_to_half2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}

// four e4m3 codes as two pairs of halves
__device__ __forceinline__ void uk_e4m3x4_to_half2(uint32_t codes, uint32_t* lo, uint32_t* hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(*lo), "=r"(*hi)
      : "r"(codes));
}

// two halves as e4m3 codes, round to nearest even, saturating; lo in the low byte
__device__ __forceinline__ uint32_t uk_half2_to_e4m3x2(uint32_t x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t uk_mul_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// two equal halves
__device__ __forceinline__ uint32_t uk_half2_of(float x) {
  const __half2 h = __float2half2_rn(x);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two attention outputs as halves.  They are averages of binary16 values, so a
// finite one that lies above 65504 is so by rounding (of the weights) alone and
// becomes 65504; an infinity stays one.
__device__ __forceinline__ uint32_t uk_pack_finite(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t uk_pack_average(float lo, float hi) {
  uint32_t r = uk_pack_finite(lo, hi);
  if (fabsf(lo) == INFINITY) r = (r & 0xffff8000u) | 0x7c00u;
  if (fabsf(hi) == INFINITY) r = (r & 0x8000ffffu) | 0x7c000000u;
  return r;
}

// 2^(e - 127) for an exponent byte (0 counts as 2^-127: not written by the append)
__device__ __forceinline__ float uk_exp_scale(uint32_t e) { return __uint_as_float(e == 0 ? 0x00400000u : e << 23); }

namespace uk {
// sequences of one call: indexes of 32 and blocks of 128 of them stay within 31
// bits, and a kernel's pass over their lengths well within its bounded waits
constexpr int MAX_SEQS = 1 << 24;
// host checks of a cache and its block table (kv_cache.cu)
int kv_view(const uk_kv_cache* cache, const int32_t* table, int64_t table_stride, int n_seq, int max_pages,
            const char* what, UkKvView* out);
// strides of packed rows [tokens][heads][dim] in elements: multiples of 8
// and at least `least` where the extent is above one
int check_rows(const char* what, const char* name, const void* p, int64_t tokens, int heads, int64_t token_stride,
               int64_t head_stride, int64_t least);
}  // namespace uk
