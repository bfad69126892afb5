// attn_prompt.cu -- attention over packed prompts, causal or full, with grouped
// heads: O[i][h] = sum_j w_j V[j][g], w = softmax_j(scale * Q[i][h] . K[j][g])
// over the keys row i sees, in one pass with a running reference m and sum l
// per row (scores carry scale * log2 e, so every exponential is a power of two):
//   l = sum 2^(s_j - m),  o = sum 2^(s_j - m) v_j;
// m moves (l and o scaled by 2^(m - m')) only when a score passes it by 2^8.
//
// The work is bound by the tensor cores (4 dim flops per visible pair and head)
// and, nearly as much, by the exponentials (one per pair and head; the MUFU
// makes 16 per cycle and SM, a 128 x 128 tile's take as long as its two
// products at dim 128); the two wait for one another (8192 rows, 32 heads over 8 of
// 128: 3150 cycles for two tiles by 128 keys, 2048 of them products), and long
// prompts run into the power limit (1520 MHz: 517 us, 442 before the limit acts).
// A tile has 128 rows: the heads of a key head's group, side by side for each of as
// many tokens as fit (32 for groups of 4), so short sequences fill it too.  A CTA
// (one per SM) works on two tiles of one key head at a time, so that one tile's
// products run while the other's softmax does:
//   warp 10      loads (TMA): both Q tiles, then K and V blocks of 128 keys through
//                a ring in shared memory; finds the next pair of tiles meanwhile;
//   warps 8, 9   issue tcgen05.mma, a tile each: S = Q K^T for runs of 64 keys,
//                O += P V with P in TMEM;
//   warps 0-3    softmax of tile 0, a thread per row: reads a run of its S row from
//                TMEM, writes P (binary16) over it, rescales O when m moves, and at
//                the end divides by l and stores; warps 4-7 the same for tile 1.
// TMEM: S/P of tile 0 and 1 at columns 0 and 128 (even and odd runs, 64 each), O
// at 256 and 384.  A run's S is issued behind the product that reads the P in its
// place, and the tensor core runs one thread's products in order.
//
// More than PART runs of keys are taken in parts, behind each of which the softmax
// warps take out of O what it holds to 11 bits, O / l as binary16 (kept in the
// row's place in the output), and leave the rest: the tensor core goes on adding to a
// small number, and nothing is lost.  (The CTAs of a cluster share their rows: they
// keep the sums in the unused tile's TMEM, in 32 bits, and leave zero.)
//
// What lies behind a row's mask: scores are replaced before the maximum, V rows
// behind the sequence's last key are zeroed in shared memory (a zero weight
// times a NaN would be one), and where a finite sum meets a row of O that is
// not, the few masked keys of its last blocks are looked through; if one of
// them holds a NaN or an infinity the row is computed again, key by key.
//
// Every mbarrier wait is bounded (wait_until, uk_mbar_wait); a timeout sets the fault word
// read by uk_cuda_pipeline_fault() and the CTA unwinds.  Rows that are computed
// again may take longer than any limit (17.5 us a key for a warp's 32 rows): while
// they are, the time limit is put off again and again.
#include <cudaTypedefs.h>

#include <mutex>
#include <utility>

#include "attn_prompt_items.cuh"

namespace uk {
__device__ unsigned int g_attn_prompt_fault = 0;
}  // namespace uk

namespace {

using namespace uk_prompt;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float GROW = 8.f;  // scores may pass the reference by 2^8 before it moves

__device__ __forceinline__ float4 row4(const uint16_t* row, int lane, int dim) {
  if (lane * 4 >= dim) return make_float4(0.f, 0.f, 0.f, 0.f);
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(row) + lane);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  return make_float4(x.x, x.y, y.x, y.y);
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr uint64_t WAIT_NS = 2000000000ull;  // 2 s
__device__ __forceinline__ void put_off(volatile uint64_t* limit) { *limit = uk_globaltimer() + WAIT_NS; }

// A sum that carries what its additions round off (Kahan): those of equal terms
// all round the same way (2^20 keys by plain sums: 7 times the tests' bound off).
struct LongSum {
  float s = 0.f, c = 0.f;
  __device__ __forceinline__ void add(float x) {
    const float y = x - c, t = s + y;
    c = fabsf(t) < INFINITY ? (t - s) - y : 0.f;  // an infinity stays one
    s = t;
  }
  __device__ __forceinline__ void scale(float f) { s *= f, c *= f; }
};

// One row by one warp, key by key, on CUDA cores: keys [k0, end).  A lane
// holds four of the row's values.  *limit (where there is one), the
// time limit of other warps' waits, is put off every few milliseconds.
__device__ __noinline__ void attend_row(const Args& a, int64_t t, int h, int64_t k0, int64_t end,
                                        volatile uint64_t* limit) {
  const int lane = threadIdx.x & 31, g = h / a.group;
  const float4 q = row4(a.q + t * a.q_token + h * a.q_head, lane, a.dim);
  float m = -INFINITY;
  LongSum l, o[4];
  constexpr int U = 4;  // keys in flight
  for (int64_t j = k0; j < end; j += U) {
    if (limit != nullptr && ((j - k0) & 4095) == 0 && lane == 0) put_off(limit);
    float4 k[U], v[U];
    float s[U], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = j + u < end;
      k[u] = on ? row4(a.k + (j + u) * a.k_token + g * a.k_head, lane, a.dim) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[u] = on ? row4(a.v + (j + u) * a.v_token + g * a.v_head, lane, a.dim) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = uk_warp_sum(q.x * k[u].x + q.y * k[u].y + q.z * k[u].z + q.w * k[u].w) * a.scale2;
      if (j + u >= end) s[u] = -INFINITY;
      top = fmaxf(top, s[u]);
    }
    if (top > m + GROW) {
      const float f = ex2(m - top);
      m = top;
      l.scale(f);
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c].scale(f);
    }
    const float z = m == -INFINITY ? 0.f : m;
    float e = 0.f;
    float4 p = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = ex2(s[u] - z);
      e += w;
      p = make_float4(fmaf(w, v[u].x, p.x), fmaf(w, v[u].y, p.y), fmaf(w, v[u].z, p.z), fmaf(w, v[u].w, p.w));
    }
    l.add(e);
    o[0].add(p.x), o[1].add(p.y), o[2].add(p.z), o[3].add(p.w);
  }
  const float inv = l.s == 0.f ? 0.f : 1.f / l.s;
  if (lane * 4 < a.dim)
    reinterpret_cast<uint2*>(a.o + t * a.o_token + h * a.o_head)[lane] =
        make_uint2(uk_pack_average(o[0].s * inv, o[1].s * inv), uk_pack_average(o[2].s * inv, o[3].s * inv));
  if (a.lse != nullptr && lane == 0) a.lse[t * a.heads_q + h] = l.s == 0.f ? -INFINITY : (m + log2f(l.s)) * LN2;
}

// ---- what one CTA works on -----------------------------------------------------------
// runs of keys whose products the tensor core adds up in one go: its sums are
// truncated, 1e-7 of the sum for every 16 keys (2e-4 over 512 runs, 32768 keys; in one
// go 8e-4 over 131072, 7e-3 over 2^20).  Calls of at most as many keys in all run
// without the code for parts: 11 x 900 rows of dim 64 39.6 us, 41.1 with it.
constexpr int PART = 512;
// Weights enter the product as binary16, 2^7 * 2^(s - m): up to 2^15 (binary16 ends
// at 2^16), normal down to 2^-21 of the reference's.  Each is off by 2^-11 at most;
// 32-bit operands would halve the products' rate.
constexpr float SHIFT = 7.f;
// three warpgroups: two of softmax, one of the MMA and load warps (and an idle
// one).  They launch with 168 registers a thread; the softmax takes 216 (a row
// of 128 scores stays in registers) and the others keep 72.
constexpr int NUM_THREADS = 384;
constexpr int REGS_LAUNCH = 168, REGS_SOFTMAX = 216, REGS_OTHERS = 72;
static_assert(2 * REGS_SOFTMAX + REGS_OTHERS <= 3 * REGS_LAUNCH, "registers of the block");
constexpr int MMA_WARP = 8, LOAD_WARP = 10;  // MMA_WARP + t: tile t

// One warp: the first level that has items, from the longest sequence.
__device__ int first_level(const Args& a) {
  int most = 0;
  for (int b = threadIdx.x & 31; b < a.n_seq; b += 32) most = max(most, keys_of(a, b));
  return first_level_of(a, __reduce_max_sync(0xffffffffu, most));
}

// One warp: item i, or false behind the list's end.
__device__ __forceinline__ bool find_item(const Args& a, uint32_t item, Cursor& at, Item* out) {
  const int lane = threadIdx.x & 31;
  Lot lot;
  if (!find_chunk(a, item, at, [&](int level, int chunk) {
        lot = lot_of(a, level, chunk, lane);
        return __reduce_add_sync(0xffffffffu, lot.mine);
      }))
    return false;
  uint32_t incl = lot.mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  const uint32_t x = item - at.before - (incl - lot.mine);  // huge where the item lies in a lane before
  if (x < lot.mine) place_item(a, lot, x, out);
  return true;
}

template <int DP>
struct Smem {
  static constexpr int CHUNKS = DP / 64;         // 64-wide columns of a tile, one TMA box each
  static constexpr int BOX = 128 * 128;          // 128 rows of 128 bytes
  static constexpr int TILE = CHUNKS * BOX;      // a Q tile, a K or a V block
  static constexpr int STAGES = DP == 128 ? 5 : 10;
  static constexpr size_t BYTES = 1024 + (size_t)(2 + STAGES) * TILE + 768;
};

struct Ctl {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[10], kv_empty[10];
  uint64_t s_full[2][2], p_full[2][2];  // of each tile, for the even and the odd runs of keys
  uint64_t pv_done[2];                  // a run's product with V is in O
  uint64_t o_full[2], o_empty[2];
  uint64_t item_full[2], item_empty[2];
  uint64_t next;      // the answer about the next block
  uint64_t v_landed;  // a V block whose rows behind the last key are zeroed before use
  uint64_t teardown;
  alignas(16) uint8_t answer[16];
  uint32_t tmem;
  int abort;
  uint64_t limit;   // of the waits: a time
  unsigned odd[4];  // rows of a shared tile to look at again
  Item item[2];
};
static_assert(sizeof(Ctl) <= 768, "control block");
static_assert(Smem<128>::BYTES <= 232448 && Smem<64>::BYTES <= 232448, "shared memory per block on sm_100");

__device__ __forceinline__ void raise_fault(Ctl* ctl, unsigned bit) {
  atomicOr(&uk::g_attn_prompt_fault, bit);
  ctl->abort = 1;
  *(volatile uint64_t*)&ctl->limit = 0;
}

// Waits end at the block's common time limit.  It is put off when the load warp comes
// to a new item and every 64 blocks of keys, and every few milliseconds while rows
// are computed again or blocks taken over, of which there are finitely many.
__device__ __forceinline__ bool wait_until(const Ctl* ctl, uint64_t* bar, uint32_t parity) {
  if (uk_mbar_try_wait(bar, parity)) return true;
  for (uint32_t i = 1;; ++i) {
    if (uk_mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0 && uk_globaltimer() > *(const volatile uint64_t*)&ctl->limit) return false;
  }
}
// by a whole warp: the same answer in every lane
__device__ __forceinline__ bool wait_warp(Ctl* ctl, uint64_t* bar, uint32_t parity, unsigned bit) {
  if (__all_sync(0xffffffffu, wait_until(ctl, bar, parity))) return true;
  if (!*(volatile int*)&ctl->abort) raise_fault(ctl, bit);
  return false;
}
// ---- the softmax of a tile ------------------------------------------------------------
// *turn: runs of 64 keys of this tile's slot that came before, even and odd ones;
// *ends: parts of items.
// One past the last key that a token of the sequence sees.
__device__ __forceinline__ int end_of(const Args& a, const Item& it, int token) {
  const int64_t end = a.causal ? (int64_t)it.m - it.n + 1 + token : it.m;
  return (int)(end < 0 ? 0 : end > it.m ? it.m : end);
}

// A row with a finite sum that is not finite itself (one warp): it is computed
// again where one of the keys between its mask and the end of its blocks is not,
// in a column that is no NaN by a key the row does see.  (Of those only the last
// are looked at: from the first NaN of a model on, all are.  8192 rows of NaN, 32
// heads over 8 of 128: 2.4 ms, all of them computed again 551.)
__device__ __noinline__ void look_again(const Args& a, const Item& it, const Tile& tile, int row, int units,
                                        volatile uint64_t* limit) {
  const Row r(a, tile, row);
  const int lane = threadIdx.x & 31, from = end_of(a, it, r.token), to = min(units * UN, it.m);
  const uint16_t* v0 = a.v + (int64_t)it.k0 * a.v_token + it.g * a.v_head;
  constexpr int U = 8;  // keys in flight
  auto column = [](const float4& x, int c) { return c == 0 ? x.x : c == 1 ? x.y : c == 2 ? x.z : x.w; };
  unsigned bad = 0;  // of the lane's four columns
  for (int k = from; k < to; k += U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = k + u < to ? row4(v0 + (int64_t)(k + u) * a.v_token, lane, a.dim) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < 4; ++c) bad |= (unsigned)!(fabsf(column(v[u], c)) < INFINITY) << c;
  }
  const int last = max(from - BN, 0);
  for (int k = from - U; __any_sync(0xffffffffu, bad != 0) && k + U > last; k -= U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = k + u >= last ? row4(v0 + (int64_t)(k + u) * a.v_token, lane, a.dim) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (isnan(column(v[u], c))) bad &= ~(1u << c);
  }
  __syncwarp();  // the row's stores before come before these
  if (__any_sync(0xffffffffu, bad != 0))
    attend_row(a, (int64_t)it.q0 + r.token, r.head, it.k0, (int64_t)it.k0 + from, limit);
}

// A shared tile's sums in shared memory: 128 rows of DP floats (16-byte pieces
// exchanged by the row's low bits: a thread per row writes without conflicts),
// then the rows' references and sums.
template <int DP>
struct Shared {
  float* o;
  float* m;
  float* l;
  __device__ __forceinline__ explicit Shared(uint8_t* ring)
      : o((float*)ring), m((float*)(ring + 2 * Smem<DP>::TILE)), l(m + BM) {}
  __device__ __forceinline__ float* piece(int row, int c) const { return o + row * DP + (c ^ (row & 7)) * 4; }
};

// 16 values of a row of the output, as far as `left` of it go; zeros without a row
__device__ __forceinline__ void load_halves(const uint16_t* row, int left, uint32_t (&x)[16]) {
  uint4 w[2] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (k * 8 < left) w[k] = reinterpret_cast<const uint4*>(row)[k];
  const uint32_t h[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
    x[2 * k] = __float_as_uint(y.x), x[2 * k + 1] = __float_as_uint(y.y);
  }
}

// A warp's rows of O times inv, each stored by its own thread: where they were taken
// out in parts (part: what the halves that lie in `own` are multiples of), and where a
// value is not finite.  True where that is so.
template <int DP>
__device__ __noinline__ bool store_own(uint32_t o_at, float inv, uint16_t* own, float part, int dim) {
  float odd = 0.f;
#pragma unroll 1
  for (int c = 0; c < DP / 16; ++c) {
    uint32_t o[16], x[16], w[8];
    uk_tmem_ld16(o_at + c * 16, o);
    const int left = own != nullptr ? dim - c * 16 : 0;
    load_halves(own + c * 16, part != 0.f ? left : 0, x);
    uk_tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float y0 = fmaf(__uint_as_float(x[2 * k]), part, __uint_as_float(o[2 * k])) * inv;
      const float y1 = fmaf(__uint_as_float(x[2 * k + 1]), part, __uint_as_float(o[2 * k + 1])) * inv;
      odd = fmaf(y0, 0.f, fmaf(y1, 0.f, odd));
      w[k] = uk_pack_average(y0, y1);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (k * 8 < left)
        reinterpret_cast<uint4*>(own + c * 16)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  }
  return odd != 0.f;
}

template <int DP, bool kSplit, bool kParts>
__device__ __forceinline__ bool softmax_tile(const Args& a, Ctl* ctl, const Item& it, int t, uint32_t tmem,
                                             uint8_t* ring, uint32_t (&turn)[2], uint32_t* ends) {
  const Tile& tile = it.tile[t];
  if (tile.head < 0) return true;
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3;
  const int i = quad * 32 + lane;  // row of the tile
  const uint32_t lanes = (uint32_t)(quad * 32) << 16;
  const uint32_t s_at = tmem + lanes + t * BN, o_at = tmem + lanes + 256 + t * 128, sum_at = tmem + lanes + 384;
  const Row row(a, tile, i);
  // one past the last key that this row and that the tile's first token see
  const int end = end_of(a, it, row.token), clear = end_of(a, it, tile.first);
  const uint64_t scale2 = uk_f2(a.scale2, a.scale2);
  const int units = tile.units;

  const int64_t token = (int64_t)it.q0 + row.token;
  uint16_t* const own = row.on ? a.o + token * a.o_token + row.head * a.o_head : nullptr;
  float m = -INFINITY, l = 0.f, lost = 0.f;  // lost: what the additions to l have rounded off (Kahan)
  float part = 0.f;                          // what the numbers of the parts before are multiples of
  auto step = [&](int u, int h, uint32_t runs) {  // run u, of parity h; runs: of this tile's slot before it
    if (!wait_warp(ctl, &ctl->s_full[t][h], turn[h] & 1u, UK_FAULT_EPILOGUE)) return false;
    ++turn[h];
    uk_tc_fence_after();
    const uint32_t at = s_at + h * UN;
    uint32_t s[2][32];
    uk_tmem_ld32(at, s[0]);
    uk_tmem_ld32(at + 32, s[1]);
    uk_tmem_ld_wait();
    const int base = (u + (kSplit ? 2 * it.first_block : 0)) * UN;
    if (base + UN > clear) {  // some row of the tile does not see the whole run
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int k = 0; k < 32; ++k)
          if (base + c * 32 + k >= end) s[c][k] = 0xff800000u;  // -inf
    }
    float top[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      top[c] = __uint_as_float(s[c / 2][16 * (c % 2)]);
#pragma unroll
      for (int k = 1; k < 15; k += 2)
        top[c] = uk_max3_nan(top[c], __uint_as_float(s[c / 2][16 * (c % 2) + k]),
                             __uint_as_float(s[c / 2][16 * (c % 2) + k + 1]));
    }
    const float rest = uk_max3_nan(__uint_as_float(s[0][15]), __uint_as_float(s[0][31]),
                                   uk_max3_nan(__uint_as_float(s[1][15]), __uint_as_float(s[1][31]), top[0]));
    const float mt = uk_max3_nan(uk_max3_nan(top[1], top[2], top[3]), rest, rest) * a.scale2;
    // the rows of the warp move together; ones that stand for nothing have no say
    // (what they hold is whatever shared memory held)
    if (__any_sync(0xffffffffu, row.on && mt > m + GROW)) {
      const float m2 = fmaxf(m, mt);
      const float f = m2 == -INFINITY ? 1.f : ex2(m - m2);
      m = m2;
      l *= f, lost *= f;
      if (kParts) part *= f;
      if (u > 0) {
        // the run before this one may still be on its way into O
        if (!wait_warp(ctl, &ctl->pv_done[t], (runs - 1) & 1u, UK_FAULT_EPILOGUE)) return false;
        uk_tc_fence_after();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          uint32_t o[16];
          uk_tmem_ld16(o_at + c * 16, o);
          uk_tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          uk_tmem_st16(o_at + c * 16, o);
        }
      }
    }
    if (!(mt < INFINITY)) l = NAN;  // a score that is NaN or +inf: so is the softmax
    const float z = m == -INFINITY ? 0.f : SHIFT - m;
    const uint64_t z2 = uk_f2(z, z);
    uint64_t sum[2] = {uk_f2(0.f, 0.f), uk_f2(0.f, 0.f)};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t p[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint64_t x2 =
            uk_f2_fma(uk_f2(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1])), scale2, z2);
        float x, y;
        uk_f2_split(x2, &x, &y);
        x = ex2(x), y = ex2(y);
        sum[k & 1] = uk_f2_add(sum[k & 1], uk_f2(x, y));
        p[k] = pack_half(x, y);
      }
      uk_tmem_st16(at + c * 16, p);
    }
    uk_tmem_st_wait();
    uk_tc_fence_before();
    __syncwarp();
    if (lane == 0) uk_mbar_arrive(&ctl->p_full[t][h]);
    float l0, l1;
    uk_f2_split(uk_f2_add(sum[0], sum[1]), &l0, &l1);
    const float add = l0 + l1 - lost, sum_l = l + add;
    lost = sum_l - l - add;
    l = sum_l;
    return true;
  };
  // adds to 16 columns of O what was taken out of them
  auto add_parts = [&](int c, uint32_t* o) {
    uint32_t x[16];
    if constexpr (kSplit) {
      uk_tmem_ld16(sum_at + c * 16, x);
      uk_tmem_ld_wait();
    } else {
      load_halves(own + c * 16, own != nullptr ? a.dim - c * 16 : 0, x);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(fmaf(__uint_as_float(x[k]), part, __uint_as_float(o[k])));
  };
  // behind a part, before run u
  auto end_part = [&](int u) {
    if (!wait_warp(ctl, &ctl->o_full[t], *ends & 1u, UK_FAULT_EPILOGUE)) return false;
    uk_tc_fence_after();
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
    for (int c = 0; c < DP / 16; ++c) {
      uint32_t o[16];
      uk_tmem_ld16(o_at + c * 16, o);
      uk_tmem_ld_wait();
      if (u > PART) add_parts(c, o);
      if constexpr (kSplit) {
        uk_tmem_st16(sum_at + c * 16, o);
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = 0;
      } else {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float x[2] = {__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1])};
          w[k] = uk_pack_finite(x[0] * inv, x[1] * inv);  // an infinity or a NaN stays in the rest
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
          o[2 * k] = __float_as_uint(fmaf(-l, y.x, x[0])), o[2 * k + 1] = __float_as_uint(fmaf(-l, y.y, x[1]));
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (own != nullptr && c * 16 + k * 8 < a.dim)
            reinterpret_cast<uint4*>(own + c * 16)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
      }
      uk_tmem_st16(o_at + c * 16, o);
    }
    part = kSplit ? 1.f : l;
    uk_tmem_st_wait();
    uk_tc_fence_before();
    __syncwarp();
    if (lane == 0) uk_mbar_arrive(&ctl->o_empty[t]);
    ++*ends;
    return true;
  };
  for (int u = 0; u < units;) {
    if (kParts && u > 0 && !end_part(u)) return false;
    for (const int stop = kParts ? min(u + PART, units) : units; u < stop; ++u)
      if (!step(u, u & 1, turn[0] + turn[1])) return false;
  }

  // ---- O / l, the log of the sum
  const bool mine = row.on;
  if (units > 0) {
    if (!wait_warp(ctl, &ctl->o_full[t], *ends & 1u, UK_FAULT_EPILOGUE)) return false;
    uk_tc_fence_after();
  }
  if constexpr (kSplit) {
    const Shared<DP> sh(ring);  // every product has read its blocks: the ring is free
    sh.m[i] = m, sh.l[i] = l;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      uint32_t o[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) o[k] = 0;
      if (units > 0) {
        uk_tmem_ld32(o_at + c * 32, o);
        uk_tmem_ld_wait();
        if (kParts && units > PART) add_parts(2 * c, o), add_parts(2 * c + 1, o + 16);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        *reinterpret_cast<uint4*>(sh.piece(i, c * 8 + k)) =
            make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
    }
    return true;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const uint64_t inv2 = uk_f2(inv, inv), zero2 = uk_f2(0.f, 0.f);
  unsigned odd;  // rows of the warp with a finite sum, but a value that is not
  if (kParts && units > PART) {
    const bool bad = store_own<DP>(o_at, inv, own, part, a.dim);
    odd = __ballot_sync(0xffffffffu, mine && bad && l - l == 0.f);
  } else {
    uint64_t odd2 = zero2;  // NaN once a value of the row is not finite
    // Stores go by groups of four lanes: a 4 x 4 transpose of 16-byte pieces
    // between their rows turns 32 lines touched by every store into 8 (the
    // store path takes a line per cycle: 2000 cycles a tile pair at dim 64).
    const int j4 = lane & 3;
    uint16_t* out[4];  // of the group's four rows
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = (uint16_t*)__shfl_sync(0xffffffffu, (uint64_t)own, (lane & ~3) + k);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      uint32_t w[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k][0] = w[k][1] = w[k][2] = w[k][3] = 0;
      if (units > 0) {
        uint32_t o[32];
        uk_tmem_ld32(o_at + c * 32, o);
        uk_tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint64_t v = uk_f2_fma(uk_f2(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1])), inv2, zero2);
          odd2 = uk_f2_fma(v, zero2, odd2);
          float x, y;
          uk_f2_split(v, &x, &y);
          w[k / 4][k % 4] = uk_pack_finite(x, y);
        }
      }
#pragma unroll
      for (int bit = 1; bit < 4; bit *= 2)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (k & bit) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool up = lane & bit;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[k][e] : w[k + bit][e], bit);
            if (up) w[k][e] = got;
            else w[k + bit][e] = got;
          }
        }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (out[k] != nullptr && c * 32 + j4 * 8 < a.dim)
          *reinterpret_cast<uint4*>(out[k] + c * 32 + j4 * 8) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    }
    float odd0, odd1;
    uk_f2_split(odd2, &odd0, &odd1);
    odd = __ballot_sync(0xffffffffu, mine && odd0 + odd1 != 0.f && l - l == 0.f);
    if (odd != 0) {  // infinities go out as such
      __syncwarp();
      store_own<DP>(o_at, inv, odd >> lane & 1u ? own : nullptr, 0.f, a.dim);
    }
  }
  if (units > 0) {
    uk_tc_fence_before();
    __syncwarp();
    if (lane == 0) uk_mbar_arrive(&ctl->o_empty[t]);
    ++*ends;
  }
  if (mine && a.lse != nullptr)
    a.lse[token * a.heads_q + row.head] = l == 0.f ? -INFINITY : (m - SHIFT + log2f(l)) * LN2;

  // they may have met what their mask hides
  while (odd != 0) {
    const int r = __ffs(odd) - 1;
    odd &= odd - 1;
    look_again(a, it, tile, quad * 32 + r, units, &ctl->limit);
  }
  return true;
}

// ---- a shared tile: the CTAs of a cluster add up their sums, a share of the rows each -----
// The eight softmax warps: the others have given their registers away.
template <int DP>
__device__ __forceinline__ void join_shares(const Args& a, Ctl* ctl, uint8_t* ring) {
  const Shared<DP> sh(ring);
  const Item& it = ctl->item[0];
  const Tile& tile = it.tile[0];
  const int rank = (int)(blockIdx.x % a.split), rows = BM / a.split;
  for (int x = threadIdx.x; x < rows * (DP / 8); x += 256) {
    const int row = rank * rows + x / (DP / 8), d = x % (DP / 8) * 8;
    const Row r(a, tile, row);
    if (!r.on || d >= a.dim) continue;
    float mm = -INFINITY, l = 0.f, o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.f;
    for (int c = 0; c < a.split; ++c) mm = fmaxf(mm, uk_ld_dsmem_f32(uk_mapa(uk_smem_u32(sh.m + row), c)));
    for (int c = 0; c < a.split; ++c) {  // in the order of the ranks
      const float m = uk_ld_dsmem_f32(uk_mapa(uk_smem_u32(sh.m + row), c)), f = m == -INFINITY ? 1.f : ex2(m - mm);
      const float4 u = uk_ld_dsmem_f32x4(uk_mapa(uk_smem_u32(sh.piece(row, d / 4)), c));
      const float4 v = uk_ld_dsmem_f32x4(uk_mapa(uk_smem_u32(sh.piece(row, d / 4 + 1)), c));
      l += uk_ld_dsmem_f32(uk_mapa(uk_smem_u32(sh.l + row), c)) * f;
      o[0] += u.x * f, o[1] += u.y * f, o[2] += u.z * f, o[3] += u.w * f;
      o[4] += v.x * f, o[5] += v.y * f, o[6] += v.z * f, o[7] += v.w * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bool odd = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      o[k] *= inv;
      odd |= !(fabsf(o[k]) < INFINITY);
    }
    const int64_t token = (int64_t)it.q0 + r.token;
    *reinterpret_cast<uint4*>(a.o + token * a.o_token + r.head * a.o_head + d) = make_uint4(
        uk_pack_average(o[0], o[1]), uk_pack_average(o[2], o[3]), uk_pack_average(o[4], o[5]), uk_pack_average(o[6], o[7]));
    if (a.lse != nullptr && d == 0)
      a.lse[token * a.heads_q + r.head] = l == 0.f ? -INFINITY : (mm - SHIFT + log2f(l)) * LN2;
    if (odd && l - l == 0.f) atomicOr(&ctl->odd[row / 32], 1u << (row % 32));
  }
  asm volatile("bar.sync 1, 256;" ::: "memory");
  for (int row = rank * rows + (int)(threadIdx.x >> 5); row < (rank + 1) * rows; row += 8)
    if (ctl->odd[row / 32] >> (row % 32) & 1u) look_again(a, it, tile, row, it.all_units, &ctl->limit);
}

// Most blocks of the grid can lie behind the list's end, up to as many as there are
// items: a warp that has got one of them takes over others, each in less time than it
// takes to start one (1024 prompts of 64 rows, 32 heads over 8 of 128: 357 us, 1340
// without this).  Returns the number of one that is on the list after all, its item
// looked up from the start, or -1; and how many answers there were.
__device__ __noinline__ int2 drain_blocks(const Args& a, Ctl* ctl, uint32_t items, uint32_t answers, Item* out) {
  uint32_t n = 0;
  const int block = next_listed(items, [&] {
    if ((threadIdx.x & 31) == 0) {
      uk_mbar_expect_tx(&ctl->next, 16);
      uk_next_block_ask(ctl->answer, &ctl->next);
      if (n % 1024 == 0) put_off(&ctl->limit);
    }
    __syncwarp();
    // this block's memory is not given up before the answer is there
    if (!__all_sync(0xffffffffu, uk_mbar_wait(&ctl->next, (answers + n) & 1u, nullptr, WAIT_NS))) {
      raise_fault(ctl, UK_FAULT_PRODUCER);
      return -1;
    }
    ++n;
    const int got = uk_next_block(ctl->answer);
    uk_fence_proxy_async_smem();  // read before the next answer is written
    __syncwarp();
    return got;
  });
  Cursor cursor;
  if (block >= 0) find_item(a, (uint32_t)block, cursor, out);
  return make_int2(block, (int)n);
}

// ---- items and loads, one warp ---------------------------------------------------------
template <int DP, bool kSplit>
__device__ __forceinline__ void load_items(const Args& a, Ctl* ctl, uint8_t* smem, uint8_t* ring,
                                           const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                           Cursor cursor, bool any) {
  using S = Smem<DP>;
  volatile int* abort = &ctl->abort;
  const int lane = threadIdx.x & 31;
  int block = blockIdx.x;
  uint32_t n = 0, fixed = 0, q_turn[2] = {0, 0};  // blocks put into the ring, V blocks zeroed, Q tiles loaded
  bool ok = true, asked = false;
  uint32_t answers = 0;
  for (uint32_t turn = 0; ok; ++turn) {
    Item& it = ctl->item[turn & 1u];
    if (lane == 0 && !*abort) put_off(&ctl->limit);
    if (!(ok = wait_warp(ctl, &ctl->item_empty[turn & 1u], ((turn >> 1) & 1u) ^ 1u, UK_FAULT_PRODUCER))) break;
    // the first item was looked up before the barriers were up
    if (turn > 0) any = block >= 0 && find_item(a, (uint32_t)block, cursor, &it);
    if (!kSplit && !any && block >= 0) {
      const int2 next = drain_blocks(a, ctl, cursor.before, answers, &it);
      block = next.x, answers += next.y;
      any = block >= 0;
    }
    __syncwarp();
    if (lane == 0) {
      it.any = any;
      uk_mbar_arrive(&ctl->item_full[turn & 1u]);  // releases the item to the waiting warps
      if (any && !kSplit) {
        uk_mbar_expect_tx(&ctl->next, 16);
        uk_next_block_ask(ctl->answer, &ctl->next);
      }
    }
    __syncwarp();
    if (!any) break;
    asked = !kSplit;
    const int blocks = it.blocks();
    for (int j = 0; j < 2 * blocks && ok; ++j) {
      if (j == 0) {
        for (int t = 0; t < 2 && ok; ++t) {
          if (it.tile[t].units == 0) continue;
          if (!(ok = wait_warp(ctl, &ctl->q_empty[t], (q_turn[t] & 1u) ^ 1u, UK_FAULT_PRODUCER))) break;
          ++q_turn[t];
          if (lane == 0) {
            // rows behind the last token's and head's stay as they are in shared memory: nobody reads their sums
            uk_mbar_expect_tx(&ctl->q_full[t], S::CHUNKS * 128 * a.heads * a.tokens);
#pragma unroll
            for (int c = 0; c < S::CHUNKS; ++c)
              uk_tma_load_3d(smem + t * S::TILE + c * S::BOX, &tm_q, &ctl->q_full[t], c * 64, it.tile[t].head,
                             it.q0 + it.tile[t].first);
          }
          __syncwarp();
        }
        if (!ok) break;
      }
      const int s = n % S::STAGES, at = (it.first_block + (j >> 1)) * BN;  // K and V blocks alternate
      if ((j & 127) == 127 && lane == 0 && !*abort) put_off(&ctl->limit);
      if (!(ok = wait_warp(ctl, &ctl->kv_empty[s], ((n / S::STAGES) & 1u) ^ 1u, UK_FAULT_PRODUCER))) break;
      const bool fix = (j & 1) && at + BN > it.m;
      uint8_t* dst = ring + (size_t)s * S::TILE;
      uint64_t* bar = fix ? &ctl->v_landed : &ctl->kv_full[s];
      if (lane == 0) {
        uk_mbar_expect_tx(bar, S::TILE);
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c)
          uk_tma_load_3d(dst + c * S::BOX, j & 1 ? &tm_v : &tm_k, bar, c * 64, it.k0 + at, it.g);
      }
      __syncwarp();
      ++n;
      if (fix) {
        // rows behind the sequence's last key hold whatever is there, and their weight is zero
        if (!__all_sync(0xffffffffu, uk_mbar_wait(bar, fixed & 1u, nullptr, WAIT_NS)))
          raise_fault(ctl, UK_FAULT_PRODUCER);
        ++fixed;
        const int valid = it.m - at;
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c)
          for (int x = valid * 8 + lane; x < BN * 8; x += 32)
            reinterpret_cast<uint4*>(dst + c * S::BOX)[x] = make_uint4(0, 0, 0, 0);
        uk_fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) uk_mbar_arrive(&ctl->kv_full[s]);
      }
    }
    if (!ok || kSplit) break;
    if (!(ok = wait_warp(ctl, &ctl->next, answers & 1u, UK_FAULT_PRODUCER))) break;
    ++answers;
    asked = false;
    block = uk_next_block(ctl->answer);
    uk_fence_proxy_async_smem();  // read before the next answer is written
    __syncwarp();
  }
  if (!ok || *abort) {  // what is in flight lands before this block's memory is given up
    if (asked) uk_mbar_wait(&ctl->next, answers & 1u, nullptr, WAIT_NS);
    for (uint32_t x = n > S::STAGES ? n - S::STAGES : 0; x < n; ++x)
      uk_mbar_wait(&ctl->kv_full[x % S::STAGES], (x / S::STAGES) & 1u, nullptr, WAIT_NS);
    for (int t = 0; t < 2; ++t)
      if (q_turn[t] > 0) uk_mbar_wait(&ctl->q_full[t], (q_turn[t] - 1) & 1u, nullptr, WAIT_NS);
  }
}

// ---- products of tile t ----------------------------------------------------------------
// The whole warp runs the loop and one elected lane issues: with control flow
// and operands the same in every lane the descriptors stay in uniform registers
// (issued from a branch of a single lane, every product waited for its operands
// to be moved there).  The tensor core takes few products ahead, so while this
// warp waits for the softmax it would run dry; the other tile's warp feeds it
// then (one warp for both tiles left it idle 40 % of the time).
template <int DP, bool kSplit, bool kParts>
__device__ __forceinline__ void issue_products(Ctl* ctl, int t, uint8_t* smem, uint8_t* ring, uint32_t tmem) {
  using S = Smem<DP>;
  constexpr uint32_t IDESC_S = uk_idesc_f16_ab(BM, UN, 0, 0), IDESC_O = uk_idesc_f16_ab(BM, DP, 0, 1);
  const uint32_t leader = uk_elect();
  const uint64_t dq = uk_desc_sw128(uk_smem_u32(smem + t * S::TILE), 16, 1024);  // K-major: Q and K
  const uint64_t dk = uk_desc_sw128(uk_smem_u32(ring), 16, 1024);
  const uint64_t dv = uk_desc_sw128(uk_smem_u32(ring), S::BOX, 1024);  // MN-major: V
  const uint32_t s_at = tmem + t * BN, o_at = tmem + 256 + t * 128;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool ok = wait_warp(ctl, bar, parity & 1u, UK_FAULT_MMA);
    uk_tc_fence_after();
    return ok;
  };
  auto commit = [&](uint64_t* bar) { uk_umma_commit_if(leader, bar); };
  uint32_t slot = 0, phase = 0;              // the ring's next block
  uint32_t turn[2] = {0, 0}, items = 0, ends = 0;  // of this tile so far: even and odd runs, items, parts of items
  auto next_slot = [&] {
    if (++slot == S::STAGES) slot = 0, phase ^= 1u;
  };
  // S for the even (h = 0) or odd run of the K block in the ring's slot `at`
  auto scores = [&](int h, uint32_t at) {
    const uint64_t k0 = dk + at * (S::TILE >> 4) + h * (UN * 128 >> 4);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      constexpr int BOX16 = S::BOX >> 4;
      const int off = (k / 4) * BOX16 + (k % 4) * 2;
      uk_umma_f16_ss(leader, s_at + h * UN, dq + off, k0 + off, IDESC_S, k > 0);
    }
    commit(&ctl->s_full[t][h]);
  };
  bool ok = true;
  for (uint32_t item = 0; ok; ++item) {
    if (!(ok = wait(&ctl->item_full[item & 1u], item >> 1))) break;
    const Item& it = ctl->item[item & 1u];
    const int any = __reduce_max_sync(0xffffffffu, it.any);  // the same in every lane, for the compiler too
    const int own = __reduce_max_sync(0xffffffffu, it.tile[t].units);
    const int blocks = __reduce_max_sync(0xffffffffu, it.blocks());
    __syncwarp();
    if (leader) uk_mbar_arrive(&ctl->item_empty[item & 1u]);
    if (!any) break;
    // Each tile's warp gives every block back, used or not, and never before it
    // is there: an early return would stand for the other warp's.
    if (blocks > 0 && !(ok = wait(&ctl->kv_full[slot], phase))) break;
    if (own > 0) {  // the scores of the first block
      if (!(ok = wait(&ctl->q_full[t], items))) break;
      ++items;
      scores(0, slot);
      if (own > 1) scores(1, slot);
      if (own <= 2) commit(&ctl->q_empty[t]);
    }
    if (blocks > 0) {
      commit(&ctl->kv_empty[slot]);
      next_slot();
    }
    for (int j = 0; j < blocks && ok; ++j) {
      // V of this block, K of the next
      const bool more = j + 1 < blocks;
      const uint32_t sv = slot, pv = phase;
      next_slot();
      const uint32_t sk = slot, pk = phase;
      if (more) next_slot();
      const uint64_t v0 = dv + sv * (S::TILE >> 4);
      if (!(ok = wait(&ctl->kv_full[sv], pv) && (!more || wait(&ctl->kv_full[sk], pk)))) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int u = 2 * j + h;
        if (!ok || u >= own) continue;
        if ((kParts ? u % PART == 0 : u == 0) && !(ok = wait(&ctl->o_empty[t], ends ^ 1u))) continue;
        if (!(ok = wait(&ctl->p_full[t][h], turn[h]))) continue;
        ++turn[h];
#pragma unroll
        for (int k = 0; k < UN / 16; ++k)  // O += P V
          uk_umma_f16_ts(leader, o_at, s_at + h * UN + k * 8, v0 + (h * (UN / 16) + k) * (2048 >> 4), IDESC_O,
                         u > 0 || k > 0);
        commit(&ctl->pv_done[t]);
        if (u + 2 < own) {
          scores(h, sk);
          if (u + 3 == own) commit(&ctl->q_empty[t]);
        }
        if (u + 1 == own || (kParts && (u + 1) % PART == 0)) {
          commit(&ctl->o_full[t]);
          ++ends;
        }
      }
      if (!ok) break;
      commit(&ctl->kv_empty[sv]);
      if (more) commit(&ctl->kv_empty[sk]);
    }
    if (kSplit) break;
  }
  // every product issued completes before TMEM and shared memory are given up
  commit(&ctl->teardown);
  // (the other tile's warp, too, has to get there)
  while (!__all_sync(0xffffffffu, uk_mbar_wait(&ctl->teardown, 0, nullptr, WAIT_NS))) {
    if (!__any_sync(0xffffffffu, uk_globaltimer() > *(volatile uint64_t*)&ctl->limit)) continue;
    atomicOr(&uk::g_attn_prompt_fault, UK_FAULT_TEARDOWN);
    break;
  }
}

// kSplit: a cluster of a.split CTAs per tile, each with a share of its keys, and
// one tile per block (no next item).  kParts: tiles may see more than PART runs.
template <int DP, bool kSplit, bool kParts>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    k_attn_prompt(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Args a) {
  using S = Smem<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* ring = smem + 2 * S::TILE;
  Ctl* ctl = (Ctl*)(ring + (size_t)S::STAGES * S::TILE);
  // the same in every lane, for the compiler too: the branches by it are uniform
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (warp == LOAD_WARP && lane == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      uk_mbar_init(&ctl->kv_full[s], 1);
      uk_mbar_init(&ctl->kv_empty[s], 2);  // both tiles' MMA warps
    }
    for (int t = 0; t < 2; ++t) {
      uk_mbar_init(&ctl->q_full[t], 1);
      uk_mbar_init(&ctl->q_empty[t], 1);
      for (int h = 0; h < 2; ++h) {
        uk_mbar_init(&ctl->s_full[t][h], 1);
        uk_mbar_init(&ctl->p_full[t][h], 4);
      }
      uk_mbar_init(&ctl->pv_done[t], 1);
      uk_mbar_init(&ctl->o_full[t], 1);
      uk_mbar_init(&ctl->o_empty[t], 4);
      uk_mbar_init(&ctl->item_full[t], 1);
      uk_mbar_init(&ctl->item_empty[t], 10);  // 8 softmax warps, 2 MMA warps
    }
    uk_mbar_init(&ctl->next, 1);
    uk_mbar_init(&ctl->v_landed, 1);
    uk_mbar_init(&ctl->teardown, 2);
    ctl->abort = 0;
    put_off(&ctl->limit);
    for (int i = 0; i < 4; ++i) ctl->odd[i] = 0;
    uk_fence_mbar_init();
    uk_tma_prefetch_desc(&tm_q);
    uk_tma_prefetch_desc(&tm_k);
    uk_tma_prefetch_desc(&tm_v);
  }
  if (warp == MMA_WARP) {
    uk_tmem_alloc(&ctl->tmem, 512);
    uk_tmem_relinquish();
  }
  Cursor cursor;
  bool any = false;
  if (warp == LOAD_WARP) {
    if (a.levels > 0) cursor.level = first_level(a);
    any = find_item(a, kSplit ? blockIdx.x / a.split : blockIdx.x, cursor, &ctl->item[0]);
    __syncwarp();
    if (kSplit && lane == 0) {
      Item& it = ctl->item[0];
      it.any = any;  // read by every warp at the end, too
      if (any) {
        const int rank = (int)(blockIdx.x % a.split), blocks = it.tile[0].blocks();
        const int from = (int)((int64_t)blocks * rank / a.split), to = (int)((int64_t)blocks * (rank + 1) / a.split);
        it.first_block = from;
        it.all_units = it.tile[0].units;
        it.tile[0].units = to > from ? min(it.all_units, 2 * to) - 2 * from : 0;
      }
    }
  }
  uk_tc_fence_before();
  __syncthreads();
  uk_tc_fence_after();
  const uint32_t tmem = ctl->tmem;

  if (warp < 8) {
    uk_regs_up<REGS_SOFTMAX>();
    uint32_t turn[2] = {0, 0}, ends = 0;
    for (uint32_t item = 0;; ++item) {
      if (!wait_warp(ctl, &ctl->item_full[item & 1u], (item >> 1) & 1u, UK_FAULT_EPILOGUE)) break;
      const Item& it = ctl->item[item & 1u];
      if (!it.any || !softmax_tile<DP, kSplit, kParts>(a, ctl, it, warp >> 2, tmem, ring, turn, &ends) || kSplit) break;
      __syncwarp();
      if (lane == 0) uk_mbar_arrive(&ctl->item_empty[item & 1u]);
    }
  } else {
    uk_regs_down<REGS_OTHERS>();
    if (warp == LOAD_WARP) load_items<DP, kSplit>(a, ctl, smem, ring, tm_q, tm_k, tm_v, cursor, any);
    else if (warp < MMA_WARP + 2) issue_products<DP, kSplit, kParts>(ctl, warp - MMA_WARP, smem, ring, tmem);
  }
  __syncwarp();
  uk_tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    uk_tc_fence_after();
    uk_tmem_dealloc(tmem, 512);
  }
  if constexpr (kSplit) {
    uk_cluster_sync();  // every CTA's sums are there
    if (warp < 8 && ctl->item[0].any && !ctl->abort) join_shares<DP>(a, ctl, ring);
    __syncwarp();
    uk_cluster_sync();  // no CTA leaves while another reads its shared memory
  }
}

// Row by row, a warp each: where there are no keys (every row is zero), and for a
// negative scale, which no model has (the tiles' softmax takes the maximum before
// it scales).
__global__ void __launch_bounds__(256) k_attn_prompt_rows(const __grid_constant__ Args a) {
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t t = w / a.heads_q;
  const int h = (int)(w - t * a.heads_q);
  const int b = t < a.total_q ? uk_find_seq<true>(a.cu_q, a.n_seq, t) : -1;
  if (b < 0) return;
  const int q1 = bound(a.cu_q, b + 1, 0, (int)a.total_q);
  const int64_t k0 = bound(a.cu_k, b, 0, (int)a.total_k), k1 = k0 + keys_of(a, b);
  attend_row(a, t, h, k0, a.causal ? k1 - (q1 - 1 - t) : k1, nullptr);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
  });
  return fn;
}

// packed rows [tokens][heads][dim] as a (dim, token, head) tensor, boxes of 64 x
// `tokens` x 1 (K, V), or as (dim, head, token), boxes of 64 x `heads` x `tokens`
// (Q); columns behind dim and rows behind the last are filled with zeros
int make_map(CUtensorMap* m, const char* name, const uint16_t* base, int dim, int64_t tokens, int heads,
             int64_t token_stride, int64_t head_stride, int box_tokens, int box_heads) {
  auto fn = encode_fn();
  if (!fn) return uk::fail(UK_ECUDA, "attn_prompt: cuTensorMapEncodeTiled is unavailable from the driver");
  // a stride that nothing steps by still has to be one the map accepts
  if (tokens == 1) token_stride = dim;
  if (heads == 1) head_stride = dim;
  const bool by_head = box_heads > 0;
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)tokens, (cuuint64_t)heads};
  cuuint64_t strides[2] = {(cuuint64_t)token_stride * 2, (cuuint64_t)head_stride * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_tokens, 1};
  if (by_head) {
    std::swap(dims[1], dims[2]);
    std::swap(strides[0], strides[1]);
    box[1] = (cuuint32_t)box_heads, box[2] = (cuuint32_t)box_tokens;
  }
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<uint16_t*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return uk::fail(UK_ECUDA, "attn_prompt: no tensor map of %s (%d)", name, (int)r);
  return UK_OK;
}

template <int DP, bool kSplit, bool kParts>
int launch(const Args& a, int64_t items, cudaStream_t st) {
  CUtensorMap q, k, v;
  if (int rc = make_map(&q, "Q", a.q, a.dim, a.total_q, a.heads_q, a.q_token, a.q_head, a.tokens, a.heads)) return rc;
  if (int rc = make_map(&k, "K", a.k, a.dim, a.total_k, a.heads_kv, a.k_token, a.k_head, BN, 0)) return rc;
  if (int rc = make_map(&v, "V", a.v, a.dim, a.total_k, a.heads_kv, a.v_token, a.v_head, BN, 0)) return rc;
  static bool attr_done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(k_attn_prompt<DP, kSplit, kParts>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Smem<DP>::BYTES);
    if (e != cudaSuccess) return uk::fail(UK_ECUDA, "attn_prompt: smem attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) attr_done[dev] = true;
  }
  if constexpr (!kSplit) {
    k_attn_prompt<DP, false, kParts><<<(unsigned)items, NUM_THREADS, Smem<DP>::BYTES, st>>>(q, k, v, a);
    return uk::check_launch("attn_prompt");
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  cfg.gridDim = dim3((unsigned)(items * a.split), 1, 1);
  cfg.blockDim = dim3(NUM_THREADS, 1, 1);
  cfg.dynamicSmemBytes = Smem<DP>::BYTES;
  cfg.stream = st;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)a.split;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_attn_prompt<DP, kSplit, kParts>, q, k, v, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return uk::fail(UK_ECUDA, "attn_prompt: %s", cudaGetErrorString(e));
  }
  return UK_OK;
}

template <int DP>
int launch(const Args& a, int64_t items, cudaStream_t st) {
  if (a.total_k > PART * UN)
    return a.split > 1 ? launch<DP, true, true>(a, items, st) : launch<DP, false, true>(a, items, st);
  return a.split > 1 ? launch<DP, true, false>(a, items, st) : launch<DP, false, false>(a, items, st);
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
  // 2^25 keys: a tile's pass over them takes 0.6 s, and weights below 2^-32 of the
  // largest, which binary16 does not hold, are at most 2^-7 of the sum; queries: a
  // tile's row numbers stay within 31 bits
  if (n_seq < 0 || n_seq > uk::MAX_SEQS || total_q < 0 || total_k < 0 || total_q > 0x7fffff00 || total_k > (1 << 25))
    return uk::fail(UK_EINVAL, "attn_prompt: n_seq %d (at most 2^24), total_q %lld (2^31 - 256), total_k %lld (2^25)",
                    n_seq, (long long)total_q, (long long)total_k);
  if (heads_kv < 1 || heads_q < 1 || heads_q > 65535 || heads_q % heads_kv != 0)
    return uk::fail(UK_EINVAL, "attn_prompt: %d query heads do not divide over %d key heads", heads_q, heads_kv);
  if (dim < 8 || dim > 128 || dim % 8 != 0)
    return uk::fail(UK_EINVAL, "attn_prompt: dim %d must be a multiple of 8 from 8 to 128", dim);
  const float scale2 = scale * LOG2E;
  if (!(scale2 - scale2 == 0.f)) return uk::fail(UK_EINVAL, "attn_prompt: the scale is not finite");
  if (total_q == 0 || n_seq == 0) return UK_OK;
  if (int rc = uk::check_rows("attn_prompt", "Q", Q, total_q, heads_q, q_token_stride, q_head_stride, dim)) return rc;
  if (int rc = uk::check_rows("attn_prompt", "O", O, total_q, heads_q, o_token_stride, o_head_stride, dim)) return rc;
  if (total_k > 0) {
    if (int rc = uk::check_rows("attn_prompt", "K", K, total_k, heads_kv, k_token_stride, k_head_stride, dim))
      return rc;
    if (int rc = uk::check_rows("attn_prompt", "V", V, total_k, heads_kv, v_token_stride, v_head_stride, dim))
      return rc;
  }
  if (int rc = uk::check_device_ptr(cu_q, "cu_q")) return rc;
  if (int rc = uk::check_device_ptr(cu_k, "cu_k")) return rc;
  if (LSE != nullptr)
    if (int rc = uk::check_device_ptr(LSE, "LSE")) return rc;
  Args a{Q, K, V, O, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
         o_token_stride, o_head_stride, LSE, cu_q, cu_k, n_seq, heads_q, heads_kv, heads_q / heads_kv, dim, causal,
         total_q, total_k, scale2};
  // a zero scale: any factor that no score can raise above rounding does the same
  // and leaves hidden scores at -inf
  if (a.scale2 == 0.f) a.scale2 = 1e-30f;
  if (total_k == 0 || a.scale2 < 0.f) {
    const int64_t blocks = (total_q * heads_q + 7) / 8;
    if (blocks > 0x7fffffff) return uk::fail(UK_EINVAL, "attn_prompt: total_q * heads_q exceeds the grid");
    k_attn_prompt_rows<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(a);
    return uk::check_launch("attn_prompt");
  }
  const int64_t items = plan_items(&a, uk::sm_count());
  if (items < 0) return uk::fail(UK_EINVAL, "attn_prompt: more tiles than a grid has blocks");
  return dim > 64 ? launch<128>(a, items, (cudaStream_t)stream) : launch<64>(a, items, (cudaStream_t)stream);
}
