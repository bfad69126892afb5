// attn_decode.cu -- attention of one new token per sequence over a paged cache:
//   O[b][h] = sum_p w_p V[p][g],  w = softmax(scale * Q[b][h] . K[p][g]),
// p < seq_lens[b], g = h / (query heads per key head), in one pass over the
// cache with a running reference m, sum l and product o per head:
//   l = sum 2^(s_p - m),  o = sum 2^(s_p - m) v_p,  s = score * scale * log2 e;
// m moves (l and o scaled by 2^(m - m')) only when a score passes it by 2^8, so
// weights stay within [0, 2^15] as binary16 after a constant shift of 7.
//
// The work is bound by streaming the cache once: the floor is its bytes over
// the HBM rate.  Two kernels:
// * k_attn_decode: one resident wave of CTAs.  The (sequence, key head) pairs'
//   lengths, cut into tiles of 64 or 128 positions, are laid end to end and
//   every CTA takes an equal run of that line, whatever the lengths are: no
//   tail of long sequences, no empty CTAs.  A run that covers a pair whole
//   writes O; a pair cut by a run's end leaves (m, l, o) in the workspace, at
//   most two per CTA (the pair that entered its run, the pair that leaves it).
// * k_attn_join_few / _many: for each pair that left a run, the sum of its parts
//   in the order of the CTAs (deterministic); launched programmatically behind
//   the first.
//
// Within a CTA each of 4 warps takes its own 16 or 32 positions of a tile and
// never waits for another: rows go from global memory straight into the
// registers of the mma.sync operand that needs them, with no shared memory in
// between.  The products are S^T = K Q^T (16 positions x 8 query heads) and
// O^T += V^T P^T, so a key head's query group fills the 8 columns instead of
// padding 16 rows, and the fragments fit 16-byte loads by renaming the
// contraction index:
//   K (A operand): lane (r = lane / 4, q = lane % 4) holds 16 bytes at byte
//     16 q of positions r and r + 8; Q is loaded in the same order of d, so
//     the sum over d is the same.
//   V^T (A operand): lane (r, q) holds 16 bytes at byte 16 r of positions 2q,
//     2q + 1, 2q + 8, 2q + 9; a byte permute pairs neighbouring positions, as
//     the operand packs them, and the row index d is renamed.
//   P^T (B operand): the S^T accumulator has position and head exchanged; an
//     8 x 8 transpose between lanes (movmatrix) puts that right.
// e4m3 rows are converted to binary16 in registers, exactly.  The keys' scale
// multiplies the score; the values' multiplies the converted codes (exact, too:
// a held value is a binary16 one).  In the weight's exponent instead, where it
// costs fewer instructions, it would push the weights of rows of small values into
// binary16's subnormals beside one row of large ones.
// K of the next tile loads while the softmax and V product of this one run,
// then V of the next; page ids load one tile earlier still.
#include "kv_cache.cuh"

namespace uk {
__device__ unsigned int g_attn_decode_fault = 0;
}  // namespace uk

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int MAX_CTAS = 1024;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float GROW = 8.f;   // scores may pass the reference by 2^8 before it moves
// positions that are summed up in one go: the tensor core's sums are truncated, and l
// is a plain one (one sequence of 2^20 positions per CTA in one go: 1e-3 too small)
constexpr int PART = 1 << 15;
constexpr float SHIFT = 7.f;  // weights are held as 2^7 * 2^(s - m): up to 2^15, binary16 ends at 2^16

struct Args {
  const uint16_t* q;
  int64_t q_seq, q_head;
  uint16_t* o;
  int64_t o_seq, o_head;
  float* lse;
  const int32_t* lens;
  int n_seq, heads_q, group;  // group = query heads per key head
  int chunks;                 // runs of 8 NH query heads per key head
  float scale2;               // scale * log2 e
  float* parts;               // [ctas][2][part_floats]; also holds a pair's sum between its PARTs
  // a pair cut by the end of its first CTA's run: {b, pair, first CTA, last
  // CTA}, b = -1: none; one per pair where there are no more pairs than CTAs
  // (by_pair), else one per CTA
  int4* recs;
  int by_pair;
  int unit;  // bytes: a power of two that divides the cache's strides; rows are passed between lanes in units
};

template <int KIND, int DP>
struct Shape {
  static constexpr bool kF16 = KIND == UK_KV_F16;
  static constexpr int NT = (kF16 && DP == 128) ? 1 : 2;  // 16-position groups per warp tile
  static constexpr int WT = 16 * NT, CT = WARPS * WT;     // positions per warp and CTA tile
  static constexpr int KC = kF16 ? DP / 32 : DP / 64;     // 16-byte loads of a K row per lane
  static constexpr int VC = kF16 ? DP / 64 : 1;           // loads of a V row per lane
  static constexpr int VB = kF16 ? 16 : DP / 8;           // bytes of each (8 or 16)
  static constexpr int VW = VB / 4;                       // words of each
  static constexpr int MV = DP / 16;                      // V products per group of positions
};

__host__ __device__ constexpr int part_floats(int dp, int nh) { return 8 * nh * (dp + 2); }

__device__ __forceinline__ uint4 ldg16(const void* p, bool on) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (on)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg8(const void* p, bool on) {
  uint2 v = make_uint2(0, 0);
  if (on) asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// D (16 x 8, fp32) += A (16 x 16, f16) B (16 x 8, f16)
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 x 8 transpose of halves between the lanes of a warp
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
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

// ---- the line of tiles -------------------------------------------------------------
// A pair takes a place per tile and START places in front of them, for what
// starting and joining it costs a CTA (its first loads, the sum over the warps):
// runs of many short pairs get fewer tiles.  0 / 1 / 2 / 3 places, one B200: the
// ragged 32 x 8192 e4m3 batch 66.3 / 62.5 / 62.9 / 62.7 us, 64 ragged sequences up
// to 1000 in f16 37.6 / 31.6 / 31.5 / 32.2 us.
constexpr int START = 1;

struct Line {
  int64_t total;  // places of all pairs
  int64_t ctas;   // CTAs that take part, each with at least one place
  __device__ __forceinline__ int64_t begin(int64_t c) const { return c * total / ctas; }
  // the CTA whose run holds place x: the last c with c * total / ctas <= x
  __device__ __forceinline__ int64_t owner(int64_t x) const { return ((x + 1) * ctas - 1) / total; }
};

__device__ __forceinline__ int clamped_len(const Args& a, int64_t room, int b) {
  const int len = max(__ldg(a.lens + b), 0);
  return len > room ? (int)room : len;
}

// places of a pair of `len` positions
template <int CT>
__device__ __forceinline__ int64_t places(int len) {
  return len > 0 ? (len + CT - 1) / CT + START : 0;
}

// The line, and the sequence that holds this CTA's first place with the number
// of places (of one pair) before it.  Every thread sums a run of sequences; the
// thread whose run holds the place finds it there.
template <int CT>
__device__ Line find_begin(const Args& a, int64_t room, int pairs, int64_t* x0, int64_t* x1, int* b0, int64_t* before) {
  __shared__ int64_t warp_sum[WARPS];
  __shared__ int64_t s_before;
  __shared__ int s_b;
  const int per = (a.n_seq + THREADS - 1) / THREADS;
  const int first = min((int)threadIdx.x * per, a.n_seq), last = min(first + per, a.n_seq);
  int64_t mine = 0;
  for (int b = first; b < last; ++b) mine += places<CT>(clamped_len(a, room, b));
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, incl, o);
    if ((threadIdx.x & 31) >= o) incl += t;
  }
  if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x >> 5] = incl;
  __syncthreads();
  int64_t base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < (int)(threadIdx.x >> 5)) base += warp_sum[w];
    all += warp_sum[w];
  }
  Line line{all * pairs, 0};
  line.ctas = min((int64_t)gridDim.x, line.total);
  *x0 = *x1 = 0;
  if ((int64_t)blockIdx.x < line.ctas) {
    *x0 = line.begin(blockIdx.x);
    *x1 = line.begin(blockIdx.x + 1);
    int64_t at = base + incl - mine;  // places before this thread's run
    if (at * pairs <= *x0 && *x0 < (at + mine) * pairs) {
      int b = first;
      for (;; ++b) {
        const int64_t here = places<CT>(clamped_len(a, room, b));
        if (*x0 < (at + here) * pairs) break;  // mine bounds the sum: ends within the run
        at += here;
      }
      s_b = b;
      s_before = at;
    }
  }
  __syncthreads();
  *b0 = s_b;
  *before = s_before;
  return line;
}

// ---- the kernel -----------------------------------------------------------------------
// kWhole: page_size is a multiple of 16, so a group of 16 positions lies in one
// page and its rows are one address apart; otherwise every position's row is
// looked up by one lane and passed to the others (32 x 8192 f16 positions: 173
// against 186 us).  e4m3 takes the second form always: its exponents are looked
// up by position in any case (ragged 32 x 8192: 68 against 79 us with kWhole).
//
// kCluster: short caches of few pairs.  The eight CTAs of a cluster take a
// pair's tiles in equal shares and add their sums up through distributed shared
// memory: one launch, no workspace (use_clusters has the rule and both sides).
constexpr int CLUSTER = 8;

template <int KIND, int DP, int NH, bool kWhole, bool kCluster>
__global__ void __launch_bounds__(THREADS, NH == 1 ? 3 : 2) k_attn_decode(Args a, UkKvView c) {
  using S = Shape<KIND, DP>;
  constexpr int CT = S::CT, WT = S::WT, NT = S::NT;
  __shared__ float sm_m[WARPS][8 * NH], sm_l[WARPS][8 * NH];
  __shared__ __align__(16) float sm_o[WARPS][8 * NH][DP + 2];
  __shared__ float part_m[2][8 * NH], part_l[2][8 * NH];  // of the PARTs of a pair so far; by turns
  __shared__ float sum_m[kCluster ? 8 * NH : 1], sum_l[kCluster ? 8 * NH : 1];  // of this CTA's four warps
  __shared__ __align__(16) float sum_o[kCluster ? 8 * NH : 1][kCluster ? DP : 4];

  if (!kCluster) uk_pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
  const int64_t room = (int64_t)c.max_pages * c.page_size;
  const int pairs = c.heads * a.chunks;

  // sequences without positions have no tiles: their rows are written at the
  // end, off the way to the first loads
  auto write_empty = [&] {
    for (int b = blockIdx.x; b < a.n_seq; b += gridDim.x) {
      const int len = __ldg(a.lens + b);
      if (len > room && threadIdx.x == 0) atomicOr(&uk::g_attn_decode_fault, UK_FAULT_PAGE);
      if (len > 0 && room > 0) continue;
      for (int i = threadIdx.x; i < a.heads_q * (c.dim / 8); i += THREADS) {
        const int h = i / (c.dim / 8), d = i % (c.dim / 8);
        reinterpret_cast<uint4*>(a.o + b * a.o_seq + h * a.o_head)[d] = make_uint4(0, 0, 0, 0);
      }
      if (a.lse != nullptr)
        for (int h = threadIdx.x; h < a.heads_q; h += THREADS) a.lse[(int64_t)b * a.heads_q + h] = -INFINITY;
      if (a.by_pair)
        for (int i = threadIdx.x; i < pairs; i += THREADS) a.recs[b * pairs + i] = make_int4(-1, 0, 0, 0);
    }
  };

  int64_t x0 = 0, x1 = 0, before = 0;
  int b, len, nt, pair;
  Line line{0, 0};
  int4 rec = make_int4(-1, 0, 0, 0);
  if (kCluster) {
    pair = (int)(blockIdx.x / CLUSTER);
    b = pair / pairs;
    pair -= b * pairs;
    len = clamped_len(a, room, b), nt = (len + CT - 1) / CT;
    const int rank = (int)(blockIdx.x % CLUSTER);
    x0 = (int64_t)nt * rank / CLUSTER, x1 = (int64_t)nt * (rank + 1) / CLUSTER;
    if (threadIdx.x == 0 && rank == 0 && __ldg(a.lens + b) > room) atomicOr(&uk::g_attn_decode_fault, UK_FAULT_PAGE);
  } else {
    line = find_begin<CT>(a, room, pairs, &x0, &x1, &b, &before);
    if (x0 >= x1) {
      if (threadIdx.x == 0 && !a.by_pair) a.recs[blockIdx.x] = rec;
      write_empty();
      return;
    }
    len = clamped_len(a, room, b), nt = (len + CT - 1) / CT;
    pair = (int)((x0 - before * pairs) / (nt + START));
  }

  int64_t x = x0;
  int turn = 0;
  for (bool more = true; more;) {
    // the place of the pair's first tile, and its tiles here
    const int64_t start = kCluster ? 0 : before * pairs + (int64_t)pair * (nt + START) + START;
    const int t0 = x > start ? (int)(x - start) : 0, end = (int)min((int64_t)nt, x1 - start);
    if (!kCluster && end <= t0) break;  // only places in front of it
    const int t1 = kCluster ? end : min(end, t0 + PART / CT);  // the rest follows in the next turn
    const int g = pair / a.chunks, h0 = g * a.group + (pair % a.chunks) * 8 * NH;
    const int heads = min(8 * NH, (g + 1) * a.group - h0);  // query heads of this run

    const int32_t* table = c.table + (int64_t)b * c.table_stride;
    const int p0 = t0 * CT + warp * WT;                       // first position of this warp
    const int p1 = (int)min((int64_t)t1 * CT, (int64_t)len);  // one past the run's last

    // The rows of a warp tile at p.  kWhole: group n's page id and then the
    // byte offset of its first row, the same in every lane (-1: absent).  Else
    // lane i's own for position p + i, the offset in units (ABSENT), with its
    // exponent bytes (e4m3).  K and V load one tile ahead, page ids two (three
    // without kWhole, and rows and exponents two): an instruction that needs a
    // load stops the warp until it is there.
    constexpr int NR = kWhole ? NT : 1;
    constexpr uint32_t ABSENT = 0xffffffffu;
    struct Where {
      int64_t row[NR];
      uint32_t unit;
      uint32_t ek, ev;
    };
    auto page_of = [&](int p, int (&page)[NR]) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int pos = kWhole ? p + n * 16 : p + lane;
        page[n] = pos < p1 && (kWhole || lane < WT) ? __ldg(table + c.div.div((uint32_t)pos)) : -1;
      }
    };
    auto rows_of = [&](int p, const int (&page)[NR]) {
      Where w;
      w.unit = ABSENT, w.ek = w.ev = 127;
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int pos = kWhole ? p + n * 16 : p + lane;
        w.row[n] = -1;
        if (pos < p1 && (kWhole || lane < WT)) {
          if ((unsigned)page[n] < (uint64_t)c.pages) {
            const int off = pos - (int)c.div.div((uint32_t)pos) * c.page_size;
            w.row[n] = uk_kv_row(c, page[n], off, g);
            if (!kWhole) w.unit = (uint32_t)((uint64_t)w.row[n] / (uint32_t)a.unit);
            if (!S::kF16) {
              const int64_t at = uk_kv_exp(c, page[n], off, g);
              w.ek = __ldg(c.k_exp + at);
              w.ev = __ldg(c.v_exp + at);
            }
          } else {
            atomicOr(&uk::g_attn_decode_fault, UK_FAULT_PAGE);
          }
        }
      }
      return w;
    };

    uint4 kr[NT][2][S::KC];
    uint32_t vr[NT][4][S::VC][S::VW];
    unsigned seen = 0;  // bit 2 n + i: position 16 n + 8 i + r of the tile counts
    // a warp tile without absent positions, of rows as long as the operands:
    // nothing to check per load
    bool plain = false;
    auto get_k = [&](const uint8_t* kp, bool on, uint4 (&to)[S::KC]) {
#pragma unroll
      for (int k = 0; k < S::KC; ++k) to[k] = ldg16(kp + k * 64, on && (k * 64 + q * 16) / (S::kF16 ? 2 : 1) < c.dim);
    };
    auto get_v = [&](const uint8_t* vp, bool on, uint32_t (&to)[S::VC][S::VW]) {
#pragma unroll
      for (int k = 0; k < S::VC; ++k) {
        const bool y = on && (k * 128 + r * S::VB) / (S::kF16 ? 2 : 1) < c.dim;
        if (S::VB == 16) {
          const uint4 v = ldg16(vp + k * 128, y);
          to[k][0] = v.x, to[k][1] = v.y, to[k][S::VW - 2] = v.z, to[k][S::VW - 1] = v.w;
        } else {
          const uint2 v = ldg8(vp + k * 128, y);
          to[k][0] = v.x, to[k][1] = v.y;
        }
      }
    };
    auto load_k = [&](const Where& w, int p) {
      seen = 0;
      if constexpr (kWhole) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const bool on = w.row[n] >= 0 && p + n * 16 + i * 8 + r < p1;
            if (on) seen |= 1u << (2 * n + i);
            get_k(c.k + w.row[n] + (int64_t)(i * 8 + r) * c.token_bytes + q * 16, on, kr[n][i]);
          }
      } else {
        plain = c.dim == DP && __all_sync(0xffffffffu, lane >= WT || w.unit != ABSENT);
        const uint8_t* kq = c.k + q * 16;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t u = __shfl_sync(0xffffffffu, w.unit, n * 16 + i * 8 + r);
            const uint8_t* kp = kq + (uint64_t)u * (uint32_t)a.unit;
            if (plain) {
#pragma unroll
              for (int k = 0; k < S::KC; ++k) kr[n][i][k] = ldg16(kp + k * 64, true);
            } else {
              if (u != ABSENT) seen |= 1u << (2 * n + i);
              get_k(kp, u != ABSENT, kr[n][i]);
            }
          }
        if (plain) seen = (1u << (2 * NT)) - 1;
      }
    };
    auto load_v = [&](const Where& w, int p) {
      if constexpr (kWhole) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int x = (i >> 1) * 8 + 2 * q + (i & 1);
            get_v(c.v + w.row[n] + (int64_t)x * c.token_bytes + r * S::VB, w.row[n] >= 0 && p + n * 16 + x < p1,
                  vr[n][i]);
          }
      } else {
        const uint8_t* vq = c.v + r * S::VB;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t u = __shfl_sync(0xffffffffu, w.unit, n * 16 + (i >> 1) * 8 + 2 * q + (i & 1));
            const uint8_t* vp = vq + (uint64_t)u * (uint32_t)a.unit;
            if (plain) {
#pragma unroll
              for (int k = 0; k < S::VC; ++k) {
                if (S::VB == 16) {
                  const uint4 v = ldg16(vp + k * 128, true);
                  vr[n][i][k][0] = v.x, vr[n][i][k][1] = v.y;
                  vr[n][i][k][S::VW - 2] = v.z, vr[n][i][k][S::VW - 1] = v.w;
                } else {
                  const uint2 v = ldg8(vp + k * 128, true);
                  vr[n][i][k][0] = v.x, vr[n][i][k][1] = v.y;
                }
              }
            } else {
              get_v(vp, u != ABSENT, vr[n][i]);
            }
          }
      }
    };

    // the first tile's loads go out before Q is brought into shape
    int page[NR];
    Where rows, next;
    if (p0 < p1) {
      int first[NR], second[NR];
      page_of(p0, first);
      page_of(p0 + CT, kWhole ? page : second);
      if constexpr (!kWhole) page_of(p0 + 2 * CT, page);
      rows = rows_of(p0, first);
      load_k(rows, p0);
      load_v(rows, p0);
      if constexpr (!kWhole) next = rows_of(p0 + CT, second);
    }

    // Q in the operand's order of d; absent heads and d behind dim are zero
    uint32_t qf[NH][DP / 8];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const uint16_t* qp = a.q + b * a.q_seq + (int64_t)(h0 + n * 8 + r) * a.q_head;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        // f16: 8 values at 32 i + 8 q; e4m3: the i-th half of 16 values at 64 (i / 2) + 16 q
        const int d = S::kF16 ? i * 32 + q * 8 : (i / 2) * 64 + q * 16 + (i % 2) * 8;
        const uint4 v = ldg16(qp + d, n * 8 + r < heads && d < c.dim);
        qf[n][i * 4] = v.x, qf[n][i * 4 + 1] = v.y, qf[n][i * 4 + 2] = v.z, qf[n][i * 4 + 3] = v.w;
      }
    }

    float m[NH][2], l[NH][2], acc[S::MV][NH][4];
#pragma unroll
    for (int n = 0; n < NH; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int j = 0; j < S::MV; ++j)
#pragma unroll
      for (int n = 0; n < NH; ++n) acc[j][n][0] = acc[j][n][1] = acc[j][n][2] = acc[j][n][3] = 0.f;

    for (int p = p0; p < p1; p += CT) {
      // ---- S^T = K Q^T
      float s[NT][NH][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int w = 0; w < NH; ++w) s[n][w][0] = s[n][w][1] = s[n][w][2] = s[n][w][3] = 0.f;
        if (S::kF16) {
#pragma unroll
          for (int k = 0; k < S::KC; ++k) {
            const uint4 lo = kr[n][0][k], hi = kr[n][1][k];
#pragma unroll
            for (int w = 0; w < NH; ++w) {
              mma16816(s[n][w], lo.x, hi.x, lo.y, hi.y, qf[w][k * 4], qf[w][k * 4 + 1]);
              mma16816(s[n][w], lo.z, hi.z, lo.w, hi.w, qf[w][k * 4 + 2], qf[w][k * 4 + 3]);
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < S::KC; ++k) {
            const uint32_t lo[4] = {kr[n][0][k].x, kr[n][0][k].y, kr[n][0][k].z, kr[n][0][k].w};
            const uint32_t hi[4] = {kr[n][1][k].x, kr[n][1][k].y, kr[n][1][k].z, kr[n][1][k].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a0, a1, a2, a3;
              uk_e4m3x4_to_half2(lo[i], &a0, &a2);
              uk_e4m3x4_to_half2(hi[i], &a1, &a3);
#pragma unroll
              for (int w = 0; w < NH; ++w)
                mma16816(s[n][w], a0, a1, a2, a3, qf[w][k * 8 + 2 * i], qf[w][k * 8 + 2 * i + 1]);
            }
          }
        }
      }
      const unsigned now = seen;
      // ---- the next tile's rows and keys
      const Where now_at = rows;
      if constexpr (kWhole) {
        rows = rows_of(p + CT, page);
        page_of(p + 2 * CT, page);
      } else {
        rows = next;
        next = rows_of(p + 2 * CT, page);
        page_of(p + 3 * CT, page);
      }
      load_k(rows, p + CT);

      // ---- scores, reference and weights
      float top[NH][2];
      float ek = 1.f;    // of this lane's position: scale * 2^ek
      uint32_t ev2 = 0;  // 2^ev of an even lane's position and of the next one, as halves
      if (!S::kF16) {
        ek = a.scale2 * uk_exp_scale(now_at.ek);
        const uint32_t own = uk_half2_of(uk_exp_scale(now_at.ev));
        ev2 = __byte_perm(own, __shfl_xor_sync(0xffffffffu, own, 1), 0x7610);
      }
#pragma unroll
      for (int w = 0; w < NH; ++w) top[w][0] = top[w][1] = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float f = S::kF16 ? a.scale2 : __shfl_sync(0xffffffffu, ek, n * 16 + i * 8 + r);
          const bool on = now >> (2 * n + i) & 1u;
#pragma unroll
          for (int w = 0; w < NH; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float& v = s[n][w][2 * i + h];
              v = on ? v * f : -INFINITY;
              top[w][h] = fmaxf(top[w][h], v);
            }
        }
      bool grow = false;
#pragma unroll
      for (int w = 0; w < NH; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) grow |= top[w][h] > m[w][h] + GROW;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int w = 0; w < NH; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float t = top[w][h];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
            t = fmaxf(t, m[w][h]);
            const float f = t == -INFINITY ? 1.f : ex2(m[w][h] - t);
            m[w][h] = t;
            l[w][h] *= f;
#pragma unroll
            for (int j = 0; j < S::MV; ++j) {
              acc[j][w][h] *= f;
              acc[j][w][2 + h] *= f;
            }
          }
      }
      uint32_t pf[NT][NH][2];
#pragma unroll
      for (int w = 0; w < NH; ++w) {
        const float z0 = m[w][0] == -INFINITY ? 0.f : m[w][0] - SHIFT;
        const float z1 = m[w][1] == -INFINITY ? 0.f : m[w][1] - SHIFT;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float a0 = ex2(s[n][w][2 * i] - z0), a1 = ex2(s[n][w][2 * i + 1] - z1);
            l[w][0] += a0;
            l[w][1] += a1;
            pf[n][w][i] = transpose8(pack_half(a0, a1));
          }
      }

      // ---- O^T += V^T P^T
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (S::kF16) {
#pragma unroll
          for (int k = 0; k < S::VC; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a0 = __byte_perm(vr[n][0][k][i], vr[n][1][k][i], 0x5410);
              const uint32_t a1 = __byte_perm(vr[n][0][k][i], vr[n][1][k][i], 0x7632);
              const uint32_t a2 = __byte_perm(vr[n][2][k][i], vr[n][3][k][i], 0x5410);
              const uint32_t a3 = __byte_perm(vr[n][2][k][i], vr[n][3][k][i], 0x7632);
#pragma unroll
              for (int w = 0; w < NH; ++w) mma16816(acc[k * 4 + i][w], a0, a1, a2, a3, pf[n][w][0], pf[n][w][1]);
            }
        } else {
          const uint32_t e0 = __shfl_sync(0xffffffffu, ev2, n * 16 + 2 * q);  // of positions 2q, 2q + 1
          const uint32_t e1 = __shfl_sync(0xffffffffu, ev2, n * 16 + 8 + 2 * q);
#pragma unroll
          for (int i = 0; i < S::VW; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t sel = half ? 0x7362 : 0x5140;
              const uint32_t y0 = __byte_perm(vr[n][0][0][i], vr[n][1][0][i], sel);
              const uint32_t y1 = __byte_perm(vr[n][2][0][i], vr[n][3][0][i], sel);
              uint32_t a0, a1, a2, a3;
              uk_e4m3x4_to_half2(y0, &a0, &a1);
              uk_e4m3x4_to_half2(y1, &a2, &a3);
              a0 = uk_mul_half2(a0, e0), a1 = uk_mul_half2(a1, e0);
              a2 = uk_mul_half2(a2, e1), a3 = uk_mul_half2(a3, e1);
#pragma unroll
              for (int w = 0; w < NH; ++w)
                mma16816(acc[2 * i + half][w], a0, a1, a2, a3, pf[n][w][0], pf[n][w][1]);
            }
        }
      }
      load_v(rows, p + CT);
    }

    // ---- the four warps' parts joined in shared memory
#pragma unroll
    for (int w = 0; w < NH; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float t = l[w][h];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        const int head = w * 8 + 2 * q + h;
        if (r == 0) {
          sm_m[warp][head] = m[w][h];
          sm_l[warp][head] = t;
        }
#pragma unroll
        for (int j = 0; j < S::MV; ++j) {
          const int d = S::kF16 ? (j / 4) * 64 + r * 8 + (j % 4) * 2 : r * (DP / 8) + 2 * j;
          *reinterpret_cast<float2*>(&sm_o[warp][head][d]) = make_float2(acc[j][w][h], acc[j][w][2 + h]);
        }
      }
    __syncthreads();
    const bool entered = x0 > start, leaves = end < nt;
    const bool goes_on = t1 < end, went_on = t0 > 0 && x > x0;  // the pair's PARTs here behind and before this one
    float* part = a.parts + ((int64_t)blockIdx.x * 2 + (entered ? 0 : 1)) * part_floats(DP, NH);
    constexpr int LANES = DP / 8;  // threads per head, 8 values each
    for (int i = threadIdx.x; i < heads * LANES; i += THREADS) {
      const int head = i / LANES, d = (i % LANES) * 8;
      float mm = -INFINITY, ll = 0.f, o[8];
#pragma unroll
      for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, sm_m[w][head]);
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float mw = sm_m[w][head];
        // a warp without a reference has zero sums, or NaN ones that stay
        const float f = mw == -INFINITY ? 1.f : ex2(mw - mm);
        ll += sm_l[w][head] * f;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] += sm_o[w][head][d + k] * f;
      }
      if (!kCluster && went_on) {  // what this thread left of the PARTs before
        const float m0 = part_m[turn][head], m2 = fmaxf(mm, m0);
        const float f = mm == m2 ? 1.f : ex2(mm - m2), f0 = m0 == m2 ? 1.f : ex2(m0 - m2);
        const float4* src = reinterpret_cast<const float4*>(part + 16 * NH + head * DP + d);
        const float4 u = src[0], v = src[1];
        mm = m2, ll = ll * f + part_l[turn][head] * f0;
        o[0] = o[0] * f + u.x * f0, o[1] = o[1] * f + u.y * f0, o[2] = o[2] * f + u.z * f0, o[3] = o[3] * f + u.w * f0;
        o[4] = o[4] * f + v.x * f0, o[5] = o[5] * f + v.y * f0, o[6] = o[6] * f + v.z * f0, o[7] = o[7] * f + v.w * f0;
      }
      if (kCluster) {
        if (d == 0) sum_m[head] = mm, sum_l[head] = ll;
        *reinterpret_cast<float4*>(&sum_o[head][d]) = make_float4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<float4*>(&sum_o[head][d + 4]) = make_float4(o[4], o[5], o[6], o[7]);
      } else if (entered || leaves || goes_on) {
        if (d == 0 && goes_on) {
          part_m[turn ^ 1][head] = mm, part_l[turn ^ 1][head] = ll;
        } else if (d == 0) {
          part[head] = mm;
          part[8 * NH + head] = ll;
        }
        float4* dst = reinterpret_cast<float4*>(part + 16 * NH + head * DP + d);
        dst[0] = make_float4(o[0], o[1], o[2], o[3]);
        dst[1] = make_float4(o[4], o[5], o[6], o[7]);
      } else {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        if (d < c.dim)
          *reinterpret_cast<uint4*>(a.o + b * a.o_seq + (int64_t)(h0 + head) * a.o_head + d) =
              make_uint4(uk_pack_average(o[0] * inv, o[1] * inv), uk_pack_average(o[2] * inv, o[3] * inv),
                         uk_pack_average(o[4] * inv, o[5] * inv), uk_pack_average(o[6] * inv, o[7] * inv));
        if (a.lse != nullptr && d == 0)
          a.lse[(int64_t)b * a.heads_q + h0 + head] = ll == 0.f ? -INFINITY : (mm - SHIFT + log2f(ll)) * LN2;
      }
    }
    if constexpr (kCluster) {
      uk_cluster_sync();
      // each CTA adds up an eighth of the pair's values, in the order of the ranks
      const int i = (int)(blockIdx.x % CLUSTER) + CLUSTER * (int)threadIdx.x;
      if (i < heads * LANES) {
        const int head = i / LANES, d = (i % LANES) * 8;
        float mi[CLUSTER], mm = -INFINITY, ll = 0.f, o[8];
#pragma unroll
        for (int k = 0; k < CLUSTER; ++k) {
          mi[k] = uk_ld_dsmem_f32(uk_mapa(uk_smem_u32(&sum_m[head]), k));
          mm = fmaxf(mm, mi[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll
        for (int k = 0; k < CLUSTER; ++k) {
          const float f = mi[k] == -INFINITY ? 1.f : ex2(mi[k] - mm);
          ll += uk_ld_dsmem_f32(uk_mapa(uk_smem_u32(&sum_l[head]), k)) * f;
          const uint32_t at = uk_mapa(uk_smem_u32(&sum_o[head][d]), k);
          const float4 u = uk_ld_dsmem_f32x4(at), v = uk_ld_dsmem_f32x4(at + 16);
          o[0] += u.x * f, o[1] += u.y * f, o[2] += u.z * f, o[3] += u.w * f;
          o[4] += v.x * f, o[5] += v.y * f, o[6] += v.z * f, o[7] += v.w * f;
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        if (d < c.dim)
          *reinterpret_cast<uint4*>(a.o + b * a.o_seq + (int64_t)(h0 + head) * a.o_head + d) =
              make_uint4(uk_pack_average(o[0] * inv, o[1] * inv), uk_pack_average(o[2] * inv, o[3] * inv),
                         uk_pack_average(o[4] * inv, o[5] * inv), uk_pack_average(o[6] * inv, o[7] * inv));
        if (a.lse != nullptr && d == 0)
          a.lse[(int64_t)b * a.heads_q + h0 + head] = ll == 0.f ? -INFINITY : (mm - SHIFT + log2f(ll)) * LN2;
      }
      uk_cluster_sync();  // no CTA leaves while another reads its shared memory
      return;
    }
    turn ^= 1;
    if (!entered && !goes_on) {
      if (leaves) rec = make_int4(b, pair, blockIdx.x, (int)line.owner(start + nt - 1));
      if (a.by_pair && threadIdx.x == 0) a.recs[b * pairs + pair] = leaves ? rec : make_int4(-1, 0, 0, 0);
    }
    __syncthreads();

    x = start + t1;
    more = x < x1;
    if (more && !goes_on && ++pair == pairs) {
      pair = 0;
      before += nt + START;
      do {
        ++b;
        len = clamped_len(a, room, b);
        nt = (len + CT - 1) / CT;
      } while (nt == 0);
    }
  }
  if (threadIdx.x == 0 && !a.by_pair) a.recs[blockIdx.x] = rec;
  write_empty();
}

// A warp per (cut pair, query head of its run), the parts one after the other
// with a running reference, four loads of each kind in flight and nothing to
// wait for between warps: for pairs of few parts.
template <int DP, int NH>
__global__ void __launch_bounds__(256) k_attn_join_few(Args a, int dim) {
  uk_pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 rec = a.recs[blockIdx.x / NH];
  const int b = rec.x, pair = rec.y, first = rec.z, n = rec.w - first + 1;
  const int head = (blockIdx.x % NH) * 8 + warp;
  if (b < 0) return;
  const int g = pair / a.chunks, h = g * a.group + (pair % a.chunks) * 8 * NH + head;
  if (h >= (g + 1) * a.group) return;
  constexpr int LANES = DP / 4, PER = 32 / LANES, U = 4;  // lanes of a part's row; a warp takes PER parts at a time
  const int d4 = lane % LANES;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = lane / LANES; i0 < n; i0 += U * PER) {
    float mi[U], li[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * PER;
      mi[u] = -INFINITY, li[u] = 0.f, v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < n) {
        const float* p = a.parts + ((int64_t)(first + i) * 2 + (i == 0 ? 1 : 0)) * part_floats(DP, NH);
        mi[u] = p[head];
        li[u] = p[8 * NH + head];
        v[u] = reinterpret_cast<const float4*>(p + 16 * NH + head * DP)[d4];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float m2 = fmaxf(m, mi[u]);
      const float f = m == m2 ? 1.f : ex2(m - m2), e = mi[u] == -INFINITY ? 1.f : ex2(mi[u] - m2);
      m = m2;
      l = l * f + li[u] * e;
      o = make_float4(o.x * f + v[u].x * e, o.y * f + v[u].y * e, o.z * f + v[u].z * e, o.w * f + v[u].w * e);
    }
  }
  if (PER == 2) {  // the two halves' sums
    const float m1 = __shfl_xor_sync(0xffffffffu, m, 16), m2 = fmaxf(m, m1);
    const float f = m == -INFINITY ? 1.f : ex2(m - m2), e = m1 == -INFINITY ? 1.f : ex2(m1 - m2);
    m = m2;
    l = l * f + __shfl_xor_sync(0xffffffffu, l, 16) * e;
    o.x = o.x * f + __shfl_xor_sync(0xffffffffu, o.x, 16) * e;
    o.y = o.y * f + __shfl_xor_sync(0xffffffffu, o.y, 16) * e;
    o.z = o.z * f + __shfl_xor_sync(0xffffffffu, o.z, 16) * e;
    o.w = o.w * f + __shfl_xor_sync(0xffffffffu, o.w, 16) * e;
  }
  if (lane >= LANES) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (d4 * 4 < dim)
    reinterpret_cast<uint2*>(a.o + b * a.o_seq + (int64_t)h * a.o_head)[d4] =
        make_uint2(uk_pack_average(o.x * inv, o.y * inv), uk_pack_average(o.z * inv, o.w * inv));
  if (a.lse != nullptr && d4 == 0)
    a.lse[(int64_t)b * a.heads_q + h] = l == 0.f ? -INFINITY : (m - SHIFT + log2f(l)) * LN2;
}

// One CTA per (cut pair, query head of its run): weights of the parts, then
// their sum, the warps taking turns: for pairs of many parts.
template <int DP, int NH>
__global__ void __launch_bounds__(512) k_attn_join_many(Args a, int dim) {
  constexpr int JT = 512;
  constexpr int JW = JT / 32;
  __shared__ float wt[MAX_CTAS];
  __shared__ float red[33];
  __shared__ float4 so[JW][32];
  uk_pdl_wait();
  const int head = blockIdx.x % (8 * NH);
  const int4 rec = a.recs[blockIdx.x / (8 * NH)];
  const int b = rec.x, pair = rec.y, first = rec.z, n = rec.w - first + 1;
  if (b < 0) return;
  const int g = pair / a.chunks, h = g * a.group + (pair % a.chunks) * 8 * NH + head;
  if (h >= (g + 1) * a.group) return;
  auto part = [&](int i) { return a.parts + ((int64_t)(first + i) * 2 + (i == 0 ? 1 : 0)) * part_floats(DP, NH); };
  float mm = -INFINITY;
  for (int i = threadIdx.x; i < n; i += JT) mm = fmaxf(mm, part(i)[head]);
  mm = uk_block_max<JT>(mm, red);
  float ll = 0.f;
  for (int i = threadIdx.x; i < n; i += JT) {
    const float mw = part(i)[head], f = mw == -INFINITY ? 1.f : ex2(mw - mm);
    wt[i] = f;
    ll += f * part(i)[8 * NH + head];
  }
  ll = uk_block_sum<JT>(ll, red);  // ends with a barrier: wt is complete
  constexpr int LANES = DP / 4, PER = 32 / LANES;  // a warp takes PER parts at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d4 = lane % LANES;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp * PER + lane / LANES; i < n; i += JW * PER) {
    const float4 v = reinterpret_cast<const float4*>(part(i) + 16 * NH + head * DP)[d4];
    const float f = wt[i];
    o = make_float4(o.x + f * v.x, o.y + f * v.y, o.z + f * v.z, o.w + f * v.w);
  }
  so[warp][lane] = o;
  __syncthreads();
  if (threadIdx.x < LANES) {
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < JW; ++w)
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const float4 v = so[w][k * LANES + d4];
        o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
      }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    if (d4 * 4 < dim)
      reinterpret_cast<uint2*>(a.o + b * a.o_seq + (int64_t)h * a.o_head)[d4] =
          make_uint2(uk_pack_average(o.x * inv, o.y * inv), uk_pack_average(o.z * inv, o.w * inv));
    if (a.lse != nullptr && d4 == 0)
      a.lse[(int64_t)b * a.heads_q + h] = ll == 0.f ? -INFINITY : (mm - SHIFT + log2f(ll)) * LN2;
  }
}

// ---- host side ------------------------------------------------------------------------

// query heads per key head above 8 run as 16 wide: the cache is read once for
// 16 of them, at twice the registers
int heads_nh(int group) { return group > 8 ? 2 : 1; }
int padded_dim(int dim) { return dim > 64 ? 128 : 64; }
int ctas_per_sm(int nh) { return nh == 1 ? 3 : 2; }

int grid_ctas(int nh) {
  const int n = uk::sm_count() * ctas_per_sm(nh);
  return n < MAX_CTAS ? n : MAX_CTAS;
}

size_t workspace_bytes_for(int ctas, int dp, int nh) {
  return (size_t)ctas * (sizeof(int4) + 2 * sizeof(float) * part_floats(dp, nh));
}

// Clusters of eight CTAs per pair, or the even split and its join?  The lengths are
// not known here, the table's room is.  Clusters while they all run at once (two
// CTAs per SM) and a CTA's share of the room, room / 8, is at most as many
// positions as eight per CTA of the grid.  Measured on one B200 in a graph, 8 key
// heads of 128, clusters against the split: 1 sequence of 500 4.5 / 7.7 us, 4000
// 10.3 / 11.5, 8000 15.9 / 13.6; 4 sequences of 500 5.8 / 10.0, 16000 47.6 / 49.7;
// 7 sequences (448 CTAs) of 2000 16.8 / 16.5, 13 of 500 15.1 / 12.7.
bool use_clusters(int64_t pairs, int64_t room) {
  const int64_t ctas = pairs * CLUSTER;
  return ctas <= 2 * uk::sm_count() && room / CLUSTER <= 8 * ctas;
}

template <int DP, int NH>
int launch_join(const Args& a, int dim, int ctas, cudaStream_t st) {
  const int64_t all = (int64_t)a.n_seq * (a.heads_q / a.group) * a.chunks;
  // 16 warps per head where a pair can have many parts (one sequence of 131071
  // with two key heads, 148 parts a pair: 7.5 us against 17.4 by four warps);
  // else a warp per head
  const bool many = a.by_pair && ctas / all >= 16;
  const int64_t recs = a.by_pair ? all : ctas;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  cfg.gridDim = dim3((unsigned)(recs * (many ? 8 * NH : NH)), 1, 1);
  cfg.blockDim = dim3(many ? 512 : 256, 1, 1);
  cfg.stream = st;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = many ? cudaLaunchKernelEx(&cfg, k_attn_join_many<DP, NH>, a, dim)
                             : cudaLaunchKernelEx(&cfg, k_attn_join_few<DP, NH>, a, dim);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return uk::fail(UK_ECUDA, "attn_decode: %s", cudaGetErrorString(e));
  }
  return UK_OK;
}

template <int KIND, int DP, int NH, bool kWhole>
int launch(const Args& a, const UkKvView& c, int ctas, cudaStream_t st) {
  const int64_t all = (int64_t)a.n_seq * c.heads * a.chunks;
  if (use_clusters(all, (int64_t)c.max_pages * c.page_size)) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    cfg.gridDim = dim3((unsigned)(all * CLUSTER), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.stream = st;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = CLUSTER;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k_attn_decode<KIND, DP, NH, kWhole, true>, a, c);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return uk::fail(UK_ECUDA, "attn_decode: %s", cudaGetErrorString(e));
    }
    return UK_OK;
  }
  k_attn_decode<KIND, DP, NH, kWhole, false><<<(unsigned)ctas, THREADS, 0, st>>>(a, c);
  if (int rc = uk::check_launch("attn_decode")) return rc;
  return launch_join<DP, NH>(a, c.dim, ctas, st);
}

// every group of 16 positions in one page (kWhole)
bool whole_groups(const UkKvView& c) { return c.kind == UK_KV_F16 && c.page_size % 16 == 0; }

template <int KIND, int DP, int NH>
int launch(const Args& a, const UkKvView& c, int ctas, cudaStream_t st) {
  if constexpr (KIND == UK_KV_F16)
    if (whole_groups(c)) return launch<KIND, DP, NH, true>(a, c, ctas, st);
  return launch<KIND, DP, NH, false>(a, c, ctas, st);
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
  if (heads_q <= 0 || heads_kv <= 0 || dim <= 0 || dim > 128) return 0;
  const int nh = heads_nh(heads_q / heads_kv);
  return workspace_bytes_for(grid_ctas(nh), padded_dim(dim), nh);
}

extern "C" int uk_cuda_attn_decode_f16(const uint16_t* Q, int64_t q_seq_stride, int64_t q_head_stride,
                                       const uk_kv_cache* cache, const int32_t* block_table, int64_t table_stride,
                                       int max_pages, const int32_t* seq_lens, int n_seq, int heads_q, float scale,
                                       uint16_t* O, int64_t o_seq_stride, int64_t o_head_stride, float* LSE,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  if (n_seq < 0 || n_seq > uk::MAX_SEQS || heads_q < 1 || heads_q > 65535)
    return uk::fail(UK_EINVAL, "attn_decode: n_seq %d (at most 2^24), heads_q %d (at most 65535)", n_seq, heads_q);
  const float scale2 = scale * LOG2E;
  if (!(scale2 - scale2 == 0.f)) return uk::fail(UK_EINVAL, "attn_decode: the scale is not finite");
  UkKvView c;
  if (int rc = uk::kv_view(cache, block_table, table_stride, n_seq, max_pages, "attn_decode", &c)) return rc;
  if (heads_q % cache->heads != 0)
    return uk::fail(UK_EINVAL, "attn_decode: %d query heads do not divide over %d key heads", heads_q, cache->heads);
  if (n_seq == 0) return UK_OK;
  if (int rc = uk::check_rows("attn_decode", "Q", Q, n_seq, heads_q, q_seq_stride, q_head_stride, 0)) return rc;
  if (int rc = uk::check_rows("attn_decode", "O", O, n_seq, heads_q, o_seq_stride, o_head_stride, cache->dim))
    return rc;
  if (int rc = uk::check_device_ptr(seq_lens, "seq_lens")) return rc;
  if (LSE != nullptr)
    if (int rc = uk::check_device_ptr(LSE, "LSE")) return rc;
  if (int rc = uk::check_device_ptr(workspace, "workspace")) return rc;
  const int group = heads_q / cache->heads, nh = heads_nh(group), ctas = grid_ctas(nh), dp = padded_dim(cache->dim);
  const size_t need = workspace_bytes_for(ctas, dp, nh);
  if (workspace_bytes < need || !uk::aligned16(workspace))
    return uk::fail(UK_EINVAL, "attn_decode: workspace of %zu bytes, %zu wanted, 16-byte aligned", workspace_bytes,
                    need);
  Args a{Q, q_seq_stride, q_head_stride, O, o_seq_stride, o_head_stride, LSE, seq_lens, n_seq, heads_q, group,
         (group + 8 * nh - 1) / (8 * nh), scale2, nullptr, (int4*)workspace, 0, 0};
  a.by_pair = (int64_t)n_seq * cache->heads * a.chunks <= ctas;
  // rows cross lanes as 32-bit multiples of the strides' common power of two
  int64_t strides = 4096;
  if (c.pages > 1) strides |= c.page_bytes;
  if (c.page_size > 1) strides |= c.token_bytes;
  if (c.heads > 1) strides |= c.head_bytes;
  a.unit = (int)(strides & -strides);
  // (in 128 bits: nothing bounds the strides).  Whole groups go by 64-bit offsets:
  // there the limit only catches strides that cannot be meant, 4 TiB from end to end.
  const __int128 far = (__int128)(c.pages - 1) * c.page_bytes + (__int128)(c.page_size - 1) * c.token_bytes +
                       (__int128)(c.heads - 1) * c.head_bytes;
  if (c.pages > 0 && far / a.unit >= 0xffffffffll && (!whole_groups(c) || far >= (__int128)1 << 42))
    return uk::fail(UK_EINVAL, "attn_decode: a pool of %.3g bytes with strides of multiples of %d bytes only",
                    (double)far, a.unit);
  a.parts = reinterpret_cast<float*>(a.recs + ctas);
  const cudaStream_t st = (cudaStream_t)stream;
  switch ((cache->kind == UK_KV_E4M3 ? 4 : 0) + (dp == 128 ? 2 : 0) + (nh - 1)) {
    case 0: return launch<UK_KV_F16, 64, 1>(a, c, ctas, st);
    case 1: return launch<UK_KV_F16, 64, 2>(a, c, ctas, st);
    case 2: return launch<UK_KV_F16, 128, 1>(a, c, ctas, st);
    case 3: return launch<UK_KV_F16, 128, 2>(a, c, ctas, st);
    case 4: return launch<UK_KV_E4M3, 64, 1>(a, c, ctas, st);
    case 5: return launch<UK_KV_E4M3, 64, 2>(a, c, ctas, st);
    case 6: return launch<UK_KV_E4M3, 128, 1>(a, c, ctas, st);
    default: return launch<UK_KV_E4M3, 128, 2>(a, c, ctas, st);
  }
}
