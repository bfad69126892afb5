// attn_prompt_items.cuh -- what the blocks of the prompt attention work on: the
// list of items (pairs of tiles) of a packed batch, an item by its number, and the
// numbers that blocks take over from one another.  Everything but the sums over a
// warp compiles for the host too, where the list is tested.
#pragma once

#include "kv_cache.cuh"

namespace uk_prompt {

constexpr int BM = 128, BN = 128;  // rows of a tile, keys of a block
constexpr int UN = 64;             // keys of a softmax step (half a block)

struct Args {
  const uint16_t *q, *k, *v;
  uint16_t* o;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  float* lse;
  const int32_t *cu_q, *cu_k;
  int n_seq, heads_q, heads_kv, group, dim, causal;
  int64_t total_q, total_k;
  float scale2;
  int levels;  // of the order of work
  int tiles;   // of an item: 2, or 1 where pairs would leave SMs without work
  int split;   // CTAs (a cluster) that share a tile's keys
  // a tile is `tokens` query tokens by `heads` query heads of one key head, the
  // heads of a token side by side; `chunks` tiles make the key head's group
  int tokens, heads, chunks;
  UkFastDiv by_tokens, by_heads, by_chunks, by_kv;  // by tokens, heads, chunks and heads_kv
};

struct Tile {
  int head;    // its first query head; -1: no tile
  int heads;   // query heads it has
  int first;   // its first token within the sequence
  int tokens;  // tokens it has
  int units;   // runs of 64 keys that some row of it sees
  __host__ __device__ __forceinline__ int blocks() const { return (units + 1) / 2; }
};
// row i of a tile: token i / a.heads of it, head i % a.heads
struct Row {
  int token, head;
  bool on;
  __host__ __device__ __forceinline__ Row(const Args& a, const Tile& t, int i) {
    token = (int)a.by_heads.div((uint32_t)i);
    head = i - token * a.heads;
    on = token < t.tokens && head < t.heads;
    token += t.first, head += t.head;
  }
};
struct Item {
  Tile tile[2];
  int g;             // key head
  int q0, k0, n, m;  // the sequence: its first rows, query and key counts
  int any;           // 0: there is no further item
  int first_block;   // the first block of keys that this CTA works on
  int all_units;     // tile 0's runs of keys, of which tile[0].units are this CTA's
  __host__ __device__ __forceinline__ int blocks() const { return max(tile[0].blocks(), tile[1].blocks()); }
};

// How a call's work is cut: fills in `levels` to `by_kv`, the rest of *a given.
// Returns the blocks (clusters, where split > 1) that hold the items whatever the
// lengths are, or -1 where a grid has not as many.
inline int64_t plan_items(Args* a, int sms) {
  a->levels = 0, a->tiles = 2, a->split = 1;
  // the order of work: a level per power of two of the keys a tile can see; with
  // many sequences every level is a long search, and the order matters less
  if (a->n_seq <= 1024)
    while ((a->total_k + UN - 1) / UN >> a->levels) ++a->levels;
  const int64_t seqs = a->n_seq < a->total_q ? a->n_seq : a->total_q;
  // the heads of a group in as few tiles as hold them, a tile's rows filled up with tokens
  a->chunks = (a->group + BM - 1) / BM;
  a->heads = (a->group + a->chunks - 1) / a->chunks;
  a->tokens = BM / a->heads;
  a->by_tokens = UkFastDiv::make(a->tokens), a->by_heads = UkFastDiv::make(a->heads);
  a->by_chunks = UkFastDiv::make(a->chunks), a->by_kv = UkFastDiv::make(a->heads_kv);
  // at most this many query blocks and pairs of tiles
  const int64_t most = (a->total_q + (a->tokens - 1) * seqs) / a->tokens;
  const int64_t q_blocks = most < a->total_q ? most : a->total_q, tiles = q_blocks * a->chunks * a->heads_kv;
  if (tiles > 0x7fffffff) return -1;
  // Few tiles: where all of them can run at once, a tile per block instead of a
  // pair (one alone takes two thirds of a pair's time), and its keys shared by a
  // cluster of 2, 4 or 8 blocks while the SMs last and every one keeps four blocks
  // of keys on average.  One B200, 32 heads over 8 of 128: 512 rows 17.9 us in
  // pairs, 14.6 in single tiles (1024 rows, 256 tiles: 25.2 against 26.8); 200 rows
  // behind 8000 keys 124 us in pairs, 92 in single tiles, 60 shared by two.
  if (tiles > sms) return (q_blocks * a->chunks + seqs) / 2 * a->heads_kv;
  a->tiles = 1;
  const int64_t blocks = a->total_k / a->n_seq / BN;
  while (a->split < 8 && tiles * a->split * 2 <= sms && blocks >= 8 * a->split) a->split *= 2;
  return tiles;
}

// The list of items, by the work of a pair's first tile: first those of at least
// 2^(levels - 1) runs of keys, then of half as many, and so on, at the end the
// rest (blocks take items as they come free, so the last ones should be short).
// Within a level: sequences in order; in each the pairs of its tiles, the tiles
// going from the last tokens to the first and through the group's heads, for
// every key head.  A block's items come in nearly rising order, so the search goes
// on from where the last one ended: 32 sequences at a time, a lane each.  (By the
// machine's long division a step of it took 2 us: 80 prompts of 84 rows, 21 heads
// over 7 of 64, 82 us.)
struct Cursor {
  int level = 0, chunk = 0;
  uint32_t before = 0;  // items before this level's chunk; items are fewer than 2^31
};

// The first level that has items when the longest sequence has `most` keys.
__host__ __device__ __forceinline__ int first_level_of(const Args& a, int most) {
  int bits = 0;
  while ((most + UN - 1) / UN >> bits) ++bits;
  return a.levels - bits;
}

__host__ __device__ __forceinline__ int bound(const int32_t* cu, int i, int lo, int hi) {
#ifdef __CUDA_ARCH__
  return min(max(__ldg(cu + i), lo), hi);
#else
  return cu[i] < lo ? lo : cu[i] > hi ? hi : cu[i];
#endif
}
// keys of sequence b
__host__ __device__ __forceinline__ int keys_of(const Args& a, int b) {
  const int k0 = bound(a.cu_k, b, 0, (int)a.total_k);
  return bound(a.cu_k, b + 1, k0, (int)a.total_k) - k0;
}

// A lane's sequence of a chunk of 32, and its items of a level.
struct Lot {
  int q0, k0, n, m, blocks;
  uint32_t above, mine;  // pairs (of a key head) of the levels before; items
};

__host__ __device__ __forceinline__ Lot lot_of(const Args& a, int level, int chunk, int lane) {
  const int b = chunk * 32 + lane;
  int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
  if (b < a.n_seq) {
    const int most_q = (int)a.total_q, most_k = (int)a.total_k;
    q0 = bound(a.cu_q, b, 0, most_q), q1 = bound(a.cu_q, b + 1, q0, most_q);
    k0 = bound(a.cu_k, b, 0, most_k), k1 = bound(a.cu_k, b + 1, k0, most_k);
  }
  const int n = q1 - q0, m = k1 - k0, blocks = (int)a.by_tokens.div((uint32_t)(n + a.tokens - 1));
  // pairs whose first tile sees at least `units` runs of keys
  auto pairs = [&](int units) -> uint32_t {
    uint32_t tiles = blocks;
    if (units > 0) {
      const int64_t end = (int64_t)(units - 1) * UN;  // its last row sees more keys than that
      if (a.causal) {
        const int64_t x = end - m + n;
        tiles = x >= n ? 0 : blocks - (x > 0 ? (int)a.by_tokens.div((uint32_t)x) : 0);
      } else if (m <= end) {
        tiles = 0;
      }
    }
    return (tiles * a.chunks + a.tiles - 1) >> (a.tiles - 1);  // by 1 or 2
  };
  const uint32_t above = level == 0 ? 0 : pairs(1 << (a.levels - level));
  const uint32_t here = pairs(level == a.levels ? 0 : 1 << (a.levels - 1 - level)) - above;
  return Lot{q0, k0, n, m, blocks, above, here * a.heads_kv};
}

// Moves the cursor to the level's chunk that holds the item; false behind the
// list's end, where at.before is the number of items.  count(level, chunk): the
// items there.
template <class Count>
__host__ __device__ __forceinline__ bool find_chunk(const Args& a, uint32_t item, Cursor& at, Count count) {
  const int chunks = (a.n_seq + 31) / 32;
  while (item < at.before) {  // numbers are taken over in no order
    if (--at.chunk < 0) at.chunk = chunks - 1, --at.level;
    at.before -= count(at.level, at.chunk);
  }
  for (;;) {
    if (at.level > a.levels) return false;
    const uint32_t all = count(at.level, at.chunk);
    if (item - at.before < all) return true;
    at.before += all;
    if (++at.chunk == chunks) at.chunk = 0, ++at.level;
  }
}

// Item x of a lane's.
__host__ __device__ __forceinline__ void place_item(const Args& a, const Lot& lot, uint32_t x, Item* out) {
  const uint32_t per_head = a.by_kv.div(x), pair = lot.above + per_head;
  out->g = (int)(x - per_head * a.heads_kv);
  out->q0 = lot.q0, out->k0 = lot.k0, out->n = lot.n, out->m = lot.m;
  out->first_block = 0;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint32_t e = pair * a.tiles + t;
    Tile& tile = out->tile[t];
    tile.head = -1, tile.heads = 0, tile.first = 0, tile.tokens = 0, tile.units = 0;
    if (t >= a.tiles || e >= (uint32_t)(lot.blocks * a.chunks)) continue;
    const int at_block = (int)a.by_chunks.div(e), chunk = (int)e - at_block * a.chunks;
    const int left = a.group - chunk * a.heads;
    tile.head = out->g * a.group + chunk * a.heads;
    tile.heads = left < a.heads ? left : a.heads;
    tile.first = (lot.blocks - 1 - at_block) * a.tokens;
    tile.tokens = lot.n - tile.first < a.tokens ? lot.n - tile.first : a.tokens;
    // one past the last key that its last token sees
    const int64_t end = a.causal ? (int64_t)lot.m - lot.n + tile.first + tile.tokens : lot.m;
    tile.units = end <= 0 ? 0 : (int)((end + UN - 1) / UN);
  }
}

// The list has `items` items and the grid has at least as many blocks.  A block
// that has got a number behind the list's end takes over others for as long as
// there are any: ask() is the number of a block that has not started and now never
// will, or -1 when none is left.  Nothing promises an order, so one of the list's
// may come behind one that is not, and is nobody else's: it is the result.
template <class Ask>
__host__ __device__ __forceinline__ int next_listed(uint32_t items, Ask ask) {
  for (;;) {
    const int block = ask();
    if (block < 0 || (uint32_t)block < items) return block;
  }
}

}  // namespace uk_prompt
