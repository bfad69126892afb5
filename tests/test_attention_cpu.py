"""Refusals of the cache and attention entry points, and the host arithmetic
they use (no GPU: arguments are checked before any CUDA work)."""
import ctypes as C
import subprocess

import pytest
import torch

from pathlib import Path

import unikern_b200.abi as abi

ROOT = Path(__file__).resolve().parents[1]


def cache(**kw):
    d = dict(k=None, v=None, k_exp=None, v_exp=None, page_stride=0, token_stride=0, head_stride=0, pages=0, page_size=16,
             heads=2, dim=64, kind=abi.UK_KV_F16)
    d.update(kw)
    return C.byref(abi.KvCacheStruct(*[d[f[0]] for f in abi.KvCacheStruct._fields_]))


def append(c, total=4, max_pages=0, n_seq=1, ts=8):
    return abi.lib().uk_cuda_kv_append_f16(None, 128, 64, None, 128, 64, total, c, None, ts, max_pages, None, None,
                                           n_seq, None)


def gather(c, total=4, max_pages=0, n_seq=1, ts=8):
    return abi.lib().uk_cuda_kv_gather_f16(c, None, ts, max_pages, None, None, n_seq, None, 128, 64, None, 128, 64, total,
                                           None)


def decode(c, heads_q=4, n_seq=1, scale=1.0, max_pages=0):
    return abi.lib().uk_cuda_attn_decode_f16(None, 256, 64, c, None, 8, max_pages, None, n_seq, heads_q, scale, None, 256,
                                             64, None, None, 0, None)


def prompt(n_seq=1, tq=4, tk=4, hq=4, hk=2, dim=64, scale=1.0):
    return abi.lib().uk_cuda_attn_prompt_f16(None, 256, 64, None, 128, 64, None, 128, 64, None, None, n_seq, tq, tk, hq,
                                             hk, dim, scale, 1, None, 256, 64, None, None)


BAD = [dict(kind=2), dict(kind=-1), dict(dim=0), dict(dim=4), dict(dim=136), dict(dim=60), dict(dim=24, kind=1),
       dict(heads=0), dict(page_size=0), dict(pages=-1), dict(heads=70000),
       dict(pages=2, page_stride=8), dict(pages=2, page_stride=4100), dict(token_stride=32, pages=1),
       dict(head_stride=60, token_stride=128), dict(kind=1, token_stride=136, head_stride=64)]


@pytest.mark.parametrize("kw", BAD)
@pytest.mark.parametrize("call", [append, gather, decode])
def test_bad_caches(call, kw):
    assert call(cache(**kw)) == 2 and abi.lib().uk_cuda_last_error()


@pytest.mark.parametrize("f", [
    lambda c: append(None), lambda c: append(c, total=-1), lambda c: append(c, n_seq=-1),
    lambda c: append(c, total=1 << 32), lambda c: append(c, max_pages=-1), lambda c: append(c, max_pages=9, n_seq=2),
    lambda c: append(c, max_pages=1 << 28), lambda c: append(c),  # rows are NULL
    lambda c: gather(None), lambda c: gather(c, total=-1), lambda c: gather(c),
    lambda c: decode(None), lambda c: decode(c, heads_q=3), lambda c: decode(c, heads_q=0),
    lambda c: decode(c, n_seq=-1), lambda c: decode(c, scale=float("inf")), lambda c: decode(c, scale=float("nan")),
    lambda c: decode(c, max_pages=1), lambda c: decode(c),
    lambda c: prompt(n_seq=-1), lambda c: prompt(tq=-1), lambda c: prompt(tk=1 << 33),
    lambda c: prompt(tk=(1 << 27) + 1), lambda c: prompt(hq=3),
    lambda c: prompt(hk=0), lambda c: prompt(dim=12), lambda c: prompt(dim=256), lambda c: prompt(scale=float("nan")),
    lambda c: prompt(),
])
def test_bad_arguments(f):
    assert f(cache(token_stride=128, head_stride=64)) == 2
    assert abi.lib().uk_cuda_last_error()


@pytest.mark.parametrize("f,said", [
    # limits of the kernels' 32-bit numbers and bounded waits
    (lambda c: append(c, n_seq=(1 << 24) + 1), "n_seq"), (lambda c: gather(c, n_seq=(1 << 24) + 1), "n_seq"),
    (lambda c: decode(c, n_seq=(1 << 24) + 1), "n_seq"), (lambda c: prompt(n_seq=(1 << 24) + 1), "n_seq"),
    (lambda c: decode(c, heads_q=65536), "heads_q"), (lambda c: prompt(hq=65536), "heads"),
    (lambda c: prompt(tq=(1 << 31) - 255), "total_q"), (lambda c: prompt(tk=(1 << 25) + 1), "total_k"),
    # finite, but not times log2 e
    (lambda c: decode(c, scale=3e38), "scale"), (lambda c: prompt(scale=-3e38), "scale"),
])
def test_limits(f, said):
    assert f(cache(token_stride=128, head_stride=64)) == 2
    assert said in abi.lib().uk_cuda_last_error().decode()


def test_nothing_to_do():
    c = cache(token_stride=128, head_stride=64)
    assert append(c, total=0) == 0 and append(c, n_seq=0) == 0 and gather(c, total=0) == 0
    assert decode(c, n_seq=0) == 0 and prompt(tq=0) == 0 and prompt(n_seq=0) == 0


def test_workspace_size():
    f = abi.lib().uk_cuda_attn_decode_workspace_size
    assert f(32, 8, 128) > 0 and f(0, 1, 64) == 0 and f(4, 0, 64) == 0 and f(4, 2, -1) == 0


def h(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def i(*v):
    return torch.tensor(v, dtype=torch.int32)


POOL = (6, 16, 2, 64)


@pytest.mark.parametrize("make", [
    lambda: abi.KvCache(h(*POOL), h(6, 16, 2, 32)),
    lambda: abi.KvCache(h(6, 16, 64), h(6, 16, 64)),
    lambda: abi.KvCache(h(*POOL).float(), h(*POOL).float()),
    lambda: abi.KvCache(h(*POOL), h(6, 2, 16, 64).transpose(1, 2)),
    lambda: abi.KvCache(h(6, 16, 64, 2).transpose(2, 3), h(6, 16, 64, 2).transpose(2, 3)),
    lambda: abi.KvCache(h(*POOL).to(torch.float8_e4m3fn), h(*POOL).to(torch.float8_e4m3fn)),
    lambda: abi.KvCache(h(*POOL), h(*POOL), torch.zeros(6, 2, 16, dtype=torch.uint8),
                        torch.zeros(6, 2, 16, dtype=torch.uint8)),
    lambda: abi.KvCache(h(*POOL).to(torch.float8_e4m3fn), h(*POOL).to(torch.float8_e4m3fn),
                        torch.zeros(6, 16, 2, dtype=torch.uint8), torch.zeros(6, 16, 2, dtype=torch.uint8)),
])
def test_cache_tensors_refused(make):
    with pytest.raises(abi.UkError) as e:
        make()
    assert e.value.code == 2


@pytest.mark.parametrize("call", [
    lambda c, t: abi.kv_append(h(3, 2, 32), h(3, 2, 32), c, t, i(0, 3), i(3)),
    lambda c, t: abi.kv_append(h(3, 2, 64), h(2, 2, 64), c, t, i(0, 3), i(3)),
    lambda c, t: abi.kv_append(h(3, 2, 64).float(), h(3, 2, 64), c, t, i(0, 3), i(3)),
    lambda c, t: abi.kv_append(h(3, 2, 64), h(3, 2, 64), c, t, i(0, 3, 4), i(3)),
    lambda c, t: abi.kv_append(h(3, 2, 64), h(3, 2, 64), c, t, i(0, 3).long(), i(3)),
    lambda c, t: abi.kv_append(h(3, 2, 64), h(3, 2, 64), c, t.long(), i(0, 3), i(3)),
    lambda c, t: abi.kv_append(h(3, 2, 64), h(3, 2, 64), c, t.repeat(2, 2)[:, ::2], i(0, 3, 3), i(3, 3)),
    lambda c, t: abi.kv_gather(c, t, i(0, 3), i(3, 3), h(3, 2, 64), h(3, 2, 64)),
    lambda c, t: abi.kv_gather(c, t, i(0, 3), i(3), h(3, 2, 64).transpose(1, 2), h(3, 2, 64)),
    lambda c, t: abi.attn_decode(h(2, 4, 64), c, t, i(3), h(1, 4, 64)),
    lambda c, t: abi.attn_decode(h(1, 4, 64), c, t, i(3), h(1, 2, 64)),
    lambda c, t: abi.attn_decode(h(1, 4, 64), c, t, i(3), h(1, 4, 64), lse=torch.zeros(1, 3)),
    lambda c, t: abi.attn_decode(h(1, 4, 64), c, t, i(3), h(1, 4, 64), lse=torch.zeros(1, 4).half()),
    lambda c, t: abi.attn_prompt(h(3, 4, 64), h(3, 2, 64), h(3, 2, 32), i(0, 3), i(0, 3), h(3, 4, 64)),
    lambda c, t: abi.attn_prompt(h(3, 4, 64), h(3, 2, 64), h(3, 2, 64), i(0, 3), i(0, 1, 3), h(3, 4, 64)),
    lambda c, t: abi.attn_prompt(h(3, 4, 64), h(3, 2, 64), h(3, 2, 64), i(0, 3), i(0, 3), h(2, 4, 64)),
    lambda c, t: abi.attn_prompt(h(3, 256), h(3, 2, 64), h(3, 2, 64), i(0, 3), i(0, 3), h(3, 4, 64)),
])
def test_tensors_refused(call):
    with pytest.raises(abi.UkError) as e:
        call(abi.KvCache(h(*POOL), h(*POOL)), i(0, 1, 2)[None])
    assert e.value.code == 2


def test_host_tensors_are_not_resident():
    c = abi.KvCache(h(*POOL), h(*POOL))
    rows = abi.lib().uk_cuda_kv_append_f16(h(3, 2, 64).data_ptr(), 128, 64, h(3, 2, 64).data_ptr(), 128, 64, 3, c.ref,
                                           i(0).data_ptr(), 1, 1, i(0, 3).data_ptr(), i(3).data_ptr(), 1, None)
    assert rows == 5


def test_page_division(tmp_path):
    """The multiply-and-shift division by the page size, against / for every
    divisor up to 600 and larger ones, over numbers up to 2^31 - 1."""
    src = tmp_path / "div.cu"
    src.write_text(r'''
#include "kv_cache.cuh"
#include <cstdio>
int main() {
  unsigned ds[700]; int n = 0;
  for (unsigned d = 1; d <= 600; ++d) ds[n++] = d;
  for (unsigned d : {1023u, 1024u, 1025u, 4096u, 65535u, 65536u, 65537u, 1u << 30, (1u << 30) + 1, 2147483646u, 2147483647u})
    ds[n++] = d;
  for (int i = 0; i < n; ++i) {
    const unsigned d = ds[i];
    const UkFastDiv f = UkFastDiv::make(d);
    unsigned x = 12345;
    for (int j = 0; j < 4000; ++j) {
      x = x * 1664525u + 1013904223u;
      const unsigned q = (x >> 1) / d;
      // a random number, and the borders of its quotient
      for (unsigned v : {x >> 1, q * d, q * d + d - 1, q * d == 0 ? 0 : q * d - 1, 2147483647u - (x & 1023)})
        if (v <= 2147483647u && f.div(v) != v / d) { std::printf("%u / %u\n", v, d); return 1; }
    }
  }
  return 0;
}
''')
    from unikern_b200 import build
    exe = tmp_path / "div"
    subprocess.run([build.nvcc(), "-std=c++17", "-I", str(ROOT / "include"), "-I", str(build.CSRC), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_prompt_items_in_any_order(tmp_path):
    """The blocks of the prompt attention, each with the numbers that it takes over
    in an arbitrary order: every row of every head is worked on once, with all the
    keys it sees, and no block gives up while numbers are left."""
    src = tmp_path / "items.cu"
    src.write_text(r'''
#include "attn_prompt_items.cuh"
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
using namespace uk_prompt;

struct Sim {  // what a warp does in find_item and drain_blocks, lane by lane
  const Args& a;
  uint32_t count(int level, int chunk) const {
    uint32_t n = 0;
    for (int lane = 0; lane < 32; ++lane) n += lot_of(a, level, chunk, lane).mine;
    return n;
  }
  bool find(uint32_t item, Cursor& at, Item* out) const {
    if (!find_chunk(a, item, at, [&](int l, int c) { return count(l, c); })) return false;
    uint32_t x = item - at.before;
    for (int lane = 0; lane < 32; ++lane) {
      const Lot lot = lot_of(a, at.level, at.chunk, lane);
      if (x < lot.mine) { place_item(a, lot, x, out); return true; }
      x -= lot.mine;
    }
    return false;
  }
};

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  for (int round = 0; round < 400; ++round) {
    const int n_seq = round % 10 == 0 ? pick(1025, 1100) : round % 3 ? pick(1, 40) : pick(1, 300);
    const int kv = pick(1, 5), group = round % 7 == 0 ? pick(100, 300) : pick(1, 9), sms = pick(1, 24);
    std::vector<int32_t> cq{pick(0, 2)}, ck{pick(0, 2)};
    for (int b = 0; b < n_seq; ++b) {
      const int n = pick(0, 3) ? pick(0, 40) : pick(0, 400);
      cq.push_back(cq.back() + n);
      ck.push_back(ck.back() + std::max(0, n + (pick(0, 2) ? 0 : pick(-30, 3000))));
    }
    Args a{};
    a.cu_q = cq.data(), a.cu_k = ck.data(), a.n_seq = n_seq, a.heads_q = kv * group, a.heads_kv = kv, a.group = group;
    a.total_q = cq.back() + pick(0, 300), a.total_k = std::max(1, ck.back() + pick(0, 300)), a.causal = pick(0, 1);
    if (a.total_q == 0) continue;
    const int64_t grid = plan_items(&a, sms);
    if (grid < 0) { std::puts("grid"); return 1; }
    const Sim sim{a};
    int most = 0;
    for (int b = 0; b < n_seq; ++b) most = std::max(most, keys_of(a, b));

    // the numbers nobody has got yet, handed out from the end of `left`
    std::vector<int> left(grid);
    for (int i = 0; i < grid; ++i) left[i] = i;
    switch (round % 4) {
      case 0: std::reverse(left.begin(), left.end()); break;  // rising
      case 1: break;                                          // falling: those behind the list's end first
      default: std::shuffle(left.begin(), left.end(), rng);
    }
    auto ask = [&] {
      if (left.empty()) return -1;
      const int x = left.back();
      left.pop_back();
      return x;
    };
    std::vector<uint8_t> seen((size_t)a.total_q * a.heads_q, 0);
    int64_t worked = 0;
    auto work = [&](const Item& it) {
      ++worked;
      if (it.tile[0].head < 0) return false;
      for (const Tile& t : it.tile) {
        if (t.head < 0) continue;
        int end = 0;
        for (int i = 0; i < BM; ++i) {
          const Row r(a, t, i);
          if (!r.on) continue;
          if (r.token >= it.n || r.head / a.group != it.g) return false;
          if (seen[(size_t)(it.q0 + r.token) * a.heads_q + r.head]++) return false;
          end = std::max(end, a.causal ? it.m - it.n + 1 + r.token : it.m);
        }
        if (t.units != (end + UN - 1) / UN) return false;
      }
      return true;
    };
    struct Block { int number; Cursor at; bool any; Item it; };
    std::vector<Block> running;
    auto start = [&] {
      Block b{ask(), {}, false, {}};
      if (b.number < 0) return;
      if (a.levels > 0) b.at.level = first_level_of(a, most);
      b.any = sim.find(b.number, b.at, &b.it);
      running.push_back(b);
    };
    for (int i = 0; i < sms; ++i) start();
    while (!running.empty()) {
      const size_t i = rng() % running.size();
      Block& b = running[i];
      if (!b.any && b.number >= 0 && a.split == 1) {
        b.number = next_listed(b.at.before, ask);
        if (b.number >= 0) {
          Cursor fresh;
          b.any = sim.find(b.number, fresh, &b.it);
        }
      }
      if (!b.any) {  // leaves; another block starts in its place
        running.erase(running.begin() + i);
        start();
        continue;
      }
      if (!work(b.it)) { std::printf("round %d: item %d\n", round, b.number); return 1; }
      b.any = false;
      if (a.split > 1) { b.number = -1; continue; }  // one tile a cluster
      b.number = ask();
      b.any = b.number >= 0 && sim.find(b.number, b.at, &b.it);
    }
    for (int t = 0; t < a.total_q; ++t)
      for (int h = 0; h < a.heads_q; ++h)
        if (seen[(size_t)t * a.heads_q + h] != (t >= cq[0] && t < cq.back())) {
          std::printf("round %d: row %d head %d\n", round, t, h);
          return 1;
        }
  }
  return 0;
}
''')
    from unikern_b200 import build
    exe = tmp_path / "items"
    subprocess.run([build.nvcc(), "-O1", "-std=c++17", "--expt-relaxed-constexpr", "-I", str(ROOT / "include"), "-I",
                    str(build.CSRC), str(src), "-o", str(exe)], check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
