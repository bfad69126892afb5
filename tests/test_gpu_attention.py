"""Attention over a paged cache (one new token per sequence) and over packed
prompts on the GPU, against the definition in 64 bits; bounds in attn_testutil."""
import ctypes
import math
import random

import pytest
import torch

from attn_testutil import Pool, assert_close, attention_f64, quantise_f64, same_bits

pytestmark = pytest.mark.gpu


def abi():
    import unikern_b200.abi as a
    assert torch.cuda.is_available()
    return a


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prefix(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def fault():
    torch.cuda.synchronize()
    return abi().lib().uk_cuda_pipeline_fault()


def randn(*shape, seed=0, mul=1.0):
    return (torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * mul).half()


# ---- one new token over a paged cache -----------------------------------------------

def check_decode(pool, q, o, lse, scale, values=None, gone=None):
    """gone: per sequence a set of positions that do not count."""
    heads_q, group = q.shape[1], q.shape[1] // pool.heads
    for b, n in enumerate(pool.lens):
        k, v = (values or pool.values)[b]
        seen = torch.ones(group, n, dtype=torch.bool, device="cuda")
        if gone:
            seen[:, sorted(gone[b])] = False
        for g in range(pool.heads):
            rows = slice(g * group, (g + 1) * group)
            ro, rl, to, tl = attention_f64(q[b, rows], k[:, g], v[:, g], scale, seen)
            assert_close(o[b, rows], ro, to, "sequence %d heads of %d: o" % (b, g))
            if lse is not None:
                assert_close(lse[b, rows], rl, tl, "sequence %d heads of %d: lse" % (b, g))


DECODE = [  # kind, layout, heads_kv, group, dim, page_size, lengths
    ("f16", "nhd", 1, 1, 8, 1, [1]),
    ("f16", "hnd", 2, 3, 24, 3, [0, 1, 2, 5, 0]),
    ("f16", "hnd", 8, 4, 128, 16, [500]),
    ("f16", "nhd", 2, 8, 64, 16, [15, 16, 17, 63, 64, 65, 127, 128, 129, 0, 1]),
    ("f16", "hnd", 1, 12, 128, 32, [1000, 31, 2049]),
    ("f16", "nhd", 2, 16, 96, 7, [333, 64]),
    ("f16", "hnd", 1, 20, 80, 256, [1500]),
    ("f16", "hnd", 1, 40, 120, 5, [77, 0, 200]),
    ("f16", "hnd", 3, 5, 104, 64, [400, 1]),
    ("e4m3", "hnd", 1, 1, 16, 1, [1, 2, 0]),
    ("e4m3", "nhd", 3, 4, 48, 5, [9, 40, 0, 333]),
    ("e4m3", "hnd", 8, 4, 128, 16, [700, 12]),
    ("e4m3", "hnd", 2, 7, 64, 32, [31, 32, 33, 95, 96, 97, 255, 256, 257, 1, 0]),
    ("e4m3", "nhd", 1, 16, 112, 24, [2000]),
    ("e4m3", "hnd", 1, 9, 80, 64, [129, 4097]),
    ("e4m3", "hnd", 1, 33, 32, 128, [300, 20]),
]


@pytest.mark.parametrize("kind,layout,heads,group,dim,page,lens", DECODE)
def test_decode(kind, layout, heads, group, dim, page, lens):
    a = abi()
    fault()
    pool = Pool(kind, layout, heads, dim, page, lens, seed=3)
    q = randn(len(lens), heads * group, dim, seed=5)
    o, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device="cuda")
    a.attn_decode(q, pool.cache, pool.table, pool.lens_t, o, lse=lse)
    assert fault() == 0
    check_decode(pool, q, o, lse, dim ** -0.5)
    # the same again: same bits; without lse; strided rows of a wider tensor
    wide = torch.full((len(lens), 3, heads * group, dim), 7.0, dtype=torch.float16, device="cuda")
    wide[:, 0] = q
    a.attn_decode(wide[:, 0], pool.cache, pool.table, pool.lens_t, wide[:, 2])
    assert same_bits(wide[:, 2], o) and (wide[:, 1] == 7).all() and same_bits(wide[:, 0], q)


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("lens", [[8191], [3000] * 9, [1] * 700, [0] * 5, [0, 0, 5000, 0, 1, 0, 640, 0, 0],
                                  [i * 13 % 700 for i in range(300)]])
def test_decode_work_split(kind, lens):
    """Lengths that the split of the work cuts in every way: within a
    sequence, between sequences, more sequences than blocks, none at all."""
    a = abi()
    pool = Pool(kind, "hnd", 2, 64, 16, lens, seed=1, table_pad=0 if max(lens) else 1)
    q = randn(len(lens), 8, 64, seed=2)
    o, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device="cuda")
    a.attn_decode(q, pool.cache, pool.table, pool.lens_t, o, lse=lse)
    check_decode(pool, q, o, lse, 64 ** -0.5)


@pytest.mark.parametrize("kind,page", [("f16", 16), ("f16", 5), ("e4m3", 32)])
@pytest.mark.parametrize("heads,group,dim", [(8, 4, 128), (2, 12, 64), (1, 1, 32), (3, 20, 112)])
def test_decode_short_tables(kind, page, heads, group, dim):
    """Few pairs and short tables: every length around the shares of a cluster,
    the same sequence beside others and alone, tables with room to spare."""
    a = abi()
    fault()
    for lens in ([0], [1], [7], [63, 0], [64, 65], [511, 512, 0], [513], [0, 0, 1000]):
        pool = Pool(kind, "hnd", heads, dim, page, lens, seed=4, table_pad=3)
        q = randn(len(lens), heads * group, dim, seed=6)
        o, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device="cuda")
        a.attn_decode(q, pool.cache, pool.table, pool.lens_t, o, lse=lse)
        check_decode(pool, q, o, lse, dim ** -0.5)
        # the same table with far more room takes the other split of the work
        wide = torch.full((len(lens), 70000 // page), -1, dtype=torch.int32, device="cuda")
        wide[:, :pool.table.shape[1]] = pool.table
        o2, lse2 = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device="cuda")
        a.attn_decode(q, pool.cache, wide, pool.lens_t, o2, lse=lse2)
        check_decode(pool, q, o2, lse2, dim ** -0.5)
    assert fault() == 0


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_decode_long(kind):
    """One long sequence, one key head: many parts joined; a strong first key
    in front of a long weak tail (weights far below the first one's)."""
    a = abi()
    n, dim = 131071, 128
    pool = Pool(kind, "nhd", 1, dim, 64, [n], seed=1)
    q = randn(1, 16, dim, seed=2)
    strong = (q[0, 0] * 2).view(1, 1, dim)  # score of head 0 about 2 |q|^2 / sqrt(dim) = 22
    first = pool.put(0, 0, 0, strong)
    k, v = pool.values[0]
    k[0:1] = first
    o, lse = torch.empty_like(q), torch.empty(1, 16, device="cuda")
    a.attn_decode(q, pool.cache, pool.table, pool.lens_t, o, lse=lse)
    check_decode(pool, q, o, lse, dim ** -0.5)


@pytest.mark.parametrize("kind,page,heads,group,dim,seqs,n", [
    ("f16", 64, 8, 4, 16, 64, 1 << 20), ("e4m3", 64, 8, 4, 16, 64, 1 << 20), ("f16", 40, 2, 12, 64, 230, 150001),
    ("e4m3", 32, 2, 20, 128, 230, 140000), ("f16", 16, 8, 1, 128, 56, 200000), ("f16", 64, 2, 4, 16, 10, 1 << 20),
    ("e4m3", 16, 1, 9, 64, 12, 1600000)])
def test_decode_sums_over_long_contexts(kind, page, heads, group, dim, seqs, n):
    """So many long sequences that a block sums whole ones up (all of them in the
    same pages), some shorter ones between them; values that do not cancel under
    weights that are nearly equal: a sum that is rounded the same way at every step
    drifts."""
    a = abi()
    fault()
    pool = Pool(kind, "hnd", heads, dim, page, [n], seed=1, fill=False)
    k = torch.zeros(n, heads, dim, device="cuda")
    k[:, :, 0] = randn(n, heads, seed=1, mul=0.1)
    k[0, :, 0] = 9.0
    k, v = pool.put(0, 0, 0, k.half()), pool.put(1, 0, 0, randn(n, heads, dim, seed=2).abs() + 0.5)
    lens = [n] * seqs
    lens[3:9] = [70000, 0, 32768, 32769, 5, 98305]
    lens[-2] = 65536
    q = torch.zeros(seqs, heads * group, dim, device="cuda").half()
    q[:, :, 0] = torch.linspace(0.01, 3, seqs, device="cuda").half()[:, None]
    o, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device="cuda")
    table = pool.table.repeat(seqs, 1)
    a.attn_decode(q, pool.cache, table, i32(lens), o, lse=lse)
    assert fault() == 0
    assert torch.isfinite(o).all() and torch.isfinite(lse[[b for b in range(seqs) if lens[b]]]).all()
    for b in [0, 1, 3, 4, 5, 6, 7, 8, seqs // 2, seqs - 3, seqs - 2, seqs - 1]:
        m = lens[b]
        for g in (0, heads - 1):
            rows = slice(g * group, (g + 1) * group)
            seen = torch.ones(group, m, dtype=torch.bool, device="cuda")
            ro, rl, to, tl = attention_f64(q[b, rows], k[:m, g], v[:m, g], dim ** -0.5, seen)
            assert_close(o[b, rows], ro, to, "sequence %d heads of %d: o" % (b, g))
            assert_close(lse[b, rows], rl, tl, "sequence %d heads of %d: lse" % (b, g))
    again = torch.full_like(q, math.nan)
    a.attn_decode(q, pool.cache, table, i32(lens), again)
    assert same_bits(again, o)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 40.0])
def test_decode_scales(scale):
    """Uniform weights, negative scales, and scores of some hundreds that rise
    along the sequence (every tile raises the maximum)."""
    a = abi()
    for kind in ("f16", "e4m3"):
        pool = Pool(kind, "hnd", 1, 64, 16, [1000, 70], seed=1)
        q = randn(2, 4, 64, seed=2)
        if scale == 40.0:
            for b, n in enumerate(pool.lens):
                up = q[b, 0].float() * torch.arange(n, device="cuda").view(n, 1, 1) / n / q[b, 0].float().norm()
                pool.values[b] = (pool.put(0, b, 0, up.half()), pool.values[b][1])
        o, lse = torch.empty_like(q), torch.empty(2, 4, device="cuda")
        a.attn_decode(q, pool.cache, pool.table, pool.lens_t, o, scale=scale, lse=lse)
        check_decode(pool, q, o, lse, scale)


def both_splits(pool):
    """The block table as it is, and with far more room: two splits of the work."""
    wide = torch.full((pool.table.shape[0], 70000 // pool.page_size), -1, dtype=torch.int32, device="cuda")
    wide[:, :pool.table.shape[1]] = pool.table
    return pool.table, wide


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("group,dim", [(4, 128), (4, 64), (12, 128), (12, 48)])
def test_decode_values_of_all_magnitudes(kind, group, dim):
    """Value rows from 2^-12 to 2^8 times normal ones in one sequence, each with
    a scale of its own in the 8-bit cache: the small rows' share is as exact."""
    a = abi()
    lens = [700, 33, 2500]
    pool = Pool(kind, "hnd", 2, dim, 16, lens, seed=3)
    g = torch.Generator("cuda").manual_seed(4)
    for b, n in enumerate(lens):
        x = torch.randn(n, 2, dim, device="cuda", generator=g)
        # columns that large rows leave to the small ones
        x[:, :, dim // 2:] *= 2.0 ** -10
        e = torch.randint(-12, 9, (n, 2, 1), device="cuda", generator=g)
        pool.values[b] = (pool.values[b][0], pool.put(1, b, 0, (x * torch.exp2(e.float())).half()))
    q = randn(len(lens), 2 * group, dim, seed=5)
    for table in both_splits(pool):
        o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        a.attn_decode(q, pool.cache, table, pool.lens_t, o, lse=lse)
        check_decode(pool, q, o, lse, dim ** -0.5)


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("n", [700, 16385])
def test_decode_one_large_value_in_front_of_a_tail(kind, n):
    """A first row of large values and weight in a few columns, zero in the
    others, in front of a tail of small values whose weights lie 14.5 bits lower
    and still make up much of the sum."""
    a = abi()
    pool = Pool(kind, "hnd", 1, 64, 16, [n], seed=1, fill=False)
    k, v = torch.zeros(n, 1, 64, device="cuda"), randn(n, 1, 64, seed=2).float().abs() * 2.0 ** -8
    k[0, 0, 0] = 14.5 * math.log(2) * 8  # times q = 1 and the scale 1 / 8
    v[0] = 0
    v[0, 0, :8] = 448 * 2.0 ** 3
    pool.values[0] = (pool.put(0, 0, 0, k.half()), pool.put(1, 0, 0, v.half()))
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.float16)
    q[..., 0] = 1
    for table in both_splits(pool):
        o, lse = torch.empty_like(q), torch.empty(1, 4, device="cuda")
        a.attn_decode(q, pool.cache, table, pool.lens_t, o, lse=lse)
        check_decode(pool, q, o, lse, 0.125)


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_decode_infinities_and_nan(kind):
    """Held NaN and infinities reach exactly the heads and columns they should;
    a key of the type's lowest value takes no weight."""
    a = abi()
    pool = Pool(kind, "hnd", 2, 32, 16, [40, 40, 40], seed=1)
    q = randn(3, 4, 32, seed=2).abs() + 0.1
    low = torch.full((1, 2, 32), -65504.0, dtype=torch.float16, device="cuda")
    pool.values[0] = (pool.values[0][0].clone(), pool.values[0][1])
    pool.values[0][0][7:8] = pool.put(0, 0, 7, low)
    v = pool.values[1][1].half()
    v[20, 1, 3], v[30, 1, 5] = math.inf if kind == "f16" else math.nan, math.nan
    pool.values[1] = (pool.values[1][0], pool.put(1, 1, 0, v))
    k = pool.values[2][0].half()
    k[11, 0, 2] = math.nan
    pool.values[2] = (pool.put(0, 2, 0, k), pool.values[2][1])
    o, lse = torch.empty_like(q), torch.empty(3, 4, device="cuda")
    a.attn_decode(q, pool.cache, pool.table, pool.lens_t, o, lse=lse)
    assert torch.isfinite(o[0]).all()
    assert torch.isfinite(o[1, :2]).all() and not torch.isfinite(o[1, 2:, 3]).any() and torch.isnan(o[1, 2:, 5]).all()
    rest = [c for c in range(32) if c not in (3, 5)]
    assert torch.isfinite(o[1][:, rest]).all()
    assert torch.isnan(o[2, :2]).all() and torch.isfinite(o[2, 2:]).all()
    pool.lens = [40]
    check_decode(pool, q, o, lse, 32 ** -0.5)


def test_exponents_of_the_callers_own():
    """Exponent bytes that the append does not write: values are rounded to binary16
    by the gather and in the value product, keys enter the scores as they are."""
    a = abi()
    fault()
    heads, dim, n = 2, 64, 700
    pool = Pool("e4m3", "hnd", heads, dim, 16, [n], seed=1)
    g = torch.Generator("cuda").manual_seed(5)
    page, off = pool.where(0, 0, n)
    held = []
    for which in range(2):
        e = torch.randint(-24, 16, (n, heads), device="cuda", generator=g)
        if which == 0:
            e = e.clamp(max=-3)  # scores of ordinary size
        x = torch.randn(n, heads, dim, device="cuda", generator=g)
        x = torch.where(e[..., None] > 8, x.clamp(-1.75, 1.75), x * 16)
        code = x.to(torch.float8_e4m3fn)
        (pool.k, pool.v)[which].view(torch.uint8)[page, off] = code.view(torch.uint8)
        pool.exps[which].transpose(1, 2)[page, off] = (e + 127).to(torch.uint8)
        held.append(code.double() * torch.exp2(e.double())[..., None])
    rounded = [h.half() for h in held]  # exact in fp32 on the way: four significant bits
    out = [torch.empty(n, heads, dim, dtype=torch.float16, device="cuda") for _ in "kv"]
    a.kv_gather(pool.cache, pool.table, i32([0, n]), pool.lens_t, *out)
    assert same_bits(out[0], rounded[0]) and same_bits(out[1], rounded[1])
    assert torch.isfinite(rounded[1]).all()
    pool.values[0] = (held[0], rounded[1].double())
    q = randn(1, heads * 4, dim, seed=2)
    for table in both_splits(pool):
        o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        a.attn_decode(q, pool.cache, table, pool.lens_t, o, lse=lse)
        check_decode(pool, q, o, lse, dim ** -0.5)
    assert fault() == 0


def test_decode_absent_pages():
    a = abi()
    fault()
    for kind in ("f16", "e4m3"):
        pool = Pool(kind, "hnd", 2, 64, 8, [50, 50, 50, 50], seed=1)
        table = pool.table.clone()
        table[0, 2] = -1
        table[1, 6] = pool.pages
        table[2, :] = 2147483647
        gone = [set(range(16, 24)), {48, 49}, set(range(50)), set()]
        q = randn(4, 4, 64, seed=2)
        o, lse = torch.empty_like(q), torch.empty(4, 4, device="cuda")
        lens = pool.lens_t.clone()
        a.attn_decode(q, pool.cache, table, lens, o, lse=lse)
        assert fault() == 64
        check_decode(pool, q, o, lse, 0.125, gone=gone)
        # lengths behind the table stop at it (the pad entries are bad ids), negative ones are empty
        lens[0], lens[3] = 2147483647, -4
        a.attn_decode(q, pool.cache, pool.table, lens, o, lse=lse)
        assert fault() == 64
        assert (o[3] == 0).all() and (lse[3] == -math.inf).all()
        far = pool.table.shape[1] * 8
        assert far > 50  # positions 50 .. 55 are held by nobody: all bits set, NaN
        full = Pool(kind, "hnd", 2, 64, 8, [56], seed=1, table_pad=0)
        ln = i32([2147483647])
        qq = q[:1].contiguous()
        o1, l1 = torch.empty_like(qq), torch.empty(1, 4, device="cuda")
        a.attn_decode(qq, full.cache, full.table, ln, o1, lse=l1)
        assert fault() == 64
        check_decode(full, qq, o1, l1, 0.125)


@pytest.mark.parametrize("kind,page", [("f16", 16), ("f16", 7), ("e4m3", 16)])
def test_decode_offsets_past_32_bits(kind, page):
    a = abi()
    fault()
    heads, dim = 2, 64
    es, dt = (2, torch.float16) if kind == "f16" else (1, torch.float8_e4m3fn)
    stride = (1 << 31) // es + 64  # elements: five pages span more than 8 GB
    k, v = (torch.empty((4 * stride + page * heads * dim) * es, dtype=torch.uint8, device="cuda").view(dt)
            .as_strided((5, page, heads, dim), (stride, heads * dim, dim, 1)) for _ in "kv")
    e = [torch.empty(5, heads, page, dtype=torch.uint8, device="cuda") if kind == "e4m3" else None for _ in "kv"]
    n = 3 * page - 2
    x = [randn(n, heads, dim, seed=i) for i in range(2)]
    table = i32([[4, 0, 3]])
    cache = a.KvCache(k, v, *e)
    a.kv_append(x[0], x[1], cache, table, i32([0, n]), i32([n]))
    held = [t.double() if kind == "f16" else quantise_f64(t)[0] for t in x]
    q = randn(1, 6, dim, seed=7)
    for room in (3, 9000):  # both splits of the work
        wide = torch.full((1, room), -1, dtype=torch.int32, device="cuda")
        wide[:, :3] = table
        o = torch.empty_like(q)
        a.attn_decode(q, cache, wide, i32([n]), o)
        seen = torch.ones(3, n, dtype=torch.bool, device="cuda")
        for g in range(heads):
            ro, _, to, _ = attention_f64(q[0, 3 * g:3 * g + 3], held[0][:, g], held[1][:, g], dim ** -0.5, seen)
            assert_close(o[0, 3 * g:3 * g + 3], ro, to, "o")
    assert fault() == 0
    # a pool whose rows 32 bits of its strides' common unit do not reach is refused
    far = a.KvCacheStruct(*[getattr(cache.struct, f[0]) for f in a.KvCacheStruct._fields_])
    far.pages, far.page_stride, far.token_stride = 1 << 30, 4096 + 8 * 16 // es, heads * dim
    ws = a.attn_decode_workspace(cache, 6)
    rc = a.lib().uk_cuda_attn_decode_f16(q.data_ptr(), q.stride(0), q.stride(1), ctypes.byref(far), table.data_ptr(), 3,
                                         3, i32([n]).data_ptr(), 1, 6, 0.125, o.data_ptr(), o.stride(0), o.stride(1),
                                         None, ws.data_ptr(), ws.numel(), None)
    assert rc == 2


@pytest.mark.parametrize("kind,page,taken", [("f16", 16, True), ("f16", 48, True), ("f16", 8, False),
                                             ("e4m3", 16, False)])
def test_decode_pools_of_small_units(kind, page, taken):
    """A pool of more than 2^32 of the units that its strides have in common: the
    form that finds groups of 16 positions by 64-bit offsets takes it.  (Only the
    pages that the table names exist.)"""
    a = abi()
    dim, heads, n = 24 if kind == "f16" else 48, 3, 100
    pool = Pool(kind, "hnd", heads, dim, page, [n], seed=1)
    q = randn(1, heads * 2, dim, seed=2)
    o, lse = torch.empty_like(q), torch.empty(1, heads * 2, device="cuda")
    far = a.KvCacheStruct(*[getattr(pool.cache.struct, f[0]) for f in a.KvCacheStruct._fields_])
    far.pages = (1 << 36) // (far.page_stride * (2 if kind == "f16" else 1)) + 2
    ws = a.attn_decode_workspace(pool.cache, heads * 2)
    t = pool.table
    rc = a.lib().uk_cuda_attn_decode_f16(q.data_ptr(), q.stride(0), q.stride(1), ctypes.byref(far), t.data_ptr(),
                                         t.stride(0), t.shape[1], pool.lens_t.data_ptr(), 1, heads * 2, dim ** -0.5,
                                         o.data_ptr(), o.stride(0), o.stride(1), lse.data_ptr(), ws.data_ptr(),
                                         ws.numel(), None)
    assert rc == (0 if taken else 2)
    if taken:
        check_decode(pool, q, o, lse, dim ** -0.5)
    # strides whose extent does not even fit 64 bits
    far.page_stride = 1 << 60
    rc = a.lib().uk_cuda_attn_decode_f16(q.data_ptr(), q.stride(0), q.stride(1), ctypes.byref(far), t.data_ptr(),
                                         t.stride(0), t.shape[1], pool.lens_t.data_ptr(), 1, heads * 2, dim ** -0.5,
                                         o.data_ptr(), o.stride(0), o.stride(1), lse.data_ptr(), ws.data_ptr(),
                                         ws.numel(), None)
    assert rc == 2


# ---- packed prompts -------------------------------------------------------------------

def check_prompt(q, k, v, cu_q, cu_k, o, lse, scale, causal):
    group = q.shape[1] // k.shape[1]
    for b in range(len(cu_q) - 1):
        n, m = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if n == 0:
            continue
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
        seen = (j <= i + m - n) if causal else (j >= 0).expand(n, m)
        qs, ks = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        for h in range(q.shape[1]):
            ro, rl, to, tl = attention_f64(q[qs, h], k[ks, h // group], v[ks, h // group], scale, seen)
            assert_close(o[qs, h], ro, to, "sequence %d head %d: o" % (b, h))
            assert_close(lse[qs, h], rl, tl, "sequence %d head %d: lse" % (b, h))


PROMPT = [  # heads_kv, group, dim, query lengths, key lengths (None: the same)
    (1, 1, 8, [1], None),
    (1, 1, 128, [128], None),
    (2, 2, 64, [1, 2, 0, 3, 127, 128, 129], None),
    (1, 3, 128, [255, 256, 257], None),
    (2, 4, 128, [77], None),
    (1, 5, 80, [300, 5], None),
    (3, 1, 72, [64, 200], None),
    (1, 2, 128, [1, 1, 5, 130, 128], [1, 500, 5, 1000, 129]),
    (1, 2, 64, [10, 200, 130, 7, 3], [4, 100, 0, 7, 260]),
    (2, 3, 24, [40, 0, 17, 140], [0, 30, 400, 139]),
    (1, 8, 96, [513], [700]),
    (1, 1, 128, [1] * 40, [i * 7 for i in range(40)]),
    (2, 20, 64, [14, 3, 200], [400, 3, 260]),
    (1, 128, 32, [1, 2, 65], [300, 2, 65]),
    (1, 130, 16, [3, 70], [3, 200]),  # more query heads of a key head than a tile has rows
    (1, 65, 40, [2, 130], None),
    (2, 33, 72, [1, 129, 64], [700, 129, 64]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim,nq,nk", PROMPT)
def test_prompt(heads, group, dim, nq, nk, causal):
    a = abi()
    fault()
    nk = nq if nk is None else nk
    # NaN rows before the first, behind the last and between nothing: they belong to nobody
    lead, tail = 5, 133
    cu_q, cu_k = [lead + c for c in prefix(nq)], [lead + c for c in prefix(nk)]
    tq, tk = cu_q[-1] + tail, cu_k[-1] + tail
    q = randn(tq, heads * group, dim, seed=1)
    kv = randn(tk, 2 * heads, dim, seed=2)  # keys beside values: strided heads
    for x, cu in ((q, cu_q), (kv, cu_k)):
        x[:lead], x[cu[-1]:] = math.nan, math.nan
    k, v = kv[:, :heads], kv[:, heads:]
    o = torch.full((tq, heads * group, 2, dim), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((tq, heads * group), 7.0, device="cuda")
    a.attn_prompt(q, k, v, i32(cu_q), i32(cu_k), o[:, :, 0], causal=causal, lse=lse)
    assert fault() == 0
    assert (o[:, :, 1] == 7).all()
    for x in (o, lse):
        assert (x[:lead] == 7).all() and (x[cu_q[-1]:] == 7).all()
    check_prompt(q, k, v, cu_q, cu_k, o[:, :, 0], lse, dim ** -0.5, causal)
    again = torch.empty_like(q)
    a.attn_prompt(q, k, v, i32(cu_q), i32(cu_k), again, causal=causal)
    rows = slice(cu_q[0], cu_q[-1])
    assert same_bits(again[rows], o[rows, :, 0])


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 30.0])
def test_prompt_scales(scale):
    a = abi()
    n, dim = 400, 64
    q, k, v = (randn(n, 2, dim, seed=s) for s in range(3))
    if scale == 30.0:  # scores that rise along the keys: the maximum moves in every tile
        up = q[-1].float() / q[-1].float().norm(dim=-1, keepdim=True)
        k = (up[None] * torch.arange(n, device="cuda")[:, None, None] / n).half()
    o, lse = torch.empty_like(q), torch.empty(n, 2, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, n]), o, scale=scale, lse=lse)
    check_prompt(q, k, v, [0, n], [0, n], o, lse, scale, True)


@pytest.mark.parametrize("equal", [True, False])
def test_prompt_row_by_row_over_a_long_context(equal):
    """A negative scale takes the rows one by one: sums of 2^20 terms, of equal
    ones behind a first key of its own weight and of random ones."""
    a = abi()
    n, m, dim = 6, 1 << 20, 8
    q, k, v = randn(n, 1, dim, seed=1), randn(m, 1, dim, seed=2), randn(m, 1, dim, seed=3)
    if equal:
        q[:, 0, 0] = torch.linspace(-4, 1, n, device="cuda").half()
        k[0], k[1:], v = 1.0, 0.0, v.abs() + 1
    o, lse = torch.empty_like(q), torch.empty(n, 1, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, m]), o, scale=-0.3, lse=lse)
    check_prompt(q, k, v, [0, n], [0, m], o, lse, -0.3, True)


def test_prompt_weak_tail():
    """A strong first key in front of many weak ones, whose weights together
    still count: they must not vanish in a narrow type."""
    a = abi()
    n, dim = 4096, 128
    q, k, v = (randn(n, 1, dim, seed=s, mul=m) for s, m in ((1, 1.0), (2, 0.05), (3, 1.0)))
    q[:, 0] = q[0, 0]
    k[0, 0] = q[0, 0] * (13.0 * math.sqrt(dim) / float(q[0, 0].float().square().sum()))  # score 13 = ln 442413
    v[1:] += 2.0
    o, lse = torch.empty_like(q), torch.empty(n, 1, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, n]), o, lse=lse)
    check_prompt(q, k, v, [0, n], [0, n], o, lse, dim ** -0.5, True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,heads,m", [
    (9600, 4, 1 << 18),  # pairs of tiles
    (9600, 1, 1 << 18),  # a tile per block
    (100, 1, 1 << 20),   # a tile's keys shared by a cluster
])
def test_prompt_sums_over_long_contexts(n, heads, m, dim):
    """Values that do not cancel under weights that are nearly equal: a sum that
    is rounded the same way at every step drifts."""
    a = abi()
    fault()
    q, k = torch.zeros(n, heads, dim, device="cuda").half(), torch.zeros(m, heads, dim, device="cuda").half()
    q[:, :, 0] = torch.linspace(0.01, 3, n, device="cuda").half()[:, None]
    k[:, :, 0] = randn(m, heads, seed=1, mul=0.1)
    k[0, :, 0] = 9.0  # the reference is this key's score: the others' weights are no powers of two
    v = randn(m, heads, dim, seed=2).abs() + 0.5
    o, lse = torch.full_like(q, math.nan), torch.full((n, heads), math.nan, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, m]), o, lse=lse)
    assert fault() == 0
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    for r in (0, n // 2, n - 40):
        rows, end = slice(r, r + 40), m - n + r + 40
        for h in (0, heads - 1):
            check_prompt(q[rows, h:h + 1], k[:end, h:h + 1], v[:end, h:h + 1], [0, 40], [0, end], o[rows, h:h + 1],
                         lse[rows, h:h + 1], dim ** -0.5, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim", [(8, 4, 128), (8, 4, 64), (6, 1, 96), (12, 3, 40)])
def test_prompt_long_contexts_among_short_ones(heads, group, dim, causal):
    """Tiles whose keys are taken in several parts, in one, and around the border
    between them, in one list."""
    a = abi()
    fault()
    nq = [300, 700, 40, 130, 0, 1200, 257]
    nk = [300, 33000, 70000, 32768, 50, 1200, 32769]
    cu_q, cu_k = [3 + c for c in prefix(nq)], [5 + c for c in prefix(nk)]
    q = randn(cu_q[-1] + 7, heads * group, dim, seed=1)
    kv = randn(cu_k[-1] + 130, 2 * heads, dim, seed=2)
    kv[cu_k[-1]:] = math.nan
    k, v = kv[:, :heads], kv[:, heads:]
    o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    a.attn_prompt(q, k, v, i32(cu_q), i32(cu_k), o, causal=causal, lse=lse)
    assert fault() == 0
    for x in (o, lse):
        assert (x[:3] == 7).all() and (x[cu_q[-1]:] == 7).all()
    for b, (n, m) in enumerate(zip(nq, nk)):
        for h in (0, heads * group - 1):
            for r in range(0, n, max(1, n - 60)):  # the first rows and the last ones
                rows = slice(cu_q[b] + r, cu_q[b] + min(n, r + 60))
                cnt = rows.stop - rows.start
                end = m - n + r + cnt if causal else m
                ks = slice(cu_k[b], cu_k[b] + end)
                check_prompt(q[rows, h:h + 1], k[ks, h // group:h // group + 1], v[ks, h // group:h // group + 1],
                             [0, cnt], [0, end], o[rows, h:h + 1], lse[rows, h:h + 1], dim ** -0.5, causal)
    again = torch.full_like(q, 7.0)
    a.attn_prompt(q, k, v, i32(cu_q), i32(cu_k), again, causal=causal)
    assert same_bits(again, o)


@pytest.mark.parametrize("heads,group,dim,n", [(8, 4, 128, 700), (8, 4, 64, 700), (1, 2, 128, 40)])
def test_prompt_long_contexts_with_infinities_and_nan(heads, group, dim, n):
    """In the first part, in the middle and behind the mask of all rows but the last."""
    a = abi()
    fault()
    m = 70000
    q, k, v = randn(n, heads * group, dim, seed=1), randn(m, heads, dim, seed=2), randn(m, heads, dim, seed=3)
    v[3, 0, 1], v[40000, 0, 2], v[40001, 0, 3], v[m - 1, 0, 4] = math.inf, -math.inf, math.nan, math.nan
    k[:, 0, :], q[:, :group] = k[:, 0, :].abs(), -q[:, :group].abs()
    k[50000, 0, 0] = math.inf  # a score of -inf: no weight
    o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, m]), o, lse=lse)
    assert fault() == 0
    x = o[:, :group]
    assert (x[..., 1] == math.inf).all() and (x[..., 2] == -math.inf).all() and torch.isnan(x[..., 3]).all()
    assert torch.isfinite(x[:-1, :, 4]).all() and torch.isnan(x[-1, :, 4]).all()
    assert torch.isfinite(lse).all() and torch.isfinite(x[..., 5:]).all() and torch.isfinite(o[:, group:]).all()
    cols = [0] + list(range(4, dim))
    sane = v.clone()
    sane[[3, 40000, 40001], 0, 1:4] = 0.0
    for r in (0, n - 30):
        rows, end = slice(r, r + 29), m - n + r + 29
        for h in (0, heads * group - 1):
            g = h // group
            qq, kk = q[rows, h].double(), k[:end, g].double()
            kk[50000] = torch.where(torch.isinf(kk[50000]), torch.full_like(kk[50000], 1e6), kk[50000])
            seen = torch.arange(end, device="cuda")[None] <= torch.arange(29, device="cuda")[:, None] + end - 29
            ro, rl, to, _ = attention_f64(qq, kk, sane[:end, g], dim ** -0.5, seen)
            kk[50000] = 0  # takes no part in the scores' bound
            _, _, to, tl = attention_f64(qq, kk, sane[:end, g], dim ** -0.5, seen)
            assert_close(o[rows, h][:, cols], ro[:, cols], to[:, cols], "rows from %d, head %d: o" % (r, h))
            assert_close(lse[rows, h], rl, tl, "rows from %d, head %d: lse" % (r, h))


def test_prompt_rows_do_not_see_behind_their_mask():
    """Infinities, NaN and the lowest value at later keys reach no earlier row;
    at keys that are seen they do."""
    a = abi()
    n, dim = 300, 64
    for where in ("k", "v"):
        for value in (math.nan, math.inf, -math.inf, -65504.0):
            q, k, v = (randn(n, 2, dim, seed=s) for s in range(3))
            x = k if where == "k" else v
            x[150, 0], x[299, 1] = value, value
            o, lse = torch.empty_like(q), torch.empty(n, 2, device="cuda")
            a.attn_prompt(q, k, v, i32([0, n]), i32([0, n]), o, lse=lse)
            check_prompt(q[:150], k[:150], v[:150], [0, 150], [0, 150], o[:150], lse[:150], dim ** -0.5, True)
            check_prompt(q[:299, 1:], k[:299, 1:], v[:299, 1:], [0, 299], [0, 299], o[:299, 1:], lse[:299, 1:],
                         dim ** -0.5, True)
            if where == "v" and value != -65504.0:
                bad = torch.isnan(o[150:, 0]) if math.isnan(value) else torch.isinf(o[150:, 0])
                assert bad.all()
                assert torch.isfinite(lse).all()


@pytest.mark.parametrize("heads,group,dim,n", [(2, 4, 128, 700), (3, 1, 72, 1500), (1, 2, 64, 3000)])
def test_prompt_nan_from_a_key_on(heads, group, dim, n):
    """All values NaN from a key on, some columns from another one on, infinities
    among them: rows before are exact, columns that only hidden keys spoil too."""
    a = abi()
    fault()
    q, k, v = randn(n, heads * group, dim, seed=1), randn(n, heads, dim, seed=2), randn(n, heads, dim, seed=3)
    at = {0: n // 2 + 3, 7: n // 2 - 50, 11: n - 1}  # the first key that spoils a column
    rest = n // 2 + 20
    for c, j in at.items():
        v[j:, 0, c] = math.nan
    v[n // 2 - 5, 0, 2] = math.inf
    v[rest:, 0, [c for c in range(dim) if c not in (2, *at)]] = math.nan
    o, lse = torch.empty_like(q), torch.empty(n, heads * group, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, n]), o, lse=lse)
    assert fault() == 0
    first = torch.tensor([at.get(c, n if c == 2 else rest) for c in range(dim)], device="cuda")
    gone = torch.arange(n, device="cuda")[:, None] >= first
    assert torch.equal(torch.isnan(o[:, :group]), gone[:, None].expand(n, group, dim))
    assert torch.equal(o[:, :group, 2] == math.inf, (torch.arange(n, device="cuda") >= n // 2 - 5)[:, None].expand(n, group))
    assert torch.isfinite(lse).all() and torch.isfinite(o[:, group:]).all()
    # each column against the definition over keys that hold nothing spoilt but what it sees
    sane = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    seen = torch.arange(n, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None]
    for h in (0, heads * group - 1):
        ro, rl, to, tl = attention_f64(q[:, h], k[:, h // group], sane[:, h // group], dim ** -0.5, seen)
        got = o[:, h].double()
        fine = torch.isfinite(got)
        assert ((got - ro).abs() <= to)[fine].all()
        assert_close(lse[:, h], rl, tl, "head %d: lse" % h)


def test_prompt_of_nan_is_not_computed_again():
    """Where every value is NaN no row is looked at key by key (a thousand times the
    time of a prompt of numbers; 5 times it without)."""
    a = abi()
    n = 8192
    q, k, v = (randn(n, h, 128, seed=h) for h in (8, 2, 2))
    o, cu = torch.empty_like(q), i32([0, n])

    def took():
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.attn_prompt(q, k, v, cu, cu, o)
        torch.cuda.synchronize()
        start.record()
        a.attn_prompt(q, k, v, cu, cu, o)
        end.record()
        torch.cuda.synchronize()
        return start.elapsed_time(end)

    clean = took()
    v.fill_(math.nan)
    assert took() < 60 * clean
    assert torch.isnan(o).all()


def test_prompt_rows_computed_again_behind_a_long_context():
    """A NaN that only the last query may see, behind so many keys that the 127
    rows before it in its tile take seconds to be computed again: the other warps
    wait for them, and go on."""
    a = abi()
    fault()
    n, m, heads, dim = 9600, 320000, 16, 8
    q, k, v = randn(n, heads, dim, seed=1), randn(m, heads, dim, seed=2), randn(m, heads, dim, seed=3)
    v[m - 1, 3, 5] = math.nan
    o, lse = torch.full_like(q, 7.0), torch.full((n, heads), 7.0, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, m]), o, lse=lse)
    assert fault() == 0
    assert torch.isnan(o[-1, 3, 5]) and torch.isnan(o).sum() == 1
    rows = slice(n - 128, n - 1)
    check_prompt(q[rows, 3:4], k[:m - 1, 3:4], v[:m - 1, 3:4], [0, 127], [0, m - 1], o[rows, 3:4], lse[rows, 3:4],
                 dim ** -0.5, True)


def test_prompt_bounds_of_the_length_arrays():
    """Row bounds outside the tensors are clamped, never read."""
    a = abi()
    q, k, v = (randn(100, 2, 32, seed=s) for s in range(3))
    o, lse = torch.full_like(q, 7.0), torch.full((100, 2), 7.0, device="cuda")
    a.attn_prompt(q, k, v, i32([-5, 1000]), i32([-7, 2000]), o, causal=False, lse=lse)
    check_prompt(q, k, v, [0, 100], [0, 100], o, lse, 32 ** -0.5, False)
    a.attn_prompt(q, k, v, i32([0, 100]), i32([60, 20]), o, lse=lse)
    assert (o == 0).all() and (lse == -math.inf).all()
    assert fault() == 0


def test_prompt_many_sequences_and_heads():
    a = abi()
    nq = [i % 5 for i in range(400)]
    nk = [n + i % 3 for i, n in enumerate(nq)]
    cu_q, cu_k = prefix(nq), prefix(nk)
    q, k, v = randn(cu_q[-1], 6, 16, seed=1), randn(cu_k[-1], 3, 16, seed=2), randn(cu_k[-1], 3, 16, seed=3)
    o, lse = torch.empty_like(q), torch.empty(cu_q[-1], 6, device="cuda")
    a.attn_prompt(q, k, v, i32(cu_q), i32(cu_k), o, lse=lse)
    check_prompt(q, k, v, cu_q, cu_k, o, lse, 0.25, True)


@pytest.mark.parametrize("seqs,heads,group,causal", [(1000, 2, 4, True), (1024, 8, 4, True), (1025, 8, 1, True),
                                                     (33, 16, 3, True), (700, 3, 7, False)])
def test_prompt_lists_of_mixed_lengths(seqs, heads, group, causal):
    """Hundreds of short prompts among long contexts and empty ones: every tile
    is found once, whatever the order its block starts in."""
    a = abi()
    fault()
    rng = random.Random(seqs)
    nq = [rng.choice([0, 1, 7, 31, 32, 33, 64, 90]) for _ in range(seqs)]
    nk = [n + rng.choice([0, 0, 0, 63, 200, 1100]) for n in nq]
    nq[-1] = nk[-1] = 129
    cu_q, cu_k = prefix(nq), prefix(nk)
    q, k, v = (randn(cu_q[-1], heads * group, 32, seed=1), randn(cu_k[-1], heads, 32, seed=2),
               randn(cu_k[-1], heads, 32, seed=3))
    o, lse = torch.full_like(q, math.nan), torch.full((cu_q[-1], heads * group), math.nan, device="cuda")
    a.attn_prompt(q, k, v, i32(cu_q), i32(cu_k), o, causal=causal, lse=lse)
    assert fault() == 0
    assert not o.isnan().any() and not lse.isnan().any()  # every row was written
    for b in rng.sample(range(seqs), 12) + [seqs - 1]:
        x, y = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        check_prompt(q[x], k[y], v[y], [0, nq[b]], [0, nk[b]], o[x], lse[x], 32 ** -0.5, causal)


def test_prompt_long():
    a = abi()
    n, dim = 3001, 128
    q, k, v = randn(n, 4, dim, seed=1), randn(n, 2, dim, seed=2), randn(n, 2, dim, seed=3)
    o, lse = torch.empty_like(q), torch.empty(n, 4, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, n]), o, lse=lse)
    check_prompt(q, k, v, [0, n], [0, n], o, lse, dim ** -0.5, True)


@pytest.mark.parametrize("n,heads,group,dim,m", [(700, 8, 4, 128, 900), (300, 2, 3, 64, 700), (40, 1, 4, 64, 5000),
                                                 (700, 8, 4, 64, 40000), (20, 2, 4, 64, 600)])
def test_prompt_averages_of_the_largest_values(n, heads, group, dim, m):
    """Columns that hold 65504 at every key, seen with weights that round up: the
    average does not become an infinity.  (Scores 3 bits above the reference.)"""
    a = abi()
    fault()
    q, k = torch.zeros(n, heads * group, dim, device="cuda").half(), torch.zeros(m, heads, dim, device="cuda").half()
    q[:, :, 0] = 1.0 + randn(n, heads * group, seed=1, mul=0.1).abs()
    k[128:, :, 0] = 3.0 * math.log(2) * math.sqrt(dim)
    v = randn(m, heads, dim, seed=2)
    v[:, :, 0], v[:, :, 1], v[:, :, 8] = 65504.0, -65504.0, 65504.0
    for scale in (dim ** -0.5, -dim ** -0.5):
        o, lse = torch.empty_like(q), torch.empty(n, heads * group, device="cuda")
        a.attn_prompt(q, k, v, i32([0, n]), i32([0, m]), o, scale=scale, lse=lse)
        assert torch.isfinite(o).all()
        rows = slice(n - 20, n)
        check_prompt(q[rows], k, v, [0, 20], [0, m], o[rows], lse[rows], scale, True)


@pytest.mark.parametrize("n,page", [(900, 16), (900, 5), (20000, 16)])
def test_decode_averages_of_the_largest_values(n, page):
    """The same over a cache, whole sequences and ones cut in parts."""
    a = abi()
    heads, group, dim, seqs = 2, 16, 64, 40
    pool = Pool("f16", "hnd", heads, dim, page, [n], seed=1, fill=False)
    k = torch.zeros(n, heads, dim, device="cuda")
    k[256:, :, 0] = 3.0 * math.log(2) * math.sqrt(dim)
    v = randn(n, heads, dim, seed=2)
    v[:, :, 0], v[:, :, 1], v[:, :, 8] = 65504.0, -65504.0, 65504.0
    k, v = pool.put(0, 0, 0, k.half()), pool.put(1, 0, 0, v)
    for count in (1, seqs):
        q = torch.zeros(count, heads * group, dim, device="cuda").half()
        q[:, :, 0] = 1.0 + randn(count, heads * group, seed=1, mul=0.1).abs()
        for table in both_splits(pool):
            o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
            a.attn_decode(q, pool.cache, table.repeat(count, 1), i32([n] * count), o, lse=lse)
            assert torch.isfinite(o).all()
            seen = torch.ones(group, n, dtype=torch.bool, device="cuda")
            for b in (0, count - 1):
                for g in range(heads):
                    rows = slice(g * group, (g + 1) * group)
                    ro, rl, to, tl = attention_f64(q[b, rows], k[:, g], v[:, g], dim ** -0.5, seen)
                    assert_close(o[b, rows], ro, to, "sequence %d heads of %d: o" % (b, g))
                    assert_close(lse[b, rows], rl, tl, "sequence %d heads of %d: lse" % (b, g))


# ---- together -------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_serving_run(kind):
    """Prompts in two chunks and then single tokens, as a server runs them:
    append, gather the context, attend over it, decode; every row against the
    attention over what the cache holds."""
    a = abi()
    fault()
    hk, group, dim, ps = 2, 4, 64, 16
    prompts, chunk, steps = [150, 40, 0, 71], 64, 5
    n_seq = len(prompts)
    rows = [[randn(p + steps, h, dim, seed=10 * b + i) for i, h in enumerate((hk * group, hk, hk))]
            for b, p in enumerate(prompts)]
    pool = Pool(kind, "hnd", hk, dim, ps, [0] * n_seq, max_len=max(prompts) + steps)
    scale, done = dim ** -0.5, [0] * n_seq
    out = [torch.zeros(p + steps, hk * group, dim, device="cuda", dtype=torch.float16) for p in prompts]
    lses = [torch.zeros(p + steps, hk * group, device="cuda") for p in prompts]
    while any(d < p for d, p in zip(done, prompts)):
        new = [min(chunk, p - d) for d, p in zip(done, prompts)]
        lens = [d + n for d, n in zip(done, new)]
        q, k, v = (torch.cat([rows[b][i][done[b]:lens[b]] for b in range(n_seq)]) for i in range(3))
        cu_q, cu_k = i32(prefix(new)), i32(prefix(lens))
        a.kv_append(k, v, pool.cache, pool.table, cu_q, i32(lens))
        ck, cv = (torch.empty(sum(lens), hk, dim, dtype=torch.float16, device="cuda") for _ in "kv")
        a.kv_gather(pool.cache, pool.table, cu_k, i32(lens), ck, cv)
        o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        a.attn_prompt(q, ck, cv, cu_q, cu_k, o, lse=lse)
        for b, c in enumerate(prefix(new)[:-1]):
            out[b][done[b]:lens[b]], lses[b][done[b]:lens[b]] = o[c:c + new[b]], lse[c:c + new[b]]
        done = lens
    ws = a.attn_decode_workspace(pool.cache, hk * group)
    for step in range(steps):
        at = [d + step for d in done]
        q, k, v = (torch.stack([rows[b][i][at[b]] for b in range(n_seq)]) for i in range(3))
        lens = i32([p + 1 for p in at])
        a.kv_append(k, v, pool.cache, pool.table, i32(range(n_seq + 1)), lens)
        o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        a.attn_decode(q, pool.cache, pool.table, lens, o, lse=lse, workspace=ws)
        for b in range(n_seq):
            out[b][at[b]], lses[b][at[b]] = o[b], lse[b]
    assert fault() == 0
    for b, p in enumerate(prompts):
        n = p + steps
        k, v = pool.get(0, b, 0, n), pool.get(1, b, 0, n)
        check_prompt(rows[b][0], k, v, [0, n], [0, n], out[b], lses[b], scale, True)


def test_two_streams_with_a_workspace_each():
    a = abi()
    pools = [Pool(kind, "hnd", 2, 128, 16, [5000, 3000], seed=s) for s, kind in enumerate(("f16", "e4m3"))]
    q = randn(2, 8, 128, seed=1)
    want, got = [], []
    for p in pools:
        want.append(torch.empty_like(q))
        a.attn_decode(q, p.cache, p.table, p.lens_t, want[-1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pools]
    for rep in range(10):
        for p, st in zip(pools, streams):
            got.append(torch.empty_like(q))
            a.attn_decode(q, p.cache, p.table, p.lens_t, got[-1], stream=st)  # its own workspace each
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert same_bits(o, want[i % 2])


def test_prompts_on_two_streams():
    a = abi()
    cu = i32([0, 700, 1500])
    sets = [[randn(1500, h, d, seed=10 * i + s) for s, h in enumerate((8, 4, 4))] for i, d in enumerate((128, 64))]
    want = [torch.empty_like(s[0]) for s in sets]
    for s, o in zip(sets, want):
        a.attn_prompt(*s, cu, cu, o)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for rep in range(8):
        for s, st in zip(sets, streams):
            got.append(torch.empty_like(s[0]))
            a.attn_prompt(*s, cu, cu, got[-1], stream=st)
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert same_bits(o, want[i % 2])
    assert fault() == 0


def test_prompt_more_keys_than_queries_ragged_groups():
    """Odd groups, where a pair of tiles spans two query blocks with different
    numbers of keys, and sequences whose tiles see no key at all between others."""
    a = abi()
    nq, nk = [300, 500, 129, 260, 1, 700], [100, 640, 0, 261, 300, 700]
    for heads, group, dim in ((2, 3, 128), (1, 5, 64), (3, 1, 128)):
        cu_q, cu_k = prefix(nq), prefix(nk)
        q = randn(cu_q[-1], heads * group, dim, seed=1)
        k, v = randn(cu_k[-1], heads, dim, seed=2), randn(cu_k[-1], heads, dim, seed=3)
        for causal in (True, False):
            o, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device="cuda")
            a.attn_prompt(q, k, v, i32(cu_q), i32(cu_k), o, causal=causal, lse=lse)
            check_prompt(q, k, v, cu_q, cu_k, o, lse, dim ** -0.5, causal)
    assert fault() == 0


@pytest.mark.parametrize("heads,group,dim", [(1, 1, 128), (1, 3, 64), (2, 4, 128), (2, 2, 40), (1, 7, 96)])
def test_prompt_few_rows_behind_long_contexts(heads, group, dim):
    """Few tiles over many keys: the keys are shared between blocks, evenly and
    not, with shares that hold no key a row sees."""
    a = abi()
    for nq, nk in (([1], [5000]), ([130], [8192]), ([200], [4097]), ([3, 0, 40], [9000, 100, 1]),
                   ([128], [2049]), ([5], [1024]), ([77, 33], [3000, 20000]), ([300], [300]), ([64], [40])):
        cu_q, cu_k = [2 + c for c in prefix(nq)], [3 + c for c in prefix(nk)]
        q = randn(cu_q[-1] + 4, heads * group, dim, seed=1)
        k, v = randn(cu_k[-1] + 200, heads, dim, seed=2), randn(cu_k[-1] + 200, heads, dim, seed=3)
        for x, cu in ((q, cu_q), (k, cu_k), (v, cu_k)):
            x[:cu[0]], x[cu[-1]:] = math.nan, math.nan
        for causal in (True, False):
            o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
            a.attn_prompt(q, k, v, i32(cu_q), i32(cu_k), o, causal=causal, lse=lse)
            check_prompt(q, k, v, cu_q, cu_k, o, lse, dim ** -0.5, causal)
            for x in (o, lse):
                assert (x[:cu_q[0]] == 7).all() and (x[cu_q[-1]:] == 7).all()
    assert fault() == 0


def test_prompt_few_rows_masked_nan():
    """The same split with NaN at the keys that the last rows alone see."""
    a = abi()
    n, m, dim = 20, 6000, 64
    q, k, v = randn(n, 2, dim, seed=1), randn(m, 2, dim, seed=2), randn(m, 2, dim, seed=3)
    v[m - 5, 0, 7], v[m - 1] = math.nan, math.inf
    o, lse = torch.empty_like(q), torch.empty(n, 2, device="cuda")
    a.attn_prompt(q, k, v, i32([0, n]), i32([0, m]), o, lse=lse)
    check_prompt(q[:15, :1], k[:m - 5, :1], v[:m - 5, :1], [0, 15], [0, m - 5], o[:15, :1], lse[:15, :1], 0.125, True)
    check_prompt(q[:19, 1:], k[:m - 1, 1:], v[:m - 1, 1:], [0, 19], [0, m - 1], o[:19, 1:], lse[:19, 1:], 0.125, True)
    assert torch.isnan(o[15:, 0, 7]).all() and not torch.isfinite(o[19]).any()


def test_captured_and_replayed():
    """Decode and prompt in one graph, replayed with other lengths and inputs;
    the workspace serves an eager call between replays."""
    a = abi()
    pool = Pool("f16", "hnd", 2, 64, 16, [900, 64, 300], seed=1)
    q, qp = randn(3, 4, 64, seed=1), randn(260, 4, 64, seed=2)
    kp, vp = randn(260, 2, 64, seed=3), randn(260, 2, 64, seed=4)
    lens, cu = pool.lens_t.clone(), i32([0, 100, 260])
    o, op = torch.empty_like(q), torch.empty_like(qp)
    lse, lp = torch.empty(3, 4, device="cuda"), torch.empty(260, 4, device="cuda")
    ws = a.attn_decode_workspace(pool.cache, 4)
    graph = torch.cuda.CUDAGraph()
    a.attn_decode(q, pool.cache, pool.table, lens, o, lse=lse, workspace=ws)
    a.attn_prompt(qp, kp, vp, cu, cu, op, lse=lp)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.attn_decode(q, pool.cache, pool.table, lens, o, lse=lse, workspace=ws)
        a.attn_prompt(qp, kp, vp, cu, cu, op, lse=lp)
    other = torch.empty_like(q)
    for step, (ln, c) in enumerate((([900, 64, 300], [0, 100, 260]), ([1, 0, 299], [3, 259, 259]),
                                    ([890, 1, 0], [0, 0, 128]))):
        lens.copy_(i32(ln))
        cu.copy_(i32(c))
        qp.copy_(randn(260, 4, 64, seed=20 + step))
        q.copy_(randn(3, 4, 64, seed=30 + step))
        graph.replay()
        a.attn_decode(q, pool.cache, pool.table, pool.lens_t, other, workspace=ws)
        torch.cuda.synchronize()
        pool.lens = ln
        vals = [tuple(x[:n] for x in kv) for kv, n in zip(pool.values, ln)]
        check_decode(pool, q, o, lse, 0.125, values=vals)
        check_prompt(qp, kp, vp, c, c, op, lp, 0.125, True)
    del graph


def test_large_grids():
    """More rows than one dimension of a grid holds."""
    a = abi()
    n = 70000
    q, k, v = randn(n, 1, 8, seed=1), randn(n, 1, 8, seed=2), randn(n, 1, 8, seed=3)
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    o = torch.empty_like(q)
    a.attn_prompt(q, k, v, cu, cu, o)
    assert same_bits(o, v)  # one key: weight one
    pool = torch.empty(n, 1, 1, 8, dtype=torch.float16, device="cuda"), torch.empty(n, 1, 1, 8, dtype=torch.float16,
                                                                                device="cuda")
    cache = a.KvCache(*pool)
    table = torch.arange(n, dtype=torch.int32, device="cuda").flip(0).view(n, 1)
    ones = torch.ones(n, dtype=torch.int32, device="cuda")
    a.kv_append(k, v, cache, table, cu, ones)
    a.attn_decode(q, cache, table, ones, o.zero_())
    assert same_bits(o, v)
    assert fault() == 0
