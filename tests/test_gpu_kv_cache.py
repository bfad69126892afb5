"""The paged key-value cache on the GPU: append (with its quantisation) and
gather, against the definition in 64 bits.  Both are exact: bits are compared."""
import math

import pytest
import torch

from attn_testutil import Pool, quantise_f64, same_bits

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


CASES = [  # kind, layout, heads, dim, page_size, lengths before, rows appended
    ("f16", "nhd", 1, 8, 1, [0, 3], [1, 2]),
    ("f16", "hnd", 3, 24, 3, [0, 5, 0, 7], [4, 0, 0, 9]),
    ("f16", "hnd", 8, 128, 16, [100, 0, 17], [1, 1, 1]),
    ("f16", "nhd", 5, 72, 24, [11], [200]),
    ("e4m3", "hnd", 1, 16, 1, [0], [1]),
    ("e4m3", "nhd", 2, 32, 5, [0, 0, 9, 16], [7, 0, 1, 33]),
    ("e4m3", "hnd", 8, 128, 16, [31, 32, 33, 0], [1, 1, 1, 1]),
    ("e4m3", "hnd", 8, 128, 16, [0, 100], [300, 77]),
    ("e4m3", "nhd", 7, 112, 64, [3], [129]),
    ("e4m3", "hnd", 4, 64, 128, [1000, 0], [5, 260]),
    ("e4m3", "nhd", 1100, 16, 2, [1, 0], [2, 3]),  # more rows per token than a block stages exponents of
    ("e4m3", "hnd", 2, 32, 16, [0] * 1500, [i % 3 for i in range(1500)]),  # more sequences than it holds bounds of
    ("f16", "hnd", 1, 16, 16, [i % 5 for i in range(1023)], [i % 2 for i in range(1023)]),
    ("f16", "nhd", 2, 64, 16, [0], [12000]),  # many tokens to a block
    ("e4m3", "hnd", 2, 96, 48, [5, 0], [7001, 5000]),
]


@pytest.mark.parametrize("kind,layout,heads,dim,page,past,new", CASES)
def test_append_then_gather(kind, layout, heads, dim, page, past, new):
    a = abi()
    fault()
    lens = [p + n for p, n in zip(past, new)]
    pool = Pool(kind, layout, heads, dim, page, past, max_len=max(lens))
    want = Pool(kind, layout, heads, dim, page, past, max_len=max(lens))
    # rows before the first and behind the last sequence belong to nobody
    lead, tail = 3, 5
    total = lead + sum(new) + tail
    g = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn(total, 2 * heads, dim, device="cuda", generator=g).half()
         * torch.exp2(torch.randint(-12, 9, (total, 2 * heads, 1), device="cuda", generator=g).float()).half()
         for _ in "kv"]
    k, v = x[0][:, :heads], x[1][:, heads:]  # strided rows
    cu = i32([lead + c for c in prefix(new)])
    a.kv_append(k, v, pool.cache, pool.table, cu, i32(lens))
    at = lead
    held = []
    for b, n in enumerate(new):
        held.append([want.put(i, b, past[b], r[at:at + n]) for i, r in enumerate((k, v))])
        at += n
    assert fault() == 0
    for got, ref in zip(pool.raw + [e for e in pool.exps if e is not None],
                        want.raw + [e for e in want.exps if e is not None]):
        assert same_bits(got, ref)  # what was written, and everything else as it was

    out = [torch.full((total, heads, dim), 7.0, dtype=torch.float16, device="cuda") for _ in "kv"]
    a.kv_gather(pool.cache, pool.table, cu, i32(lens), *out)
    at = lead
    for b, n in enumerate(new):
        for i in range(2):
            assert torch.equal(out[i][at:at + n].double(), held[b][i])
        at += n
    for o in out:
        assert (o[:lead] == 7).all() and (o[at:] == 7).all()
    # the whole of each sequence, strided destination
    whole = sum(lens)
    big = torch.full((whole, heads, 2, dim), 7.0, dtype=torch.float16, device="cuda")
    a.kv_gather(pool.cache, pool.table, i32(prefix(lens)), i32(lens), big[:, :, 0], big[:, :, 1])
    at = 0
    for b, n in enumerate(lens):
        for i in range(2):
            assert torch.equal(big[at:at + n, :, i].double(), pool.get(i, b, 0, n))
        at += n
    assert fault() == 0


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 72])
@pytest.mark.parametrize("shift,pad", [(0, 0), (8, 0), (0, 8), (16, 16), (8, 8)])
def test_gather_into_any_alignment(kind, dim, shift, pad):
    """Rows that begin on 32- and on 16-byte boundaries, and what lies between
    them left as it was."""
    a = abi()
    if kind == "e4m3" and dim % 16:
        dim = 48
    heads, n = 3, 37
    pool = Pool(kind, "hnd", heads, dim, 16, [n])
    outs, flat = [], []
    for _ in "kv":
        f = torch.full((shift + n * heads * (dim + pad),), 7.0, dtype=torch.float16, device="cuda")
        flat.append(f)
        outs.append(f[shift:].view(n, heads, dim + pad)[:, :, :dim])
    a.kv_gather(pool.cache, pool.table, i32([0, n]), i32([n]), *outs)
    assert fault() == 0
    for i in range(2):
        assert torch.equal(outs[i].double(), pool.get(i, 0, 0, n))
        assert (flat[i][:shift] == 7).all()
        assert (flat[i][shift:].view(n, heads, dim + pad)[:, :, dim:] == 7).all()


def test_quantiser_at_its_borders():
    """Maxima at and next to 448 * 2^e, zeros, subnormals, the largest values,
    infinities and NaN, one row each."""
    a = abi()
    dim = 16
    rows = []
    for e in range(-17, 9):
        for f in (1.0, 1.75, 1.75 + 2 ** -10, 1.75 - 2 ** -10, 2 - 2 ** -10):
            top = f * 2.0 ** (e + 8)
            rows.append([top if top <= 65504 else 65504.0] + [top * s / 40 for s in range(-14, 1)])
    rows += [[0.0] * dim, [-0.0] * dim, [2.0 ** -24] * dim, [2.0 ** -24, -(2.0 ** -14)] * 8, [65504.0, -65504.0] * 8,
             [61440.0, 61472.0] * 8, [math.inf] + [1.0] * 15, [-math.inf, 3e-5] * 8, [math.nan] + [2.0] * 15,
             [math.nan] * dim]
    # every e4m3 tie: midpoints of neighbouring codes at one scale
    rows += [[448.0] + [(8 + m + 0.5) * 2.0 ** x for m in range(8)] + [0.0] * 7 for x in range(-9, 5)]
    x = torch.tensor(rows, dtype=torch.float64).half().cuda()[:, None, :].contiguous()
    n = x.shape[0]
    pool = Pool("e4m3", "nhd", 1, dim, 16, [n], fill=False)
    a.kv_append(x, x, pool.cache, pool.table, i32([0, n]), i32([n]))
    held, code, e = quantise_f64(x)
    page, off = pool.where(0, 0, n)
    for which in range(2):
        assert torch.equal(pool.exps[which].transpose(1, 2)[page, off].long() - 127, e)
        got = (pool.k, pool.v)[which].view(torch.uint8)[page, off].view(torch.float8_e4m3fn).double()
        assert torch.equal(torch.isnan(got), torch.isnan(x))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(code))
    out = [torch.empty_like(x) for _ in "kv"]
    a.kv_gather(pool.cache, pool.table, i32([0, n]), i32([n]), *out)
    fine = torch.isfinite(x)
    back = out[0].double()
    assert torch.equal(torch.nan_to_num(back), torch.nan_to_num(held)) and torch.isfinite(back[~torch.isnan(x)]).all()
    # half a step of the three bits behind the leading one, or half the smallest step of the row's scale
    xs, bound = x.double(), torch.tensor([2.0 ** (k - 10) for k in range(-15, 9)], dtype=torch.float64, device="cuda")
    ok = (back - xs).abs() <= torch.maximum(xs.abs() * 2.0 ** -4, bound[e + 15].unsqueeze(-1))
    assert ok[fine].all()


def test_bad_pages_and_lengths_are_skipped():
    a = abi()
    fault()
    for kind in ("f16", "e4m3"):
        pool = Pool(kind, "hnd", 2, 32, 4, [8, 8, 8])
        before = [r.clone() for r in pool.raw]
        table = pool.table.clone()
        table[0, 1] = pool.pages  # one past the pool
        table[1, 0] = -5
        table[2, 0] = 2147483647
        rows = torch.randn(6, 2, 32, device="cuda").half()
        # rows 0-1 -> sequence 0 positions 6, 7 (page entry 1); 2-3 -> sequence 1 positions 2, 3 (entry 0);
        # 4-5 -> sequence 2 at 0, 1 (entry 0)
        a.kv_append(rows, rows, pool.cache, table, i32([0, 2, 4, 6]), i32([8, 4, 2]))
        assert fault() == 64
        for r, w in zip(pool.raw, before):
            assert same_bits(r, w)
        out = [torch.full((6, 2, 32), 7.0, dtype=torch.float16, device="cuda") for _ in "kv"]
        a.kv_gather(pool.cache, table, i32([0, 2, 4, 6]), i32([8, 4, 2]), *out)
        assert fault() == 64
        assert (out[0] == 0).all() and (out[1] == 0).all()
        # positions behind the table, below zero, and negative lengths
        far = pool.table.shape[1] * 4
        a.kv_append(rows, rows, pool.cache, pool.table, i32([0, 2, 4, 6]), i32([far + 2, 0, -3]))
        assert fault() == 64
        for r, w in zip(pool.raw, before):
            assert same_bits(r, w)
        a.kv_gather(pool.cache, pool.table, i32([0, 2, 4, 6]), i32([0, 1, -7]), *out)
        assert fault() == 0
        assert (out[0][[0, 1, 2, 4, 5]] == 0).all() and torch.equal(out[0][3].double(), pool.values[1][0][0])
        # lengths near the 31-bit end
        a.kv_append(rows, rows, pool.cache, pool.table, i32([0, 2, 4, 6]), i32([2147483647] * 3))
        assert fault() == 64
        for r, w in zip(pool.raw, before):
            assert same_bits(r, w)


def test_no_rows_and_no_pages():
    a = abi()
    pool = Pool("f16", "nhd", 2, 16, 4, [3])
    none = torch.empty(0, 2, 16, dtype=torch.float16, device="cuda")
    a.kv_append(none, none, pool.cache, pool.table, i32([0, 0]), i32([3]))
    a.kv_gather(pool.cache, pool.table, i32([0, 0]), i32([3]), none, none)
    empty = torch.empty(0, 4, 2, 16, dtype=torch.float16, device="cuda")
    cache = a.KvCache(empty, empty.clone())
    out = torch.ones(2, 2, 16, dtype=torch.float16, device="cuda")
    a.kv_gather(cache, pool.table, i32([0, 2]), i32([2]), out, out.clone())
    assert (out == 0).all() and fault() == 64


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_offsets_past_32_bits(kind):
    """Pages more than 2^32 bytes apart in one pool."""
    a = abi()
    fault()
    heads, dim, ps = 2, 32, 4
    es = 2 if kind == "f16" else 1
    stride = (1 << 32) // es // 2 + 64  # elements between pages: 3 pages span more than 2^32 bytes
    dt = torch.float16 if kind == "f16" else torch.float8_e4m3fn
    raw = torch.empty((2 * stride + ps * heads * dim) * es, dtype=torch.uint8, device="cuda")
    k = raw.view(dt).as_strided((3, ps, heads, dim), (stride, heads * dim, dim, 1))
    v = torch.empty_like(raw).view(dt).as_strided((3, ps, heads, dim), (stride, heads * dim, dim, 1))
    e = [torch.zeros(3, heads, ps, dtype=torch.uint8, device="cuda") if kind == "e4m3" else None for _ in "kv"]
    cache = a.KvCache(k, v, *e)
    table = i32([[2, 0, 1]])
    x = [torch.randn(12, heads, dim, device="cuda").half() for _ in "kv"]
    a.kv_append(x[0], x[1], cache, table, i32([0, 12]), i32([12]))
    out = [torch.empty_like(t) for t in x]
    a.kv_gather(cache, table, i32([0, 12]), i32([12]), *out)
    for t, o in zip(x, out):
        ref = t.double() if kind == "f16" else quantise_f64(t)[0]
        assert torch.equal(o.double(), ref)
    # the far page holds the first four positions
    if kind == "f16":
        assert torch.equal(k[2], x[0][:4])
    assert fault() == 0


def test_append_on_another_stream_and_in_a_graph():
    a = abi()
    pool, want = (Pool("e4m3", "hnd", 4, 64, 16, [0, 0], max_len=40) for _ in range(2))
    x = torch.zeros(2, 4, 64, device="cuda", dtype=torch.float16)
    lens, cu = i32([0, 0]), i32([0, 1, 2])
    st = torch.cuda.Stream()
    a.kv_append(x, x, want.cache, want.table, cu, i32([1, 1]))
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        a.kv_append(x, x, want.cache, want.table, cu, i32([1, 1]), stream=st)  # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens.add_(1)
        a.kv_append(x, x, pool.cache, pool.table, cu, lens)
    lens.zero_()
    for step in range(33):  # the position moves on by itself, across pages
        x.copy_(torch.randn(2, 4, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(step)))
        graph.replay()
        for i in range(2):
            for b in range(2):
                want.put(i, b, step, x[b:b + 1])
    torch.cuda.synchronize()
    for got, ref in zip(pool.raw + pool.exps, want.raw + want.exps):
        assert same_bits(got, ref)
    del graph
