"""Definitions in 64 bits and error bounds for the paged cache and the
attention operators (shared by their tests).

Bounds, per output element, for weights w_j and values v_j of the keys seen:
  |o - ref| <= 2^-11 |ref|            the rounding into binary16 (half a step)
             + 2^-11 A                each weight's rounding to binary16
             + (2 E + 2^-18) A        the scores' error E, absolute, moves each
                                      weight by at most e^(2E) - 1; exp2 and the
                                      fp32 sums stay below 2^-18
             + 2^-25                  half the smallest binary16 step
with A = sum_j w_j |v_j| and, for dim products summed in fp32 one after the
other or in any grouping, with truncation (one whole step 2^-23 each),
  E = (dim + 2) 2^-23 scale max_j sum_d |q_d k_jd|.
|lse - ref| <= E + 2^-18 + 2^-22 |ref|.
"""
import math

import torch

E4M3_MAX, VALUE_MAX, EXP_MIN = 448.0, 61440.0, -15


def attention_f64(q, k, v, scale, seen):
    """One head: q [n, d], k, v [m, d] (any type), seen [n, m] bool.  Returns
    o, lse, and the bounds of both.  Keys not seen take no part whatever they hold."""
    q, k, v = (x.double() for x in (q, k, v))
    n, m = seen.shape
    if m == 0:
        zero = torch.zeros(n, dtype=torch.float64, device=q.device)
        return torch.zeros_like(q), zero - math.inf, torch.ones_like(q), zero + 1.0
    prod = torch.where(seen[:, :, None], q[:, None, :] * k[None], torch.zeros((), dtype=torch.float64,
                                                                             device=q.device)) \
        if n * m * q.shape[1] <= 1 << 24 else None
    if prod is not None:
        s, mag = prod.sum(-1) * scale, prod.abs().sum(-1)
    else:
        s, mag = q @ k.T * scale, q.abs() @ k.abs().T
    err = (q.shape[1] + 2) * 2.0 ** -23 * abs(scale) * torch.where(seen, mag, torch.zeros_like(mag)).amax(-1)
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    any_ = seen.any(-1)
    top = torch.where(any_, s.amax(-1), torch.zeros_like(err))
    p = torch.exp(s - top[:, None])
    total = p.sum(-1)
    w = p / torch.where(any_, total, torch.ones_like(total))[:, None]
    if torch.isfinite(v).all():
        o, a = w @ v, w @ v.abs()
    else:
        wv = torch.where(seen[:, :, None], w[:, :, None] * v[None], torch.zeros((), dtype=torch.float64,
                                                                                 device=q.device))
        o, a = wv.sum(1), wv.abs().sum(1)
    lse = torch.where(any_, total.log() + top, torch.full_like(top, -math.inf))
    tol = 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2 * err[:, None] + 2.0 ** -18) * a + 2.0 ** -25
    return o, lse, tol, err + 2.0 ** -18 + 2.0 ** -22 * torch.where(any_, lse.abs(), torch.zeros_like(lse))


def quantise_f64(x):
    """(values held, codes' values, exponent) of binary16 rows x [..., d], from
    the definition: thresholds for the exponent, rounding to multiples for the code."""
    x = x.double().clamp(-VALUE_MAX, VALUE_MAX)
    top = torch.nan_to_num(x.abs(), nan=0.0).amax(-1)
    e = torch.full(top.shape, EXP_MIN, dtype=torch.int64, device=x.device)
    for k in range(EXP_MIN, 9):
        e += (top > E4M3_MAX * 2.0 ** k).long()
    two = torch.tensor([2.0 ** k for k in range(-40, 41)], dtype=torch.float64, device=x.device)
    s = two[e + 40].unsqueeze(-1)
    y = x / s
    ex = torch.frexp(torch.nan_to_num(y.abs(), nan=1.0).clamp(min=2.0 ** -6))[1]
    step = two[ex - 4 + 40]
    code = torch.round(y / step) * step
    return code * s, code, e


class Pool:
    """A paged cache with a shuffled block table: every byte of the pools that
    no position owns holds NaN (all bits set), unused table entries are bad ids."""

    def __init__(self, kind, layout, heads, dim, page_size, lens, spare_pages=2, table_pad=1, bad=-1, seed=0, fill=True,
                 max_len=None):
        from unikern_b200 import abi
        g = torch.Generator().manual_seed(seed)
        self.kind, self.heads, self.dim, self.page_size, self.lens = kind, heads, dim, page_size, list(lens)
        top = [max(n, max_len or 0) for n in lens]
        per = [-(-n // page_size) for n in top]
        self.pages = sum(per) + spare_pages
        ids = torch.randperm(self.pages, generator=g).to(torch.int32)
        table = torch.full((len(lens), max(per + [0]) + table_pad), bad, dtype=torch.int32)
        at = 0
        for b, p in enumerate(per):
            table[b, :p] = ids[at:at + p]
            at += p
        self.table_cpu, self.table = table, table.cuda()
        shape = (self.pages, page_size, heads, dim) if layout == "nhd" else (self.pages, heads, page_size, dim)
        dt = torch.float16 if kind == "f16" else torch.float8_e4m3fn
        es = 2 if kind == "f16" else 1
        self.raw = [torch.full((self.pages * page_size * heads * dim * es,), 255, dtype=torch.uint8, device="cuda")
                    for _ in "kv"]
        self.k, self.v = (r.view(dt).view(shape) for r in self.raw)
        if layout == "hnd":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.exps = [None, None]
        if kind == "e4m3":
            self.exps = [torch.full((self.pages, heads, page_size), 255, dtype=torch.uint8, device="cuda")
                         for _ in "kv"]
        self.cache = abi.KvCache(self.k, self.v, *self.exps)
        self.values = []  # per sequence: (k, v) [len, heads, dim] float64, what the cache stands for
        for b, n in enumerate(self.lens):
            rows = [torch.randn(n, heads, dim, generator=g).half().cuda() for _ in "kv"]
            self.values.append(tuple(self.put(i, b, 0, r) if fill else None for i, r in enumerate(rows)))
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def where(self, b, first, n):
        pos = torch.arange(first, first + n)
        page = self.table_cpu[b][pos // self.page_size].long().cuda()
        return page, (pos % self.page_size).cuda()

    def put(self, which, b, first, rows):
        """Writes binary16 rows [n, heads, dim] from the definition; returns the values held."""
        page, off = self.where(b, first, rows.shape[0])
        dst = (self.k, self.v)[which]
        if self.kind == "f16":
            dst[page, off] = rows
            return rows.double()
        held, code, e = quantise_f64(rows)
        # indexing of float8 tensors goes through their bytes
        dst.view(torch.uint8)[page, off] = code.float().to(torch.float8_e4m3fn).view(torch.uint8)
        self.exps[which].transpose(1, 2)[page, off] = (e + 127).to(torch.uint8)
        return held

    def get(self, which, b, first, n):
        """Values the cache stands for, read from the definition."""
        page, off = self.where(b, first, n)
        src = (self.k, self.v)[which]
        if self.kind == "f16":
            return src[page, off].double()
        code = src.view(torch.uint8)[page, off].view(torch.float8_e4m3fn).double()
        e = self.exps[which].transpose(1, 2)[page, off].long() - 127
        two = torch.tensor([2.0 ** k for k in range(-127, 129)], dtype=torch.float64, device="cuda")
        return code * two[e + 127].unsqueeze(-1)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def assert_close(got, ref, tol, what):
    got = got.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what + ": NaN elsewhere"
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), what + ": infinities"
    over = ((got - ref).abs() / tol)[fine]
    if over.numel():
        worst = over.max().item()
        assert worst <= 1.0, "%s: %.3g times the bound" % (what, worst)
