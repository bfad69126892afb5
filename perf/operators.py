"""Measured cases of the paged key-value cache and the attention operators.

Four operators, each in a plain form (elementary torch operations in 32 bits)
and, where `own` is set, as the calls of `unikern_b200.abi`:

* append  -- new tokens' keys and values written into a paged cache, as
  binary16 or as e4m3 codes with one power-of-two exponent per token and head;
* gather  -- positions of a paged cache read back as packed binary16 rows;
* decode  -- attention of one new token per sequence over a paged cache;
* prompt  -- attention over packed prompts, causal or full, grouped heads.
"""
import math

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
EXP_MIN = -15  # every binary16 value is a multiple of 2^-24 = 2^-9 * 2^-15
VALUE_MAX = 61440.0  # 240 * 2^8: the largest e4m3 multiple that is a binary16 value


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # one decode step's new tokens of a full batch, 8-bit cache: latency
        dict(name="append e4m3 32x1", op="append", kind="e4m3", seqs=32, new=1, past=1000, spread=0.9, heads_kv=8,
             dim=128, page=16, layout="hnd"),
        # some prompts, some thousand tokens in all, going into an 8-bit cache
        dict(name="append e4m3 5x1639", op="append", kind="e4m3", seqs=5, new=1639, past=0, spread=0.3, heads_kv=8,
             dim=128, page=16, layout="hnd"),
        # the context of a few requests read back before their next prompt chunk, odd sizes
        dict(name="gather f16 7x531", op="gather", kind="f16", seqs=7, new=531, past=0, spread=0.6, heads_kv=5, dim=64,
             page=32, layout="nhd"),
        # long contexts out of an 8-bit cache
        dict(name="gather e4m3 4x16384", op="gather", kind="e4m3", seqs=4, new=16384, past=0, spread=0.0, heads_kv=8,
             dim=128, page=64, layout="hnd"),
        # one request with a short context: the latency of a token
        dict(name="decode f16 1x500", op="decode", kind="f16", seqs=1, len=500, spread=0.0, heads_q=32, heads_kv=8,
             dim=128, page=16, layout="hnd"),
        # the decode chain's batch and score length: 32 tokens, 32 heads, 8192 positions
        dict(name="decode f16 32x8192", op="decode", kind="f16", seqs=32, len=8192, spread=0.0, heads_q=32, heads_kv=8,
             dim=128, page=16, layout="hnd"),
        # the same batch, ragged, out of an 8-bit cache
        dict(name="decode e4m3 32x8192 ragged", op="decode", kind="e4m3", seqs=32, len=8192, spread=0.9, heads_q=32,
             heads_kv=8, dim=128, page=32, layout="hnd"),
        # one request with a very long context and few key heads: the split over its length
        dict(name="decode f16 1x131071", op="decode", kind="f16", seqs=1, len=131071, spread=0.0, heads_q=32,
             heads_kv=2, dim=128, page=64, layout="nhd"),
        # a short prompt: latency
        dict(name="prompt 1x77", op="prompt", seqs=1, len=77, past=0, spread=0.0, heads_q=32, heads_kv=8, dim=128,
             causal=True),
        # prompts of mixed lengths packed together, small heads, odd group
        dict(name="prompt 11x900 ragged d64", op="prompt", seqs=11, len=900, past=0, spread=0.8, heads_q=21, heads_kv=7,
             dim=64, causal=True),
        # the next chunk of prompts behind a cached context
        dict(name="prompt 3x1000+5000", op="prompt", seqs=3, len=1000, past=5000, spread=0.4, heads_q=32, heads_kv=8,
             dim=128, causal=True),
        # one whole prompt
        dict(name="prompt 1x8192", op="prompt", seqs=1, len=8192, past=0, spread=0.0, heads_q=32, heads_kv=8, dim=128,
             causal=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "decode", "decode", "prompt", "prompt"])
    kind = rng.choice(["f16", "e4m3"])
    heads_kv = rng.choice([1, 2, 3, 4, 5, 7, 8, 12])
    dim = rng.choice([64, 128, 128, 32, 80, 96, 112])
    c = dict(op=op, seqs=_log(rng, 1, 64), heads_kv=heads_kv, dim=dim, spread=rng.choice([0.0, 0.5, 0.95]))
    if op != "prompt":
        c.update(kind=kind, page=rng.choice([8, 16, 16, 32, 48, 64, 128, 256]), layout=rng.choice(["hnd", "nhd"]))
    if op in ("append", "gather"):
        c["new"] = _log(rng, 1, max(1, min(16384, 65536 // c["seqs"])))
        c["past"] = rng.choice([0, 0, _log(rng, 1, 1500)])
    else:
        c["heads_q"] = heads_kv * rng.choice([1, 2, 3, 4, 4, 8] if heads_kv > 2 else [1, 4, 8, 12, 16, 20])
        if op == "decode":
            most = 32 * 8192 * 8 * 128 // (c["seqs"] * heads_kv * dim)
            c["len"] = _log(rng, 1, min(131071, most))
        else:
            # at most the work of the largest listed case, 2^31 scores of 128-wide heads
            c["seqs"] = min(c["seqs"], 24)
            c["causal"] = rng.random() < 0.75
            most = int(math.sqrt((2 ** 31 if c["causal"] else 2 ** 30) / (c["seqs"] * c["heads_q"])))
            c["len"] = _log(rng, 1, max(2, min(8191, most)))
            room = 2 ** 30 // (c["seqs"] * c["heads_q"] * c["len"]) - c["len"]
            c["past"] = _log(rng, 1, min(room, 16384)) if room > 1 and rng.random() < 0.4 else 0
    return c


def _lengths(n, top, spread):
    """n lengths up to `top`, the first of them `top`; the others fall by at
    most the share `spread`, by the fractional parts of multiples of the golden
    section: the same for every seed."""
    return [max(1, int(top * (1.0 - spread * ((i * 0.6180339887498949) % 1.0)))) if top > 0 else 0 for i in range(n)]


def _counts(case):
    """(new or query tokens, tokens held in all) of each sequence."""
    if case["op"] == "decode":
        held = _lengths(case["seqs"], case["len"], case["spread"])
        return [1] * case["seqs"], held
    new = _lengths(case["seqs"], case["new"] if "new" in case else case["len"], case["spread"])
    past = _lengths(case["seqs"], case["past"], case["spread"])
    return new, [a + b for a, b in zip(new, past)]


def _prefix(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    new, held = _counts(case)
    hk, d = case["heads_kv"], case["dim"]
    s = dict(case=case)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    half = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)  # noqa: E731
    s["cu_new"], s["held"] = i32(_prefix(new)), i32(held)
    total = sum(new)
    if case["op"] == "prompt":
        s["cu_held"] = i32(_prefix(held))
        s["q"] = half(total, case["heads_q"], d)
        # keys and values come out of one projection: heads of K beside heads of V
        kv = half(sum(held), 2 * hk, d)
        s["k"], s["v"] = kv[:, :hk], kv[:, hk:]
        s["o"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(total, case["heads_q"], device=DEV)
        s["max_new"], s["max_held"] = max(new), max(held)
        return s
    # a pool of pages with some free ones, handed out in no order
    ps = case["page"]
    per = [-(-h // ps) for h in held]
    n_pages = sum(per) + 3
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(held), max(per)), -1, dtype=torch.int32, device=DEV)
    for b, (p, at) in enumerate(zip(per, _prefix(per))):
        table[b, :p] = ids[at:at + p]
    s["table"] = table
    shape = (n_pages, ps, hk, d) if case["layout"] == "nhd" else (n_pages, hk, ps, d)
    for name in ("k", "v"):
        x = half(*shape)
        if case["layout"] == "hnd":
            x = x.transpose(1, 2)
        if case["kind"] == "e4m3":
            code, e = _quantise(x.float())
            # (page, head, token), the tokens of a page side by side
            s["cache_%s_exp" % name] = e.transpose(1, 2).contiguous()
            held_codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device=DEV)
            held_codes = held_codes.transpose(1, 2) if case["layout"] == "hnd" else held_codes
            held_codes.copy_(code)
            x = held_codes
        s["cache_" + name] = x
    if case["op"] == "append":
        s["k"], s["v"] = half(total, hk, d), half(total, hk, d)
    elif case["op"] == "gather":
        s["k"], s["v"] = (torch.empty(total, hk, d, dtype=torch.float16, device=DEV) for _ in "kv")
    else:
        s["q"] = half(case["seqs"], case["heads_q"], d)
        s["o"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(case["seqs"], case["heads_q"], device=DEV)
        s["max_held"] = max(held)
    if own:
        from unikern_b200 import abi
        s["cache"] = abi.KvCache(s["cache_k"], s["cache_v"], s.get("cache_k_exp"), s.get("cache_v_exp"))
        if case["op"] == "decode":
            s["workspace"] = abi.attn_decode_workspace(s["cache"], case["heads_q"])
    return s


# ---- the plain forms -----------------------------------------------------------

def _two(e):
    """2^e in 32 bits for whole e in [-126, 127]: the exponent field itself (a
    power function may be off in the last place)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """e4m3 codes of x (last axis a head's values) and the exponent byte e of
    their scale 2^(e - 127): the smallest power of two that keeps them in range."""
    x = x.clamp(-VALUE_MAX, VALUE_MAX)
    m, e = torch.frexp(x.abs().amax(-1) / E4M3_MAX)
    e = torch.where(m == 0.5, e - 1, e).clamp(min=EXP_MIN)
    e = torch.where(m == 0.0, torch.full_like(e, EXP_MIN), e)
    return (x * _two(-e).unsqueeze(-1)).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _slots(s, total):
    """Of each packed token: its sequence and its position there."""
    t = torch.arange(total, device=DEV)
    cu = s["cu_new"].long()
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, t - cu[b + 1] + s["held"].long()[b]


def _held(s, name, page, at):
    """Rows of the cache in 32 bits: page and offset index arrays of one shape."""
    x = s["cache_" + name][page, at].float()
    e = s.get("cache_%s_exp" % name)
    if e is not None:
        x = x * _two(e.transpose(1, 2)[page, at].int() - 127).unsqueeze(-1)
    return x


def _softmax_product(scores, values):
    """softmax(scores) @ values and the logarithm of the softmax's sum; a row
    of -inf gives zeros and -inf."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, values) / torch.where(total > 0, total, torch.ones_like(total))
    return o, (total.log() + top).squeeze(-1)


def _plain_append(s):
    b, pos = _slots(s, s["k"].shape[0])
    ps = s["case"]["page"]
    page, at = s["table"].long()[b, pos // ps], pos % ps
    out = {}
    for name in ("k", "v"):
        cache, e = s["cache_" + name], s.get("cache_%s_exp" % name)
        if e is None:
            cache[page, at] = s[name]
        else:
            code, exp = _quantise(s[name].float())
            cache.view(torch.uint8)[page, at] = code.view(torch.uint8)
            e.transpose(1, 2)[page, at] = exp
            out[name + "_exp"] = e
        out[name] = cache
    return out


def _plain_gather(s):
    b, pos = _slots(s, s["k"].shape[0])
    ps = s["case"]["page"]
    page, at = s["table"].long()[b, pos // ps], pos % ps
    return {name: _held(s, name, page, at).to(torch.float16) for name in ("k", "v")}


def _plain_decode(s):
    c = s["case"]
    n, hq, hk, d = c["seqs"], c["heads_q"], c["heads_kv"], c["dim"]
    pos = torch.arange(s["max_held"], device=DEV)
    page, at = s["table"].long()[:, pos // c["page"]].clamp(min=0), (pos % c["page"]).expand(n, -1)
    k = _held(s, "k", page, at).permute(0, 2, 3, 1)
    q = s["q"].float().view(n, hk, hq // hk, d)
    scores = torch.matmul(q, k) / math.sqrt(d)
    hidden = pos >= s["held"].unsqueeze(1)
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    o, lse = _softmax_product(scores, _held(s, "v", page, at).transpose(1, 2))
    return {"o": o.reshape(n, hq, d).to(torch.float16), "lse": lse.reshape(n, hq)}


def _plain_prompt(s):
    c = s["case"]
    n, hq, hk, d = c["seqs"], c["heads_q"], c["heads_kv"], c["dim"]
    lq, lk = s["max_new"], s["max_held"]
    cu_q, cu_k = s["cu_new"].long(), s["cu_held"].long()
    len_q, len_k = cu_q.diff(), cu_k.diff()
    i, j = torch.arange(lq, device=DEV), torch.arange(lk, device=DEV)

    def padded(x, cu, lens, at):  # packed rows as (sequence, head, token, dim)
        rows = cu[:-1, None] + torch.minimum(at, (lens - 1).clamp(min=0)[:, None])
        return x[rows.clamp(max=x.shape[0] - 1)].float().transpose(1, 2)

    q = padded(s["q"], cu_q, len_q, i).reshape(n, hk, hq // hk * lq, d)
    k = padded(s["k"], cu_k, len_k, j)
    scores = torch.matmul(q, k.transpose(2, 3)).view(n, hk, hq // hk, lq, lk)
    scores.mul_(1.0 / math.sqrt(d))
    hidden = (j >= len_k[:, None])[:, None, :]
    if c["causal"]:
        hidden = hidden | (j > i[:, None] + (len_k - len_q)[:, None, None])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores = scores.view(n, hk, hq // hk * lq, lk)
    o, lse = _softmax_product(scores, padded(s["v"], cu_k, len_k, j))
    t = torch.arange(s["q"].shape[0], device=DEV)
    b = torch.searchsorted(cu_q, t, right=True) - 1
    o, lse = o.view(n, hq, lq, d)[b, :, t - cu_q[b]], lse.view(n, hq, lq)[b, :, t - cu_q[b]]
    return {"o": o.to(torch.float16), "lse": lse}


# ---- the framework's calls --------------------------------------------------------

def _own(s):
    from unikern_b200 import abi
    op = s["case"]["op"]
    if op == "append":
        abi.kv_append(s["k"], s["v"], s["cache"], s["table"], s["cu_new"], s["held"])
        out = {"k": s["cache_k"], "v": s["cache_v"]}
        if s["case"]["kind"] == "e4m3":
            out.update(k_exp=s["cache_k_exp"], v_exp=s["cache_v_exp"])
        return out
    if op == "gather":
        abi.kv_gather(s["cache"], s["table"], s["cu_new"], s["held"], s["k"], s["v"])
        return {"k": s["k"], "v": s["v"]}
    if op == "decode":
        abi.attn_decode(s["q"], s["cache"], s["table"], s["held"], s["o"], lse=s["lse"], workspace=s["workspace"])
    else:
        abi.attn_prompt(s["q"], s["k"], s["v"], s["cu_new"], s["cu_held"], s["o"], causal=s["case"]["causal"],
                        lse=s["lse"])
    return {"o": s["o"], "lse": s["lse"]}


def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "gather": _plain_gather, "decode": _plain_decode,
            "prompt": _plain_prompt}[s["case"]["op"]](s)


# ---- what cannot be left out ---------------------------------------------------------

def work(case):
    new, held = _counts(case)
    hk, d = case["heads_kv"], case["dim"]
    held_row = 0 if case["op"] == "prompt" else hk * (d + 1 if case["kind"] == "e4m3" else 2 * d)  # of K or V
    if case["op"] in ("append", "gather"):
        rows = sum(new)
        return {"bytes": 2 * rows * (2 * hk * d + held_row), "flops": 4 * rows * hk * d}
    hq = case["heads_q"]
    if case["op"] == "decode":
        small = case["seqs"] * hq * (4 * d + 4)
        return {"bytes": 2 * sum(held) * held_row + small, "flops": 4 * sum(held) * hq * d}
    if case["causal"]:
        pairs = sum(n * (h - n) + n * (n + 1) // 2 for n, h in zip(new, held))
    else:
        pairs = sum(n * h for n, h in zip(new, held))
    return {"bytes": sum(new) * hq * (4 * d + 4) + 4 * sum(held) * hk * d, "flops": 4 * pairs * hq * d}


# ---- the definitions in 64 bits --------------------------------------------------------

def _exact_two(e):
    """2^e in 64 bits, exactly."""
    return torch.tensor([2.0 ** k for k in range(-64, 65)], dtype=torch.float64, device=DEV)[e.long() + 64]


def _exact_codes(x):
    """Per value of x the e4m3 value it is held as, and the scale's exponent byte."""
    x = x.double().clamp(-VALUE_MAX, VALUE_MAX)
    top = x.abs().amax(-1)
    e = torch.full_like(top, EXP_MIN)
    for k in range(EXP_MIN, 9):
        e += (top > E4M3_MAX * 2.0 ** k).double()
    y = x / _exact_two(e).unsqueeze(-1)
    # 3 bits behind the leading one, down to the steps of the smallest normal value 2^-6
    step = _exact_two(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    return torch.round(y / step) * step, (e + 127).to(torch.uint8)


def _exact_row(s, name, b, pos):
    ps = s["case"]["page"]
    pages = s["table"][b].tolist()
    page = torch.tensor([pages[p // ps] for p in pos], device=DEV)
    at = torch.tensor([p % ps for p in pos], device=DEV)
    x = s["cache_" + name][page, at].double()
    e = s.get("cache_%s_exp" % name)
    if e is not None:
        x = x * _exact_two(e.permute(0, 2, 1)[page, at].long() - 127).unsqueeze(-1)
    return x


def _exact_attention(q, k, v, first):
    """One head: q (n, d), k and v (m, d); row i sees the keys up to first + i."""
    sc = (q @ k.T) / math.sqrt(q.shape[1])
    if first is not None:
        i = torch.arange(q.shape[0], device=DEV)[:, None] + first
        sc = torch.where(torch.arange(k.shape[0], device=DEV)[None] <= i, sc, torch.full_like(sc, -math.inf))
    lse = torch.logsumexp(sc, -1)
    w = torch.exp(sc - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None])
    return w @ v, lse


def exact(case, seed):
    s = prepare(case, seed)
    new, held = _counts(case)
    op, hk, d = case["op"], case["heads_kv"], case["dim"]
    at = _prefix(new)
    if op == "append":
        out = {}
        for name in ("k", "v"):
            cache = s["cache_" + name].double()
            e = s.get("cache_%s_exp" % name)
            for b, (n, h) in enumerate(zip(new, held)):
                pages, ps = s["table"][b].tolist(), case["page"]
                page = torch.tensor([pages[p // ps] for p in range(h - n, h)], device=DEV)
                off = torch.tensor([p % ps for p in range(h - n, h)], device=DEV)
                rows = s[name][at[b]:at[b + 1]]
                if e is None:
                    cache[page, off] = rows.double()
                else:
                    codes, exps = _exact_codes(rows)
                    cache[page, off] = codes
                    e.permute(0, 2, 1)[page, off] = exps
            out[name] = cache
            if e is not None:
                out[name + "_exp"] = e
        return out
    if op == "gather":
        return {name: torch.cat([_exact_row(s, name, b, range(h - n, h)) for b, (n, h) in enumerate(zip(new, held))])
                for name in ("k", "v")}
    hq = case["heads_q"]
    o = torch.empty(sum(new), hq, d, dtype=torch.float64, device=DEV)
    lse = torch.empty(sum(new), hq, dtype=torch.float64, device=DEV)
    from_k = _prefix(held)
    for b, (n, h) in enumerate(zip(new, held)):
        if op == "decode":
            k, v = _exact_row(s, "k", b, range(h)), _exact_row(s, "v", b, range(h))
        else:
            k, v = (s[x][from_k[b]:from_k[b + 1]].double() for x in "kv")
        rows = slice(at[b], at[b + 1])
        for head in range(hq):
            kv = head // (hq // hk)
            first = h - n if op == "prompt" and case["causal"] else None
            o[rows, head], lse[rows, head] = _exact_attention(s["q"][rows, head].double(), k[:, kv], v[:, kv], first)
    return {"o": o, "lse": lse}
