"""Timed cases of what a step of many requests needs beside the projections: rotary positions for its queries and keys,
pages for its new tokens, a key/value cache held in 4 bits, and attention over that cache.

Token counts run from one query (a step that adds a token) over prompts (hundreds of rows) and chunks of a clip (a few
thousand) to a whole clip (19200 rows, with 521 prompt rows before them); heads are those of the H3 block (56 x 128), of
the hidden-5120 block (40 x 128, also with 8 key/value heads that 5 query heads share) and generic ones of 64 and 256.

A cache of 4 bits is a pool of pages, one page a block of 64 tokens, and a table of pages for each sequence:
  k, v [pages, heads, 64, dim / 2] uint8: element 2 j in the low half of byte j, as a sign bit and the place of the value
  among 0, 0.5, 1, 1.5, 2, 3, 4, 6;
  k_scale, v_scale [pages, heads, dim / 32, 64] uint8: e + 127 of the factor 2^e of each 32 elements of a token (above 252:
  not a number).  e is the least of -125 .. 125 for which no element is above 7 2^e; values round to the nearest, to even.

Free pages are a stack, free[0 .. count - 1], taken from its end.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 64   # tokens of a block, and of a page
GROUP = 32   # elements that share a scale
BF16 = torch.bfloat16

# The largest listed attention: no drawn case has more (query, token, head) pairs, or elements of cache.
_MAX_PAIRS = 4800 * 19721 * 56
_MAX_CACHE = 4 * 131072 * 8 * 128


def listed():
    return [
        # Queries and keys of one more token in each of 8 sequences: latency counts.
        {"name": "rope_token", "kind": "rope", "n": 8, "rows": 1, "before": 2477, "heads": 56, "kv": 56, "dim": 128, "rot": 128,
         "interleaved": False, "factor": 1.0, "inverse": False, "inplace": True, "ragged": True},
        # Chunks of 4 uneven sequences far into long contexts: half of each head, in pairs of neighbours, 5 query heads to a
        # key head, frequencies scaled for 16 times the length, into new tensors.
        {"name": "rope_chunk_2401", "kind": "rope", "n": 4, "rows": 2401, "before": 131072, "heads": 40, "kv": 8, "dim": 128, "rot": 64,
         "interleaved": True, "factor": 16.0, "inverse": False, "inplace": False, "ragged": True},
        # A whole clip's gradients, turned back: the largest.
        {"name": "rope_clip_19200", "kind": "rope", "n": 1, "rows": 19200, "before": 521, "heads": 56, "kv": 56, "dim": 128, "rot": 128,
         "interleaved": False, "factor": 1.0, "inverse": True, "inplace": True, "ragged": False},
        # One more token in each of 256 sequences: a few of them need a page.
        {"name": "pages_token_256", "kind": "extend", "n": 256, "rows": 1, "before": 19721, "blocks": 2048, "ragged": True},
        # 32 prompts come and go: pages taken for them, and given back.
        {"name": "pages_prompts_521", "kind": "admit", "n": 32, "rows": 521, "before": 0, "blocks": 309, "ragged": True},
        # 8 clips behind what their sequences hold already: the largest.
        {"name": "pages_clips_19200", "kind": "admit", "n": 8, "rows": 19200, "before": 521, "blocks": 2048, "ragged": True},
        # One more token in each of 8 sequences, into partly filled blocks, and back: latency counts.
        {"name": "write4_token", "kind": "write", "n": 8, "rows": 1, "before": 2477, "heads": 56, "dim": 128, "ragged": True},
        # A whole clip of H3's block behind its prompt, so that its first block is partly filled: the largest write.
        {"name": "write4_clip_19200", "kind": "write", "n": 1, "rows": 19200, "before": 521, "heads": 56, "dim": 128, "ragged": False},
        # A single query over a clip and its prompt: every head reads its own keys and values once.
        {"name": "attend4_token", "kind": "attend", "n": 1, "rows": 1, "tokens": 19721, "heads": 56, "kv": 56, "dim": 128,
         "causal": True, "ragged": False},
        # A step of 16 sequences of uneven lengths, 5 query heads to a key/value head.
        {"name": "attend4_tokens_16", "kind": "attend", "n": 16, "rows": 1, "tokens": 32768, "heads": 40, "kv": 8, "dim": 128,
         "causal": True, "ragged": True},
        # Two prompts of uneven lengths, each over itself.
        {"name": "attend4_prompt_512", "kind": "attend", "n": 2, "rows": 512, "tokens": 512, "heads": 40, "kv": 40, "dim": 128,
         "causal": True, "ragged": True},
        # A chunk of a clip over the clip and its prompt: the largest product.
        {"name": "attend4_chunk_4800", "kind": "attend", "n": 1, "rows": 4800, "tokens": 19721, "heads": 56, "kv": 56, "dim": 128,
         "causal": False, "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choices(["rope", "extend", "admit", "write", "attend"], [3, 1, 2, 2, 5])[0]
    if kind in ("extend", "admit"):
        n = _log(rng, 1, 256)
        rows = rng.choice([1, rng.randint(1, 3)]) if kind == "extend" else _log(rng, 1, 8 * 19200 // n)
        before = rng.choice([0, _log(rng, 1, 19721)])
        # a pass of "extend" leaves its tokens there: room for many passes
        blocks = 2048 if kind == "extend" else -(-(rows + before) // BLOCK) + rng.randint(0, 300)
        return {"kind": kind, "n": n, "rows": rows, "before": before, "blocks": blocks, "ragged": n > 1 and rng.random() < 0.7}
    heads, kv, dim = rng.choice([(56, 56, 128), (56, 56, 128), (40, 40, 128), (40, 8, 128), (24, 24, 64), (20, 20, 256), (20, 4, 256)])
    n = rng.choice([1, 1, 1, 2, 3, 8, 16])
    ragged = n > 1 and rng.random() < 0.7
    if kind == "rope":
        rows = _log(rng, 1, 19200 // n * 56 * 128 // (heads * dim))
        rot = rng.choice([dim, dim, dim // 2, dim // 4, rng.randint(1, dim // 2) * 2])
        factor = rng.choice([1.0, 1.0, 4.0, 16.0])
        # (a factor grows the result, in place with every pass)
        return {"kind": kind, "n": n, "rows": rows, "before": rng.choice([0, _log(rng, 1, 1000000)]), "heads": heads, "kv": kv, "dim": dim,
                "rot": rot, "interleaved": rng.random() < 0.5, "factor": factor, "inverse": rng.random() < 0.3,
                "inplace": factor == 1.0 and rng.random() < 0.8, "ragged": ragged}
    if kind == "write":
        rows = _log(rng, 1, 19200 // n)
        return {"kind": kind, "n": n, "rows": rows, "before": rng.choice([0, _log(rng, 1, 4800)]), "heads": kv, "dim": dim,
                "ragged": ragged}
    rows = rng.choice([1, rng.randint(1, 16), _log(rng, 16, 4800), _log(rng, 16, 4800)])
    rows = min(rows, _MAX_CACHE // (n * kv * dim), math.isqrt(_MAX_PAIRS * 128 // (n * heads * dim)))
    most = min(131072, _MAX_CACHE // (n * kv * dim), _MAX_PAIRS * 128 // (n * heads * dim * rows))
    return {"kind": kind, "n": n, "rows": rows, "tokens": _log(rng, rows, most), "heads": heads, "kv": kv, "dim": dim,
            "causal": rng.random() < 0.6, "ragged": ragged}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _keys(g, n, rows, heads, dim):
    """N(0, 1) around a centre of each run of 64 tokens, as neighbouring patches and words are alike."""
    x = torch.randn(n, rows, heads, dim, generator=g, device="cuda")
    centre = torch.randn(n, -(-rows // BLOCK), heads, dim, generator=g, device="cuda") * 0.5
    return x.add_(centre.repeat_interleave(BLOCK, 1)[:, :rows]).to(BF16)


def _lengths(g, n, most, least, ragged):
    """Lengths of n sequences: the first is the longest, the others (ragged) anything down to `least`."""
    t = torch.full((n,), most, device="cuda", dtype=torch.int32)
    if ragged and n > 1:
        t[1:] = torch.randint(least, most + 1, (n - 1,), generator=g, device="cuda", dtype=torch.int32)
    return t


def _tables(g, n, blocks):
    """Pages of each sequence, in no order, from a pool with a few more."""
    return torch.randperm(n * blocks + 3, generator=g, device="cuda")[:n * blocks].reshape(n, blocks).to(torch.int32)


def _cache(g, tables, heads, dim):
    """A cache whose blocks hold keys and values of 4 bits; the pages of no sequence hold old ones."""
    pages = tables.numel() + 3
    got = {}
    for name in ("k", "v"):
        x = _keys(g, 1, pages * BLOCK, heads, dim).reshape(pages, BLOCK, heads, dim).transpose(1, 2)
        got[name], scale = _quantize(x)
        got[name + "_scale"] = scale.transpose(2, 3).contiguous()
    return got


def _frequencies(rot, factor, base=10000.0, window=8192):
    """(radians a token of each pair, in 64 bits, factor of the result).  For contexts of `factor` times `window` tokens, pairs
    that turn less than once in the window are slowed by the factor, those that turn 32 times and more are left, and the
    others lie between; the result grows by 1 + 0.1 ln factor."""
    f = base ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / -rot)
    if factor == 1.0:
        return f, 1.0
    at = lambda turns: rot * math.log(window / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    keep = 1 - ((torch.arange(rot // 2, device="cuda", dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f * (keep + (1 - keep) / factor), 1 + 0.1 * math.log(factor)


def prepare(case, seed):
    g, kind, n = _gen(seed), case["kind"], case["n"]
    st = {"case": case}
    if kind == "rope":
        rows, heads, kv, dim = case["rows"], case["heads"], case["kv"], case["dim"]
        # views of a projection's output: query heads, key heads, value heads of each token
        qkv = torch.randn(n, rows, heads + 2 * kv, dim, generator=g, device="cuda").to(BF16)
        st["q"], st["k"] = qkv[:, :, :heads], qkv[:, :, heads:heads + kv]
        counts, start = _lengths(g, n, rows, 1, case["ragged"]), _lengths(g, n, case["before"], case["before"] // 2, case["ragged"])
        r = torch.arange(rows, device="cuda", dtype=torch.int32)
        st["positions"] = torch.where(r < counts[:, None], start[:, None] + r, -1)  # -1: no row of the sequence
        st["freqs"], st["amplitude"] = _frequencies(case["rot"], case["factor"])
        return st
    if kind in ("extend", "admit"):
        rows, before, blocks = case["rows"], case["before"], case["blocks"]
        st["counts"] = _lengths(g, n, rows, 1, case["ragged"])
        st["lens"] = _lengths(g, n, before, before // 2, case["ragged"])
        st["before"] = st["lens"].clone()
        have = (st["lens"] + BLOCK - 1) // BLOCK
        pages = n * blocks
        stack = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        held = torch.arange(blocks, device="cuda") < have[:, None]
        place = (torch.cumsum(held.reshape(-1), 0).reshape(n, blocks) - 1).clamp_min(0)
        st["tables"] = torch.where(held, stack[pages - 1 - place], -1).to(torch.int32)
        st["count"] = (pages - have.sum()).to(torch.int32).reshape(1)
        st["free"] = stack
        return st
    if kind == "write":
        rows, before, heads, dim = case["rows"], case["before"], case["heads"], case["dim"]
        st["tables"] = _tables(g, n, -(-(rows + before) // BLOCK))
        st["cache"] = _cache(g, st["tables"], heads, dim)
        st["counts"] = _lengths(g, n, rows, 1, case["ragged"])
        st["starts"] = _lengths(g, n, before, before // 2, case["ragged"])
        st["lens"] = st["counts"] + st["starts"]
        kv = torch.stack([_keys(g, n, rows, heads, dim), _keys(g, n, rows, heads, dim) * 2], 2)
        st["k"], st["v"] = kv[:, :, 0], kv[:, :, 1]
        return st
    rows, tokens, heads, kv, dim = (case[k] for k in ("rows", "tokens", "heads", "kv", "dim"))
    st["tables"] = _tables(g, n, -(-tokens // BLOCK))
    st["cache"] = _cache(g, st["tables"], kv, dim)
    st["counts"] = _lengths(g, n, rows, 1, case["ragged"])
    st["lens"] = _lengths(g, n, tokens, rows, case["ragged"])
    if rows == tokens:
        st["lens"] = st["counts"].clone()  # prompts over themselves
    st["q"] = _keys(g, n, rows, heads, dim)
    return st


# ------------------------------------------------------------------ plain forms


def _quantize(x):
    """x [..., dim] -> (bytes [..., dim / 2], scales [..., dim / 32])."""
    x = x.float().unflatten(-1, (-1, GROUP))
    a = x.abs().amax(-1)
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1)
    e = torch.where(a == 0, -125, (e - 3 + (m > 0.875).to(e.dtype)).clamp(-125, 125))
    bad = ~torch.isfinite(a)
    y = torch.where(bad[..., None], 0.0, torch.ldexp(x, -e[..., None]))
    t = y.abs()
    code = torch.where(t < 2, torch.round(2 * t), torch.where(t < 4, 2 + torch.round(t), 4 + torch.round(t / 2))).clamp_max(7)
    code = (code.to(torch.uint8) + 8 * torch.signbit(y).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.where(bad, 255, e + 127).to(torch.uint8)


def _values(q, scale, dtype=torch.float32):
    """bytes [..., dim / 2] and scales [..., dim / 32] -> [..., dim]."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda", dtype=dtype)
    x = table[torch.stack([q & 15, q >> 4], -1).flatten(-2).int()].unflatten(-1, (-1, GROUP))
    f = torch.ldexp(torch.ones((), device="cuda", dtype=dtype), scale.int() - 127)
    return (x * torch.where(scale > 252, math.nan, f)[..., None]).flatten(-2)


def _plain_rope(st):
    case, rot = st["case"], st["case"]["rot"]
    at = st["positions"]
    # 64 bits: far positions have thousands of turns
    angle = at.double()[..., None] * st["freqs"]
    c, s = (f(angle).mul_(st["amplitude"]).float()[:, :, None] for f in (torch.cos, torch.sin))
    if case["inverse"]:
        s = -s
    there = (at >= 0)[..., None, None]
    out = []
    for x in (st["q"], st["k"]):
        y = x if case["inplace"] else x.clone(memory_format=torch.contiguous_format)
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["interleaved"] else (x[..., :rot // 2], x[..., rot // 2:rot])
        af, bf = a.float(), b.float()
        pair = [torch.where(there, z.to(BF16), w) for z, w in ((af * c - bf * s, a), (af * s + bf * c, b))]
        y[..., :rot] = torch.stack(pair, -1).flatten(-2) if case["interleaved"] else torch.cat(pair, -1)
        out.append(y)
    return out


def _plain_extend(st):
    n, blocks = st["tables"].shape
    rows, pages = st["case"]["rows"], st["free"].shape[0]
    c = st["counts"].long().clamp(0, rows)
    old = st["lens"].long().clamp_min(0)
    have = (old + BLOCK - 1) // BLOCK
    fits = old + c <= BLOCK * blocks
    want = torch.where(fits, (old + c + BLOCK - 1) // BLOCK - have, 0)
    upto = torch.cumsum(want, 0)
    given = fits & (upto <= st["count"])
    granted = torch.where(given, c, 0)
    b = torch.arange(blocks, device="cuda")
    new = given[:, None] & (b >= have[:, None]) & (b < (have + want)[:, None])
    place = st["count"].long() - 1 - ((upto - want)[:, None] + b - have[:, None])
    st["tables"].copy_(torch.where(new, st["free"][place.clamp(0, pages - 1)], st["tables"]))
    st["count"].sub_((want * given).sum().int())
    st["lens"].copy_(torch.where(st["lens"] < 0, 0, st["lens"]) + granted.int())
    r = torch.arange(rows, device="cuda")
    at = torch.where(r < granted[:, None], old[:, None] + r, -1)
    page = st["tables"].long().gather(1, (at // BLOCK).clamp(0, blocks - 1))
    slots = torch.where((at >= 0) & (page >= 0) & (page < pages), page * BLOCK + at % BLOCK, -1)
    return granted.int(), at.int(), slots


def _plain_release(st, keep):
    n, blocks = st["tables"].shape
    pages = st["free"].shape[0]
    old = st["lens"].long().clamp_min(0)
    left = torch.minimum(old, keep.long().clamp_min(0))
    b = torch.arange(blocks, device="cuda")
    gone = (b >= ((left + BLOCK - 1) // BLOCK)[:, None]) & (b < ((old + BLOCK - 1) // BLOCK)[:, None])
    good = gone & (st["tables"] >= 0) & (st["tables"] < pages)
    place = st["count"] + torch.cumsum(good.reshape(-1).long(), 0) - 1
    place = torch.where(good.reshape(-1) & (place < pages), place, pages)
    grown = torch.nn.functional.pad(st["free"], (0, 1)).scatter_(0, place, st["tables"].reshape(-1))
    st["free"].copy_(grown[:pages])
    st["count"].copy_((st["count"] + good.sum()).clamp_max(pages))
    st["tables"].masked_fill_(gone, -1)
    st["lens"].copy_(left)


def _plain_write(st):
    cache, rows = st["cache"], st["k"].shape[1]
    r = torch.arange(rows, device="cuda")
    who, row = torch.nonzero(r < st["counts"][:, None], as_tuple=True)
    at = st["starts"].long()[who] + row
    page, off = st["tables"].long()[who, at // BLOCK], at % BLOCK
    heads = torch.arange(st["k"].shape[2], device="cuda")
    for name in ("k", "v"):
        q, scale = _quantize(st[name][who, row])
        cache[name][page[:, None], heads, off[:, None]] = q
        cache[name + "_scale"].transpose(2, 3)[page[:, None], heads, off[:, None]] = scale


def _plain_read(st, length):
    cache, tables = st["cache"], st["tables"].long()
    at = st["starts"].long()[:, None] + torch.arange(length, device="cuda")
    page = tables.gather(1, (at // BLOCK).clamp_max(tables.shape[1] - 1))
    there = (at < st["lens"].long()[:, None])[..., None, None]
    k, v = (_values(cache[x][page, :, at % BLOCK], cache[x + "_scale"][page, :, :, at % BLOCK]) for x in ("k", "v"))
    return torch.where(there, k, 0.0).to(BF16), torch.where(there, v, 0.0).to(BF16)


def _plain_attention(st):
    case, cache = st["case"], st["cache"]
    n, rows, heads, dim = st["q"].shape
    kv, page = cache["k"].shape[1], st["tables"].long()
    lens, counts = st["lens"].long(), st["counts"].long()
    span = page.shape[1] * BLOCK
    k, v = (_values(cache[x][page], cache[x + "_scale"][page].transpose(3, 4)).transpose(1, 2).reshape(n, kv, 1, span, dim) for x in ("k", "v"))
    q = (st["q"].float() * dim ** -0.5).reshape(n, rows, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    s = q @ k.transpose(3, 4)
    t = torch.arange(span, device="cuda")
    r = torch.arange(rows, device="cuda")
    hidden = (t >= lens[:, None])[:, None] | (r >= counts[:, None])[..., None]
    if case["causal"]:
        hidden = hidden | (t > ((lens - counts)[:, None] + r)[..., None])
    s.masked_fill_(hidden[:, None, None], -math.inf)
    top = s.amax(4, keepdim=True)
    s.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = s.sum(4, keepdim=True)
    o = (s @ v) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(n, rows, heads, dim).to(BF16)


# ------------------------------------------------------------------ one pass


def _package():
    at = os.path.join(os.getcwd(), "minimax-h3-multi-dgx-spark_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import h3mi
    return h3mi


def run(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "rope":
        if own:
            h3mi = _package()
            f = h3mi.rotary_ if case["inplace"] else h3mi.rotary
            return f(st["q"], st["k"], st["positions"], st["freqs"], interleaved=case["interleaved"], inverse=case["inverse"],
                     amplitude=st["amplitude"])
        return _plain_rope(st)
    if kind in ("extend", "admit"):  # "admit": the sequences' new tokens are dropped again
        if own:
            h3mi = _package()
            pool = h3mi.KVPool(st["free"], st["count"])
            granted, positions, slots = h3mi.kv_extend_(pool, st["tables"], st["lens"], case["rows"], counts=st["counts"])
            if kind == "admit":
                h3mi.kv_release_(pool, st["tables"], st["lens"], st["before"])
        else:
            granted, positions, slots = _plain_extend(st)
            if kind == "admit":
                _plain_release(st, st["before"])
        return {"granted": granted, "positions": positions, "slots": slots, "tables": st["tables"], "lens": st["lens"],
                "free": st["free"], "count": st["count"]}
    if kind == "write":  # write, then the tokens read back
        if own:
            h3mi = _package()
            cache = h3mi.KVCache4(**st["cache"])
            h3mi.kv_write_(cache, st["k"], st["v"], st["tables"], st["lens"], counts=st["counts"])
            k, v = h3mi.kv_read(cache, st["tables"], st["lens"], case["rows"], starts=st["starts"])
        else:
            _plain_write(st)
            k, v = _plain_read(st, case["rows"])
        return {"k": k, "v": v, "k_scale": st["cache"]["k_scale"], "v_scale": st["cache"]["v_scale"]}
    if own:
        h3mi = _package()
        return h3mi.kv_attention(st["q"], h3mi.KVCache4(**st["cache"]), st["tables"], st["lens"], causal=case["causal"],
                                 counts=st["counts"])
    return _plain_attention(st)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    """Bytes and operations at the longest lengths of the case (the others of a ragged batch are about half as long)."""
    n, kind = case["n"], case["kind"]
    share = (1 + (n - 1) * 0.5) / n if case.get("ragged") else 1.0
    if kind == "rope":
        tokens, heads = n * share * case["rows"], case["heads"] + case["kv"]
        # in place the turned elements, else all of every row
        e = tokens * heads * case["rot"] if case["inplace"] else n * case["rows"] * heads * case["dim"]
        return {"bytes": int(4 * e + 4 * n * case["rows"] + 4 * case["rot"]), "flops": int(3 * tokens * heads * case["rot"])}
    if kind in ("extend", "admit"):
        # lengths and counts, positions and slots; a page of each new block off the stack and into the table, and back
        pages = n * share * case["rows"] / BLOCK
        return {"bytes": int(n * 20 + n * case["rows"] * 12 + pages * (8 if kind == "extend" else 20)), "flops": 0}
    dim = case["dim"]
    row = dim * 0.5 + dim / GROUP  # bytes of a token and head, of keys or of values
    if kind == "write":
        # bf16 read, 4 bits written; those read, and bf16 written, zeros behind the sequences' ends too
        e = n * case["heads"] * case["rows"]
        return {"bytes": int(2 * e * (share * (2 * dim + 2 * row) + 2 * dim)), "flops": 0}
    rows, tokens, heads, kv = (case[k] for k in ("rows", "tokens", "heads", "kv"))
    seen = tokens
    if case["causal"]:
        seen = tokens - (rows - 1) / 2 if rows < tokens else (tokens + 1) / 2
    return {"bytes": int(2 * n * share * tokens * kv * row + 4 * n * rows * heads * dim * share),
            "flops": int(4 * n * share * rows * heads * dim * seen)}


# ------------------------------------------------------------------ from the definition, in 64 bits


def _exact_rope(st):
    case, rot = st["case"], st["case"]["rot"]
    half = rot // 2
    turn = torch.polar(torch.full((), st["amplitude"], device="cuda", dtype=torch.float64), st["positions"].double()[..., None] * st["freqs"])
    if case["inverse"]:
        turn = turn.conj()
    first = torch.arange(half, device="cuda") * 2 if case["interleaved"] else torch.arange(half, device="cuda")
    second = first + (1 if case["interleaved"] else half)
    out = []
    for x in (st["q"], st["k"]):
        y = x.double().clone(memory_format=torch.contiguous_format)
        for i in range(y.shape[0]):
            rows = torch.nonzero(st["positions"][i] >= 0)[:, 0]
            z = torch.complex(y[i][rows][..., first], y[i][rows][..., second]) * turn[i, rows, None]
            part = y[i][rows]
            part[..., first], part[..., second] = z.real, z.imag
            y[i][rows] = part
        out.append(y)
    return out


def _exact_write(st):
    """Token by token: the nearest value, of two as near the one whose place is even."""
    rows = st["k"].shape[1]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda", dtype=torch.float64)
    out = {"k_scale": None, "v_scale": None}
    for name in ("k", "v"):
        got = torch.zeros(st[name].shape, device="cuda", dtype=torch.float64)
        for i in range(got.shape[0]):
            count = int(st["counts"][i])
            for lo in range(0, count, 1024):
                x = st[name][i, lo:min(lo + 1024, count)].double().unflatten(-1, (-1, GROUP))
                f = 2.0 ** torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -125) / 7)).clamp(-125, 125)
                far = (x.abs() / f)[..., None] - grid
                far = far.abs() + torch.tensor([0, 1e-9] * 4, device="cuda", dtype=torch.float64)
                got[i, lo:lo + 1024][:x.shape[0]] = (grid[far.argmin(-1)] * f * x.sign()).flatten(-2)
        out[name] = got
    return out


def _exact_attention(st):
    case, c = st["case"], st["cache"]
    n, rows, heads, dim = st["q"].shape
    group = heads // case["kv"]
    out = torch.zeros(n, rows, heads, dim, device="cuda", dtype=torch.float64)
    for i in range(n):
        end, count = int(st["lens"][i]), int(st["counts"][i])
        page = st["tables"][i, :-(-end // BLOCK)].long()
        t, at = torch.arange(end, device="cuda"), end - count + torch.arange(count, device="cuda")
        hide = t > at[:, None] if case["causal"] else None
        for h in range(case["kv"]):
            k, v = (_values(c[x][page, h], c[x + "_scale"][page, h].transpose(1, 2), torch.float64).flatten(0, 1)[:end] for x in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                s = st["q"][i, :count, j].double() @ k.t() * dim ** -0.5
                out[i, :count, j] = torch.softmax(s if hide is None else s.masked_fill_(hide, -math.inf), 1) @ v
    return torch.nan_to_num(out)  # rows that see no token are zero


def exact(case, seed):
    kind = case["kind"]
    if kind in ("extend", "admit"):
        return None  # whole numbers
    st = prepare(case, seed)
    return _exact_rope(st) if kind == "rope" else _exact_write(st) if kind == "write" else _exact_attention(st)
