"""Timed cases of the 8-bit key/value cache: writing it, reading it back, and attention over it.

Token counts run from one query (a step that adds a token) over prompts (hundreds of rows) and chunks of a clip (a few
thousand) to a whole clip (19200 or 38400 rows, with 521 prompt rows before them); heads are those of the H3 block
(56 x 128), of the hidden-5120 block (40 x 128, also with 8 key/value heads that 5 query heads share) and generic ones
of 64 and 256.

A cache is a pool of pages, one page a block of 64 tokens, and a table of pages for each sequence:
  k [pages, heads, 64, dim] int8, v [pages, heads, dim, 64] int8 (values transposed),
  k_scale, v_scale [pages, heads] fp32, k_sum [pages, heads, dim] int16 (sum of the block's 8-bit keys).
"""
import math
import os
import sys

import torch

own = False

BLOCK = 64   # tokens of a block, and of a page
TILE = 128   # query rows that share a selection
BF16 = torch.bfloat16

# The largest listed attention: no drawn case has more (query, token, head) pairs, or elements of cache.
_MAX_PAIRS = 4800 * 19721 * 56
_MAX_CACHE = 4 * 131072 * 8 * 128


def listed():
    return [
        # One more token in each of 8 sequences: the smallest write, into partly filled blocks; latency counts.
        {"name": "write_token", "kind": "write", "n": 8, "rows": 1, "before": 2477, "heads": 56, "dim": 128, "ragged": True},
        # A share of a clip behind 521 prompt rows, so that its first block is partly filled.
        {"name": "write_chunk_2401", "kind": "write", "n": 1, "rows": 2401, "before": 521, "heads": 56, "dim": 128, "ragged": False},
        # A whole clip of H3's block: the largest write.
        {"name": "write_clip_19200", "kind": "write", "n": 1, "rows": 19200, "before": 0, "heads": 56, "dim": 128, "ragged": False},
        # A prompt's keys and values, taken back out for a block that runs on bf16.
        {"name": "read_prompt_521", "kind": "read", "n": 1, "length": 521, "heads": 40, "dim": 128},
        # A whole clip's.
        {"name": "read_clip_19200", "kind": "read", "n": 1, "length": 19200, "heads": 56, "dim": 128},
        # A single query over a clip and its prompt: every head reads its own keys and values once.
        {"name": "attend_token", "kind": "attend", "n": 1, "rows": 1, "tokens": 19721, "heads": 56, "kv": 56, "dim": 128,
         "causal": True, "ragged": False},
        # A step of 16 sequences of uneven lengths, 5 query heads to a key/value head.
        {"name": "attend_tokens_16", "kind": "attend", "n": 16, "rows": 1, "tokens": 32768, "heads": 40, "kv": 8, "dim": 128,
         "causal": True, "ragged": True},
        # Two prompts of uneven lengths, each over itself.
        {"name": "attend_prompt_512", "kind": "attend", "n": 2, "rows": 512, "tokens": 512, "heads": 40, "kv": 40, "dim": 128,
         "causal": True, "ragged": True},
        # A chunk of a clip over the clip and its prompt: the largest product.
        {"name": "attend_chunk_4800", "kind": "attend", "n": 1, "rows": 4800, "tokens": 19721, "heads": 56, "kv": 56, "dim": 128,
         "causal": False, "ragged": False},
        # A step of 4 sequences over long caches, each over the 64 blocks that its query selects.
        {"name": "sparse_tokens_4", "kind": "sparse", "n": 4, "rows": 1, "tokens": 131072, "heads": 40, "kv": 8, "dim": 128,
         "causal": True, "ragged": True, "top": 64},
        # A small model's chunk over a quarter of its blocks.
        {"name": "sparse_chunk_1201", "kind": "sparse", "n": 1, "rows": 1201, "tokens": 9600, "heads": 24, "kv": 24, "dim": 64,
         "causal": True, "ragged": False, "top": 38},
        # H3's chunk over a sixth of a long clip.
        {"name": "sparse_chunk_2401", "kind": "sparse", "n": 1, "rows": 2401, "tokens": 38921, "heads": 56, "kv": 56, "dim": 128,
         "causal": False, "ragged": False, "top": 100},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choices(["write", "read", "attend", "sparse"], [2, 1, 4, 3])[0]
    heads, kv, dim = rng.choice([(56, 56, 128), (56, 56, 128), (40, 40, 128), (40, 8, 128), (24, 24, 64), (20, 20, 256), (20, 4, 256)])
    n = rng.choice([1, 1, 1, 2, 3, 8, 16])
    ragged = n > 1 and rng.random() < 0.7
    if kind == "write":
        rows = _log(rng, 1, 19200 // n)
        return {"kind": kind, "n": n, "rows": rows, "before": rng.choice([0, _log(rng, 1, 4800)]), "heads": kv, "dim": dim,
                "ragged": ragged}
    if kind == "read":
        return {"kind": kind, "n": n, "length": _log(rng, 1, 19200 // n), "heads": kv, "dim": dim}
    rows = rng.choice([1, rng.randint(1, 16), _log(rng, 16, 4800), _log(rng, 16, 4800)])
    rows = min(rows, _MAX_CACHE // (n * kv * dim), math.isqrt(_MAX_PAIRS * 128 // (n * heads * dim)))
    most = min(131072, _MAX_CACHE // (n * kv * dim), _MAX_PAIRS * 128 // (n * heads * dim * rows))
    tokens = _log(rng, rows, most)
    case = {"kind": kind, "n": n, "rows": rows, "tokens": tokens, "heads": heads, "kv": kv, "dim": dim, "causal": rng.random() < 0.6,
            "ragged": ragged}
    return case if kind == "attend" else {**case, "top": _log(rng, 3, min(256, max(4, tokens // BLOCK)))}


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
    """A cache whose blocks hold keys and values, quantized a block at a time; the pages of no sequence hold old ones."""
    pages = tables.numel() + 3
    got = {}
    for name in ("k", "v"):
        x = _keys(g, 1, pages * BLOCK, heads, dim).reshape(pages, BLOCK, heads, dim).transpose(1, 2)
        s = x.abs().amax((2, 3)).float() / 127
        q = torch.round(x.float() / s[:, :, None, None]).clamp_(-127, 127).to(torch.int8)
        got[name] = (q if name == "k" else q.transpose(2, 3)).contiguous()
        got[name + "_scale"] = s
    got["k_sum"] = got["k"].sum(2, dtype=torch.int16)
    return got


def prepare(case, seed):
    g, kind, n = _gen(seed), case["kind"], case["n"]
    st = {"case": case}
    if kind == "write":
        rows, before, heads, dim = case["rows"], case["before"], case["heads"], case["dim"]
        blocks = -(-(rows + before) // BLOCK)
        st["tables"] = _tables(g, n, blocks)
        st["cache"] = _cache(g, st["tables"], heads, dim)
        st["counts"] = _lengths(g, n, rows, 1, case["ragged"])
        st["lens"] = st["counts"] + _lengths(g, n, before, before // 2, case["ragged"])
        # views of a projection's output: key heads, then value heads, of each token
        kv = torch.stack([_keys(g, n, rows, heads, dim), _keys(g, n, rows, heads, dim) * 2], 2)
        st["k"], st["v"] = kv[:, :, 0], kv[:, :, 1]
        st["starts"] = (st["lens"] - st["counts"]) // BLOCK * BLOCK  # back from the first block that changes
        return st
    if kind == "read":
        blocks = -(-case["length"] // BLOCK)
        st["tables"] = _tables(g, n, blocks)
        st["cache"] = _cache(g, st["tables"], case["heads"], case["dim"])
        st["lens"] = _lengths(g, n, case["length"], 1, n > 1)
        st["starts"] = torch.zeros_like(st["lens"])
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



def _quantize(x, s):
    """The 8-bit values (as fp32) of x under scales s that broadcast with it."""
    q = torch.round(x / s).clamp_(-127, 127)
    return torch.where((s > 0) & torch.isfinite(s), q, torch.zeros_like(q))


def _write_one(x, old, s_old, fresh, new, kept):
    """x [n, blocks, 64, heads, dim] fp32, zero where no token is new; old [n, blocks, heads, 64, dim] ints as fp32;
    s_old [n, blocks, heads]; fresh [n, blocks]; new, kept [n, blocks, 64]: the tokens written now, and those before."""
    a = x.abs().amax((2, 4)) / 127
    r = a / s_old
    m, e = torch.frexp(r)
    fold = torch.where(r > 1, e - (m == 0.5).to(e.dtype), torch.zeros_like(e))  # least k with 2^k >= r
    again = fresh[:, :, None] | (s_old == 0) | ~(r <= 256)
    s = torch.where(again, a, torch.ldexp(s_old, fold))
    s = torch.where(~fresh[:, :, None] & ~torch.isfinite(s_old), s_old, s)
    fold = torch.where(again, torch.full_like(fold, 16), fold)
    held = torch.round(torch.ldexp(old, -fold[..., None, None])) * kept[:, :, None, :, None]
    q = _quantize(x.transpose(2, 3), s[..., None, None])
    return torch.where(new[:, :, None, :, None], q, held), s


def _plain_write(st):
    cache, tables, lens, counts = st["cache"], st["tables"], st["lens"].long(), st["counts"].long()
    n, rows = st["k"].shape[:2]
    start = lens - counts
    b = (start // BLOCK)[:, None] + torch.arange((rows + 126) // BLOCK, device="cuda")
    at = b[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")
    new = (at >= start[:, None, None]) & (at < lens[:, None, None])
    kept = at < start[:, None, None]
    live = new.any(2)
    page = tables.long().gather(1, b.clamp_max(tables.shape[1] - 1))
    row = (at - start[:, None, None]).clamp_(0, rows - 1)
    who = torch.arange(n, device="cuda")[:, None, None]
    fresh = start[:, None] <= b * BLOCK
    for name in ("k", "v"):
        x = st[name][who, row].float() * new[..., None, None]
        old = cache[name][page]
        if name == "v":
            old = old.transpose(3, 4)
        q, s = _write_one(x, old.float(), cache[name + "_scale"][page], fresh, new, kept)
        q = q.to(torch.int8)
        cache[name][page[live]] = (q if name == "k" else q.transpose(3, 4))[live]
        cache[name + "_scale"][page[live]] = s[live]
        if name == "k":
            cache["k_sum"][page[live]] = q.sum(3, dtype=torch.int16)[live]


def _plain_read(st, length):
    cache, tables = st["cache"], st["tables"].long()
    at = st["starts"].long()[:, None] + torch.arange(length, device="cuda")
    page = tables.gather(1, (at // BLOCK).clamp_max(tables.shape[1] - 1))
    there = (at < st["lens"].long()[:, None])[..., None, None]
    k = cache["k"][page, :, at % BLOCK].float() * cache["k_scale"][page][..., None]
    v = cache["v"][page, :, :, at % BLOCK].float() * cache["v_scale"][page][..., None]
    return torch.where(there, k, 0.0).to(BF16), torch.where(there, v, 0.0).to(BF16)


def _plain_select(st):
    case, cache = st["case"], st["cache"]
    n, rows, heads, dim = st["q"].shape
    kv, top = cache["k"].shape[1], case["top"]
    tiles = -(-rows // TILE)
    lens, counts = st["lens"].long(), st["counts"].long()
    page = st["tables"].long()
    row = torch.arange(tiles * TILE, device="cuda").reshape(tiles, TILE)
    # 64 bits: the sums are whole multiples of their smallest term, so no order of adding them rounds
    q = torch.nn.functional.pad(st["q"].double(), (0, 0, 0, 0, 0, tiles * TILE - rows))
    q = q * (row.reshape(-1) < counts[:, None])[..., None, None]
    p = q.reshape(n, tiles, TILE, kv, heads // kv, dim).sum((2, 4))
    most = p.abs().amax(3, keepdim=True)
    qi = torch.where((most > 0) & torch.isfinite(most), torch.round(p * 1023 / most), torch.zeros_like(p))
    dot = qi.transpose(1, 2) @ cache["k_sum"][page].double().permute(0, 2, 3, 1)  # [n, kv, tiles, blocks], whole numbers
    b = torch.arange(page.shape[1], device="cuda")
    held = (lens[:, None] - b * BLOCK).clamp(1, BLOCK).float()
    score = dot.float() * (cache["k_scale"][page] / held[..., None]).transpose(1, 2)[:, :, None]
    score = torch.where(torch.isnan(score), -math.inf, score)
    live = torch.minimum(row[:, -1] + 1, counts[:, None]) - row[:, 0]  # rows of each tile
    first = (lens - counts)[:, None] + row[:, 0]
    if case["causal"]:
        mine = (b >= first[..., None] // BLOCK) & (b <= (first + live - 1)[..., None] // BLOCK)
        score = torch.where(mine[:, None], math.inf, score)
        seen = (b <= (first + live - 1)[..., None] // BLOCK) & (live > 0)[..., None]
    else:
        seen = (b * BLOCK < lens[:, None])[:, None] & (live > 0)[..., None]
    score = torch.where(seen[:, None], score, -math.inf)
    take = min(top, page.shape[1])
    best = torch.sort(score, dim=3, descending=True, stable=True).indices[..., :take]
    best = torch.where(seen[:, None].expand_as(score).gather(3, best), best, page.shape[1]).sort(3).values
    best = torch.where(best == page.shape[1], -1, best)
    return torch.nn.functional.pad(best, (0, top - take), value=-1).transpose(1, 2).contiguous().to(torch.int32)


def _plain_attention(st, blocks=None):
    case, cache = st["case"], st["cache"]
    n, rows, heads, dim = st["q"].shape
    kv, page = cache["k"].shape[1], st["tables"].long()
    lens, counts = st["lens"].long(), st["counts"].long()
    span = page.shape[1] * BLOCK
    k = (cache["k"][page].float() * cache["k_scale"][page][..., None, None]).transpose(1, 2).reshape(n, kv, 1, span, dim)
    v = (cache["v"][page].float() * cache["v_scale"][page][..., None, None]).transpose(3, 4).transpose(1, 2).reshape(n, kv, 1, span, dim)
    q = (st["q"].float() * dim ** -0.5).reshape(n, rows, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    s = q @ k.transpose(3, 4)
    t = torch.arange(span, device="cuda")
    r = torch.arange(rows, device="cuda")
    hidden = (t >= lens[:, None])[:, None] | (r >= counts[:, None])[..., None]
    if case["causal"]:
        hidden = hidden | (t > ((lens - counts)[:, None] + r)[..., None])
    hidden = hidden[:, None, None]
    if blocks is not None:
        taken = torch.zeros(n, blocks.shape[1], kv, page.shape[1] + 1, device="cuda", dtype=torch.bool)
        taken.scatter_(3, torch.where(blocks < 0, page.shape[1], blocks).long(), True)
        taken = taken[..., :-1].transpose(1, 2).repeat_interleave(BLOCK, 3).repeat_interleave(TILE, 2)[:, :, :rows]
        hidden = hidden | ~taken[:, :, None]
    s.masked_fill_(hidden, -math.inf)
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
    if kind == "write":  # write, then the changed blocks' tokens read back
        length = case["rows"] + BLOCK - 1
        if own:
            h3mi = _package()
            cache = h3mi.KVCache(**st["cache"])
            h3mi.kv_write_(cache, st["k"], st["v"], st["tables"], st["lens"], counts=st["counts"])
            k, v = h3mi.kv_read(cache, st["tables"], st["lens"], length, starts=st["starts"])
        else:
            _plain_write(st)
            k, v = _plain_read(st, length)
        return {"k": k, "v": v, "k_scale": st["cache"]["k_scale"], "v_scale": st["cache"]["v_scale"], "k_sum": st["cache"]["k_sum"]}
    if kind == "read":
        if own:
            h3mi = _package()
            return h3mi.kv_read(h3mi.KVCache(**st["cache"]), st["tables"], st["lens"], case["length"], starts=st["starts"])
        return _plain_read(st, case["length"])
    if own:
        h3mi = _package()
        cache, blocks = h3mi.KVCache(**st["cache"]), None
        if kind == "sparse":
            blocks = h3mi.kv_select(st["q"], cache, st["tables"], st["lens"], case["top"], causal=case["causal"], counts=st["counts"])
        o = h3mi.kv_attention(st["q"], cache, st["tables"], st["lens"], causal=case["causal"], counts=st["counts"], blocks=blocks)
    else:
        blocks = _plain_select(st) if kind == "sparse" else None
        o = _plain_attention(st, blocks)
    return o if kind == "attend" else {"blocks": blocks, "out": o}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    """Bytes and operations at the longest lengths of the case (the others of a ragged batch are about half as long)."""
    n, dim, kind = case["n"], case["dim"], case["kind"]
    share = (1 + (n - 1) * 0.5) / n if case.get("ragged") or (kind == "read" and n > 1) else 1.0
    if kind in ("write", "read"):
        e = n * share * case["heads"] * dim
        if kind == "read":
            return {"bytes": int(e * case["length"] * 2 * (1 + 2 / share)), "flops": 0}
        blocks = -(-case["rows"] // BLOCK)
        # k and v read and their bytes written, sums and scales; then the bytes read back and bf16 written
        return {"bytes": int(e * (case["rows"] * 2 * (2 + 1 + 1) + blocks * 2 + 8 * blocks / dim)
                             + n * case["heads"] * dim * (case["rows"] + BLOCK - 1) * 4), "flops": 0}
    rows, tokens, heads, kv = (case[k] for k in ("rows", "tokens", "heads", "kv"))
    seen = tokens
    if case["causal"]:
        seen = tokens - (rows - 1) / 2 if rows < tokens else (tokens + 1) / 2
    rest = 4 * n * rows * heads * dim * share
    if kind == "attend":
        return {"bytes": int(2 * n * share * tokens * kv * dim + rest), "flops": int(4 * n * share * rows * heads * dim * seen)}
    tiles, blocks = -(-rows // TILE), -(-tokens // BLOCK)
    picked = min(case["top"], blocks)
    read = min(tokens, tiles * picked * BLOCK)
    return {"bytes": int(2 * n * share * kv * dim * (read + blocks) + rest + 4 * n * tiles * kv * case["top"]),
            "flops": int(4 * n * rows * heads * dim * min(seen, picked * BLOCK) * share + 2 * n * share * tiles * blocks * kv * dim)}


# ------------------------------------------------------------------ from the definition, in 64 bits


def _exact_write(st):
    """(k, v) [n, rows + 63, heads, dim] and the scales of every page, token by token of each sequence's changed blocks."""
    cache, rows = st["cache"], st["k"].shape[1]
    out = {"k_sum": None}
    for name in ("k", "v"):
        ints = cache[name].double() if name == "k" else cache[name].double().transpose(2, 3)
        scale = cache[name + "_scale"].double()
        got = torch.zeros(st["k"].shape[0], rows + BLOCK - 1, *st["k"].shape[2:], device="cuda", dtype=torch.float64)
        for i in range(got.shape[0]):
            end, count = int(st["lens"][i]), int(st["counts"][i])
            start, base = end - count, (end - count) // BLOCK * BLOCK
            x = st[name][i, :count].double()
            for b in range(start // BLOCK, -(-end // BLOCK)):
                lo, hi = max(start, b * BLOCK), min(end, (b + 1) * BLOCK)
                page, off = int(st["tables"][i, b]), lo - b * BLOCK
                new = x[lo - start:hi - start].transpose(0, 1)  # [heads, tokens, dim]
                # a scale is stored in 32 bits
                a = (new.abs().amax((1, 2)) / 127).float().double()
                s, held = a, torch.zeros_like(ints[page, :, :off])
                if off:
                    r = a / scale[page]
                    k = torch.ceil(torch.log2(r.clamp_min(1)))
                    keep = r <= 256
                    s = torch.where(keep, scale[page] * 2 ** k, a)
                    held = torch.where(keep[:, None, None], torch.round(ints[page, :, :off] / (2 ** k)[:, None, None]), held)
                q = torch.round(new / s[:, None, None]).clamp(-127, 127)
                scale[page] = s
                got[i, b * BLOCK - base:hi - base] = (torch.cat([held, q], 1) * s[:, None, None]).transpose(0, 1)
        out[name], out[name + "_scale"] = got, scale
    return out


def _exact_heads(st, page):
    """Keys and values [kv, tokens, dim] of one sequence in 64 bits."""
    c = st["cache"]
    k = (c["k"][page].double() * c["k_scale"][page].double()[..., None, None]).transpose(0, 1)
    v = (c["v"][page].double() * c["v_scale"][page].double()[..., None, None]).transpose(2, 3).transpose(0, 1)
    return k.reshape(k.shape[0], -1, k.shape[3]), v.reshape(v.shape[0], -1, v.shape[3])


def _exact_picked(st, i, h, first, count, nb):
    """A truth value for each block of sequence i: whether the tile with rows first.. of kv head h takes it."""
    case, c = st["case"], st["cache"]
    n, rows, heads, dim = st["q"].shape
    group, end = heads // c["k"].shape[1], int(st["lens"][i])
    rows_of = st["q"][i, first:min(first + TILE, count), h * group:(h + 1) * group].double()
    p = rows_of.sum((0, 1))
    qi = torch.round(p * 1023 / p.abs().max())
    page = st["tables"][i, :nb].long()
    held = (end - BLOCK * torch.arange(nb, device="cuda")).clamp(1, BLOCK).double()
    score = (c["k_sum"][page, h].double() @ qi) * c["k_scale"][page, h].double() / held
    seen = nb
    if case["causal"]:
        lo, hi = end - count + first, end - count + min(first + TILE, count) - 1
        seen = hi // BLOCK + 1
        score[lo // BLOCK:seen] = math.inf
    order = torch.sort(score[:seen], descending=True, stable=True).indices[:case["top"]]
    return torch.zeros(nb, device="cuda", dtype=torch.bool).index_fill_(0, order, True)


def _exact_attention(st):
    case = st["case"]
    n, rows, heads, dim = st["q"].shape
    group = heads // case["kv"]
    out = torch.zeros(n, rows, heads, dim, device="cuda", dtype=torch.float64)
    for i in range(n):
        end, count = int(st["lens"][i]), int(st["counts"][i])
        nb = -(-end // BLOCK)
        k, v = _exact_heads(st, st["tables"][i, :nb].long())
        t, at = torch.arange(end, device="cuda"), end - count + torch.arange(count, device="cuda")
        for h in range(case["kv"]):
            hide = t > at[:, None] if case["causal"] else None
            if case["kind"] == "sparse":
                took = torch.stack([_exact_picked(st, i, h, f, count, nb) for f in range(0, count, TILE)])
                gone = ~took.repeat_interleave(BLOCK, 1)[:, :end].repeat_interleave(TILE, 0)[:count]
                hide = gone if hide is None else hide | gone
            for j in range(h * group, (h + 1) * group):
                s = st["q"][i, :count, j].double() @ k[h, :end].t() * dim ** -0.5
                p = torch.softmax(s if hide is None else s.masked_fill_(hide, -math.inf), 1)
                out[i, :count, j] = p @ v[h, :end]
    return torch.nan_to_num(out)  # rows that see no token are zero


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "write":
        return _exact_write(st)
    if kind == "read":
        k = torch.zeros(case["n"], case["length"], case["heads"], case["dim"], device="cuda", dtype=torch.float64)
        v = torch.zeros_like(k)
        for i in range(case["n"]):
            end = int(st["lens"][i])
            a, b = _exact_heads(st, st["tables"][i, :-(-end // BLOCK)].long())
            k[i, :end], v[i, :end] = a[:, :end].transpose(0, 1), b[:, :end].transpose(0, 1)
        return k, v
    o = _exact_attention(st)
    return o if kind == "attend" else {"blocks": None, "out": o}
