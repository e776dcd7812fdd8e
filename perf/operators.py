"""Cases for measuring the serving operators: the plan of a step over a paged cache, the 4-bit paged cache (writing, reading back,
attention over it) and the log probabilities of tokens.

`run` computes each operator in its plain form (elementary torch operations in 32 bits) where `own` is false, and calls the package where
it is true.  Layout of the 4-bit cache, which both sides read: uint8 [pages, kv_heads, page_size, 40 G] with G = ceil(head_dim / 32)
groups of 32 values, page_size a multiple of 16.  The bytes of one (page, head) are page_size / 16 tiles of 16 tokens, each
  key codes    [16 tokens][4 t][G g][4 bytes]                  nibble n (0..7) of the word (t, g) is dim 32 g + 8 t + n
  value codes  [2 h][8 c][4 t][G g][2 parity][2 bytes]         token 8 h + 2 t + parity; nibble n (0..3) is dim 32 g + 4 c + n
  parameters   [16 tokens][key scales G, key minima G, value scales G, value minima G] fp16
and a value is code * scale + minimum.
"""
import math
import random

import torch

own = False

DEV = "cuda"
GROUP = 32


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 16 requests: one token each, a page now and then, and the row lists that the paged Llama block reads
        {"name": "plan_decode_b16", "op": "plan", "batch": 16, "ctx": 2048, "prompt_share": 0.0, "prompt": 1, "page": 16, "rows": True, "lens": 1},
        # a step of continuous batching: decoding requests among prompt chunks, long contexts
        {"name": "plan_mixed_b256", "op": "plan", "batch": 256, "ctx": 8192, "prompt_share": 0.2, "prompt": 512, "page": 64, "rows": True, "lens": 2},
        # the new token of 16 decoding requests, 32 heads of 128
        {"name": "append_decode_b16", "op": "append", "tokens": 16, "heads": 32, "dim": 128, "page": 16, "dtype": "float16", "lens": 3},
        # a prompt over 32 heads of 80, keys and values cut out of a fused projection
        {"name": "append_prompt_500_d80", "op": "append", "tokens": 500, "heads": 32, "dim": 80, "page": 32, "dtype": "float16", "lens": 4},
        # the prompts of one step, grouped heads
        {"name": "append_prompts_8191", "op": "append", "tokens": 8191, "heads": 8, "dim": 128, "page": 64, "dtype": "bfloat16", "lens": 5},
        # one request decoding: latency, few rows, split along the cache
        {"name": "attend_b1_4096", "op": "attend", "batch": 1, "ctx": 4096, "ragged": False, "q": 1, "heads": 32, "kv_heads": 32, "dim": 128, "page": 16, "dtype": "float16", "lens": 6},
        # the batch of the paged Llama block, ragged
        {"name": "attend_b16_ragged", "op": "attend", "batch": 16, "ctx": 4096, "ragged": True, "q": 1, "heads": 32, "kv_heads": 32, "dim": 128, "page": 16, "dtype": "float16", "lens": 7},
        # a full server: many long requests, grouped heads
        {"name": "attend_gqa_b64_8192", "op": "attend", "batch": 64, "ctx": 8192, "ragged": True, "q": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bfloat16", "lens": 8},
        # a few drafted tokens a request are checked at once; heads of 80
        {"name": "attend_verify_d80", "op": "attend", "batch": 8, "ctx": 2048, "ragged": True, "q": 6, "heads": 32, "kv_heads": 32, "dim": 80, "page": 32, "dtype": "float16", "lens": 9},
        # chunks of prompts over what the cache holds already
        {"name": "attend_prompt_chunks", "op": "attend", "batch": 3, "ctx": 4096, "ragged": True, "q": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bfloat16", "lens": 10},
        # the token just decoded, from the decoder's own fp32 logits
        {"name": "logprobs_token", "op": "logprobs", "rows": 1, "vocab": 50304, "pad": 0, "top": 5, "dtype": "float32"},
        # a scored prompt
        {"name": "logprobs_prompt_2047", "op": "logprobs", "rows": 2047, "vocab": 50304, "pad": 0, "top": 20, "dtype": "float16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "logprobs"])
    lens = rng.randrange(1000, 1 << 20)
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "plan":
        return {"op": op, "batch": _log(rng, 1, 256), "ctx": _log(rng, 16, 8192), "prompt_share": rng.choice([0.0, 0.2, 0.5]), "prompt": _log(rng, 2, 512), "page": page,
                "rows": rng.random() < 0.7, "lens": lens}
    if op == "append":
        heads = rng.choice([1, 2, 4, 5, 8, 32])
        return {"op": op, "tokens": _log(rng, 1, 65528 // heads), "heads": heads, "dim": rng.choice([64, 80, 96, 128]), "page": page, "dtype": dtype, "lens": lens}
    if op == "attend":
        kv_heads = rng.choice([1, 2, 4, 8, 32])
        heads = kv_heads * rng.choice([1, 2, 4, 5, 8] if kv_heads <= 8 else [1])
        q = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 700)])
        ctx = _log(rng, 16, 16384)
        most = min(16 * 4096 * 32 // (ctx * kv_heads), 3 * 1024 * 32 * 2048 // (q * heads * ctx)) if q > 16 else 16 * 4096 * 32 // (ctx * kv_heads)
        return {"op": op, "batch": _log(rng, 1, max(1, min(64, most))), "ctx": ctx, "ragged": rng.random() < 0.7, "q": q, "heads": heads, "kv_heads": kv_heads,
                "dim": rng.choice([64, 80, 96, 128]), "page": page, "dtype": dtype, "lens": lens}
    vocab = _log(rng, 1000, 200000)
    return {"op": op, "rows": _log(rng, 1, max(1, min(4096, 2047 * 50304 // vocab // 2))), "vocab": vocab, "pad": rng.choice([0, 0, 1, 24]), "top": rng.choice([0, 1, 5, 20, 32]),
            "dtype": rng.choice(["float16", "bfloat16", "float32"])}


def _plan_lens(c):
    r = random.Random(c["lens"])
    new = [r.randint(2, max(2, c["prompt"])) if r.random() < c["prompt_share"] else 1 for _ in range(c["batch"])]
    cached = [r.randint(0, max(0, c["ctx"] - n)) for n in new]
    return cached, new


def _attend_lens(c):
    """(kv_lens, query counts): every request has its new tokens in the cache already."""
    r = random.Random(c["lens"])
    kv = [r.randint(1, c["ctx"]) if c["ragged"] else c["ctx"] for _ in range(c["batch"])]
    q = [min(n, c["q"] if c["q"] <= 1 or not c["ragged"] else r.randint(max(1, c["q"] // 2), c["q"])) for n in kv]
    return kv, q


def _pages(lens, page):
    return [-(-n // page) for n in lens]


# ----------------------------------------------------------------------------------------------------------- prepare
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(lens, page, pool, g):
    """A block table of rows of shuffled pages, and the pages that no row uses (shuffled too)."""
    n = _pages(lens, page)
    width = max(max(n), 1)
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    col = torch.arange(width, device=DEV)
    count = torch.tensor(n, device=DEV)
    at = (count.cumsum(0) - count)[:, None] + col
    table = torch.where(col < count[:, None], order[at.clamp(max=pool - 1)], torch.full_like(at, -1, dtype=torch.int32))
    return table.contiguous(), order[sum(n):].contiguous()


def _random_cache(pages, heads, page, dim, g):
    """Codes and parameters as rows of unit scale have them."""
    G = -(-dim // GROUP)
    cache = torch.randint(0, 256, (pages, heads, page // 16, 640 * G), dtype=torch.uint8, device=DEV, generator=g)
    n = (pages, heads, page // 16, 16, 2, 1, G)
    scale = torch.rand(n, device=DEV, generator=g) * 0.15 + 0.2
    low = -torch.rand(n, device=DEV, generator=g) - 1.6
    cache[..., 512 * G:] = torch.cat([scale, low], dim=-2).half().reshape(pages, heads, page // 16, 64 * G).view(torch.uint8)
    return cache.view(pages, heads, page, 40 * G)


def prepare(c, seed):
    g = _gen(seed)
    s = dict(c)
    if c["op"] == "plan":
        cached, new = _plan_lens(c)
        total = [a + b for a, b in zip(cached, new)]
        page = c["page"]
        pool = sum(_pages(total, page)) + 64
        table, free = _table(cached, page, pool, g)
        wide = torch.full((c["batch"], max(_pages(total, page)) + 3), -1, dtype=torch.int32, device=DEV)
        keep = min(wide.shape[1], table.shape[1])
        wide[:, :keep] = table[:, :keep]
        return s | {"cached": _ints(cached), "new": _ints(new), "table": wide, "free": free, "free_count": _ints([free.numel()]),
                    "max_tokens": sum(new) + 5, "max_rows": sum(total) + 7 if c["rows"] else 0}
    if c["op"] == "append":
        T, H, D, page = c["tokens"], c["heads"], c["dim"], c["page"]
        pool = -(-T // page) + 8
        kv = torch.randn(T, 3, H, D, device=DEV, generator=g) * torch.exp(0.5 * torch.randn(1, 3, H, D, device=DEV, generator=g))
        kv = kv.to(getattr(torch, c["dtype"]))  # a fused projection: the keys and values are cut out of it
        order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
        if T <= 64:  # single tokens land on pages of their own; prompts fill pages from their start
            pool = max(pool, T)
            order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
            slots = order[:T] * page + torch.randint(0, page, (T,), device=DEV, generator=g, dtype=torch.int32)
        else:
            at = torch.arange(T, device=DEV, dtype=torch.int32)
            slots = order[(at // page).long()] * page + at % page
        G = -(-D // GROUP)
        return s | {"key": kv[:, 1], "value": kv[:, 2], "slots": slots, "cache": torch.zeros(pool, H, page, 40 * G, dtype=torch.uint8, device=DEV)}
    if c["op"] == "attend":
        kv, q = _attend_lens(c)
        pool = sum(_pages(kv, c["page"])) + 3
        table, _ = _table(kv, c["page"], pool, g)
        qkv = torch.randn(sum(q), c["heads"] + 2 * c["kv_heads"], c["dim"], device=DEV, generator=g).to(getattr(torch, c["dtype"]))
        starts = [0]
        for n in q:
            starts.append(starts[-1] + n)
        return s | {"query": qkv[:, :c["heads"]], "cache": _random_cache(pool, c["kv_heads"], c["page"], c["dim"], g), "table": table, "kv_lens": _ints(kv),
                    "starts": _ints(starts), "max_q": max(q), "width": max(kv)}
    x = torch.randn(c["rows"], c["vocab"] + c["pad"], device=DEV, generator=g) * 2.5
    x = x.to(getattr(torch, c["dtype"]))[:, :c["vocab"]]
    return s | {"logits": x, "tokens": torch.randint(0, c["vocab"], (c["rows"],), device=DEV, generator=g)}


# --------------------------------------------------------------------------------------------------------------- run
def run(s):
    return {"plan": _plan, "append": _append, "attend": _attend, "logprobs": _logprobs}[s["op"]](s)


def _plan(s):
    page = s["page"]
    if own:
        import clusterfusionplus_b200 as cf
        p = cf.paged_kv_plan(s["cached"], s["new"], s["table"], s["free"], s["free_count"], page, s["max_tokens"], s["max_rows"])
        return {"table": s["table"], "kv_lens": p.kv_lens, "qo_indptr": p.qo_indptr, "positions": p.positions, "slot_map": p.slot_map,
                "kv_indptr": p.kv_indptr, "kv_indices": p.kv_indices, "free_count": p.free_count, "status": p.status}
    table, free = s["table"], s["free"]
    cached, new = s["cached"].long(), s["new"].long()
    total = cached + new
    have, need = (cached + page - 1) // page, (total + page - 1) // page
    grow = need - have
    ends = grow.cumsum(0)
    rows = torch.zeros((), dtype=torch.bool, device=DEV) if s["max_rows"] == 0 else total.sum() > s["max_rows"]
    status = ((ends[-1] > s["free_count"][0]).int() + 2 * (need.max() > table.shape[1]).int() + 4 * (new.sum() > s["max_tokens"]).int() + 8 * rows.int()
              + 16 * ((cached < 0) | (new < 0)).any().int())
    ok = status == 0
    col = torch.arange(table.shape[1], device=DEV)
    fresh = (col >= have[:, None]) & (col < need[:, None]) & ok
    at = s["free_count"] - 1 - ((ends - grow)[:, None] + col - have[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))

    def per_row(lens, count, first):
        """For `count` rows dealt out to the requests in order: whether it is dealt, its position and its slot."""
        ends = lens.cumsum(0)
        j = torch.arange(count, device=DEV)
        req = torch.searchsorted(ends, j, right=True).clamp(max=lens.numel() - 1)
        dealt = (j < ends[-1]) & ok
        pos = torch.where(dealt, first[req] + j - (ends - lens)[req], torch.zeros_like(j))
        held = table[req, (pos // page).clamp(max=table.shape[1] - 1)].long()
        return pos, torch.where(dealt & (held >= 0), held * page + pos % page, torch.full_like(j, -1)).int()

    def indptr(lens):
        return torch.where(ok, torch.cat([torch.zeros_like(lens[:1]), lens.cumsum(0)]), torch.zeros_like(lens[:1])).int()

    positions, slot_map = per_row(new, s["max_tokens"], cached)
    _, kv_indices = per_row(total, s["max_rows"], torch.zeros_like(cached))
    return {"table": table, "kv_lens": torch.where(ok, total, cached).int(), "qo_indptr": indptr(new), "positions": positions, "slot_map": slot_map,
            "kv_indptr": indptr(total), "kv_indices": kv_indices, "free_count": torch.where(ok, s["free_count"] - ends[-1], s["free_count"]).int(),
            "status": status.reshape(1).int()}


def _quantised(x):
    """codes [.., G, 32] (int32), scale and minimum [.., G] (fp16) of x [.., D]."""
    D = x.shape[-1]
    G = -(-D // GROUP)
    x = x.float().clamp(-65504.0, 65504.0)
    pad = G * GROUP - D
    low_side = torch.nn.functional.pad(x, (0, pad), value=math.inf).unflatten(-1, (G, GROUP))
    high_side = torch.nn.functional.pad(x, (0, pad), value=-math.inf).unflatten(-1, (G, GROUP))
    low = low_side.amin(-1).half()
    scale = ((high_side.amax(-1) - low.float()) / 15.0).half()
    x = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (G, GROUP))
    step = scale.float()[..., None]
    codes = torch.where(step > 0, torch.round((x - low.float()[..., None]) / torch.where(step > 0, step, torch.ones_like(step))), torch.zeros_like(x))
    real = (torch.arange(G * GROUP, device=x.device) < D).view(G, GROUP)
    return torch.where(real, codes.clamp(0, 15), torch.zeros_like(codes)).int(), scale, low


def _nibbles(codes):
    """Bytes of codes whose last axis holds their two halves."""
    return (codes[..., 0] | (codes[..., 1] << 4)).to(torch.uint8)


def _append(s):
    cache, D = s["cache"], s["dim"]
    if own:
        import clusterfusionplus_b200 as cf
        cf.kv4_append(s["key"], s["value"], s["slots"], cache)
        return cf.kv4_read(cache, s["slots"], D, s["key"].dtype)
    pages, H, page, _ = cache.shape
    T = s["slots"].numel()
    G = -(-D // GROUP)
    slot = s["slots"].long()
    which, tile, row = slot // page, slot % page // 16, slot % 16
    tiles = cache.view(pages, H, page // 16, 640 * G)
    kc, ks, km = _quantised(s["key"])
    vc, vs, vm = _quantised(s["value"])
    keys = tiles[..., :256 * G].unflatten(-1, (16, 16 * G))
    keys[which, :, tile, row] = _nibbles(kc.view(T, H, G, 4, 4, 2)).transpose(2, 3).reshape(T, H, 16 * G)
    values = tiles[..., 256 * G:512 * G].unflatten(-1, (2, 8, 4, G, 2, 2))
    values[which, :, tile, row // 8, :, row % 8 // 2, :, row % 2] = _nibbles(vc.view(T, H, G, 8, 2, 2)).transpose(2, 3)
    params = tiles[..., 512 * G:].unflatten(-1, (16, 8 * G))
    params[which, :, tile, row] = torch.stack([ks, km, vs, vm], dim=2).reshape(T, H, 4 * G).view(torch.uint8)
    got = _unpacked(tiles[which, :, tile], D)  # what the cache holds now, at these slots
    pick = row.view(T, 1, 1, 1).expand(T, H, 1, D)
    return tuple(x.gather(2, pick).squeeze(2).to(s["key"].dtype) for x in got)


def _unpacked(tiles, D):
    """(keys, values) [.., 16, D] in 32 bits of tiles [.., 640 G]."""
    G = tiles.shape[-1] // 640
    lead = tiles.shape[:-1]
    params = tiles[..., 512 * G:].contiguous().view(torch.float16).unflatten(-1, (16, 2, 2, G, 1)).float()

    def split(x):
        return torch.stack([x & 15, x >> 4], dim=-1)

    k = split(tiles[..., :256 * G].unflatten(-1, (16, 4, G, 4))).transpose(-4, -3).reshape(*lead, 16, G, GROUP).float()
    n = len(lead)
    v = split(tiles[..., 256 * G:512 * G].unflatten(-1, (2, 8, 4, G, 2, 2)))  # h, c, t, g, parity, byte, half
    v = v.permute(*range(n), n, n + 2, n + 4, n + 3, n + 1, n + 5, n + 6).reshape(*lead, 16, G, GROUP).float()
    return tuple((x * params[..., :, i, 0, :, :] + params[..., :, i, 1, :, :]).flatten(-2)[..., :D] for i, x in enumerate((k, v)))


def _attend(s):
    q, cache, table, D = s["query"], s["cache"], s["table"], s["dim"]
    if own:
        import clusterfusionplus_b200 as cf
        return cf.kv4_attention(q, cache, table, s["kv_lens"], s["starts"], max_q_len=s["max_q"])
    pages, Hkv, page, _ = cache.shape
    B, Hq = s["kv_lens"].numel(), q.shape[1]
    L, n = s["width"], s["max_q"]
    held = table[:, :-(-L // page)].clamp(min=0).long()
    tiles = cache.view(pages, Hkv, page // 16, -1)[held]                                  # [B, pages, Hkv, tiles, bytes]
    k, v = _unpacked(tiles.transpose(1, 2).reshape(B, Hkv, -1, tiles.shape[-1]), D)       # [B, Hkv, tiles, 16, D]
    k, v = k.flatten(2, 3)[:, :, :L], v.flatten(2, 3)[:, :, :L]
    first, count, kv = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long(), s["kv_lens"].long()
    i = torch.arange(n, device=DEV)
    rows = (first[:, None] + i).clamp(max=q.shape[0] - 1)
    x = q[rows].float().view(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    score = (x @ k.transpose(2, 3)).view(B, Hkv, Hq // Hkv, n, L) / math.sqrt(D)
    seen = torch.arange(L, device=DEV) <= (kv - count)[:, None, None] + i[:, None]         # [B, n, L]
    score = torch.where(seen[:, None, None], score, torch.full_like(score, -math.inf))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    y = (p.flatten(2, 3) @ v).view(B, Hkv, Hq // Hkv, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)
    return y[i < count[:, None]].to(q.dtype)


def _logprobs(s):
    x, tokens, k = s["logits"], s["tokens"], s["top"]
    if own:
        import clusterfusionplus_b200 as cf
        r = cf.token_logprobs(x, tokens, k)
        return {"logprobs": r.logprobs, "entropy": r.entropy} | ({"top_logprobs": r.top_logprobs, "top_tokens": r.top_tokens} if k else {})
    x = x.float()
    V = x.shape[1]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    r = {"logprobs": (x.gather(1, tokens[:, None]) - lse)[:, 0], "entropy": torch.log(total[:, 0]) - (e * (x - top)).sum(-1) / total[:, 0]}
    if k:  # the greatest, the lowest index first among equals: one integer key a value
        bits = (x + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + torch.arange(V - 1, -1, -1, device=DEV)
        at = V - 1 - (torch.topk(key, k, dim=-1).values & 0xFFFFFFFF)
        r |= {"top_logprobs": x.gather(1, at) - lse, "top_tokens": at}
    return r


# -------------------------------------------------------------------------------------------------------------- work
def work(c):
    if c["op"] == "plan":
        cached, new = _plan_lens(c)
        total = [a + b for a, b in zip(cached, new)]
        fresh = sum(_pages(total, c["page"])) - sum(_pages(cached, c["page"]))
        rows = sum(total) + 7 if c["rows"] else 0
        # lengths in and out, both row lists, fresh pages read and written, pages looked up, positions and slots, rows
        look = sum(_pages(total, c["page"])) if c["rows"] else sum(_pages(new, c["page"]))
        return {"bytes": 4 * (3 * c["batch"] + 2 * (c["batch"] + 1) + 3) + 8 * fresh + 4 * look + 12 * (sum(new) + 5) + 4 * rows, "flops": 0}
    if c["op"] == "append":
        n, G = c["tokens"] * c["heads"], -(-c["dim"] // GROUP)
        # keys and values in (2 x 2 bytes a value), codes and parameters written and read again, keys and values out
        return {"bytes": n * (4 * c["dim"] + 2 * (c["dim"] + 8 * G) + 4 * c["dim"]) + 4 * c["tokens"], "flops": 8 * n * c["dim"]}
    if c["op"] == "attend":
        kv, q = _attend_lens(c)
        G = -(-c["dim"] // GROUP)
        pairs = sum(n * m - m * (m - 1) // 2 for n, m in zip(kv, q))
        return {"bytes": sum(kv) * c["kv_heads"] * (c["dim"] + 8 * G) + 4 * sum(q) * c["heads"] * c["dim"] + 4 * sum(_pages(kv, c["page"])) + 8 * c["batch"],
                "flops": 4 * c["dim"] * c["heads"] * pairs}
    size = {"float16": 2, "bfloat16": 2, "float32": 4}[c["dtype"]]
    return {"bytes": c["rows"] * (c["vocab"] * size + 8 + 8 + 12 * c["top"]), "flops": 5 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------------------------------------------------- exact
def exact(c, seed):
    """From the definitions, in 64 bits."""
    if c["op"] == "plan":
        return None  # whole numbers
    s = prepare(c, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[c["op"]](s)


def _exact_append(s):
    def stored(x):
        T, H, D = x.shape
        out = torch.empty(T, H, D, dtype=torch.float64, device=DEV)
        for a in range(0, D, GROUP):
            part = x[:, :, a:a + GROUP].double()
            low = part.min(-1, keepdim=True).values.half().double()
            step = ((part.max(-1, keepdim=True).values - low) / 15).half().double()
            code = torch.round((part - low) / step).clamp(0, 15) if bool((step > 0).all()) else torch.where(step > 0, torch.round((part - low) / step), 0 * part).clamp(0, 15)
            out[:, :, a:a + GROUP] = code * step + low
        return out

    return stored(s["key"]), stored(s["value"])


def _exact_rows(tile, D):
    """Keys and values [n, 16, D] of tiles [n, 640 G], value by value from the layout's description."""
    G = tile.shape[1] // 640
    r = torch.arange(16, device=DEV)[:, None]
    d = torch.arange(D, device=DEV)[None]
    g, e = d // 32, d % 32
    at = r * 16 * G + (e // 8) * 4 * G + g * 4 + e % 8 // 2
    k = (tile[:, at].int() >> (4 * (d % 2))) & 15
    at = 256 * G + ((((r // 8) * 8 + e // 4) * 4 + r % 8 // 2) * G + g) * 4 + (r % 2) * 2 + e % 4 // 2
    v = (tile[:, at].int() >> (4 * (d % 2))) & 15
    par = tile[:, 512 * G:].contiguous().view(torch.float16).double().view(-1, 16, 4 * G)
    pick = lambda i: par[:, r, i * G + g]  # noqa: E731
    return k.double() * pick(0) + pick(1), v.double() * pick(2) + pick(3)


def _exact_attend(s):
    q, cache, D = s["query"].double(), s["cache"], s["dim"]
    pages, Hkv, page, _ = cache.shape
    per = q.shape[1] // Hkv
    starts, lens = s["starts"].tolist(), s["kv_lens"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for b, L in enumerate(lens):
        a, e = starts[b], starts[b + 1]
        held = s["table"][b, :-(-L // page)].long()
        for h in range(Hkv):
            k, v = _exact_rows(cache[held, h].reshape(held.numel() * (page // 16), -1), D)
            k, v = k.reshape(-1, D)[:L], v.reshape(-1, D)[:L]
            sc = torch.einsum("nhd,ld->hnl", q[a:e, h * per:(h + 1) * per], k) * D ** -0.5
            late = torch.arange(L, device=DEV)[None] > torch.arange(L - (e - a), L, device=DEV)[:, None]
            out[a:e, h * per:(h + 1) * per] = torch.einsum("hnl,ld->nhd", torch.softmax(sc.masked_fill(late, -math.inf), -1), v)
    return out


def _exact_logprobs(s):
    at, k = s["tokens"], s["top"]
    rows = [], [], []
    for x in s["logits"].split(256):
        lp = torch.log_softmax(x.double(), -1)
        rows[0].append(lp)
        rows[1].append(-(lp.exp() * lp).sum(-1))
        rows[2].append(torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :k])
        rows[0][-1] = torch.cat([lp.gather(1, at[sum(n.shape[0] for n in rows[0][:-1]):][:x.shape[0], None]), lp.gather(1, rows[2][-1])], 1)
    lp = torch.cat(rows[0])
    r = {"logprobs": lp[:, 0], "entropy": torch.cat(rows[1])}
    return r | ({"top_logprobs": lp[:, 1:], "top_tokens": torch.cat(rows[2])} if k else {})
