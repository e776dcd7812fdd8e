"""Plain restatements of the serving operators (numpy / 64-bit torch on the CPU), written from their definitions: the plan of a step
over a paged cache, the 4-bit cache, attention over it, and log probabilities of tokens."""
from __future__ import annotations

import math

import numpy as np
import torch

GROUP = 32


# ---------------------------------------------------------------------------------------------------- plan of a step
def plan(cached, new, table, free, count, page, max_tokens, max_rows):
    """Lists in, dict of lists out; `table` (list of rows) is not modified, the result has its own."""
    table = [list(r) for r in table]
    width = len(table[0])
    status = 0
    pages = lambda n: -(-n // page)  # noqa: E731
    good = [c >= 0 and n >= 0 and c + n < 1 << 31 for c, n in zip(cached, new)]
    if not all(good):
        status |= 16
    need = [pages(c + n) if g else 0 for c, n, g in zip(cached, new, good)]
    have = [pages(c) if g else 0 for c, g in zip(cached, good)]
    if any(n > width for n in need):
        status |= 2
    avail = count
    if not 0 <= count <= len(free) or sum(need) - sum(have) > avail:
        status |= 1
    if sum(n for n, g in zip(new, good) if g) > max_tokens:
        status |= 4
    rows = sum(c + n for c, n, g in zip(cached, new, good) if g)
    if rows > (max_rows if max_rows else (1 << 31) - 1):
        status |= 8
    B = len(cached)
    out = {"table": table, "kv_lens": list(cached), "qo_indptr": [0] * (B + 1), "kv_indptr": [0] * (B + 1), "positions": [], "slot_map": [],
           "kv_indices": [], "free_count": count, "status": status}
    if status == 0:
        for b in range(B):
            for col in range(have[b], need[b]):
                avail -= 1
                table[b][col] = free[avail]
            out["kv_lens"][b] = cached[b] + new[b]
            out["qo_indptr"][b + 1] = out["qo_indptr"][b] + new[b]
            out["kv_indptr"][b + 1] = out["kv_indptr"][b] + cached[b] + new[b]
            slot = lambda p: table[b][p // page] * page + p % page if table[b][p // page] >= 0 else -1  # noqa: E731
            for p in range(cached[b], cached[b] + new[b]):
                out["positions"].append(p)
                out["slot_map"].append(slot(p))
            if max_rows:
                out["kv_indices"] += [slot(p) for p in range(cached[b] + new[b])]
        out["free_count"] = count - (sum(need) - sum(have))
    out["positions"] += [0] * (max_tokens - len(out["positions"]))
    out["slot_map"] += [-1] * (max_tokens - len(out["slot_map"]))
    out["kv_indices"] += [-1] * (max_rows - len(out["kv_indices"]))
    return out


# ------------------------------------------------------------------------------------------------------ 4-bit cache
def groups(dim):
    return -(-dim // GROUP)


def quantise(x):
    """codes [.., D] (uint8), scale and minimum [.., G] (float16) of x [.., D] (float32 array of fp16 / bf16 values)."""
    x = np.asarray(x, dtype=np.float32)
    D = x.shape[-1]
    codes = np.zeros(x.shape, np.uint8)
    scale = np.zeros(x.shape[:-1] + (groups(D),), np.float16)
    low = np.zeros_like(scale)
    for g in range(groups(D)):
        part = x[..., 32 * g:32 * g + 32]
        bad = ~np.isfinite(part).all(-1)
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            part = np.fmin(np.fmax(part, np.float32(-65504)), np.float32(65504))
            m = part.min(-1).astype(np.float16)
            s = ((part.max(-1) - m.astype(np.float32)) / np.float32(15)).astype(np.float16)
            beyond = m.astype(np.float64) + 15 * s.astype(np.float64) > 65504   # the largest value would not be an fp16 number: one step lower
            s = np.where(beyond, np.nextafter(s, np.float16(0)), s)
            c = np.rint((part - m.astype(np.float32)[..., None]) / s.astype(np.float32)[..., None])
        c = np.where((s[..., None] > 0) & ~bad[..., None], np.clip(np.nan_to_num(c), 0, 15), 0)
        codes[..., 32 * g:32 * g + 32] = c.astype(np.uint8)
        scale[..., g], low[..., g] = np.where(bad, np.float16(np.nan), s), m
    return codes, scale, low


def nibble(D, token, dim, value):
    """(byte, shift) of a code inside a tile of 16 tokens."""
    G = groups(D)
    g, e = divmod(dim, 32)
    if not value:
        word, n = token * 4 * G + (e // 8) * G + g, e % 8
        return 4 * word + n // 2, 4 * (n % 2)
    h, t, parity = token // 8, token % 8 // 2, token % 2
    word, n = 64 * G + ((h * 8 + e // 4) * 4 + t) * G + g, e % 4
    return 4 * word + 2 * parity + n // 2, 4 * (n % 2)


def param(D, token, which, g):
    """Byte of a parameter inside a tile; which: key scale, key minimum, value scale, value minimum."""
    G = groups(D)
    return 512 * G + token * 8 * G + 2 * (which * G + g)


def _indices(D):
    """Gather indices (byte, shift) [2][16][D] of a tile."""
    at = np.zeros((2, 16, D), np.int64)
    sh = np.zeros((2, 16, D), np.int64)
    for v in range(2):
        for t in range(16):
            for d in range(D):
                at[v, t, d], sh[v, t, d] = nibble(D, t, d, v)
    return at, sh


def store(cache, slot, key, value):
    """Writes key and value [H, D] (float32) to row `slot` of cache [pages, H, page, 40 G] (uint8 array), in place."""
    pages, H, page, _ = cache.shape
    D = key.shape[-1]
    G = groups(D)
    p, at = divmod(slot, page)
    tile, t = divmod(at, 16)
    for h in range(H):
        raw = cache[p, h].reshape(-1)[tile * 640 * G:(tile + 1) * 640 * G]
        for v, x in enumerate((key[h], value[h])):
            c, s, m = quantise(x)
            full = np.zeros(32 * G, np.uint8)
            full[:D] = c
            for d in range(32 * G):
                byte, shift = nibble(D, t, d, v)
                raw[byte] = (raw[byte] & (0xF0 >> shift)) | (full[d] << shift)
            for g in range(G):
                for which, val in ((2 * v, s[g]), (2 * v + 1, m[g])):
                    raw[param(D, t, which, g):param(D, t, which, g) + 2] = np.frombuffer(np.float16(val).tobytes(), np.uint8)


def unpack(cache, D):
    """(keys, values) float64 [pages, H, page, D] of a cache (uint8 tensor or array)."""
    cache = np.ascontiguousarray(cache.cpu().numpy() if torch.is_tensor(cache) else cache)
    pages, H, page, _ = cache.shape
    G = groups(D)
    tiles = cache.reshape(pages, H, page // 16, 640 * G)
    at, sh = _indices(D)
    par = np.ascontiguousarray(tiles[..., 512 * G:]).view(np.float16).reshape(pages, H, page // 16, 16, 4, G).astype(np.float64)
    g = np.arange(D) // 32
    out = []
    for v in range(2):
        code = (tiles[..., at[v]] >> sh[v]) & 15
        with np.errstate(invalid="ignore"):  # rows that were never written may hold anything
            out.append((code * par[..., 2 * v, :][..., g] + par[..., 2 * v + 1, :][..., g]).reshape(pages, H, page, D))
    return tuple(torch.from_numpy(o) for o in out)


# --------------------------------------------------------------------------------------------------------- attention
def attention(query, keys, values, table, kv_lens, starts, scale, out=None):
    """float64 [rows, Hq, D]; keys / values [pages, Hkv, page, D] from unpack(); rows no request owns keep `out`.  Pages outside the cache
    are not there."""
    q = query.double().cpu()
    pages, Hkv, page, D = keys.shape
    per = q.shape[1] // Hkv
    out = torch.zeros(q.shape, dtype=torch.float64) if out is None else out.double().cpu().clone()
    for b, L in enumerate(kv_lens):
        n = starts[b + 1] - starts[b]
        there = [p for p in range(max(L, 0)) if p // page < len(table[b]) and 0 <= table[b][p // page] < pages]
        pick = torch.tensor([table[b][p // page] * page + p % page for p in there], dtype=torch.long)
        k = keys.transpose(1, 2).reshape(pages * page, Hkv, D)[pick]
        v = values.transpose(1, 2).reshape(pages * page, Hkv, D)[pick]
        for i in range(n):
            m = sum(p <= L - n + i for p in there)
            row = starts[b] + i
            if m == 0:
                out[row] = 0
                continue
            s = torch.einsum("hgd,lhd->hgl", q[row].view(Hkv, per, D), k[:m]) * scale
            out[row] = torch.einsum("hgl,lhd->hgd", torch.softmax(s, -1), v[:m]).reshape(-1, D)
    return out


# --------------------------------------------------------------------------------------------------- log probabilities
def logprobs(logits, tokens, k):
    """(logprobs, entropy, top_logprobs, top_tokens), float64."""
    x = logits.double().cpu()
    V = x.shape[1]
    lp = torch.log_softmax(x, -1)
    plogp = torch.where(lp == -math.inf, torch.zeros_like(lp), lp.exp() * lp)
    got = torch.tensor([lp[r, t] if 0 <= t < V else (-math.inf if not torch.isnan(lp[r]).any() else math.nan) for r, t in enumerate(tokens)], dtype=torch.float64)
    ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :k]   # stable: equal values by the lower index; NaN first
    return got, -plogp.sum(-1), lp.gather(1, ids), ids
