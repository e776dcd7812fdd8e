"""Serving a batch over a paged cache: the plan of a step, the cache held in 4 bits with the attention that reads it, and the
log probabilities of tokens.

One step of a server, all of it on the GPU and capturable (nothing is read back by the host):

    plan = cf.paged_kv_plan(cached_lens, new_lens, block_table, free_pages, free_count, page_size, max_tokens)
    cf.kv4_append(key, value, plan.slot_map, cache)                        # every layer
    out = cf.kv4_attention(query, cache, block_table, plan.kv_lens, plan.qo_indptr, max_q_len=longest)
    ...
    scored = cf.token_logprobs(logits, tokens, top_k=5)

The lists of a plan made with max_rows are what llama_decoder_layer_batch_decode_sglang takes as paged_kv_indptr,
paged_kv_indices and positions.  The reference's batched entry point (include/pybind.cpp:90-106) leaves all of this to its
caller.  Like the rest of the package these functions validate, allocate their results and launch on torch's current stream.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ._lib import CF_DTYPE_BF16, CF_DTYPE_FP16, CF_DTYPE_FP32, check, lib
from .api import _stream

_HALVES = {torch.float16: CF_DTYPE_FP16, torch.bfloat16: CF_DTYPE_BF16}
_LOGITS = {**_HALVES, torch.float32: CF_DTYPE_FP32}


def _on_device(t, name: str, device: int, dims: int) -> None:
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name}: expected a torch.Tensor")
    if t.get_device() != device:
        raise RuntimeError(f"{name}: tensor is on {t.device} but the current device is cuda:{device}" if t.is_cuda
                           else f"{name}: expected a CUDA tensor, got {t.device}")
    if t.dim() != dims:
        raise RuntimeError(f"{name}: expected {dims} dimension{'s' * (dims > 1)}, got shape {tuple(t.shape)}")


def _ints(t, name: str, device: int, n: int = -1) -> int:
    """Pointer of a contiguous int32 vector (of n entries)."""
    _on_device(t, name, device, 1)
    if t.dtype is not torch.int32:
        raise RuntimeError(f"{name}: expected dtype torch.int32, got {t.dtype}")
    if n >= 0 and t.shape[0] != n:
        raise RuntimeError(f"{name}: expected {n} entries, got {t.shape[0]}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name}: expected a contiguous tensor")
    return t.data_ptr()


def _table(t, name: str, device: int, batch: int) -> int:
    _on_device(t, name, device, 2)
    if t.dtype is not torch.int32:
        raise RuntimeError(f"{name}: expected dtype torch.int32, got {t.dtype}")
    if t.shape[0] != batch or t.stride(1) != 1 or (batch > 1 and t.stride(0) < t.shape[1]):
        raise RuntimeError(f"{name}: expected [{batch}, pages] rows of consecutive entries, got shape {tuple(t.shape)} with strides {t.stride()}")
    return t.data_ptr()


def _rows(t, name: str, device: int, dims: int, step: int) -> int:
    """Pointer of rows whose last axis is contiguous and whose other strides are multiples of `step` elements."""
    _on_device(t, name, device, dims)
    if t.dtype not in _HALVES:
        raise RuntimeError(f"{name}: expected dtype torch.float16 or torch.bfloat16, got {t.dtype}")
    s = t.stride()
    if s[2] != 1 or s[0] % step or s[1] % step or min(s) < 0:
        raise RuntimeError(f"{name}: expected a contiguous last axis and strides in multiples of {step} elements, got {s}")
    return t.data_ptr()


def _cache_shape(cache, device: int, heads: int, head_dim: int) -> Tuple[int, int]:
    _on_device(cache, "cache", device, 4)
    if cache.dtype is not torch.uint8 or not cache.is_contiguous():
        raise RuntimeError("cache: expected a contiguous uint8 tensor (see kv4_cache)")
    pages, h, page, width = cache.shape
    if h != heads or width != 40 * ((head_dim + 31) // 32):
        raise RuntimeError(f"cache: expected [pages, {heads}, page_size, {40 * ((head_dim + 31) // 32)}] for {heads} heads of {head_dim}, got {tuple(cache.shape)}")
    return pages, page


class PagedKvPlan(NamedTuple):
    """What paged_kv_plan computes (int32, positions int64)."""
    kv_lens: torch.Tensor      # [batch] cached + new tokens
    qo_indptr: torch.Tensor    # [batch + 1] first new token of every request
    positions: torch.Tensor    # [max_tokens] position of every new token in its request; 0 behind the last
    slot_map: torch.Tensor     # [max_tokens] cache row of every new token; -1 behind the last
    kv_indptr: torch.Tensor    # [batch + 1] first cached row of every request in kv_indices
    kv_indices: torch.Tensor   # [max_rows] cache rows of every request; -1 behind the last
    free_count: torch.Tensor   # [1] pages left on the free list
    status: torch.Tensor       # [1] 0, or CF_PLAN_* bits: nothing was planned


def paged_kv_plan(cached_lens, new_lens, block_table, free_pages, free_count, page_size: int, max_tokens: int, max_rows: int = 0) -> PagedKvPlan:
    """Plans a step in which request b, holding cached_lens[b] tokens, gets new_lens[b] more (int32 [batch], batch up to 4096).

    block_table int32 [batch, columns] is completed in place by the pages that the new tokens need; they come from the top of
    free_pages[: free_count[0]] (int32, free_count of one entry), request by request.  The result's free_count is what is left:
    pass it, and the result's kv_lens as cached_lens, to the next step.  max_tokens bounds the new tokens of the step; with max_rows > 0 the cache
    rows of all requests are listed too (kv_indices), the form that llama_decoder_layer_batch_decode_sglang reads.

    All or nothing: if the pages, the table's columns, max_tokens or max_rows do not suffice, or a length is negative, nothing
    changes, the lists come back empty and status[0] holds CF_PLAN_* bits.  Read it where the host waits anyway."""
    dev = torch.cuda.current_device()
    batch = cached_lens.shape[0] if isinstance(cached_lens, torch.Tensor) and cached_lens.dim() == 1 else -1
    cp, np_ = _ints(cached_lens, "cached_lens", dev), _ints(new_lens, "new_lens", dev, batch)
    tp = _table(block_table, "block_table", dev, batch)
    fp, fc = _ints(free_pages, "free_pages", dev), _ints(free_count, "free_count", dev, 1)
    max_tokens, max_rows = int(max_tokens), int(max_rows)
    if max_tokens < 0 or max_rows < 0:
        raise RuntimeError(f"max_tokens {max_tokens} and max_rows {max_rows} must not be negative")
    rows_room = (max_rows + 3) // 4 * 4  # keeps what follows aligned
    buf = torch.empty(rows_room + max_tokens + 3 * batch + 4, dtype=torch.int32, device=cached_lens.device)
    kv_indices, _, slot_map, kv_lens, qo, kv_indptr, left, status = buf.split_with_sizes(
        (max_rows, rows_room - max_rows, max_tokens, batch, batch + 1, batch + 1, 1, 1))
    positions = torch.empty(max_tokens, dtype=torch.int64, device=cached_lens.device)
    base = buf.data_ptr()
    slots = base + 4 * rows_room
    lens = slots + 4 * max_tokens
    check(lib.cf_paged_kv_plan(cp, np_, batch, tp, block_table.shape[1], block_table.stride(0) if batch > 1 else block_table.shape[1], fp, free_pages.shape[0],
                               fc, lens + 4 * (3 * batch + 2), int(page_size), lens, lens + 4 * batch, positions.data_ptr(), slots, max_tokens,
                               lens + 4 * (2 * batch + 1), base, max_rows, lens + 4 * (3 * batch + 3), _stream()))
    return PagedKvPlan(kv_lens, qo, positions, slot_map, kv_indptr, kv_indices, left, status)


def paged_kv_release(finished, kv_lens, block_table, free_pages, free_count, page_size: int):
    """Gives the pages of the requests with finished[b] != 0 (int32 [batch]) back: the first ceil(kv_lens[b] / page_size) entries of their
    table rows go on top of free_pages and become -1.  Returns (free_count, status), int32 [1] each; all or nothing like paged_kv_plan."""
    dev = torch.cuda.current_device()
    batch = kv_lens.shape[0] if isinstance(kv_lens, torch.Tensor) and kv_lens.dim() == 1 else -1
    lp, dp = _ints(kv_lens, "kv_lens", dev), _ints(finished, "finished", dev, batch)
    tp = _table(block_table, "block_table", dev, batch)
    fp, fc = _ints(free_pages, "free_pages", dev), _ints(free_count, "free_count", dev, 1)
    left, status = torch.empty(2, dtype=torch.int32, device=kv_lens.device).split_with_sizes((1, 1))
    check(lib.cf_paged_kv_release(dp, lp, batch, tp, block_table.shape[1], block_table.stride(0) if batch > 1 else block_table.shape[1], fp, free_pages.shape[0], fc,
                                  left.data_ptr(), int(page_size), status.data_ptr(), _stream()))
    return left, status


def kv4_cache(pages: int, kv_heads: int, page_size: int, head_dim: int, device=None) -> torch.Tensor:
    """An empty paged cache held in 4 bits: uint8 [pages, kv_heads, page_size, 40 * ceil(head_dim / 32)], 5 bits a value (32 values share an
    fp16 scale and minimum).  page_size is a multiple of 16, head_dim a multiple of 8 in 16..128."""
    if page_size < 16 or page_size % 16 or head_dim < 16 or head_dim > 128 or head_dim % 8:
        raise RuntimeError(f"page_size {page_size} must be a multiple of 16, head_dim {head_dim} a multiple of 8 in 16..128")
    return torch.zeros(pages, kv_heads, page_size, 40 * ((head_dim + 31) // 32), dtype=torch.uint8, device="cuda" if device is None else device)


def kv4_append(key, value, slot_map, cache) -> None:
    """Writes key and value [tokens, kv_heads, head_dim] (fp16 or bf16; slices of a fused projection are fine) to the cache's rows
    slot_map (int32 [tokens]; below 0: skipped).  No two tokens of a call may name the same row.  A row beyond the cache is
    skipped and reported by device_status()."""
    dev = torch.cuda.current_device()
    kp, vp = _rows(key, "key", dev, 3, 4), _rows(value, "value", dev, 3, 4)
    tokens, heads, dim = key.shape
    if value.shape != key.shape or value.dtype != key.dtype:
        raise RuntimeError(f"value: expected {tuple(key.shape)} of {key.dtype} like key, got {tuple(value.shape)} of {value.dtype}")
    pages, page = _cache_shape(cache, dev, heads, dim)
    ks, vs = key.stride(), value.stride()
    check(lib.cf_kv4_append(kp, vp, _HALVES[key.dtype], tokens, heads, dim, ks[0], ks[1], vs[0], vs[1], _ints(slot_map, "slot_map", dev, tokens),
                            cache.data_ptr(), pages, page, _stream()))


def kv4_read(cache, slot_map, head_dim: int, dtype=torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(key, value), each [tokens, kv_heads, head_dim] of `dtype`: what the cache's rows slot_map hold (zeros for a row below 0).  The rows of
    a request, in order, are the contiguous caches that the batch-1 blocks read."""
    dev = torch.cuda.current_device()
    sp = _ints(slot_map, "slot_map", dev)
    if dtype not in _HALVES:
        raise RuntimeError(f"dtype: expected torch.float16 or torch.bfloat16, got {dtype}")
    heads, dim, tokens = cache.shape[1] if isinstance(cache, torch.Tensor) and cache.dim() == 4 else -1, int(head_dim), slot_map.shape[0]
    pages, page = _cache_shape(cache, dev, heads, dim)
    key = torch.empty(tokens, heads, dim, dtype=dtype, device=cache.device)
    value = torch.empty_like(key)
    check(lib.cf_kv4_read(cache.data_ptr(), pages, page, heads, dim, sp, tokens, key.data_ptr(), value.data_ptr(), _HALVES[dtype], _stream()))
    return key, value


def kv4_attention(query, cache, block_table, kv_lens, qo_indptr=None, max_q_len: int = 1, scale: Optional[float] = None, out=None) -> torch.Tensor:
    """Causal attention of query [rows, heads, head_dim] (fp16 or bf16, a slice of a fused projection is fine) over the paged 4-bit cache;
    [rows, heads, head_dim].  heads is a multiple of the cache's heads.

    Request b owns the rows qo_indptr[b] : qo_indptr[b + 1] (int32 [batch + 1]; None: row b).  They are its last tokens and in the cache
    already: of n queries the i-th sees the first kv_lens[b] - n + i + 1 tokens of the pages block_table[b].  A query that sees
    none gives zeros.  Rows that no request owns are left as they were in `out` (undefined without `out`).  max_q_len: the most rows
    of a request; a hint for the size of the launch, the result does not depend on it.  scale: 1 / sqrt(head_dim) if None."""
    dev = torch.cuda.current_device()
    qp = _rows(query, "query", dev, 3, 8)
    rows, heads, dim = query.shape
    batch = kv_lens.shape[0] if isinstance(kv_lens, torch.Tensor) and kv_lens.dim() == 1 else -1
    lp = _ints(kv_lens, "kv_lens", dev)
    ip = None if qo_indptr is None else _ints(qo_indptr, "qo_indptr", dev, batch + 1)
    tp = _table(block_table, "block_table", dev, batch)
    kv_heads = cache.shape[1] if isinstance(cache, torch.Tensor) and cache.dim() == 4 else -1
    pages, page = _cache_shape(cache, dev, kv_heads, dim)
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=query.dtype, device=query.device)
    else:
        _on_device(out, "out", dev, 3)
        if out.shape != query.shape or out.dtype != query.dtype or not out.is_contiguous():
            raise RuntimeError(f"out: expected a contiguous {tuple(query.shape)} of {query.dtype}, got {tuple(out.shape)} of {out.dtype}")
    qs = query.stride()
    check(lib.cf_kv4_attention(qp, _HALVES[query.dtype], rows, heads, dim, qs[0], qs[1], cache.data_ptr(), pages, page, kv_heads, tp, block_table.shape[1],
                               block_table.stride(0) if batch > 1 else block_table.shape[1], lp, ip, batch, int(max_q_len),
                               dim ** -0.5 if scale is None else float(scale), out.data_ptr(), _stream()))
    return out


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # [rows] fp32: log probability of the given token
    entropy: torch.Tensor       # [rows] fp32, natural logarithm
    top_logprobs: torch.Tensor  # [rows, top_k] fp32, greatest first
    top_tokens: torch.Tensor    # [rows, top_k] int64; equal probabilities by the lower token


def token_logprobs(logits, tokens, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of tokens (int32 or int64 [rows]) under softmax(logits) ([rows, vocab] or [vocab]; fp16, bf16 or fp32, rows may be
    apart), the entropy of each row and its top_k (up to 32) most probable tokens.  A token outside the vocabulary has log
    probability -inf; a row with +inf or NaN, or with nothing but -inf, gives NaN.  Takes PythiaDecoder.logits as it is."""
    dev = torch.cuda.current_device()
    if isinstance(logits, torch.Tensor) and logits.dim() == 1:
        logits = logits[None]
    _on_device(logits, "logits", dev, 2)
    _on_device(tokens, "tokens", dev, 1)
    rows, vocab = logits.shape
    if logits.dtype not in _LOGITS:
        raise RuntimeError(f"logits: expected float16, bfloat16 or float32, got {logits.dtype}")
    if logits.stride(1) != 1 and vocab > 1:
        raise RuntimeError(f"logits: expected a contiguous last axis, got strides {logits.stride()}")
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.shape[0] != rows or not tokens.is_contiguous():
        raise RuntimeError(f"tokens: expected {rows} contiguous int32 or int64 entries, got {tuple(tokens.shape)} of {tokens.dtype}")
    top_k = int(top_k)
    if top_k < 0 or top_k > 32 or top_k > vocab:
        raise RuntimeError(f"top_k {top_k} outside 0..{min(32, vocab)}")
    both = torch.empty(2, rows, dtype=torch.float32, device=logits.device)
    top_lp = torch.empty(rows, top_k, dtype=torch.float32, device=logits.device)
    top_id = torch.empty(rows, top_k, dtype=torch.int64, device=logits.device)
    lp, entropy = both.unbind()
    check(lib.cf_token_logprobs(logits.data_ptr(), _LOGITS[logits.dtype], rows, vocab, logits.stride(0), tokens.data_ptr(), tokens.element_size(), top_k,
                                both.data_ptr(), both.data_ptr() + 4 * rows, top_lp.data_ptr(), top_id.data_ptr(), _stream()))
    return TokenLogprobs(lp, entropy, top_lp, top_id)
