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

import functools
from typing import NamedTuple, Optional, Tuple

import torch

from ._lib import CF_DTYPE_BF16, CF_DTYPE_FP16, CF_DTYPE_FP32, check, lib

_HALVES = {torch.float16: CF_DTYPE_FP16, torch.bfloat16: CF_DTYPE_BF16}
_LOGITS = {**_HALVES, torch.float32: CF_DTYPE_FP32}
_I32, _I64 = torch.int32, torch.int64
_current_device = torch.cuda.current_device
# The steps that these calls make are short (a few microseconds on the GPU), so the checks below look at a tensor once when it is in order
# and find out what is wrong only when it is not.  current_stream() builds a Stream object (3 us); this is the number in it.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _complain(t, name: str, device: int, dims: int, dtypes, what: str) -> None:
    """Raises what is wrong with a tensor that failed its check."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name}: expected a torch.Tensor")
    if t.get_device() != device:
        raise RuntimeError(f"{name}: tensor is on {t.device} but the current device is cuda:{device}" if t.is_cuda
                           else f"{name}: expected a CUDA tensor, got {t.device}")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name}: expected dtype {' or '.join(map(str, dtypes))}, got {t.dtype}")
    if t.dim() != dims:
        raise RuntimeError(f"{name}: expected {dims} dimension{'s' * (dims > 1)}, got shape {tuple(t.shape)}")
    raise RuntimeError(f"{name}: expected {what}, got shape {tuple(t.shape)} with strides {t.stride()}")


def _ints(t, name: str, device: int, n: int = -1) -> int:
    """Pointer of a contiguous int32 vector (of n entries)."""
    if isinstance(t, torch.Tensor) and t.dtype is _I32 and t.get_device() == device and t.dim() == 1 and t.is_contiguous() and (n < 0 or t.numel() == n):
        return t.data_ptr()
    return _complain(t, name, device, 1, (_I32,), "a contiguous tensor" if n < 0 else f"{n} contiguous entries")


def _table(t, name: str, device: int, batch: int) -> Tuple[int, int, int]:
    """Pointer, columns and distance of the rows of a block table."""
    if isinstance(t, torch.Tensor) and t.dtype is _I32 and t.get_device() == device and t.dim() == 2:
        rows, width = t.shape
        apart, step = t.stride()
        if rows == batch and (step == 1 or width == 1) and (apart >= width or batch == 1):
            return t.data_ptr(), width, apart if batch > 1 else width
    return _complain(t, name, device, 2, (_I32,), f"[{batch}, pages] rows of consecutive entries")


def _rows(t, name: str, device: int, step: int) -> Tuple[int, int, int]:
    """Pointer and strides of [rows, heads, head_dim] whose last axis is contiguous and whose other strides are multiples of `step` elements."""
    if isinstance(t, torch.Tensor) and t.dtype in _HALVES and t.get_device() == device and t.dim() == 3:
        s0, s1, s2 = t.stride()
        if s2 == 1 and s0 % step == 0 and s1 % step == 0:
            return t.data_ptr(), s0, s1
    return _complain(t, name, device, 3, tuple(_HALVES), f"a contiguous last axis and strides in multiples of {step} elements")


def _cache(t, device: int, heads: int, head_dim: int) -> Tuple[int, int, int, int]:
    """Pointer, pages, heads (any if `heads` is negative) and page size of a 4-bit cache."""
    width = 40 * ((head_dim + 31) // 32)
    if isinstance(t, torch.Tensor) and t.dtype is torch.uint8 and t.get_device() == device and t.dim() == 4 and t.is_contiguous():
        pages, h, page, w = t.shape
        if w == width and (heads < 0 or h == heads):
            return t.data_ptr(), pages, h, page
    return _complain(t, "cache", device, 4, (torch.uint8,), f"contiguous [pages, {heads if heads >= 0 else 'kv_heads'}, page_size, {width}] for heads of {head_dim} (see kv4_cache)")


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
    dev = _current_device()
    cp = _ints(cached_lens, "cached_lens", dev)
    batch = cached_lens.numel()
    np_ = _ints(new_lens, "new_lens", dev, batch)
    tp, width, apart = _table(block_table, "block_table", dev, batch)
    fp, fc = _ints(free_pages, "free_pages", dev), _ints(free_count, "free_count", dev, 1)
    max_tokens, max_rows = int(max_tokens), int(max_rows)
    if max_tokens < 0 or max_rows < 0:
        raise RuntimeError(f"max_tokens {max_tokens} and max_rows {max_rows} must not be negative")
    rows_room = (max_rows + 3) // 4 * 4  # keeps what follows aligned
    buf = cached_lens.new_empty(rows_room + max_tokens + 3 * batch + 4)
    positions = torch.empty(max_tokens, dtype=_I64, device=cached_lens.device)
    kv_indices, _, slot_map, kv_lens, qo, kv_indptr, left, status = buf.split_with_sizes(
        (max_rows, rows_room - max_rows, max_tokens, batch, batch + 1, batch + 1, 1, 1))
    base = buf.data_ptr()
    slots = base + 4 * rows_room
    lens = slots + 4 * max_tokens
    check(lib.cf_paged_kv_plan(cp, np_, batch, tp, width, apart, fp, free_pages.numel(), fc, lens + 4 * (3 * batch + 2), int(page_size), lens, lens + 4 * batch,
                               positions.data_ptr(), slots, max_tokens, lens + 4 * (2 * batch + 1), base, max_rows, lens + 4 * (3 * batch + 3),
                               _raw_stream(dev)))
    return PagedKvPlan(kv_lens, qo, positions, slot_map, kv_indptr, kv_indices, left, status)


def paged_kv_release(finished, kv_lens, block_table, free_pages, free_count, page_size: int):
    """Gives the pages of the requests with finished[b] != 0 (int32 [batch]) back: the first ceil(kv_lens[b] / page_size) entries of their
    table rows go on top of free_pages and become -1.  Returns (free_count, status), int32 [1] each; all or nothing like paged_kv_plan."""
    dev = _current_device()
    lp = _ints(kv_lens, "kv_lens", dev)
    batch = kv_lens.numel()
    dp = _ints(finished, "finished", dev, batch)
    tp, width, apart = _table(block_table, "block_table", dev, batch)
    fp, fc = _ints(free_pages, "free_pages", dev), _ints(free_count, "free_count", dev, 1)
    left, status = kv_lens.new_empty(2).split_with_sizes((1, 1))
    check(lib.cf_paged_kv_release(dp, lp, batch, tp, width, apart, fp, free_pages.numel(), fc, left.data_ptr(), int(page_size), status.data_ptr(), _raw_stream(dev)))
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
    dev = _current_device()
    kp, k0, k1 = _rows(key, "key", dev, 4)
    vp, v0, v1 = _rows(value, "value", dev, 4)
    tokens, heads, dim = key.shape
    if value.shape != key.shape or value.dtype is not key.dtype:
        raise RuntimeError(f"value: expected {tuple(key.shape)} of {key.dtype} like key, got {tuple(value.shape)} of {value.dtype}")
    cp, pages, _, page = _cache(cache, dev, heads, dim)
    check(lib.cf_kv4_append(kp, vp, _HALVES[key.dtype], tokens, heads, dim, k0, k1, v0, v1, _ints(slot_map, "slot_map", dev, tokens), cp, pages, page,
                            _raw_stream(dev)))


def kv4_read(cache, slot_map, head_dim: int, dtype=torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(key, value), each [tokens, kv_heads, head_dim] of `dtype`: what the cache's rows slot_map hold (zeros for a row below 0).  The rows of
    a request, in order, are the contiguous caches that the batch-1 blocks read."""
    dev = _current_device()
    sp = _ints(slot_map, "slot_map", dev)
    if dtype not in _HALVES:
        raise RuntimeError(f"dtype: expected torch.float16 or torch.bfloat16, got {dtype}")
    tokens, head_dim = slot_map.numel(), int(head_dim)
    cp, pages, heads, page = _cache(cache, dev, -1, head_dim)
    shape, where = (tokens, heads, head_dim), cache.device
    key, value = torch.empty(shape, dtype=dtype, device=where), torch.empty(shape, dtype=dtype, device=where)
    check(lib.cf_kv4_read(cp, pages, page, heads, head_dim, sp, tokens, key.data_ptr(), value.data_ptr(), _HALVES[dtype], _raw_stream(dev)))
    return key, value


@functools.lru_cache(maxsize=1024)
def _attention_workspace(batch: int, heads: int, kv_heads: int, head_dim: int, max_tokens: int, max_q_len: int) -> int:
    return lib.cf_kv4_attention_workspace(batch, heads, kv_heads, head_dim, max_tokens, max_q_len)


def kv4_attention(query, cache, block_table, kv_lens, qo_indptr=None, max_q_len: int = 1, scale: Optional[float] = None, out=None) -> torch.Tensor:
    """Causal attention of query [rows, heads, head_dim] (fp16 or bf16, a slice of a fused projection is fine) over the paged 4-bit cache;
    [rows, heads, head_dim].  heads is a multiple of the cache's heads.

    Request b owns the rows qo_indptr[b] : qo_indptr[b + 1] (int32 [batch + 1]; None: row b).  They are its last tokens and in the cache
    already: of n queries the i-th sees the first kv_lens[b] - n + i + 1 tokens of the pages block_table[b].  A query that sees
    none gives zeros.  Rows that no request owns are left as they were in `out` (undefined without `out`).  max_q_len: the most rows
    of a request; a hint for the size of the launch, the result does not depend on it.  scale: 1 / sqrt(head_dim) if None."""
    dev = _current_device()
    qp, q0, q1 = _rows(query, "query", dev, 8)
    rows, heads, dim = query.shape
    lp = _ints(kv_lens, "kv_lens", dev)
    batch = kv_lens.numel()
    ip = None if qo_indptr is None else _ints(qo_indptr, "qo_indptr", dev, batch + 1)
    tp, width, apart = _table(block_table, "block_table", dev, batch)
    cp, pages, kv_heads, page = _cache(cache, dev, -1, dim)
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=query.dtype, device=query.device)
    elif not isinstance(out, torch.Tensor) or out.get_device() != dev or out.shape != query.shape or out.dtype is not query.dtype or not out.is_contiguous():
        _complain(out, "out", dev, 3, (query.dtype,), f"a contiguous {tuple(query.shape)}")
    need = _attention_workspace(batch, heads, kv_heads, dim, width * page, int(max_q_len))
    work = torch.empty(need, dtype=torch.uint8, device=query.device) if need else None  # of this call alone: graphs and streams share nothing
    check(lib.cf_kv4_attention(qp, _HALVES[query.dtype], rows, heads, dim, q0, q1, cp, pages, page, kv_heads, tp, width, apart, lp, ip, batch, int(max_q_len),
                               dim ** -0.5 if scale is None else float(scale), work.data_ptr() if need else None, need, out.data_ptr(), _raw_stream(dev)))
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
    dev = _current_device()
    if isinstance(logits, torch.Tensor) and logits.dim() == 1:
        logits = logits[None]
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _LOGITS or logits.get_device() != dev or logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        _complain(logits, "logits", dev, 2, tuple(_LOGITS), "a contiguous last axis")
    rows, vocab = logits.shape
    if not isinstance(tokens, torch.Tensor) or tokens.dtype not in (_I32, _I64) or tokens.get_device() != dev or tokens.dim() != 1 or tokens.numel() != rows or not tokens.is_contiguous():
        _complain(tokens, "tokens", dev, 1, (_I32, _I64), f"{rows} contiguous entries")
    top_k = int(top_k)
    if top_k < 0 or top_k > 32 or top_k > vocab:
        raise RuntimeError(f"top_k {top_k} outside 0..{min(32, vocab)}")
    where = logits.device
    buf = torch.empty(rows * (2 + top_k), dtype=torch.float32, device=where)
    lp, entropy, top_lp = buf.split_with_sizes((rows, rows, rows * top_k))
    top_id = torch.empty((rows, top_k), dtype=_I64, device=where)
    at = buf.data_ptr()
    check(lib.cf_token_logprobs(logits.data_ptr(), _LOGITS[logits.dtype], rows, vocab, logits.stride(0), tokens.data_ptr(), 8 if tokens.dtype is _I64 else 4, top_k,
                                at, at + 4 * rows, at + 8 * rows, top_id.data_ptr(), _raw_stream(dev)))
    return TokenLogprobs(lp, entropy, top_lp.view(rows, top_k), top_id)
