"""Serving a batch over a paged cache: the plan of a step, the cache held in 4 bits with the attention that reads it, and the
log probabilities of tokens.

One step of a server, all of it on the GPU and capturable (nothing is read back by the host):

    plan = cf.paged_kv_plan(cached_lens, new_lens, block_table, free_pages, free_count, page_size, max_tokens)
    cf.kv4_append(key, value, plan.slot_map, cache)                        # every layer
    out = cf.kv4_attention(query, cache, block_table, plan.kv_lens, plan.qo_indptr, max_q_len=longest)
    ...
    scored = cf.token_logprobs(logits, tokens, top_k=5)

A plan made with max_rows and max_tokens = batch, in which every request gets one token, is what llama_decoder_layer_batch_decode_sglang
takes: kv_indptr, kv_indices and positions as they are.  That block always writes one token a request, to the last row of its list, so a request
that gets no token in a step must hold none (cached 0: its list is empty and nothing is written) or be left out of the plan.  With
such idle requests positions, which has one entry a token, is not one a request: pass (plan.kv_lens - 1).clamp(min=0).long().  Of a plan that
did not fit the block writes nothing either.  The reference's batched entry point (include/pybind.cpp:90-106) leaves all of this to its
caller.  Like the rest of the package these functions validate, allocate their results and launch on torch's current stream.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ._lib import serving_binding

# The steps that these calls make are short (a few microseconds on the GPU): the tensors are checked, and the results allocated, in
# csrc/serving_binding.cpp.
class _Calls:
    """The calls of that module, which the first of them loads."""

    def __getattr__(self, name):
        if name not in ("plan", "release", "append", "read", "attention", "logprobs"):
            raise AttributeError(name)
        module = serving_binding()
        self.__dict__.update({n: getattr(module, n) for n in ("plan", "release", "append", "read", "attention", "logprobs")})
        return self.__dict__[name]


_call = _Calls()
_workspace = None  # bytes of kv4_attention's workspace; None: what cf_kv4_attention_workspace says


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

    All or nothing: if the pages, the table's columns, max_tokens or max_rows do not suffice, a length is negative, or free_count is not one
    that free_pages can have, nothing changes, the lists come back empty and status[0] holds CF_PLAN_* bits.  Read it where the host waits anyway.  The results share one
    allocation: keeping one of them keeps all."""
    return PagedKvPlan._make(_call.plan(cached_lens, new_lens, block_table, free_pages, free_count, page_size, max_tokens, max_rows))


def paged_kv_release(finished, kv_lens, block_table, free_pages, free_count, page_size: int):
    """Gives the pages of the requests with finished[b] != 0 (int32 [batch]) back: the first ceil(kv_lens[b] / page_size) entries of their
    table rows go on top of free_pages and become -1.  Returns (free_count, status), int32 [1] each; all or nothing like paged_kv_plan.
    Pages are not counted: one that several requests name goes onto the list with each of them."""
    return _call.release(finished, kv_lens, block_table, free_pages, free_count, page_size)


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
    _call.append(key, value, slot_map, cache)


def kv4_read(cache, slot_map, head_dim: int, dtype=torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(key, value), each [tokens, kv_heads, head_dim] of `dtype`: what the cache's rows slot_map hold (zeros for a row below 0).  The rows of
    a request, in order, are the contiguous caches that the batch-1 blocks read."""
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise RuntimeError(f"dtype: expected torch.float16 or torch.bfloat16, got {dtype}")
    return _call.read(cache, slot_map, head_dim, dtype is torch.bfloat16)


def kv4_attention(query, cache, block_table, kv_lens, qo_indptr=None, max_q_len: int = 1, scale: Optional[float] = None, out=None) -> torch.Tensor:
    """Causal attention of query [rows, heads, head_dim] (fp16 or bf16, a slice of a fused projection is fine) over the paged 4-bit cache;
    [rows, heads, head_dim].  heads is a multiple of the cache's heads.

    Request b owns the rows qo_indptr[b] : qo_indptr[b + 1] (int32 [batch + 1]; None: row b).  They are its last tokens and in the cache
    already: of n queries the i-th sees the first kv_lens[b] - n + i + 1 tokens of the pages block_table[b].  A query that sees
    none gives zeros.  Rows that no request owns are left as they were in `out` (undefined without `out`), which must not overlap the queries.  scale:
    1 / sqrt(head_dim) if None.

    How the work is dealt out is chosen by max_q_len, the most rows of a request, and by the columns of block_table, the most pages of one: neither
    changes what is computed, but both should fit the step.  Of a table as wide as the longest context pass the columns in use,
    block_table[:, :n] (8 requests of up to 2048 tokens with 6 queries each: 26 us in a table for 131072 tokens, 21 in its first columns).  Requests of
    a few rows and long chunks of prompts are better two calls, with the same `out` and the parts of each list: with the n decoding requests first,
    query, block_table[:n], kv_lens[:n], qo_indptr[: n + 1] and the same from n (63 requests of up to 8192 tokens beside a chunk of 512: 566 us in one
    call, 243 in two)."""
    return _call.attention(query, cache, block_table, kv_lens, qo_indptr, max_q_len, scale, out, _workspace)


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # [rows] fp32: log probability of the given token
    entropy: torch.Tensor       # [rows] fp32, natural logarithm
    top_logprobs: torch.Tensor  # [rows, top_k] fp32, greatest first
    top_tokens: torch.Tensor    # [rows, top_k] int64; equal probabilities by the lower token


def token_logprobs(logits, tokens, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of tokens (int32 or int64 [rows]) under softmax(logits) ([rows, vocab] or [vocab]; fp16, bf16 or fp32, rows may be
    apart), the entropy of each row and its top_k (up to 32) most probable tokens.  A token outside the vocabulary has log
    probability -inf; a row with +inf or NaN, or with nothing but -inf, gives NaN.  Takes PythiaDecoder.logits as it is."""
    return TokenLogprobs._make(_call.logprobs(logits, tokens, top_k))
