"""Serving with the sparse-regular patterns: a paged cache of keys and values, and attention over it.

No counterpart in the reference, which attends over whole sequences.  A query at position i attends to the keys
``i - k * stride >= 0`` with ``k < taps`` (``taps=0``: all of them), the causal patterns of ``acsr_helpers``:

  full causal                        taps=0, stride=1
  create_causal_windowed_mask(n, p)  taps=p + 1, stride=1
  create_strided_mask(n, s)          taps=0, stride=s      (but a row alone in its column attends to itself, where the
                                                           reference's metadata describe column 0)
  create_dilated_mask(n, t, s)       taps=t, stride=s

A cache is two tensors (pages, K/V heads, page size, head size), at any strides but a contiguous last dimension; token j of
request b is row ``j % page_size`` of page ``block_table[b, j // page_size]``.  Entries of the block table outside
``[0, pages)`` are pages that are not there: nothing is written to them and their keys are not attended to.

The launchers work with lengths that are on the device only, read nothing back, and can be captured in a CUDA graph.  They
have no gradients.
``PagedAttention`` keeps the buffers that they need.
"""
from __future__ import annotations

from typing import Any

import torch
import torch.nn as nn

import splat_native as _n


def rpaged_tables_launcher(ctx_lens: torch.Tensor, q_lens: torch.Tensor, block_table: torch.Tensor,
                           free_pages: torch.Tensor, free_span: torch.Tensor, page_size: int, kv_lens: torch.Tensor,
                           q_start: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor, requests: torch.Tensor,
                           free_span_out: torch.Tensor) -> None:
    """Bookkeeping of a step, on the device.  Request b has ctx_lens[b] tokens in the cache and brings q_lens[b] (int32;
    negative ones count as 0).

    Pages that it needs in addition come from a ring of free ones, in the order of the requests: ``free_pages[i % len]`` for
    ``free_span[0] <= i < free_span[1]`` (int64).  Their entries are written into block_table (requests, width) int32, which
    otherwise stays as it is.  Written besides: kv_lens (int32, ctx + q), q_start (int32, requests + 1: exclusive sums of
    q_lens), for every row of tokens slots (int64: page * page_size + row), positions and requests (int32) -- rows behind the
    last request get -1, 0 and -1 -- and free_span_out (int64: what is left of free_span, and how many pages were
    missing).  A page that is missing, because the ring is empty or the table too narrow, leaves -1 in the table and
    in the slots.  Pages are taken, and entered in the table, for all that q_lens says, also for tokens that slots has no row
    for.  free_span_out is an array of its own, so that a call can be repeated."""
    _n.paged_tables(ctx_lens, q_lens, block_table, free_pages, free_span, page_size, kv_lens, q_start, slots, positions,
                    requests, free_span_out)


def rpaged_append_launcher(q, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           slots: torch.Tensor, q_out=None, *, positions=None, inv_freq=None, sections=None,
                           interleaved: bool = False) -> None:
    """k, v (tokens, K/V heads, d) into the rows `slots` (int64) of the cache; q (tokens, heads, d), or None, into q_out,
    which may be q itself.  With positions ((axes, tokens) or (tokens), int32 or int64) and inv_freq, q and k are turned
    on the way, as by ``r_rotary.rrotary``.  Slots outside the cache are left out; two tokens may not have the same slot."""
    _n.paged_append(q, k, v, k_cache, v_cache, slots, q_out, positions, inv_freq, sections, interleaved)


def rpaged_attention_launcher(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                              kv_lens: torch.Tensor, output: torch.Tensor, *, q_start=None, max_q_len=None,
                              scale: float = 1.0, taps: int = 0, stride: int = 1, softcap: float = 0.0, slopes=None,
                              lse=None) -> torch.Tensor:
    """Attention of the step's queries over the cache, which already holds their own keys and values.

    q (tokens, heads, d), heads a multiple of the cache's, d up to 256.  Request b's queries are the rows ``q_start[b]`` to
    ``q_start[b + 1] - 1`` (int32; without q_start one token for each request), its last tokens of the kv_lens[b] (int32)
    there are.  Scores: ``scale * q.k`` (default 1, as everywhere here), with ``softcap > 0`` capped to
    ``softcap * tanh(x / softcap)``, less ``slopes[head] * (i - j)`` if slopes (float32, heads) are given.  output (tokens,
    heads, d): softmax times V, zeros for a query without a key.  lse: float32 (tokens, heads), receives the natural
    log-sum-exp of the scores, -inf without a key.  Scores and sums are held in 32 bits; with 16-bit operands probabilities are
    rounded to their type before they are multiplied with V.  Rows that belong to no request are left as they are.  max_q_len: no
    request brings more tokens; it only helps to choose the kernel.  Returns output."""
    _n.paged_attention(q, k_cache, v_cache, block_table, kv_lens, output, q_start, max_q_len, scale, taps, stride, softcap,
                       slopes, lse)
    return output


class PagedAttention(nn.Module):
    """Cache, tables and buffers of the launchers above, for up to max_requests requests of up to max_len tokens and steps of
    up to max_tokens new ones.

    A step: ``begin_step(ctx_lens, q_lens)`` once, then ``forward(q, k, v, layer)`` for every layer.  Rows of q, k and v are
    the requests' new tokens behind one another; rows behind the last one are left alone.  ctx_lens are what the last step left, or 0
    behind a ``release``, or less behind a ``rewind``.  ``forward`` returns the
    module-owned output buffer (the same tensor on every call).  Everything runs on the current stream without reading
    anything back and can be captured; two graphs that use one module share its buffers, so they may not run at the same time."""

    def __init__(self, num_pages: int, page_size: int, num_heads: int, num_kv_heads: int, head_dim: int,
                 max_requests: int, max_tokens: int, max_len: int, GPU_ID: Any, out_dtype: torch.dtype, *,
                 num_layers: int = 1, scale: float = 1.0, taps: int = 0, stride: int = 1, softcap: float = 0.0, slopes=None,
                 inv_freq=None, sections=None, interleaved: bool = False, lse: bool = False):
        super().__init__()
        self.device = dev = _n.resolve_device(GPU_ID)
        self.page_size, self.scale, self.taps, self.stride, self.softcap = page_size, scale, taps, stride, softcap
        self.slopes, self.inv_freq, self.sections, self.interleaved = slopes, inv_freq, sections, interleaved

        def ints(*shape, dtype=torch.int32, fill=0):
            return torch.full(shape, fill, dtype=dtype, device=dev)

        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.k_cache, self.v_cache = (torch.zeros(shape, dtype=out_dtype, device=dev) for _ in range(2))
        self.block_table = ints(max_requests, -(-max_len // page_size), fill=-1)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=dev)
        self.free_span = torch.tensor([0, num_pages], dtype=torch.int64, device=dev)
        self.free_span_out = ints(3, dtype=torch.int64)
        self.kv_lens, self.q_start = ints(max_requests), ints(max_requests + 1)
        self.slots, self.positions, self.requests = ints(max_tokens, dtype=torch.int64), ints(max_tokens), ints(max_tokens)
        self.q_turned, self.output = (torch.zeros((max_tokens, num_heads, head_dim), dtype=out_dtype, device=dev)
                                      for _ in range(2))
        self.lse = torch.zeros((max_tokens, num_heads), dtype=torch.float32, device=dev) if lse else None
        self.max_q_len = max_tokens
        _n.status_word(dev)

    def begin_step(self, ctx_lens: torch.Tensor, q_lens: torch.Tensor, max_q_len=None) -> None:
        """ctx_lens, q_lens: int32 (max_requests), tokens in the cache and new ones; 0 and 0 for a request that is not there.
        The new ones are max_tokens together at most: beyond them nothing is appended, and requests whose rows do not all fit are
        not answered (``release`` them).  max_q_len: no request brings more; without it kernels for long ones are launched, too."""
        rpaged_tables_launcher(ctx_lens, q_lens, self.block_table, self.free_pages, self.free_span, self.page_size,
                               self.kv_lens, self.q_start, self.slots, self.positions, self.requests, self.free_span_out)
        self.free_span.copy_(self.free_span_out[:2])
        self.max_q_len = self.slots.shape[0] if max_q_len is None else max_q_len

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, layer: int = 0, positions=None) -> torch.Tensor:
        """q (max_tokens, heads, d), k and v (max_tokens, K/V heads, d).  positions: (axes, max_tokens) where they are not
        the tokens' places in their requests."""
        kc, vc = self.k_cache[layer], self.v_cache[layer]
        if self.inv_freq is None:
            rpaged_append_launcher(None, k, v, kc, vc, self.slots)
        else:
            rpaged_append_launcher(q, k, v, kc, vc, self.slots, self.q_turned, inv_freq=self.inv_freq, sections=self.sections,
                                   positions=self.positions if positions is None else positions, interleaved=self.interleaved)
            q = self.q_turned
        return rpaged_attention_launcher(q, kc, vc, self.block_table, self.kv_lens, self.output, q_start=self.q_start,
                                         max_q_len=self.max_q_len, scale=self.scale, taps=self.taps, stride=self.stride,
                                         softcap=self.softcap, slopes=self.slopes, lse=self.lse)

    def missing_pages(self) -> int:
        """How many pages the last step was short of (reads the device)."""
        return int(self.free_span_out[2])

    def release(self, request: int, length: int) -> None:
        """Request `request`, of `length` tokens, is done: all of its pages are free again, those of tokens that it did not keep
        among them."""
        row = self.block_table[request]
        if not 0 <= -(-length // self.page_size) <= row.shape[0]:
            raise ValueError("release: the request cannot have had so many tokens")
        self._give_back(row, row >= 0)                     # (not those that it never got)

    def rewind(self, ctx_lens: torch.Tensor) -> None:
        """Requests go on behind ctx_lens tokens (int32, max_requests), fewer than they had where drafted tokens were refused: the
        pages behind them are free again.  Before ``begin_step`` with these ctx_lens, which would take new pages in their place."""
        held = (ctx_lens.clamp(min=0).long() + self.page_size - 1) // self.page_size
        behind = torch.arange(self.block_table.shape[1], device=ctx_lens.device) >= held[:, None]
        self._give_back(self.block_table.view(-1), (behind & (self.block_table >= 0)).view(-1))

    def _give_back(self, entries: torch.Tensor, gone: torch.Tensor) -> None:
        """Of the table's entries (a view) those that `gone` marks: pages to the end of the ring."""
        order = torch.argsort(gone.to(torch.int32), descending=True, stable=True)[:self.free_pages.shape[0]]
        at = (self.free_span[1] + torch.arange(order.shape[0], device=entries.device)) % self.free_pages.shape[0]
        self.free_pages[at] = torch.where(gone[order], entries[order], self.free_pages[at])
        self.free_span[1] += gone.sum()
        entries.masked_fill_(gone, -1)

    def check_status(self) -> None:
        """Synchronises and raises if a kernel reported a wait that ran out."""
        _n.check_status_word(self.device)
