"""A paged KV cache in 8 bits for a batch of requests, beside ``dsa.DecodeKVCache``
(one sequence's contiguous cache).

``PagedKVCache`` holds the pages of all layers (the same page of every layer
belongs to the same tokens), the block tables, the requests' lengths and the
stack of free pages, all on the GPU; nothing synchronizes, so a whole serving
step can be captured into a HIP graph:

    step = cache.step(new, tokens)             # tables, slots, positions of the new tokens
    for layer in range(n):
        o = cache.update(step, q, k, v, scale, layer=layer)   # write k, v, then attend
    cache.trim(keep)                           # rejected drafts, ended requests

The reference keeps a contiguous bf16 cache for each sequence
(``mosaicvm/model/dsa_layers.py:393-400``) and has no counterpart of these.
"""
from __future__ import annotations

import torch

from .. import ops


class PagedKVCache:
    """``pages`` pages of ``page_size`` tokens (a multiple of 64) for up to
    ``max_requests`` requests of up to ``max_length`` tokens, ``layers`` layers of
    ``kv_heads`` heads of ``head_dim`` (64, 128 or 256).  A token takes 2 kv_heads
    head_dim bytes a layer, a block of 64 tokens 2 kv_heads bytes of scales."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, max_requests: int, max_length: int,
                 page_size: int = 64, layers: int = 1, device="cuda"):
        if page_size % ops.PAGED_BLOCK or not ops.PAGED_BLOCK <= page_size <= 4096:
            raise ValueError(f"page_size {page_size} must be a multiple of {ops.PAGED_BLOCK} up to 4096")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim {head_dim} must be 64, 128 or 256")
        if min(pages, kv_heads, max_requests, max_length, layers) < 1:
            raise ValueError("pages, kv_heads, max_requests, max_length and layers must be positive")
        dev = torch.device(device)
        nb = page_size // ops.PAGED_BLOCK
        self.page_size, self.kv_heads, self.head_dim = page_size, kv_heads, head_dim
        self.codes = torch.zeros(layers, pages, nb, kv_heads, 2, ops.PAGED_BLOCK * head_dim, dtype=torch.uint8, device=dev)
        self.scales = torch.full((layers, pages, nb, kv_heads, 2), 127, dtype=torch.uint8, device=dev)
        self.block_table = torch.full((max_requests, -(-max_length // page_size)), -1, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=dev)

    def step(self, new: torch.Tensor, tokens: int, out: ops.PagedStep | None = None) -> ops.PagedStep:
        """``new`` [max_requests] int32: how many tokens each request adds (0: it
        rests), in a buffer of ``tokens`` rows.  Takes the pages and commits the lengths."""
        s = ops.paged_step(self.lengths, new, self.block_table, tokens, self.page_size, self.free_pages,
                           self.free_count, out)
        self.lengths.copy_(s.lengths)
        self.free_count.copy_(s.free_count)
        return s

    def write(self, step: ops.PagedStep, k: torch.Tensor, v: torch.Tensor, layer: int = 0) -> None:
        ops.paged_kv_write(k, v, self.codes[layer], self.scales[layer], self.block_table, step.starts, step.seq_lens)

    def attend(self, step: ops.PagedStep, q: torch.Tensor, softmax_scale: float, sink: torch.Tensor | None = None,
               window: int = 0, max_new: int | None = None, layer: int = 0,
               workspace: ops.MoEWorkspace | None = None) -> torch.Tensor:
        return ops.paged_attention(q, self.codes[layer], self.scales[layer], self.block_table, step.starts,
                                   step.seq_lens, softmax_scale, sink, window, max_new, workspace=workspace)

    def update(self, step: ops.PagedStep, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float,
               sink: torch.Tensor | None = None, window: int = 0, max_new: int | None = None, layer: int = 0,
               workspace: ops.MoEWorkspace | None = None) -> torch.Tensor:
        """Write the step's keys and values of one layer, then attend: the new tokens see themselves."""
        self.write(step, k, v, layer)
        return self.attend(step, q, softmax_scale, sink, window, max_new, layer, workspace)

    def trim(self, keep: torch.Tensor) -> None:
        """Shorten request r to ``keep[r]`` tokens (0 releases it) and take its pages back, which have to be
        its own: keep those of a prefix that it shares (``ops.paged_trim``)."""
        lengths, count = ops.paged_trim(self.lengths, keep, self.block_table, self.page_size, self.free_pages,
                                        self.free_count)
        self.lengths.copy_(lengths)
        self.free_count.copy_(count)
