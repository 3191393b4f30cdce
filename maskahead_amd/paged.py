"""A paged 4-bit KV cache for a batch of requests of their own lengths.

``PackedKVCache`` keeps one length for all its batch rows, as the reference's cache does
(cache.py:94-96), and a batch of ragged requests then needs a cache, and a launch, each.
``PagedKVCache`` holds every request's tokens in pages of one pool per layer; block tables,
lengths and the ring of free pages lie on the GPU, so a step of the whole batch -- plan,
attention and append of every layer, commit -- is enqueued without a look at a length, and
can be captured in a HIP graph and replayed while the requests grow.

Codes, scales and zeros equal ``PackedKVCache``'s with ``residual_tokens=0`` for the same
tokens, bit for bit: whole groups of 32 are 4-bit, the newest length % 32 tokens 16-bit.

    cache.begin_append(new_lens, tokens=T)                 # int32 [B] on the GPU, 0 = idle
    for layer ...:
        out = cache.attend(layer, q, k, v)                 # [stored | this block]
        cache.stage_layer(layer, k, v)
    cache.commit_append()
    cache.release(finished)                                # bool [B]: their pages go back
"""

from __future__ import annotations

import torch

from ._native import KernelUnavailableError
from .kernels.paged import (GROUP, PagedPrefix, append_pages, check_plan, dequantize_pages, paged_attention,
                            plan_pages, record_bytes)


class PagedKVCache:
    """num_pages pages of page_tokens tokens (a multiple of 32), shared by batch_size requests
    of at most max_tokens tokens each; the same pages of every layer belong to one request.

    lengths int32 [B], block_table int32 [B, width], free_ring and ring_state are the kernels'
    own (``kernels.paged.plan_pages``); pool uint8 [L, pages, Hkv, page_tokens / 32, 40 D],
    k_tail and v_tail [L, B, Hkv, 32, D]."""

    def __init__(self, *, num_layers: int, batch_size: int, num_kv_heads: int, head_dim: int, num_pages: int,
                 max_tokens: int, page_tokens: int = 64, device: torch.device | str = "cuda",
                 compute_dtype: torch.dtype = torch.bfloat16) -> None:
        if min(num_layers, batch_size, num_kv_heads, head_dim, num_pages, max_tokens) <= 0:
            raise ValueError("all cache dimensions must be positive")
        if page_tokens <= 0 or page_tokens % GROUP:
            raise ValueError(f"page_tokens must be a positive multiple of {GROUP}")
        if head_dim not in (64, 128):
            raise KernelUnavailableError(f"head_dim {head_dim} is not built (64, 128)")
        if compute_dtype not in (torch.bfloat16, torch.float16):
            raise KernelUnavailableError(f"compute dtype {compute_dtype} is not built (bf16, f16)")
        self.num_layers, self.batch_size = int(num_layers), int(batch_size)
        self.num_kv_heads, self.head_dim = int(num_kv_heads), int(head_dim)
        self.num_pages, self.max_tokens, self.page_tokens = int(num_pages), int(max_tokens), int(page_tokens)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise KernelUnavailableError(f"a paged cache lives on the GPU, not on {self.device}")
        self.compute_dtype = compute_dtype
        dev, lead = self.device, (num_layers, batch_size, num_kv_heads)
        self.pool = torch.empty((num_layers, num_pages, num_kv_heads, page_tokens // GROUP, record_bytes(head_dim)),
                                device=dev, dtype=torch.uint8)
        self.k_tail = torch.empty(lead + (GROUP, head_dim), device=dev, dtype=compute_dtype)
        self.v_tail = torch.empty_like(self.k_tail)
        self.block_table = torch.full((batch_size, -(-max_tokens // page_tokens)), -1, device=dev, dtype=torch.int32)
        self.lengths = torch.zeros((batch_size,), device=dev, dtype=torch.int32)
        self.free_ring = torch.arange(num_pages, device=dev, dtype=torch.int32)
        self.ring_state = torch.tensor([0, num_pages, 0, 0], device=dev, dtype=torch.int32)
        self.prefixes = [self.prefix(i) for i in range(num_layers)]
        self._plan: tuple | None = None     # (new_lens, slots, ends, staged layers) of an append in progress

    def _check_layer(self, layer: int) -> None:
        if not 0 <= layer < self.num_layers:
            raise IndexError(layer)

    def prefix(self, layer: int, *, mask: torch.Tensor | None = None) -> PagedPrefix:
        """The kernels' descriptor of one layer, with an optional mask of dead entries."""
        self._check_layer(layer)
        return PagedPrefix(self.pool[layer], self.k_tail[layer], self.v_tail[layer], self.block_table, self.lengths,
                           mask=mask)

    def _check_readable(self, layer: int) -> None:
        """A staged layer's tail holds the new tokens while lengths are still the old ones."""
        self._check_layer(layer)
        if self._plan is not None and layer in self._plan[3]:
            raise RuntimeError(f"layer {layer} was staged: it can be read again after commit_append")

    @property
    def append_in_progress(self) -> bool:
        return self._plan is not None

    # -- one step -------------------------------------------------------------------------
    def begin_append(self, new_lens: torch.Tensor, tokens: int) -> torch.Tensor:
        """Open an append of new_lens[b] (0 .. tokens) tokens to every layer and give their pages
        to the requests.  Returns the slots [B, tokens] (``plan_pages``).  A plan that cannot be
        met (a negative count among what it refuses) stores nothing and leaves every length as it is; ``check`` reports it.  new_lens is
        read until the commit: it must not change before."""
        if self._plan is not None:
            raise RuntimeError("another cache append is already in progress")
        if tokens <= 0:
            raise ValueError("tokens must be positive")
        slots, ends = plan_pages(self.lengths, new_lens, self.block_table, self.free_ring, self.ring_state,
                                 page_tokens=self.page_tokens, tokens=tokens, give_back=False)
        self._plan = (new_lens, slots, ends, set())
        return slots

    def stage_layer(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Write one layer's new tokens, key and value [B, Hkv, T, D] (rows behind a request's
        new_lens are not read).  The layer is not read again before the commit."""
        if self._plan is None:
            raise RuntimeError("begin_append must be called before stage_layer")
        new_lens, slots, _, staged = self._plan
        if layer in staged:
            raise RuntimeError(f"layer {layer} was staged twice")
        self._check_layer(layer)
        append_pages(self.prefixes[layer], key, value, new_lens, slots)
        staged.add(layer)

    def commit_append(self) -> None:
        """Take the new lengths, when every layer has been staged."""
        if self._plan is None:
            raise RuntimeError("no append is in progress")
        missing = set(range(self.num_layers)) - self._plan[3]
        if missing:
            raise RuntimeError(f"cannot commit: layers not staged: {sorted(missing)}")
        self.lengths.copy_(self._plan[2])
        self._plan = None

    def abort_append(self) -> None:
        """Give the step up before any layer was staged (a staged layer's tails are already the
        new ones): its pages go back."""
        if self._plan is None:
            return
        _, _, ends, staged = self._plan
        if staged:
            raise RuntimeError(f"cannot abort: layers {sorted(staged)} were staged")
        plan_pages(ends, self.lengths - ends, self.block_table, self.free_ring, self.ring_state,
                   page_tokens=self.page_tokens, tokens=0)
        self._plan = None

    def release(self, finished: torch.Tensor) -> None:
        """Drop the requests that finished [B] (bool, on the GPU) names: length 0, pages free."""
        if self._plan is not None:
            raise RuntimeError("release during an append")
        if finished.dtype != torch.bool or tuple(finished.shape) != (self.batch_size,):
            raise ValueError(f"finished must be a bool [{self.batch_size}] tensor")
        _, ends = plan_pages(self.lengths, torch.where(finished, -self.lengths, 0).to(torch.int32), self.block_table,
                             self.free_ring, self.ring_state, page_tokens=self.page_tokens, tokens=0)
        self.lengths.copy_(ends)

    def check(self) -> None:
        """Raise RuntimeError for a plan that could not be met since the last check (waits)."""
        check_plan(self.ring_state)

    # -- reading --------------------------------------------------------------------------
    def attend(self, layer: int, query: torch.Tensor, current_key: torch.Tensor | None = None,
               current_value: torch.Tensor | None = None, *, new_lens: torch.Tensor | None = None,
               scaling: float | None = None, causal_block: int = 0, mask: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """``paged_attention`` of one layer over [stored | block]; new_lens defaults to that of
        the append in progress.  RuntimeError between a layer's stage_layer and the commit."""
        if new_lens is None and self._plan is not None:
            new_lens = self._plan[0]
        self._check_readable(layer)
        prefix = self.prefixes[layer] if mask is None else self.prefix(layer, mask=mask)
        return paged_attention(query, prefix, current_key, current_value, new_lens=new_lens, scaling=scaling,
                               causal_block=causal_block, out=out)

    def dequantize_layer(self, layer: int, tokens: int, *, starts: torch.Tensor | None = None,
                         dtype: torch.dtype | None = None):
        """``dequantize_pages`` of one layer: [B, Hkv, tokens, D] K and V.  RuntimeError between a
        layer's stage_layer and the commit."""
        self._check_readable(layer)
        return dequantize_pages(self.prefixes[layer], tokens, starts=starts, dtype=dtype)


__all__ = ["PagedKVCache"]
