"""A paged key/value cache for serving requests of different ages: the page pools of every attention layer, the block
table, the lengths and the free list, and one step of a batch over them.

The reference's streaming state (model.py:352-366) holds one dense window per stream and moves all streams in lock step
(`conformer_amd.streaming.StreamCache` is its ring form).  Here a request holds as many pages as its length needs,
starts and ends on its own, and may bring any number of rows per step:

    cache = KVPages(layers=17, pages=4096, kv_heads=4, head_dim=64, batch=64, max_tokens=8192)
    step = cache.plan(new_lens, rows)                 # new_lens int32 [64] on the GPU, rows = their sum
    for i in range(17):
        cache.write(i, k, v)                          # the rows' keys and values, [rows][4][64]
        out = cache.attend(i, q, max_rows=8)          # [rows][heads][64]
    tokens = ops.sample_tokens(logits, u, temperature, top_k, top_p)

Nothing here synchronises; all state advances on the device, in place, so a step can be captured into a HIP graph and
replayed (`rows` is then the capacity of the step: rows that belong to nobody get slot -1 and zeros).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import ops

Tensor = torch.Tensor


class Step(NamedTuple):
    """What `KVPages.plan` found: where the rows go (int64 [rows], -1: nowhere), where requests begin in them (int32
    [batch + 1]), and which requests got their pages (bool [batch])."""
    slots: Tensor
    cu_rows: Tensor
    granted: Tensor


class KVPages:
    """`pages` pages of `page_size` tokens (a power of two, 16 to 1024) shared by `batch` table rows, for `layers` layers of
    `kv_heads` heads of `head_dim` (at most 128, a multiple of 8); a request holds up to `max_tokens` tokens."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, batch: int, max_tokens: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(layers, pages, kv_heads, head_dim, batch, max_tokens) < 1:
            raise ValueError("KVPages: every size must be positive")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"KVPages: the page size must be a power of two, 16 to 1024, not {page_size}")
        if head_dim > 128 or head_dim % 8:
            raise ValueError(f"KVPages: head_dim must be at most 128 and a multiple of 8, not {head_dim}")
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"KVPages: dtype must be float32 or bfloat16, not {dtype}")
        self.page_size, self.layers, self.batch = page_size, layers, batch
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=device)      # what nobody has written is never read
        self.v_pages = torch.empty(shape, dtype=dtype, device=device)
        self.block_table = torch.full((batch, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=device)
        self.kv_lens = torch.zeros((batch,), dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self.step: Optional[Step] = None

    def plan(self, new_lens: Tensor, rows: int, finished: Optional[Tensor] = None) -> Step:
        """Opens a step: table row b brings new_lens[b] rows (int32 [batch], 0 for none), after `finished` rows (bool
        [batch]) gave their pages back.  A request that finds too few pages is refused whole, keeps its length and can
        come again; its rows of this step go nowhere and their attention output means nothing."""
        self.step = Step(*ops.kv_page_plan_(self.kv_lens, new_lens, finished, self.block_table, self.free_pages,
                                            self.free_count, self.page_size, rows))
        return self.step

    def _open(self) -> Step:
        if self.step is None:
            raise RuntimeError("KVPages: no step is open; call plan() first")
        return self.step

    def write(self, layer: int, k: Tensor, v: Tensor) -> None:
        """The step's keys and values of a layer, [rows][kv_heads][head_dim], into their slots."""
        ops.kv_page_write_(k, v, self.k_pages[layer], self.v_pages[layer], self._open().slots)

    def attend(self, layer: int, q: Tensor, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
               causal: bool = True, max_rows: int = 0) -> Tensor:
        """Attention of the step's rows [rows][heads][head_dim] over everything their requests hold in a layer, the rows'
        own keys included (write them first); see `ops.kv_page_attention`.  scale: 1 / sqrt(head_dim) if not given."""
        step = self._open()
        if q.shape[0] != step.slots.shape[0]:                 # the last requests' rows would sit at other positions
            raise ValueError(f"KVPages: {q.shape[0]} rows of q in a step of {step.slots.shape[0]}")
        if scale is None:
            scale = q.shape[-1] ** -0.5
        return ops.kv_page_attention(q, self.k_pages[layer], self.v_pages[layer], self.block_table, self.kv_lens,
                                     step.cu_rows, scale, window, sinks, causal, max_rows)
