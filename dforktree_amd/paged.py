"""A paged KV cache for the full-attention layers beside the GDN layers.

``PagedKV`` keeps what a serving loop would keep: the layers' pages, one
block table, the ring of free pages and the requests' committed lengths, all
on the device.  A step is

    plan = kv.plan(new_len, rows=..., n_new=...)  # pages, slots, positions
    for layer ...:
        kv.append(layer, k, v, plan)              # before the attention
        o = kv.attend(layer, q, plan)
    kv.commit(new_len)                            # all that have a place, or for a draft tree:
    kv.accept(layer, k, v, plan, path)            # each layer's accepted path, then
    kv.commit(path_len)

A request that the plan refuses (plan["status"]: DFT_STATUS_PAGES when the
pages ran out, DFT_STATUS_TABLE when its row of the block table is full) takes
no part in the step: nothing of it is written, its rows see no key, and
``commit`` adds nothing to its prefix, so the same tokens can be planned again
once there are pages.  One whose rows were cut (DFT_STATUS_SPAN) commits what
was left of them.

The kernels run on the current stream, nothing here waits for the device, and
``held``, ``free_pos``, ``prefix`` and ``served`` are updated in place: a step
of fixed sizes, captured in a HIP graph, goes on from where the replay before
it ended.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops


class PagedKV:
    """Pages of ``page_size`` tokens for ``layers`` layers and ``batch``
    requests of at most ``columns`` pages each.  Every layer's keys and
    values [pages, page_size, heads, head_dim] share one block table."""

    def __init__(self, layers: int, batch: int, columns: int, pages: int, page_size: int, heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        shape = (layers, pages, page_size, heads, head_dim)
        self.keys, self.values = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.page_size = page_size
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((batch, columns), -1, **i32)
        self.held, self.prefix = torch.zeros(batch, **i32), torch.zeros(batch, **i32)
        self.served = torch.zeros(batch, **i32)  # the last plan's tokens that have places and are not committed
        self.free_pages = torch.arange(pages, **i32)
        self.free_pos = torch.tensor([0, pages], dtype=torch.int64, device=device)

    def plan(self, new_len: torch.Tensor, *, rows: int, n_new: int, trim: bool = False,
             depth: Optional[torch.Tensor] = None, anc_bits: Optional[torch.Tensor] = None) -> dict:
        """Room for new_len[b] tokens behind every request's prefix
        (``ops.page_plan``): rows, their total or more, and n_new, the most of
        one request, are known on the host.  ``trim`` first returns the pages
        that a rejected draft left, and all of a request that has ended (its
        prefix set to 0, nothing new); ``depth`` and ``anc_bits`` are a draft
        tree's (``ops.tree_struct``)."""
        p = ops.page_plan(self.prefix, new_len, self.block_table, self.held, self.free_pages, self.free_pos,
                          page_size=self.page_size, rows=rows, trim=trim, depth=depth)
        p["served"] = (p["seq_len"] - self.prefix).clamp_(min=0)  # a refused request's seq_len is 0
        self.served.copy_(p["served"])
        self.held.copy_(p["held"])
        self.free_pos.copy_(p["free_pos"])
        return p | {"n_new": n_new, "anc_bits": anc_bits}

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: dict) -> None:
        """The new rows' keys and values [rows, heads, head_dim] into their pages."""
        ops.kv_append(k, v, self.keys[layer], self.values[layer], plan["slots"])

    def attend(self, layer: int, q: torch.Tensor, plan: dict, **kw) -> torch.Tensor:
        """The new rows' attention over their request's tokens, the new ones
        included: causal, or a tree's where the plan has its anc_bits.  Rows
        past the plan's last (rows above the tokens' total) are uninitialised
        unless ``o`` is given, a refused request's rows 0."""
        return ops.paged_attention(q, self.keys[layer], self.values[layer], self.block_table, plan["seq_len"],
                                   cu_seqlens=plan["cu_seqlens"], n_new=plan["n_new"], anc_bits=plan["anc_bits"], **kw)

    def accept(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: dict, path: torch.Tensor) -> None:
        """The keys and values of an accepted path to the places right behind
        the prefix.  path [batch, columns]: rows of k and v (the step's), -1
        past a request's last one; what is longer than the rows that the plan
        has of a request is left out, as ``commit`` leaves it out."""
        if not plan["slots"].numel():  # no row, so no place either
            return
        cu = plan["cu_seqlens"].long()
        at = cu[:-1, None] + torch.arange(path.shape[1], device=path.device)
        slots = plan["slots"][at.clamp_max(plan["slots"].numel() - 1)]
        ops.kv_append(k, v, self.keys[layer], self.values[layer], torch.where(at < cu[1:, None], slots, -1), rows=path)

    def commit(self, length: torch.Tensor, plan: Optional[dict] = None) -> None:
        """The prefixes grow by length[b] of the step's tokens, as far as the
        last plan gave them places: none of a refused request's.  With several
        plans in a step every commit names its ``plan``."""
        left = self.served if plan is None else plan["served"]
        length = torch.minimum(length, left)
        self.prefix += length
        left -= length
