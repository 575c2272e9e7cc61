"""A paged key / value cache held in 4 bits, and attention over it.  The reference's blocks keep fp16 keys and values
(modeling/llama/llama_qblocks.py:104-150); one vector of 128 takes 66 bytes here instead of 256.

A serving loop, all of it on the GPU and free to be recorded into a graph:

    pages = KVPages(num_pages, 64, max_requests, pages_per_request, device="cuda")      # one for the model
    caches = [W4KVCache(num_pages, 64, kv_heads, head_dim, device="cuda") for _ in layers]
    ...
    step = pages.assign(new_tokens, max_tokens)          # new_tokens int32 [max_requests]; -1 where a request has ended
    for layer, cache in zip(layers, caches):
        q, k, v = layer.qkv(x)                           # rows in the order of the requests, then the rotary embedding
        cache.store(k, v, step.slots)
        a = cache.attend(q, pages.table, pages.lengths, cu_q=step.cu)
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

from .. import _capi, ops


class KVStep(NamedTuple):
    """What a step's tokens need to know: `slots` int64 [max_tokens] their places in the caches (-1: none), `positions`
    int32 [max_tokens] their positions in their requests, `cu` int32 [max_requests + 1] the first token of each request,
    `refused` int32 [max_requests] 1 where a request found no room and has to be asked for again."""
    slots: torch.Tensor
    positions: torch.Tensor
    cu: torch.Tensor
    refused: torch.Tensor


class KVPages(nn.Module):
    """Which pages of the caches each request holds: `table` int32 [max_requests, pages_per_request], `lengths`
    int32 [max_requests], and the free pages as a stack, `free_pages` int32 [num_pages] with `free_count` int32 [1] entries.
    All layers' caches share it."""

    def __init__(self, num_pages, page_size, max_requests, pages_per_request, device=None):
        super().__init__()
        self.num_pages = num_pages
        self.page_size = page_size
        self.register_buffer("table", torch.full((max_requests, pages_per_request), -1, dtype=torch.int32, device=device), persistent=False)
        self.register_buffer("lengths", torch.zeros(max_requests, dtype=torch.int32, device=device), persistent=False)
        self.register_buffer("free_pages", torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device), persistent=False)
        self.register_buffer("free_count", torch.full((1,), num_pages, dtype=torch.int32, device=device), persistent=False)

    def assign(self, new_tokens: torch.Tensor, max_tokens: int) -> KVStep:
        """Pages and places for new_tokens[r] more tokens of every request r (int32, on the GPU; 0: none in this step, negative:
        the request has ended and gives its pages back).  Ended requests come first, then the others in order; one that finds
        too few pages, or no room in its row of the table or in max_tokens, is refused and stays as it was."""
        return KVStep(*ops.kv_assign_pages(new_tokens, self.lengths, self.table, self.free_pages, self.free_count, self.page_size,
                                           max_tokens))

    def __repr__(self):
        return f"KVPages(num_pages={self.num_pages}, page_size={self.page_size}, max_requests={self.table.shape[0]})"


class W4KVCache(nn.Module):
    """One layer's pool of pages: int4 codes with one fp16 scale for each token's key and value vector of a head, layout as in
    uniql_kv4_cache of the C header.  head_dim and v_head_dim from 1 to 128, page_size 16, 32, 64, 128 or 256."""

    def __init__(self, num_pages, page_size, num_kv_heads, head_dim, v_head_dim=None, device=None):
        super().__init__()
        self.num_pages = num_pages
        self.page_size = page_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.v_head_dim = head_dim if v_head_dim is None else v_head_dim
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("pages must hold 16, 32, 64, 128 or 256 tokens")
        if not (1 <= self.head_dim <= 128 and 1 <= self.v_head_dim <= 128):
            raise ValueError("heads must be 1 to 128 wide")
        if num_pages < 1 or num_kv_heads < 1:
            raise ValueError("the cache must have at least one page and one head")

        def pool(dtype, *shape):
            return torch.zeros(num_pages, num_kv_heads, *shape, dtype=dtype, device=device)

        self.register_buffer("k_codes", pool(torch.int32, page_size, (self.head_dim + 31) // 32 * 4), persistent=False)
        self.register_buffer("k_scales", pool(torch.float16, page_size), persistent=False)
        self.register_buffer("v_codes", pool(torch.int32, page_size // 4, (self.v_head_dim + 31) // 32 * 4, 4), persistent=False)
        self.register_buffer("v_scales", pool(torch.float16, page_size), persistent=False)

    # The native handle of the four tensors, with the tensors that it was made of: made at the first call, and anew where the
    # module holds others (0.2 us a call; a buffer may be replaced past the attributes: register_buffer, a functional call).
    def _native(self):
        buffers = self._buffers
        held = self.__dict__.get("_handle")
        if (held is None or held[1] is not buffers["k_codes"] or held[2] is not buffers["k_scales"]
                or held[3] is not buffers["v_codes"] or held[4] is not buffers["v_scales"]):
            tensors = buffers["k_codes"], buffers["k_scales"], buffers["v_codes"], buffers["v_scales"]
            held = self.__dict__["_handle"] = (_capi.host().KvPool(*tensors, self.head_dim, self.v_head_dim), *tensors)
        return held[0]

    # (the tensors of before are let go at once, not at the next call)
    def __setattr__(self, name, value):
        if name in ("k_codes", "k_scales", "v_codes", "v_scales", "head_dim", "v_head_dim"):
            self.__dict__.pop("_handle", None)
        super().__setattr__(name, value)

    def _apply(self, fn, recurse=True):
        self.__dict__.pop("_handle", None)
        return super()._apply(fn, recurse)

    def __getstate__(self):
        state = self.__dict__.copy()
        state.pop("_handle", None)
        return state

    def store(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantises k [tokens, kv heads, head_dim] and v [tokens, kv heads, v_head_dim] into the places `slots` (int64 [tokens]; -1
        is left out, none may occur twice)."""
        self._native().store(k, v, slots, ops._stream_of(k, "k"))

    def load(self, table: torch.Tensor, cu: torch.Tensor, rows: int, starts: torch.Tensor | None = None,
             k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None):
        """(k, v) in fp16, packed by request: rows cu[r] .. cu[r + 1] are the positions from starts[r] (0 when None) on.  For
        prompts taken in pieces: prompt_attention(q, *load(..), cu_q, cu) sees what attend would."""
        return self._native().load(table, cu, rows, starts, k_out, v_out, ops._stream_of(table, "table"))

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, cu_q: torch.Tensor | None = None,
               scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of each request's newest tokens, q [rows, q heads, head_dim], over its pages; the tokens' own keys and values
        have been stored and count in `lengths`.  cu_q int32 [requests + 1]: rows of each request (None: one each).
        Returns [rows, q heads, v_head_dim]."""
        return self._native().attend(q, table, lengths, cu_q, scale, out, ops._stream_of(q, "q"), ops._accumulator)

    def __repr__(self):
        return (f"W4KVCache(num_pages={self.num_pages}, page_size={self.page_size}, num_kv_heads={self.num_kv_heads}, "
                f"head_dim={self.head_dim}, v_head_dim={self.v_head_dim})")
