"""Paged KV cache: a pool of fixed-size pages per layer plus a block table per sequence
(replaces the reference's concat-and-grow ``KVCache``, crates/axonml-llm/src/attention.rs:19-86).
With ``dtype=torch.int8`` pages hold eight bits a value and one magnitude per page and head (half the
bytes to keep and to read; laid out as ``ops.paged.kv_write_int8`` says)."""
from __future__ import annotations

import torch

from ..ops import paged


class OutOfPages(RuntimeError):
    pass


class PagedKVCache:
    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 max_seqs: int, max_pages_per_seq: int, device, dtype=torch.bfloat16):
        self.num_layers, self.num_pages, self.page_size = num_layers, num_pages, page_size
        self.max_seqs, self.max_pages_per_seq = max_seqs, max_pages_per_seq
        self.int8 = dtype == torch.int8
        if self.int8:
            if page_size % 16 or head_dim % 16 or (torch.device(device).type == "cuda" and head_dim not in (64, 128, 256)):
                raise ValueError(f"an int8 cache needs pages of a multiple of 16 tokens (not {page_size}) and a head_dim of 64, 128 or "
                                 f"256 on a GPU, a multiple of 16 elsewhere (not {head_dim})")
            self.k = torch.zeros((num_layers, num_pages, num_kv_heads, page_size, head_dim), dtype=dtype, device=device)
            self.v = torch.zeros((num_layers, num_pages, num_kv_heads, page_size // 16, head_dim, 16), dtype=dtype, device=device)
            self.k_amax = torch.zeros((num_layers, num_pages, num_kv_heads), dtype=torch.float32, device=device)
            self.v_amax = torch.zeros_like(self.k_amax)
        else:
            shape = (num_layers, num_pages, page_size, num_kv_heads, head_dim)
            self.k = torch.zeros(shape, dtype=dtype, device=device)
            self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.block_table = torch.zeros((max_seqs, max_pages_per_seq), dtype=torch.int32, device=device)
        self._table_host = torch.zeros((max_seqs, max_pages_per_seq), dtype=torch.int32)
        self._free_pages = list(range(num_pages - 1, -1, -1))
        self._free_slots = list(range(max_seqs - 1, -1, -1))
        self._pages_of: dict[int, list] = {}
        self.lens: dict[int, int] = {}

    def write(self, layer: int, k, v, table, starts, seq, positions) -> None:
        """New K/V rows ``[T, Hkv, D]`` of the sequences whose block-table rows are ``table`` ``[B, max_pages]``, the same
        number of consecutive tokens for each from position ``starts`` ``[B]`` on; ``seq`` / ``positions`` ``[T]`` say the
        same token by token."""
        if self.int8:
            paged.kv_write_int8(k, v, self.k[layer], self.v[layer], self.k_amax[layer], self.v_amax[layer], table, starts)
        else:
            paged.kv_write(k, v, self.k[layer], self.v[layer], table, seq, positions, self.page_size)

    def attend(self, layer: int, q, table, ctx):
        """Attention of one query token per sequence, ``q`` ``[B, Hq, D]``, over the first ``ctx`` ``[B]`` tokens."""
        if self.int8:
            return paged.decode_attention_int8(q, self.k[layer], self.v[layer], self.k_amax[layer], self.v_amax[layer], table, ctx)
        return paged.decode_attention(q, self.k[layer], self.v[layer], table, ctx, self.page_size)

    def pages_free(self) -> int: return len(self._free_pages)
    def occupancy(self) -> float: return 1.0 - len(self._free_pages) / self.num_pages
    def can_admit(self, tokens: int) -> bool:
        return bool(self._free_slots) and (tokens + self.page_size - 1) // self.page_size <= len(self._free_pages)

    def allocate_seq(self) -> int:
        if not self._free_slots:
            raise OutOfPages("no free sequence slot")
        s = self._free_slots.pop()
        self._pages_of[s], self.lens[s] = [], 0
        return s

    def reserve(self, slot: int, new_len: int) -> None:
        """Makes sure ``slot`` owns enough pages for ``new_len`` tokens."""
        need = (new_len + self.page_size - 1) // self.page_size
        pages = self._pages_of[slot]
        if need > self.max_pages_per_seq:
            raise OutOfPages("sequence exceeds the maximum context")
        changed = False
        while len(pages) < need:
            if not self._free_pages:
                raise OutOfPages("KV cache is full")
            p = self._free_pages.pop()
            self._table_host[slot, len(pages)] = p
            pages.append(p)
            changed = True
        if changed:
            self.block_table[slot].copy_(self._table_host[slot], non_blocking=True)
        self.lens[slot] = new_len

    def free_seq(self, slot: int) -> None:
        self._free_pages.extend(reversed(self._pages_of.pop(slot, [])))
        self.lens.pop(slot, None)
        self._free_slots.append(slot)
