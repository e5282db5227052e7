"""Paged KV cache kernels (``csrc/kernels/paged_attn.cu``): scatter new K/V rows into pages, decode
attention through a block table; the same over a cache held in int8 with one magnitude for each page
and head (``csrc/kernels/paged_int8.cu``).  CPU tensors use the same maths with torch ops."""
from __future__ import annotations

import functools
import math

import torch

from .. import _native as N
from .int8 import MAX_ROWS, TINY, _no_gradient


def kv_write(k, v, k_cache, v_cache, block_table, seq_ids, positions, page_size: int) -> None:
    """k, v: [T, Hkv, D]; caches: [pages, page_size, Hkv, D]; block_table: [B, max_pages] int32;
    seq_ids / positions: [T] int32 (sequence and position of every token)."""
    T, Hkv, D = k.shape
    if k.is_cuda and N.have_gpu() and k.dtype == torch.bfloat16:
        if k.stride(2) != 1 or k.stride(1) != D:
            k = k.contiguous()
        if v.stride(2) != 1 or v.stride(1) != D:
            v = v.contiguous()
        rc = N.cuda().ax_paged_kv_write(N.ptr(k), N.ptr(v), N.ptr(k_cache), N.ptr(v_cache), N.ptr(block_table),
                                        N.ptr(seq_ids), N.ptr(positions), T, Hkv, D, N.c_int64(k.stride(0)),
                                        N.c_int64(v.stride(0)), page_size, block_table.shape[1], N.stream_ptr())
        N.check(rc, "ax_paged_kv_write")
        return
    pages = block_table[seq_ids.long(), (positions // page_size).long()].long()
    slots = (positions % page_size).long()
    k_cache[pages, slots] = k.to(k_cache.dtype)
    v_cache[pages, slots] = v.to(v_cache.dtype)


def decode_attention(q, k_cache, v_cache, block_table, ctx_lens, page_size: int, scale: float | None = None):
    """q: [B, Hq, D] -> [B, Hq, D]; every sequence attends to its first ``ctx_lens[b]`` cached tokens."""
    B, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    if q.is_cuda and N.have_gpu() and q.dtype == torch.bfloat16 and D == 128 and Hq // Hkv in (1, 2, 4, 8):
        q = q.contiguous()
        out = torch.empty_like(q)
        # context splits: enough CTAs for two per SM, at most one split per 32 tokens of capacity
        capacity = block_table.shape[1] * page_size
        splits = max(1, min(296 // max(B * Hkv, 1), (capacity + 31) // 32, 64))
        ws = torch.empty(B * Hq * splits * (D + 2), dtype=torch.float32, device=q.device) if splits > 1 else None
        rc = N.cuda().ax_paged_decode_attention(N.ptr(q), N.ptr(k_cache), N.ptr(v_cache), N.ptr(out), N.ptr(block_table),
                                                N.ptr(ctx_lens), B, Hq, Hkv, D, page_size, block_table.shape[1],
                                                N.c_float(scale), N.c_int64(q.stride(0)), N.c_int64(out.stride(0)),
                                                splits, N.ptr(ws) if ws is not None else None, k_cache.shape[0],
                                                N.ptr(N.status_word(q.device)), N.ptr(None), N.ptr(None), N.ptr(None), N.stream_ptr())
        N.check(rc, "ax_paged_decode_attention")
        return out
    outs = []
    G = Hq // Hkv
    for b in range(B):
        n = int(ctx_lens[b])
        pos = torch.arange(n, device=q.device)
        pages = block_table[b, (pos // page_size).long()].long()
        kk = k_cache[pages, (pos % page_size).long()].float().repeat_interleave(G, dim=1)   # [n, Hq, D]
        vv = v_cache[pages, (pos % page_size).long()].float().repeat_interleave(G, dim=1)
        s = torch.einsum("hd,nhd->hn", q[b].float(), kk) * scale
        outs.append(torch.einsum("hn,nhd->hd", torch.softmax(s, -1), vv))
    return torch.stack(outs).to(q.dtype)


# ------------------------------------------------------------------------------ cache in 8 bits
_I8, _I32, _F32 = torch.int8, torch.int32, torch.float32
_MAX_TILES = 0x7f000000      # 16-token tiles, over sequences and KV heads, that one launch of the attention can number


def _check_int8_cache(k_cache, v_cache, k_amax, v_amax, block_table):
    """``(pages, Hkv, page_size, D, GPU index or -1)`` of a consistent int8 cache."""
    if k_cache.dtype is not _I8 or v_cache.dtype is not _I8:
        raise TypeError("the caches must be int8")
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be [pages, Hkv, page_size, D], not {tuple(k_cache.shape)}")
    pages, Hkv, P, D = k_cache.shape
    if P % 16 or P == 0 or D % 16 or D == 0 or Hkv == 0:
        raise ValueError(f"page_size {P} and head_dim {D} must be multiples of 16, and {Hkv} KV heads not none")
    if v_cache.shape != (pages, Hkv, P // 16, D, 16):
        raise ValueError(f"v_cache must be [pages, Hkv, page_size / 16, D, 16], not {tuple(v_cache.shape)}")
    if k_amax.shape != (pages, Hkv) or v_amax.shape != (pages, Hkv):
        raise ValueError(f"k_amax and v_amax must be [pages, Hkv] = {(pages, Hkv)}")
    if k_amax.dtype is not _F32 or v_amax.dtype is not _F32:
        raise TypeError("k_amax and v_amax must be fp32")
    if block_table.dim() != 2 or block_table.dtype is not _I32:
        raise TypeError("block_table must be int32 [B, max_pages]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_amax.is_contiguous() and v_amax.is_contiguous()):
        raise ValueError("the caches and their magnitudes must be contiguous")
    dev = k_cache.get_device()
    if v_cache.get_device() != dev or k_amax.get_device() != dev or v_amax.get_device() != dev or block_table.get_device() != dev:
        raise ValueError("the caches, their magnitudes and the block table must be on one device")
    return pages, Hkv, P, D, dev


def _int32_vector(t, n: int, name: str, index: int):
    if t.dtype is not _I32 or t.dim() != 1 or t.shape[0] != n or t.get_device() != index:
        raise ValueError(f"{name} must be int32 [{n}] on the cache's device")
    return t if t.is_contiguous() else t.contiguous()


def kv_write_int8(k, v, k_cache, v_cache, k_amax, v_amax, block_table, starts, cu_seqlens=None) -> None:
    """Writes new K/V rows ``[T, Hkv, D]`` (bf16 or fp32) into an int8 cache, in place.

    ``k_cache`` is ``[pages, Hkv, page_size, D]``, ``v_cache`` ``[pages, Hkv, page_size / 16, D, 16]``, and a
    stored ``q`` of page ``p``, head ``h`` stands for ``q * amax[p, h] / 127``.  Sequence ``b`` (a row of
    ``block_table`` ``[B, max_pages]``) brings tokens ``cu_seqlens[b] .. cu_seqlens[b + 1]`` (without
    ``cu_seqlens``: ``T / B`` each) at positions ``starts[b], starts[b] + 1, ...``; rows of ``k`` / ``v`` behind
    ``cu_seqlens[B]`` are ignored.  A page's magnitude grows to the largest value it holds, and what it held
    before is rounded to the new grid; a page written from its first slot starts anew.  ``cu_seqlens`` must not
    decrease, and two sequences of one call must not write to the same page.  On a GPU a sequence that does not fit its table or a
    page number outside the cache is skipped and reported by ``_native.check_status()``."""
    pages, Hkv, P, D, index = _check_int8_cache(k_cache, v_cache, k_amax, v_amax, block_table)
    if k.dim() != 3 or k.shape[1:] != (Hkv, D) or v.shape != k.shape or v.dtype is not k.dtype:
        raise ValueError(f"k and v must be [T, {Hkv}, {D}] of one type, not {tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
    if k.get_device() != index or v.get_device() != index:
        raise ValueError("k and v must be on the cache's device")
    if k.requires_grad or v.requires_grad:
        _no_gradient()
    T, (B, width) = k.shape[0], block_table.shape
    starts = _int32_vector(starts, B, "starts", index)
    cu = 0
    if cu_seqlens is not None:
        cu_seqlens = _int32_vector(cu_seqlens, B + 1, "cu_seqlens", index)
        cu = cu_seqlens.data_ptr()
    elif B == 0 or T % B:
        raise ValueError(f"without cu_seqlens, {T} tokens must divide evenly over {B} sequences")
    if index < 0:
        _kv_write_int8_cpu(k, v, k_cache, v_cache, k_amax, v_amax, block_table, starts, cu_seqlens)
        return
    if k.dtype is torch.bfloat16:
        kind, vec = 1, 8
    elif k.dtype is _F32:
        kind, vec = 0, 4
    else:
        raise TypeError(f"k and v must be bf16 or fp32 on a GPU, not {k.dtype}")
    if D > 512 or Hkv > 65535 or P * D > 1 << 30 or T > MAX_ROWS:
        raise ValueError(f"head_dim {D}, {Hkv} KV heads, page_size {P} or {T} tokens are more than the kernel takes (512, 65535, 2^30 / head_dim, {MAX_ROWS})")
    if T == 0 or B == 0:
        return
    (kt, kh, k1), (vt, vh, v1) = k.stride(), v.stride()
    if k1 != 1 or kt % vec or kh % vec or k.data_ptr() % 16:
        k = k.clone(memory_format=torch.contiguous_format)
        kt, kh, _ = k.stride()
    if v1 != 1 or vt % vec or vh % vec or v.data_ptr() % 16:
        v = v.clone(memory_format=torch.contiguous_format)
        vt, vh, _ = v.stride()
    table = block_table if block_table.is_contiguous() else block_table.contiguous()
    N.launch("ax_kv_write_int8", index, kind, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, k_cache.data_ptr(), v_cache.data_ptr(), k_amax.data_ptr(),
             v_amax.data_ptr(), table.data_ptr(), starts.data_ptr(), cu, T, B, Hkv, D, P, width, pages, N.status_ptr(index))


def _kv_write_int8_cpu(k, v, k_cache, v_cache, k_amax, v_amax, block_table, starts, cu_seqlens) -> None:
    T, B, P, D = k.shape[0], block_table.shape[0], k_cache.shape[2], k_cache.shape[3]
    cu = cu_seqlens.tolist() if cu_seqlens is not None else [b * (T // B) for b in range(B + 1)]
    table = block_table.tolist()
    for b, start in enumerate(starts.tolist()):
        n = cu[b + 1] - cu[b]
        if n <= 0:
            continue
        if start < 0 or cu[b] < 0 or cu[b + 1] > T or start + n > block_table.shape[1] * P:
            raise ValueError(f"sequence {b}: tokens {cu[b]}..{cu[b + 1]} at position {start} do not fit")
        if any(not 0 <= p < k_cache.shape[0] for p in table[b][start // P:(start + n - 1) // P + 1]):
            raise ValueError(f"sequence {b}: the block table names a page outside the cache")
        pos = start
        while pos < start + n:
            page, lo = table[b][pos // P], pos % P
            cnt = min(P - lo, start + n - pos)
            src = cu[b] + pos - start
            for x, cache, amax, is_v in ((k, k_cache, k_amax, False), (v, v_cache, v_amax, True)):
                rows = cache[page].transpose(-1, -2).reshape(-1, P, D).clone() if is_v else cache[page]
                new = x[src:src + cnt].transpose(0, 1).float()
                old = amax[page].clone() if lo else torch.zeros_like(amax[page])
                grown = torch.maximum(old, new.abs().amax((1, 2)))
                grown = torch.where(grown < TINY, torch.zeros_like(grown), grown)
                one = torch.where(grown > 0, grown, torch.ones_like(grown)).double()[:, None, None]
                if lo:
                    kept = (rows[:, :lo].double() * old[:, None, None] / one).round().nan_to_num_(0.0).to(torch.int8)
                    rows[:, :lo] = torch.where((grown > old)[:, None, None], kept, rows[:, :lo])
                rows[:, lo:lo + cnt] = (new.double() * 127.0 / one).round().nan_to_num_(0.0).to(torch.int8)
                amax[page] = grown
                if is_v:
                    cache[page] = rows.view(-1, P // 16, 16, D).transpose(-1, -2)
            pos += cnt


def decode_attention_int8(q, k_cache, v_cache, k_amax, v_amax, block_table, ctx_lens, scale: float | None = None):
    """Attention of one query token per sequence over an int8 cache (laid out as ``kv_write_int8``
    says): ``q`` bf16 ``[B, Hq, D]`` -> ``[B, Hq, D]``, each sequence over its first ``ctx_lens[b]`` tokens; an
    empty context gives zeros.  On a GPU D is 64, 128 or 256; any number of query heads per KV head; a
    sequence's table has room for at most 2^31 / KV heads tiles of 16 tokens (with more than 16 query heads per KV head, as often less).  A
    page number outside the cache and a context longer than the table are reported by
    ``_native.check_status()`` and not read."""
    pages, Hkv, P, D, index = _check_int8_cache(k_cache, v_cache, k_amax, v_amax, block_table)
    B, width = block_table.shape
    if q.dim() != 3 or q.shape[0] != B or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % Hkv:
        raise ValueError(f"q must be [{B}, a multiple of {Hkv}, {D}], not {tuple(q.shape)}")
    if q.get_device() != index:
        raise ValueError("q must be on the cache's device")
    if q.requires_grad:
        _no_gradient()
    Hq = q.shape[1]
    ctx_lens = _int32_vector(ctx_lens, B, "ctx_lens", index)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if index < 0:
        return _decode_attention_int8_cpu(q, k_cache, v_cache, k_amax, v_amax, block_table, ctx_lens, scale)
    if q.dtype is not torch.bfloat16:
        raise TypeError(f"q must be bf16 on a GPU, not {q.dtype}")
    if D not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256 on a GPU, not {D}")
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty_like(q)
    table = block_table if block_table.is_contiguous() else block_table.contiguous()
    each = _int8_sequences(B, Hq // Hkv, Hkv, width, P)
    for b0 in range(0, B, each):
        n = min(each, B - b0)
        size = _int8_workspace(index, n, Hq, Hkv, D, width, P)
        ws = k_amax.new_empty(size) if size else None
        N.launch("ax_decode_int8", index, q.data_ptr() + b0 * Hq * D * 2, k_cache.data_ptr(), v_cache.data_ptr(), k_amax.data_ptr(),
                 v_amax.data_ptr(), table.data_ptr() + b0 * width * 4, ctx_lens.data_ptr() + b0 * 4, out.data_ptr() + b0 * Hq * D * 2, n, Hq, Hkv,
                 D, P, width, pages, scale, ws.data_ptr() if size else 0, N.status_ptr(index))
    return out


def _int8_sequences(B: int, G: int, Hkv: int, width: int, P: int) -> int:
    """Sequences of one launch, in shares as even as they can be: the kernel keeps a running count for each of at most 1024
    in shared memory, and numbers the 16-token tiles that a launch's tables have room for in 31 bits."""
    tiles = Hkv * (1 if G <= 8 else -(-G // 16)) * width * (P // 16)
    most = min(1024, _MAX_TILES // max(tiles, 1))
    if most == 0:
        raise ValueError(f"a table of {width} pages of {P} tokens with {Hkv} KV heads and {G} query heads each is more than the kernel takes "
                         f"({_MAX_TILES} tiles of 16 tokens and up to 16 query heads)")
    return -(-B // -(-B // most)) if B else 1


@functools.lru_cache(maxsize=4096)
def _int8_workspace(index: int, *shape) -> int:
    """Floats that the attention kernel wants beside its outputs, by shape and GPU."""
    with torch.cuda.device(index):
        return N.cuda().ax_decode_int8_workspace(*shape)


def _decode_attention_int8_cpu(q, k_cache, v_cache, k_amax, v_amax, block_table, ctx_lens, scale):
    B, Hq, D = q.shape
    Hkv, P = k_cache.shape[1], k_cache.shape[2]
    out = torch.zeros((B, Hq, D), dtype=torch.float32)
    for b, n in enumerate(ctx_lens.tolist()):
        if n == 0:
            continue
        if not 0 < n <= block_table.shape[1] * P:
            raise ValueError(f"sequence {b}: context {n} does not fit its table")
        pg = block_table[b, :(n + P - 1) // P].long()
        if int(pg.min()) < 0 or int(pg.max()) >= k_cache.shape[0]:
            raise ValueError(f"sequence {b}: the block table names a page outside the cache")
        kk = (k_cache[pg].float() * (k_amax[pg] / 127.0)[:, :, None, None]).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        vv = (v_cache[pg].float() * (v_amax[pg] / 127.0)[:, :, None, None, None]).permute(1, 0, 2, 4, 3).reshape(Hkv, -1, D)[:, :n]
        s = torch.einsum("hgd,hnd->hgn", q[b].float().view(Hkv, -1, D), kk) * scale
        out[b] = torch.einsum("hgn,hnd->hgd", torch.softmax(s, -1), vv).reshape(Hq, D)
    return out.to(q.dtype)
