"""Operators over a paged KV cache (MI355X): the pages of several sequences' keys and values, each sequence with a length
and a row of page numbers of its own.

Next to the contiguous cache's ``rope_kv_cache_write``, ``gqa_flash_decode_mps`` and ``compact_tree_kv`` (``ops``); the
reference has no kernels for pages (its PagedKVCache, axiomlm/engine/paged_cache.py:4-120, gathers them with tensor
indexing).  All compute runs in libaxm.so.

A layer's pages are ``k_cache`` / ``v_cache`` (P, Hkv, page_size, width): fp16 with width hd, or uint8 codes (FP8
E4M3FN: hd, INT4: hd/2) with fp16 ``k_scales`` / ``v_scales`` (P, Hkv, page_size, hd/64).  Pages may be strided (a view of a
larger pool); what is inside a page is contiguous.  ``block_table`` (B, max_pages) int32: slot s of sequence b is row
``s % page_size`` of page ``block_table[b, s // page_size]``.  Head size 64 or 128, page size a power of two from 16 to
1024.  Table, lengths, positions and slots are read on the device: captured graphs replay with new ones.  Numbers that
are out of range there (a page outside the pool, a sequence outside the table) are skipped and never followed.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .ops import _kv_code, on_device


def _ints(who: str, name: str, t: torch.Tensor, device: torch.device, n: int) -> torch.Tensor:
    """A device array of n int32 (int64 is converted)."""
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{who}: {name} must be an int32 or int64 tensor on {device}")
    if t.dim() != 1 or t.numel() != n:
        raise ValueError(f"{who}: {name} has shape {tuple(t.shape)}, expected ({n},)")
    return t.to(torch.int32).contiguous()


def _inside_page_contiguous(t: torch.Tensor) -> bool:
    """Whether the last three dimensions are laid out densely (strides of dimensions of one element do not matter)."""
    want = 1
    for size, stride in zip(reversed(t.shape[-3:]), reversed(t.stride()[-3:])):
        if size != 1 and stride != want:
            return False
        want *= size
    return True


def _page_stride(t: torch.Tensor, dim: int) -> int:
    """Bytes from one index of `dim` to the next; of a dimension of one, its dense size."""
    n = t.stride(dim) if t.size(dim) > 1 else t[(0,) * (dim + 1)].numel()
    return n * t.element_size()


def _describe(who: str, k, v, ks, vs, kv_dtype: str, block_table):
    """Checked axm_paged_kv of one layer, and the tensors that it points into."""
    code = _kv_code(kv_dtype)
    for name, t in (("k_cache", k), ("v_cache", v)):
        _lib.require_gpu(t, who)
        if t.dim() != 4 or t.dtype not in ((torch.float16,) if code == 0 else
                                           (torch.uint8, torch.float8_e4m3fn) if code == 1 else (torch.uint8,)):
            raise ValueError(f"{who}: {name} must be (pages, n_kv_head, page_size, width) of {kv_dtype} rows, got "
                             f"{tuple(t.shape)} {t.dtype}")
        if not _inside_page_contiguous(t):
            raise ValueError(f"{who}: {name}'s pages must be contiguous inside")
    if k.shape != v.shape or k.device != v.device or _page_stride(k, 0) != _page_stride(v, 0):
        raise ValueError(f"{who}: k_cache and v_cache differ in shape, device or page stride")
    P, Hkv, page, width = k.shape
    hd = width * 2 if code == 2 else width
    if 0 in k.shape:
        raise ValueError(f"{who}: empty cache {tuple(k.shape)}")
    scale_stride = 0
    if code:
        for name, t in (("k_scales", ks), ("v_scales", vs)):
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{who}: quantized KV cache needs k_scales and v_scales")
            if (t.dtype != torch.float16 or t.device != k.device or tuple(t.shape) != (P, Hkv, page, hd // 64)
                    or not _inside_page_contiguous(t)):
                raise ValueError(f"{who}: {name} must be fp16 {(P, Hkv, page, hd // 64)} on {k.device}, contiguous "
                                 "inside a page")
        scale_stride = _page_stride(ks, 0)
        if scale_stride != _page_stride(vs, 0):
            raise ValueError(f"{who}: k_scales and v_scales differ in page stride")
    if (not isinstance(block_table, torch.Tensor) or block_table.device != k.device or block_table.dim() != 2
            or block_table.dtype != torch.int32):
        raise ValueError(f"{who}: block_table must be a (sequences, pages) int32 tensor on {k.device}")
    table = block_table.contiguous()
    B, max_pages = table.shape
    d = _lib.PagedKv(k.data_ptr(), v.data_ptr(), ks.data_ptr() if code else None, vs.data_ptr() if code else None,
                     table.data_ptr(), _page_stride(k, 0), scale_stride, code, Hkv, hd, page, P, B, max_pages)
    return d, table


def rope_paged_kv_cache_write(qkv: torch.Tensor, freqs_cis: torch.Tensor, k_cache: torch.Tensor,
                              v_cache: torch.Tensor, block_table: torch.Tensor, positions: torch.Tensor, q_dim: int,
                              kv_dim: int, head_dim: int, slots: torch.Tensor | None = None,
                              seq_ids: torch.Tensor | None = None, qkv_bias: torch.Tensor | None = None,
                              k_scales: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                              kv_dtype: str = "fp16") -> None:
    """Fused bias + RoPE + cache write of T tokens of any sequences (prompts and single tokens together).

    qkv (T, q_dim + 2 kv_dim) fp16, rows may be strided; the query part is biased and rotated in place.  Token t of
    sequence ``seq_ids[t]`` (t where None) is rotated at ``positions[t]`` (modulo the rows of freqs_cis) and its key and
    value land at slot ``slots[t]`` (``positions[t]`` where None; they differ once tokens have been evicted).  A token with a
    slot below zero, or a sequence, slot or page out of range, is padding: its row and the cache stay as they are.
    No slot may be given twice.  freqs_cis: complex (rope_len, hd/2) or its real view (rope_len, hd/2, 2).  Rounding as
    ``rope_kv_cache_write_quantized``; FP8 codes saturate, and a group whose scale rounds to zero is stored as zeros."""
    who = "rope_paged_kv_cache_write"
    _lib.require_gpu(qkv, who)
    d, _table = _describe(who, k_cache, v_cache, k_scales, v_scales, kv_dtype, block_table)
    dev = qkv.device
    width = int(q_dim) + 2 * int(kv_dim)
    if qkv.dtype != torch.float16 or qkv.dim() != 2 or qkv.size(1) != width or (width > 1 and qkv.stride(1) != 1):
        raise ValueError(f"{who}: qkv must be fp16 (tokens, q_dim + 2 kv_dim = {width}) with contiguous rows, got "
                         f"{tuple(qkv.shape)} {qkv.dtype}")
    if dev != k_cache.device:
        raise ValueError(f"{who}: qkv is on {dev}, the cache on {k_cache.device}")
    if head_dim != d.head_dim or kv_dim != d.n_kv_head * d.head_dim:
        raise ValueError(f"{who}: kv_dim {kv_dim} of heads of {head_dim} does not match the cache's {d.n_kv_head} heads "
                         f"of {d.head_dim}")
    T = qkv.size(0)
    if T == 0:
        return
    pos = _ints(who, "positions", positions, dev, T)
    sl = None if slots is None else _ints(who, "slots", slots, dev, T)
    seq = None if seq_ids is None else _ints(who, "seq_ids", seq_ids, dev, T)
    fr = torch.view_as_real(freqs_cis) if freqs_cis.is_complex() else freqs_cis
    fr = fr.to(device=dev, dtype=torch.float32).contiguous()
    if fr.dim() != 3 or fr.size(0) < 1 or tuple(fr.shape[1:]) != (head_dim // 2, 2):
        raise ValueError(f"{who}: freqs_cis of shape {tuple(freqs_cis.shape)} for heads of {head_dim}")
    bias = None if qkv_bias is None else qkv_bias.to(device=dev, dtype=torch.float16).contiguous()
    if bias is not None and bias.numel() != width:
        raise ValueError(f"{who}: qkv_bias has {bias.numel()} elements, expected {width}")
    with on_device(dev):
        _lib.check(_lib.lib().axm_rope_paged_kv_write(
            qkv.data_ptr(), qkv.stride(0) if T > 1 else width, T, fr.data_ptr(), fr.size(0), pos.data_ptr(),
            _lib.ptr(sl), _lib.ptr(seq), _lib.ptr(bias), ctypes.byref(d), int(q_dim), _lib.stream_of(dev)), who)


def gqa_paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                     seq_lens: torch.Tensor, k_scales: torch.Tensor | None = None,
                     v_scales: torch.Tensor | None = None, kv_dtype: str = "fp16",
                     mass: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over slots [0, seq_lens[b]) of its pages (``gqa_flash_decode_mps`` for
    sequences of different lengths): q (B, Hq, hd) or (B, Hq, 1, hd) fp16, rows may be strided (the query part of a
    qkv tensor); Hq a multiple, up to 64, of Hkv.  Returns fp16 of q's shape; a sequence of length 0 gives zeros.

    mass (fp32 (B, Hkv, M), M >= max_pages * page_size, contiguous): the softmax weights of every slot, summed over the
    query heads of the KV head, are added to it: the account that ``evict_paged_kv`` goes by."""
    who = "gqa_paged_decode"
    _lib.require_gpu(q, who)
    d, _table = _describe(who, k_cache, v_cache, k_scales, v_scales, kv_dtype, block_table)
    dev, hd = q.device, d.head_dim
    if q.dim() not in (3, 4) or (q.dim() == 4 and q.size(2) != 1) or q.size(0) != d.n_seqs or q.size(-1) != hd:
        raise ValueError(f"{who}: q of shape {tuple(q.shape)} for {d.n_seqs} sequences and heads of {hd}")
    Hq = q.size(1)
    if dev != k_cache.device:
        raise ValueError(f"{who}: q is on {dev}, the cache on {k_cache.device}")
    if Hq < 1 or Hq % d.n_kv_head or Hq // d.n_kv_head > 64:
        raise ValueError(f"{who}: {Hq} query heads for {d.n_kv_head} KV heads")
    lens = _ints(who, "seq_lens", seq_lens, dev, d.n_seqs)
    out = torch.empty(q.shape, dtype=torch.float16, device=dev)
    if d.n_seqs == 0:
        return out
    if d.max_pages == 0:
        return out.zero_()
    M = 0
    if mass is not None:
        M = mass.size(-1) if isinstance(mass, torch.Tensor) and mass.dim() == 3 else -1
        if (M < d.max_pages * d.page_size or tuple(mass.shape[:2]) != (d.n_seqs, d.n_kv_head)
                or mass.dtype != torch.float32 or mass.device != dev or not mass.is_contiguous()):
            raise ValueError(f"{who}: mass must be contiguous fp32 ({d.n_seqs}, {d.n_kv_head}, at least "
                             f"{d.max_pages * d.page_size}) on {dev}")
    qc = q.to(torch.float16)
    ld = qc.stride(0)
    if qc.stride(-1) != 1 or (Hq > 1 and qc.stride(1) != hd) or qc.data_ptr() % 16 or (d.n_seqs > 1 and ld % 8) \
            or (d.n_seqs > 1 and ld < Hq * hd):
        qc = qc.contiguous()
        if qc.data_ptr() % 16:
            qc = qc.clone()
    ld = qc.stride(0) if d.n_seqs > 1 else Hq * hd
    with on_device(dev):
        L = _lib.lib()
        need = L.axm_paged_decode_workspace_bytes(d.n_seqs, Hq, d.n_kv_head, hd, d.page_size, d.max_pages,
                                                  mass is not None)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(L.axm_paged_flash_decode(qc.data_ptr(), ld, ctypes.byref(d), lens.data_ptr(), out.data_ptr(), Hq,
                                            _lib.ptr(mass), M, _lib.ptr(ws), need, _lib.stream_of(dev)), who)
    return out


def evict_paged_kv(cache: torch.Tensor, scales: torch.Tensor | None, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, mass: torch.Tensor, budget: int, recent: int):
    """Cut every sequence longer than ``budget`` down to it, in all layers: per layer and KV head its last ``recent``
    slots stay and, of those before, the ``budget - recent`` with the largest ``mass`` (equal ones: the lower slot; NaN
    below every number).  Kept rows move, in order, to slots 0 .. budget - 1 of the sequence's pages, in place.

    cache (L, 2, P, Hkv, page_size, width) fp16 or uint8 codes (width hd: FP8, hd/2: INT4, told apart by the scales' last
    dimension), scales (L, 2, P, Hkv, page_size, hd/64) or None; mass (L, B, Hkv, M) fp32, M >= max_pages * page_size.
    Returns (kept, lens, mass): int32 (L, B, Hkv, budget) the slots that the rows come from, -1 behind the last; int32 (B,)
    min(seq_lens, budget); fp32 the kept slots' mass, zeros behind.  The given mass and seq_lens stay as they are.
    Keys stay rotated at the positions they had: the next token's position goes on counting, its slot is the new length.
    The pages of a sequence over the budget must belong to it alone."""
    who = "evict_paged_kv"
    _lib.require_gpu(cache, who)
    if cache.dim() != 6 or cache.size(1) != 2:
        raise ValueError(f"{who}: cache must be (layers, 2, pages, n_kv_head, page_size, width), got "
                         f"{tuple(cache.shape)}")
    if cache.dtype == torch.float16:
        kv_dtype = "fp16"
    elif not isinstance(scales, torch.Tensor) or scales.dim() != 6 or scales.shape[:5] != cache.shape[:5]:
        raise ValueError(f"{who}: quantized KV cache needs scales (layers, 2, pages, n_kv_head, page_size, hd / 64)")
    else:
        kv_dtype = "fp8" if scales.size(5) * 64 == cache.size(5) else "int4"
    L = cache.size(0)
    if L < 1:
        raise ValueError(f"{who}: cache without layers")
    quant = kv_dtype != "fp16"
    d, table = _describe(who, cache[0, 0], cache[0, 1], scales[0, 0] if quant else None,
                         scales[0, 1] if quant else None, kv_dtype, block_table)
    dev, B, H = cache.device, d.n_seqs, d.n_kv_head
    budget, recent = int(budget), int(recent)
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"{who}: budget {budget} must be positive and recent {recent} within it")
    if (not isinstance(mass, torch.Tensor) or mass.dtype != torch.float32 or mass.device != dev or mass.dim() != 4
            or tuple(mass.shape[:3]) != (L, B, H) or mass.size(3) < d.max_pages * d.page_size):
        raise ValueError(f"{who}: mass must be fp32 ({L}, {B}, {H}, at least {d.max_pages * d.page_size}) on {dev}")
    lens = _ints(who, "seq_lens", seq_lens, dev, B)
    mass = mass.contiguous()
    kept = torch.empty((L, B, H, budget), dtype=torch.int32, device=dev)
    out_lens = torch.empty(B, dtype=torch.int32, device=dev)
    out_mass = torch.empty_like(mass)
    if B == 0:
        return kept, out_lens, out_mass
    if d.max_pages == 0:
        return kept.fill_(-1), out_lens.zero_(), out_mass.zero_()
    with on_device(dev):
        _lib.check(_lib.lib().axm_evict_paged_kv(
            ctypes.byref(d), L, _page_stride(cache, 0), _page_stride(scales, 0) if quant else 0, lens.data_ptr(),
            mass.data_ptr(), mass.size(3), budget, recent, out_mass.data_ptr(), kept.data_ptr(), out_lens.data_ptr(),
            _lib.stream_of(dev)), who)
    return kept, out_lens, out_mass
