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

import struct

import torch

from .. import _lib
from .ops import KV_CODES, _kv_code, on_device

_PAGED_KV = struct.Struct("5P2q7i4x")  # axm_paged_kv (include/axm.h)


def _ints(who: str, name: str, t: torch.Tensor, device: torch.device, n: int) -> torch.Tensor:
    """A device array of n int32 (int64 is converted; what does not fit stays out of range)."""
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{who}: {name} must be an int32 or int64 tensor on {device}")
    if t.dim() != 1 or t.numel() != n:
        raise ValueError(f"{who}: {name} has shape {tuple(t.shape)}, expected ({n},)")
    if t.dtype == torch.int64:
        t = t.clamp(-2**31, 2**31 - 1).to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _page_stride(who: str, name: str, t: torch.Tensor) -> int:
    """Bytes from one page to the next (the fourth last dimension); what is inside a page must be dense (strides of
    dimensions of one element do not matter)."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 4:
        shape, stride = shape[-4:], stride[-4:]
    dense = shape[1] * shape[2] * shape[3]
    if not (stride[3] == 1 and stride[2] == shape[3] and stride[1] == shape[2] * shape[3]):
        want = 1
        for size, step in zip(reversed(shape[1:]), reversed(stride[1:])):
            if size != 1 and step != want:
                raise ValueError(f"{who}: {name}'s pages must be contiguous inside")
            want *= size
    return (stride[0] if shape[0] > 1 else dense) * t.element_size()


def _table(who: str, t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 2 or t.device != device:
        raise ValueError(f"{who}: block_table must be a (sequences, pages) int32 tensor on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _describe(who: str, k, v, ks, vs, kv_dtype: str, block_table):
    """Checked axm_paged_kv of one layer (packed), (B, Hkv, hd, page size, pages of a row of the table), the cache's device
    and the table, which has to live until the call."""
    code = KV_CODES.get(kv_dtype)
    if code is None:
        code = _kv_code(kv_dtype)
    for name, t in (("k_cache", k), ("v_cache", v)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            _lib.require_gpu(t, who)
        if t.dim() != 4 or (t.dtype != torch.float16 if code == 0 else t.dtype != torch.uint8 and
                            (code == 2 or t.dtype != torch.float8_e4m3fn)):
            raise ValueError(f"{who}: {name} must be (pages, n_kv_head, page_size, width) of {kv_dtype} rows, got "
                             f"{tuple(t.shape)} {t.dtype}")
    shape = k.shape
    P, Hkv, page, width = shape
    if v.shape != shape or 0 in shape:
        raise ValueError(f"{who}: k_cache {tuple(shape)} and v_cache {tuple(v.shape)} must be alike and not empty")
    dev = k.device
    stride = _page_stride(who, "k_cache", k)
    if v.device != dev or _page_stride(who, "v_cache", v) != stride:
        raise ValueError(f"{who}: k_cache and v_cache differ in device or page stride")
    hd = width * 2 if code == 2 else width
    scale_stride = 0
    if code:
        want = (P, Hkv, page, hd // 64)
        for name, t in (("k_scales", ks), ("v_scales", vs)):
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{who}: quantized KV cache needs k_scales and v_scales")
            if t.dtype != torch.float16 or t.shape != want or t.device != dev:
                raise ValueError(f"{who}: {name} must be fp16 {want} on {dev}, got {tuple(t.shape)} {t.dtype}")
        scale_stride = _page_stride(who, "k_scales", ks)
        if _page_stride(who, "v_scales", vs) != scale_stride:
            raise ValueError(f"{who}: k_scales and v_scales differ in page stride")
    table = _table(who, block_table, dev)
    B, max_pages = table.shape
    d = _PAGED_KV.pack(k.data_ptr(), v.data_ptr(), ks.data_ptr() if code else 0, vs.data_ptr() if code else 0,
                       table.data_ptr(), stride, scale_stride, code, Hkv, hd, page, P, B, max_pages)
    return d, (B, Hkv, hd, page, max_pages), dev, table


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
    d, (_, Hkv, hd, _, _), dev, table = _describe(who, k_cache, v_cache, k_scales, v_scales, kv_dtype, block_table)
    width = q_dim + 2 * kv_dim
    if not isinstance(qkv, torch.Tensor) or qkv.device != dev:
        _lib.require_gpu(qkv, who)
        raise ValueError(f"{who}: qkv is on {qkv.device}, the cache on {dev}")
    if qkv.dtype != torch.float16 or qkv.dim() != 2 or qkv.shape[1] != width or qkv.stride(1) != 1:
        raise ValueError(f"{who}: qkv must be fp16 (tokens, q_dim + 2 kv_dim = {width}) with contiguous rows, got "
                         f"{tuple(qkv.shape)} {qkv.dtype}")
    if head_dim != hd or kv_dim != Hkv * hd:
        raise ValueError(f"{who}: kv_dim {kv_dim} of heads of {head_dim} does not match the cache's {Hkv} heads of {hd}")
    T = qkv.shape[0]
    if T == 0:
        return
    pos = _ints(who, "positions", positions, dev, T)
    sl = None if slots is None else _ints(who, "slots", slots, dev, T)
    seq = None if seq_ids is None else _ints(who, "seq_ids", seq_ids, dev, T)
    fr = torch.view_as_real(freqs_cis) if freqs_cis.is_complex() else freqs_cis
    if fr.dtype != torch.float32 or fr.device != dev or not fr.is_contiguous():
        fr = fr.to(device=dev, dtype=torch.float32).contiguous()
    shape = fr.shape
    if len(shape) != 3 or shape[0] < 1 or shape[1] * 2 != hd or shape[2] != 2:
        raise ValueError(f"{who}: freqs_cis of shape {tuple(freqs_cis.shape)} for heads of {head_dim}")
    bias = None if qkv_bias is None else qkv_bias.to(device=dev, dtype=torch.float16).contiguous()
    if bias is not None and bias.numel() != width:
        raise ValueError(f"{who}: qkv_bias has {bias.numel()} elements, expected {width}")
    with on_device(dev.index):
        rc = _lib.lib().axm_rope_paged_kv_write(
            qkv.data_ptr(), qkv.stride(0) if T > 1 else width, T, fr.data_ptr(), shape[0], pos.data_ptr(),
            None if sl is None else sl.data_ptr(), None if seq is None else seq.data_ptr(),
            None if bias is None else bias.data_ptr(), d, q_dim, _lib.raw_stream(dev.index))
    if rc:
        _lib.check(rc, who)


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
    d, (B, Hkv, hd, page, max_pages), dev, table = _describe(who, k_cache, v_cache, k_scales, v_scales, kv_dtype,
                                                             block_table)
    if not isinstance(q, torch.Tensor) or q.device != dev:
        _lib.require_gpu(q, who)
        raise ValueError(f"{who}: q is on {q.device}, the cache on {dev}")
    shape = q.shape
    if len(shape) not in (3, 4) or (len(shape) == 4 and shape[2] != 1) or shape[0] != B or shape[-1] != hd:
        raise ValueError(f"{who}: q of shape {tuple(shape)} for {B} sequences and heads of {hd}")
    Hq = shape[1]
    if Hq < 1 or Hq % Hkv or Hq // Hkv > 64:
        raise ValueError(f"{who}: {Hq} query heads for {Hkv} KV heads")
    lens = _ints(who, "seq_lens", seq_lens, dev, B)
    out = torch.empty_like(q, dtype=torch.float16, memory_format=torch.contiguous_format)
    if B == 0:
        return out
    if max_pages == 0:
        return out.zero_()
    M = 0
    if mass is not None:
        M = mass.shape[2] if isinstance(mass, torch.Tensor) and mass.dim() == 3 else -1
        if (M < max_pages * page or mass.shape[0] != B or mass.shape[1] != Hkv or mass.dtype != torch.float32
                or mass.device != dev or not mass.is_contiguous()):
            raise ValueError(f"{who}: mass must be contiguous fp32 ({B}, {Hkv}, at least {max_pages * page}) on {dev}")
    qc = q if q.dtype == torch.float16 else q.to(torch.float16)
    stride = qc.stride()
    ld = stride[0] if B > 1 else Hq * hd
    if stride[-1] != 1 or (Hq > 1 and stride[1] != hd) or ld % 8 or ld < Hq * hd or qc.data_ptr() % 16:
        qc, ld = qc.clone(memory_format=torch.contiguous_format), Hq * hd
    with on_device(dev.index):
        L = _lib.lib()
        need = L.axm_paged_decode_workspace_bytes(B, Hq, Hkv, hd, page, max_pages, 0 if mass is None else 1)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        rc = L.axm_paged_flash_decode(qc.data_ptr(), ld, d, lens.data_ptr(), out.data_ptr(), Hq,
                                      None if mass is None else mass.data_ptr(), M,
                                      None if ws is None else ws.data_ptr(), need, _lib.raw_stream(dev.index))
    if rc:
        _lib.check(rc, who)
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
    if not isinstance(cache, torch.Tensor) or not cache.is_cuda:
        _lib.require_gpu(cache, who)
    shape = cache.shape
    if len(shape) != 6 or shape[1] != 2 or shape[0] < 1:
        raise ValueError(f"{who}: cache must be (layers, 2, pages, n_kv_head, page_size, width), got {tuple(shape)}")
    dev = cache.device
    L, _, P, H, page, width = shape
    quant = cache.dtype != torch.float16
    code, hd, item = 0, width, 2
    stride, scale_stride = cache.stride(), (0, 0)
    scale_page, scale_ptr = 0, 0
    if quant:
        groups = scales.shape[5] if isinstance(scales, torch.Tensor) and scales.dim() == 6 else 0
        code, hd, item = (1, width, 1) if groups * 64 == width else (2, 2 * width, 1)
        if (cache.dtype not in (torch.uint8, torch.float8_e4m3fn) or not groups or groups * 64 != hd
                or scales.shape[:5] != shape[:5] or scales.dtype != torch.float16 or scales.device != dev):
            raise ValueError(f"{who}: quantized KV cache (uint8 codes) needs fp16 scales (layers, 2, pages, n_kv_head, "
                             "page_size, hd / 64)")
        scale_stride, scale_page, scale_ptr = scales.stride(), _page_stride(who, "scales", scales), scales.data_ptr()
    if 0 in shape:
        raise ValueError(f"{who}: empty cache {tuple(shape)}")
    table = _table(who, block_table, dev)
    B, max_pages = table.shape
    ptr = cache.data_ptr()
    d = _PAGED_KV.pack(ptr, ptr + stride[1] * item, scale_ptr, scale_ptr + scale_stride[1] * 2, table.data_ptr(),
                       _page_stride(who, "cache", cache), scale_page, code, H, hd, page, P, B, max_pages)
    budget, recent = int(budget), int(recent)
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"{who}: budget {budget} must be positive and recent {recent} within it")
    if (not isinstance(mass, torch.Tensor) or mass.dtype != torch.float32 or mass.device != dev or mass.dim() != 4
            or mass.shape[:3] != (L, B, H) or mass.shape[3] < max_pages * page):
        raise ValueError(f"{who}: mass must be fp32 ({L}, {B}, {H}, at least {max_pages * page}) on {dev}")
    lens = _ints(who, "seq_lens", seq_lens, dev, B)
    if not mass.is_contiguous():
        mass = mass.contiguous()
    kept = torch.empty((L, B, H, budget), dtype=torch.int32, device=dev)
    out_lens, out_mass = torch.empty_like(lens), torch.empty_like(mass)
    if B == 0:
        return kept, out_lens, out_mass
    if max_pages == 0:
        return kept.fill_(-1), out_lens.zero_(), out_mass.zero_()
    with on_device(dev.index):
        rc = _lib.lib().axm_evict_paged_kv(
            d, L, stride[0] * item, scale_stride[0] * 2, lens.data_ptr(),
            mass.data_ptr(), mass.shape[3], budget, recent, out_mass.data_ptr(), kept.data_ptr(), out_lens.data_ptr(),
            _lib.raw_stream(dev.index))
    if rc:
        _lib.check(rc, who)
    return kept, out_lens, out_mass
