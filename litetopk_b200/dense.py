"""The dense side of latent attention: writing the paged cache, attending to all of it, and the prefill of prompts.

``append_kv`` writes the rows that ``mla_decode`` reads (and, flattened to ``[rows, 656]`` or ``[rows, 576]``, that
``prepare_kv`` and ``sparse_prefill`` take); ``mla_prefill`` is the expanded form, over keys and values of every head.

Like the operators of :mod:`litetopk_b200.api` these are thin wrappers over the C ABI: asynchronous on the current stream of
their tensors' device, checked here and in C, without a CPU path, and without host synchronisation, so that they can be captured in a
CUDA graph and replayed on new contents (lengths, pages, positions) of the same tensors.  The reference has no counterpart of
them.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import check
from .api import _empty, _need, _on_device, _ptr, _status, _workspace_bytes

_INDEX = (torch.int32, torch.int64)
ROW_BYTES = {torch.bfloat16: 1152, torch.uint8: 656}


def _same_device(dev: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} must be on {dev} like the first argument, got {t.device}")


def _cache(kv_cache: torch.Tensor):
    """(packed, blocks, block size, bytes between blocks) of a paged cache; a 2-D one is a single run of rows (blocks of one)."""
    _need(kv_cache, "kv_cache", (torch.bfloat16, torch.uint8))
    packed = kv_cache.dtype == torch.uint8
    width, item = (656, 1) if packed else (576, 2)
    if kv_cache.dim() not in (2, 3) or kv_cache.shape[-1] != width:
        raise ValueError("kv_cache must be [blocks, block_size, 576] bf16 or [blocks, block_size, 656] uint8 (or 2-D rows)")
    if kv_cache.stride(-1) != 1:
        raise ValueError("kv_cache needs unit inner stride")
    if kv_cache.dim() == 2:
        return packed, kv_cache.shape[0], 1, kv_cache.stride(0) * item
    if kv_cache.shape[1] < 1 or (kv_cache.shape[1] > 1 and kv_cache.stride(1) != width):
        raise ValueError("rows of a block of kv_cache must be dense")
    return packed, kv_cache.shape[0], kv_cache.shape[1], kv_cache.stride(0) * item


def _apart(t: torch.Tensor, name: str) -> None:
    steps = sorted((step, size) for step, size in zip(t.stride()[:-1], t.shape[:-1]) if size > 1)
    end = t.shape[-1]
    for step, size in steps:
        if step < end:
            raise ValueError(f"{name} must not overlap itself")
        end += step * (size - 1)


def append_kv(kv_c: torch.Tensor, k_rope: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, slots: torch.Tensor,
              kv_cache: torch.Tensor, *, interleaved: bool = True, q_rope: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> None:
    """Write T tokens' rows into a paged latent cache, the 64 rope dims turned by the tokens' positions; in the same launch turn
    the queries' rope dims.

    kv_c [T, 512] bf16 (normalised latents), k_rope [T, 64] bf16, positions [T] and slots [T] int32 or int64, cos_sin
    [n_positions, 64] f32: cosines of the 32 angles, then their sines.  kv_cache [blocks, block_size, 576] bf16, or
    [blocks, block_size, 656] uint8 packed rows (512 e4m3 codes, 4 f32 scales, 64 bf16; scales are powers of two, so that
    dequantised rows are exact in bf16); a slot is block * block_size + place in it.  2-D caches are rows.

    ``interleaved``: dims (2i, 2i + 1) are a pair, else (i, i + 32).  ``q_rope`` [T, heads, 64] bf16 is turned into
    ``q_out`` of that shape (any views with unit inner stride: the last 64 dims of projected and of absorbed queries; the same
    view for in place), ``k_rope`` once more into ``k_out`` [T, 64] where that is given.  Neither may overlap itself.

    Tokens with a slot that is negative or beyond the cache are padding: no row is written for them.  No two tokens may have the same
    slot.  Tokens whose position is not in ``cos_sin`` are left out altogether.
    """
    if (host := _lib.host()) is not None:
        r = host.append_kv(kv_c, k_rope, positions, cos_sin, slots, kv_cache, interleaved, q_rope, q_out, k_out)
        if r is not None:
            if r is not True:
                check(r, "append_kv")
            return
    _need(kv_c, "kv_c", torch.bfloat16, 2)
    _need(k_rope, "k_rope", torch.bfloat16, 2)
    _need(positions, "positions", _INDEX, 1)
    _need(slots, "slots", _INDEX, 1)
    _need(cos_sin, "cos_sin", torch.float32, 2)
    dev, T = kv_c.device, kv_c.shape[0]
    if kv_c.shape[1] != 512 or k_rope.shape != (T, 64) or positions.shape[0] != T or slots.shape[0] != T or cos_sin.shape[1] != 64:
        raise ValueError("kv_c must be [T, 512], k_rope [T, 64], positions and slots [T], cos_sin [n_positions, 64]")
    if kv_c.stride(1) != 1 or k_rope.stride(1) != 1 or cos_sin.stride(1) != 1 or (T > 1 and not (positions.is_contiguous() and slots.is_contiguous())):
        raise ValueError("kv_c, k_rope and cos_sin need unit inner stride, positions and slots must be contiguous")
    packed, blocks, block, pitch = _cache(kv_cache)
    if (q_rope is None) != (q_out is None):
        raise ValueError("q_rope and q_out must be given together")
    qs = qo = (0, 0)
    heads = 0
    if q_rope is not None:
        _need(q_rope, "q_rope", torch.bfloat16, 3)
        _need(q_out, "q_out", torch.bfloat16, 3)
        heads = q_rope.shape[1]
        if q_rope.shape != (T, heads, 64) or q_out.shape != q_rope.shape or q_rope.stride(2) != 1 or q_out.stride(2) != 1 or heads < 1:
            raise ValueError("q_rope and q_out must be [T, heads, 64] with unit inner stride")
        _apart(q_out, "q_out")
        qs, qo = q_rope.stride()[:2], q_out.stride()[:2]
    if k_out is not None:
        _need(k_out, "k_out", torch.bfloat16, 2)
        if k_out.shape != (T, 64) or k_out.stride(1) != 1:
            raise ValueError("k_out must be [T, 64] with unit inner stride")
        _apart(k_out, "k_out")
    _same_device(dev, k_rope=k_rope, positions=positions, cos_sin=cos_sin, slots=slots, kv_cache=kv_cache, q_rope=q_rope, q_out=q_out, k_out=k_out)
    if T == 0:
        return
    check(_on_device(dev, _lib.lib().litedsa_append_kv, _ptr(kv_c), kv_c.stride(0), _ptr(k_rope), k_rope.stride(0), _ptr(positions),
                     positions.dtype == torch.int64, _ptr(cos_sin), cos_sin.shape[0], cos_sin.stride(0), _ptr(slots),
                     slots.dtype == torch.int64, _ptr(kv_cache), packed, blocks, block, pitch, bool(interleaved), _ptr(q_rope), *qs,
                     _ptr(q_out), *qo, heads, _ptr(k_out), 0 if k_out is None else k_out.stride(0), T), "append_kv")


def mla_decode(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, sm_scale: float, *,
               out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None):
    """Absorbed latent attention of every sequence's newest tokens over all of its cached rows.

    q [B, heads, 576] bf16, or [B, q_len, heads, 576] for several tokens a sequence (any strides that are multiples of 8, unit
    inner stride; 1 to 128 heads).  kv_cache as :func:`append_kv` writes it, block_size a multiple of 16.  block_table [B, columns]
    int32, seq_lens [B] int32: a sequence's keys, its new tokens among them; token j of q_len sees the first
    ``seq_lens - q_len + 1 + j``.  Keys are the 576 dims of a row, values its first 512.

    Returns ``(out [B, (q_len,) heads, 512] bf16, lse [B, (q_len,) heads] f32)``, written into ``out`` / ``lse`` when given
    (contiguous).  A row that sees no key: out = 0, lse = +inf; one with a score that is NaN or +inf: NaN in both.  Lengths are clamped to what a
    row of the table can hold.  A cached value that is infinite or NaN can reach the earlier of its sequence's new tokens, although they may not see it.
    """
    if out is None and lse is None and (host := _lib.host()) is not None:
        r = host.mla_decode(q, kv_cache, block_table, seq_lens, sm_scale)
        if r is not None:
            if type(r) is int:
                check(r, "mla_decode")
            return r
    _need(q, "q", torch.bfloat16)
    _need(block_table, "block_table", torch.int32, 2)
    _need(seq_lens, "seq_lens", torch.int32, 1)
    if q.dim() not in (3, 4) or q.shape[-1] != 576 or q.stride(-1) != 1:
        raise ValueError("q must be [B, heads, 576] or [B, q_len, heads, 576] with unit inner stride")
    dev, B, heads = q.device, q.shape[0], q.shape[-2]
    q_len = q.shape[1] if q.dim() == 4 else 1
    if not 1 <= heads <= 128 or q_len < 1:
        raise ValueError("q must have 1 to 128 heads and at least one token a sequence")
    if block_table.shape[0] != B or seq_lens.shape[0] != B or (block_table.shape[1] > 1 and block_table.stride(1) != 1) or \
            (B > 1 and seq_lens.stride(0) != 1):
        raise ValueError("block_table must be [B, columns] with unit inner stride and seq_lens a contiguous [B]")
    packed, blocks, block, pitch = _cache(kv_cache)
    if kv_cache.dim() != 3 or block % 16:
        raise ValueError("kv_cache must be [blocks, block_size, 576 | 656] with a block_size that is a multiple of 16")
    shape = q.shape[:-1]
    if out is None:
        out = _empty((*shape, 512), torch.bfloat16, dev)
    else:
        _need(out, "out", torch.bfloat16)
        if out.shape != (*shape, 512) or not out.is_contiguous():
            raise ValueError("out must be a contiguous [B, (q_len,) heads, 512] bf16 tensor")
    if lse is None:
        lse = _empty(tuple(shape), torch.float32, dev)
    else:
        _need(lse, "lse", torch.float32)
        if lse.shape != shape or not lse.is_contiguous():
            raise ValueError("lse must be a contiguous [B, (q_len,) heads] f32 tensor")
    _same_device(dev, kv_cache=kv_cache, block_table=block_table, seq_lens=seq_lens, out=out, lse=lse)
    if B == 0:
        return out, lse
    ws = _empty((max(_workspace_bytes("litedsa_mla_decode_workspace", dev.index, q_len, heads), 1),), torch.uint8, dev)
    check(_on_device(dev, _lib.lib().litedsa_mla_decode, _ptr(q), q.stride(0), q.stride(1) if q.dim() == 4 else 0, q.stride(-2),
                     _ptr(kv_cache), packed, blocks, block, pitch, _ptr(block_table), block_table.stride(0), block_table.shape[1],
                     _ptr(seq_lens), float(sm_scale), _ptr(out), _ptr(lse), B, q_len, heads, _ptr(ws), ws.numel()), "mla_decode")
    return out, lse


def mla_decode_status(reset: bool = False, device=None):
    """Status block of the decode kernel (see :func:`litetopk_b200.attn_status`)."""
    return _status("litedsa_mla_decode_status", reset, device)


def mla_prefill(q: torch.Tensor, k_nope: torch.Tensor, k_rope: torch.Tensor, v: torch.Tensor, sm_scale: float, *,
                cu_seqlens_q: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = True,
                out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None):
    """Expanded latent attention over a batch of sequences: scores ``sm_scale * (q[..., :128] . k_nope + q[..., 128:] . k_rope)``.

    q [Tq, heads, 192], k_nope and v [Tk, heads, 128], k_rope [Tk, 64] (one for all heads), all bf16; any strides but 0 that are multiples
    of 8, unit inner stride (k_nope and v may be views of one projection).  Sequence b has queries ``cu_seqlens_q[b] : cu_seqlens_q[b + 1]`` and
    keys ``cu_seqlens_k[b] : cu_seqlens_k[b + 1]`` (int32 [B + 1], entries that do not fall; both None: one sequence of all).  ``causal``: its queries are its last tokens,
    query i of n sees the first ``m - n + 1 + i`` of its m keys.  ``sm_scale`` must not be negative.

    Returns ``(out [Tq, heads, 128] bf16, lse [Tq, heads] f32)``, written into ``out`` / ``lse`` when given (contiguous).  A row that sees
    no key: out = 0, lse = +inf; one with a score that is NaN or +inf: NaN in both.  A value that is infinite or NaN can reach rows of its sequence
    that share a block of 128 keys with it, although they may not see it.  Rows that are no sequence's (behind ``cu_seqlens_q[-1]``) are not written.
    """
    if out is None and lse is None and (host := _lib.host()) is not None:
        r = host.mla_prefill(q, k_nope, k_rope, v, sm_scale, cu_seqlens_q, cu_seqlens_k, causal)
        if r is not None:
            if type(r) is int:
                check(r, "mla_prefill")
            return r
    for t, n, d in ((q, "q", 3), (k_nope, "k_nope", 3), (k_rope, "k_rope", 2), (v, "v", 3)):
        _need(t, n, torch.bfloat16, d)
        if t.stride(-1) != 1:
            raise ValueError(f"{n} needs unit inner stride")
        if any(size > 1 and step == 0 for size, step in zip(t.shape, t.stride())):
            raise ValueError(f"{n} must not be expanded")
    dev, (Tq, heads, d), Tk = q.device, q.shape, k_rope.shape[0]
    if d != 192 or heads < 1 or k_nope.shape != (Tk, heads, 128) or v.shape != (Tk, heads, 128) or k_rope.shape[1] != 64:
        raise ValueError("q must be [Tq, heads, 192], k_nope and v [Tk, heads, 128], k_rope [Tk, 64]")
    if not sm_scale >= 0:
        raise ValueError("sm_scale must not be negative")
    B = 1
    if (cu_seqlens_q is None) != (cu_seqlens_k is None):
        raise ValueError("cu_seqlens_q and cu_seqlens_k must be given together")
    if cu_seqlens_q is not None:
        _need(cu_seqlens_q, "cu_seqlens_q", torch.int32, 1)
        _need(cu_seqlens_k, "cu_seqlens_k", torch.int32, 1)
        B = cu_seqlens_q.shape[0] - 1
        if B < 0 or cu_seqlens_k.shape[0] != B + 1 or not (cu_seqlens_q.is_contiguous() and cu_seqlens_k.is_contiguous()):
            raise ValueError("cu_seqlens_q and cu_seqlens_k must be contiguous [B + 1]")
    if out is None:
        out = _empty((Tq, heads, 128), torch.bfloat16, dev)
    else:
        _need(out, "out", torch.bfloat16)
        if out.shape != (Tq, heads, 128) or not out.is_contiguous():
            raise ValueError("out must be a contiguous [Tq, heads, 128] bf16 tensor")
    if lse is None:
        lse = _empty((Tq, heads), torch.float32, dev)
    else:
        _need(lse, "lse", torch.float32)
        if lse.shape != (Tq, heads) or not lse.is_contiguous():
            raise ValueError("lse must be a contiguous [Tq, heads] f32 tensor")
    _same_device(dev, k_nope=k_nope, k_rope=k_rope, v=v, cu_seqlens_q=cu_seqlens_q, cu_seqlens_k=cu_seqlens_k, out=out, lse=lse)
    if Tq == 0 or B == 0:
        return out, lse
    need = _workspace_bytes("litedsa_mla_prefill_workspace", dev.index, Tq, Tk, heads)
    ws = _empty((need,), torch.uint8, dev) if need else None
    check(_on_device(dev, _lib.lib().litedsa_mla_prefill, _ptr(q), q.stride(0), q.stride(1), _ptr(k_nope), k_nope.stride(0), k_nope.stride(1),
                     _ptr(k_rope), k_rope.stride(0), _ptr(v), v.stride(0), v.stride(1), _ptr(cu_seqlens_q), _ptr(cu_seqlens_k), B,
                     float(sm_scale), bool(causal), _ptr(out), _ptr(lse), Tq, Tk, heads, _ptr(ws), need), "mla_prefill")
    return out, lse


def mla_prefill_status(reset: bool = False, device=None):
    """Status block of the prefill kernel (see :func:`litetopk_b200.attn_status`)."""
    return _status("litedsa_mla_prefill_status", reset, device)
