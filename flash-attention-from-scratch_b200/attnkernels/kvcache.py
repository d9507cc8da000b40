"""The 4-bit paged cache and the eviction of cached tokens.

A long-context decode is bound by the bytes of its cache. Two ways to fewer of
them, each beside the fp16 paged decode and together:

* A cache held in 4 bits: paged_append_kv4 quantises new tokens into their
  slots, paged_decode_kv4 attends over the rows as they are (80 bytes for the 256
  that a token's K or V of head_dim 128 takes in fp16), paged_read_kv4 gives
  slots' values back. A row holds groups of 32 values with an fp16 scale and an
  fp16 low, value = low + scale * code; the layout is in include/attn_b200.h.

* Eviction by accumulated attention weight: paged_decode_weights (or
  paged_decode_kv4 with `weights`) adds every token's softmax weight to a total
  per cache slot, and paged_evict keeps each head's tokens with the largest
  totals, next to the first and the last ones.

    weights = torch.zeros(num_blocks, H_kv, block_size, device="cuda")
    ...
    paged_append_kv4(k, v, k_cache, v_cache, slots, weights=weights)
    out = paged_decode_kv4(q, k_cache, v_cache, tables, lens, max_len, weights=weights)
    ...
    lens, kept = paged_evict((k_cache, v_cache), weights, tables, lens, max_len, new_tables,
                             keep=2048, recent=256, sinks=4)

No counterparts in the reference. Like the rest of the package these need a B200
and run on the current stream of their tensors' device; caches, totals and
tables are used in place and must be contiguous.
"""
from __future__ import annotations

import math

import torch

from . import load_extension, _check_decode, _decode_args

_FLOATS = (torch.float16, torch.bfloat16)


def kv4_row_bytes(head_dim):
    """Bytes of one 4-bit row: the last dim of a 4-bit cache (80 at head_dim 128, 40 at 64)."""
    if head_dim not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    return head_dim // 2 + head_dim // 8


def _check_kv4_caches(k_cache, v_cache, head_dim=None):
    """head_dim of a pair of 4-bit caches."""
    dims = {kv4_row_bytes(d): d for d in (64, 128)}
    for c in (k_cache, v_cache):
        if c.dtype != torch.uint8 or c.dim() != 4 or c.shape[-1] not in dims:
            raise ValueError("4-bit caches must be uint8 [num_blocks, H_kv, block_size, "
                             "kv4_row_bytes(head_dim)]")
        if not c.is_contiguous():
            raise ValueError("4-bit caches must be contiguous")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    d = dims[k_cache.shape[-1]]
    if head_dim is not None and d != head_dim:
        raise ValueError("head_dim must be 64 or 128 and match the cache")
    return d


def _check_weights(weights, num_blocks, hkv, block_size):
    if weights.dtype != torch.float32 or tuple(weights.shape) != (num_blocks, hkv, block_size) \
            or not weights.is_contiguous():
        raise ValueError("weights must be contiguous fp32 [num_blocks, H_kv, block_size]")


def _check_devices(*tensors):
    if not all(t.is_cuda for t in tensors):
        raise ValueError("tensors must be CUDA tensors")
    if len({t.device for t in tensors}) != 1:
        raise ValueError("tensors must be on one device")


def _check_lens(q_batch, block_tables, context_lens):
    if block_tables.dim() != 2 or context_lens.dim() != 1:
        raise ValueError("block_tables must be [B, max_blocks], context_lens [B]")
    if block_tables.shape[0] != q_batch or context_lens.shape[0] != q_batch:
        raise ValueError("block_tables and context_lens must have a row per sequence")


def _index32(t, device):
    return t.to(device=device, dtype=torch.int32).contiguous()


def _check_slots(slots, tokens):
    if slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64):
        raise ValueError("slots must be an int64 or int32 vector")
    if tokens is not None and slots.shape[0] != tokens:
        raise ValueError("slots must have one entry per token")


def _dense_rows(t):
    """t, or a copy of it where its rows are not 16-byte pieces that the kernel can load."""
    ok = t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 and \
        t.data_ptr() % 16 == 0
    return t if ok else t.contiguous()


def paged_append_kv4(k, v, k_cache, v_cache, slots, weights=None):
    """Quantise new tokens into a 4-bit paged cache.

    k, v:     [T, H_kv, D] fp16 or bf16, D in {64, 128} (any strides; a slice of a fused
              projection is read where it is)
    k_cache, v_cache: uint8 [num_blocks, H_kv, block_size, kv4_row_bytes(D)], written in place
    slots:    [T] int64 (or int32), page * block_size + offset of each token; below 0: the token
              is skipped (padding). The slots of a call must differ.
    weights:  optional fp32 [num_blocks, H_kv, block_size], set to 0 in the written slots

    Per group of 32 dims: low = min, scale = (max - low) / 15 (both fp16), codes rounded to
    nearest even. A group with an infinity, a NaN or a value beyond fp16's range reads back as
    NaN. A slot past the cache is not written and shows in device_status().
    """
    if k.dtype not in _FLOATS or v.dtype != k.dtype or k.dim() != 3 or k.shape != v.shape:
        raise ValueError("k and v must be fp16 or bf16 tensors of one shape [T, H_kv, D]")
    if k.shape[-1] not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    _check_kv4_caches(k_cache, v_cache, k.shape[-1])
    if k_cache.shape[1] != k.shape[1]:
        raise ValueError("k and the cache must have the same kv heads")
    _check_slots(slots, k.shape[0])
    tensors = [k, v, k_cache, v_cache, slots]
    if weights is not None:
        _check_weights(weights, *k_cache.shape[:3])
        tensors.append(weights)
    _check_devices(*tensors)
    if k.shape[0] == 0:
        return
    load_extension().kv4_append(_dense_rows(k), _dense_rows(v), k_cache, v_cache,
                                slots.to(torch.int64).contiguous(), weights)


def paged_read_kv4(k_cache, v_cache, slots, dtype=torch.float16):
    """Values of slots of a 4-bit paged cache: (k, v), each [T, H_kv, D] of `dtype` (fp16 or
    bf16), low + scale * code rounded once. A negative slot, or one past the cache (which also
    shows in device_status()), reads as zeros."""
    d = _check_kv4_caches(k_cache, v_cache)
    if dtype not in _FLOATS:
        raise ValueError("dtype must be fp16 or bf16")
    _check_slots(slots, None)
    _check_devices(k_cache, v_cache, slots)
    if slots.shape[0] == 0:
        return tuple(torch.empty(0, k_cache.shape[1], d, dtype=dtype, device=k_cache.device)
                     for _ in range(2))
    return load_extension().kv4_read(k_cache, v_cache, slots.to(torch.int64).contiguous(), d, dtype)


def paged_decode_kv4(q, k_cache, v_cache, block_tables, context_lens, max_context_len,
                     scale=None, weights=None):
    """Decode attention over a 4-bit paged cache: paged_decode with its arguments, but

    q:            [B, H, D] (or [B, H, 1, D]) fp16 or bf16; H / H_kv any whole number from 1 to 8
    k_cache:      uint8 [num_blocks, H_kv, block_size, kv4_row_bytes(D)] (v_cache the same);
                  block_size even at D = 64
    context_lens: 0 gives a row of zeros; lengths above max_context_len are cut to it
    weights:      optional fp32 [num_blocks, H_kv, block_size]: each token's softmax weight,
                  summed over the query heads of its kv head, is added to its slot's total
    There is no partition size: the context is split over the GPU's warps in equal runs.
    Returns q's shape and type.
    """
    if q.dtype not in _FLOATS:
        raise ValueError("q must be fp16 or bf16")
    if q.dim() == 4:
        if q.shape[2] != 1:
            raise ValueError("a 4-D decode q must be [B, H, 1, D]")
        q3 = q.reshape(q.shape[0], q.shape[1], q.shape[3])
    elif q.dim() == 3:
        q3 = q
    else:
        raise ValueError("q must be [B, H, D] (or [B, H, 1, D])")
    if q3.shape[-1] not in (64, 128):
        raise ValueError("head_dim must be 64 or 128 and match the cache")
    _check_kv4_caches(k_cache, v_cache, q3.shape[-1])
    _check_lens(q3.shape[0], block_tables, context_lens)
    tensors = [q, k_cache, v_cache]
    if weights is not None:
        _check_weights(weights, *k_cache.shape[:3])
        tensors.append(weights)
    _check_devices(*tensors)
    if q3.shape[0] == 0 or max_context_len == 0:
        return torch.zeros_like(q)
    scale = 1.0 / math.sqrt(q3.shape[-1]) if scale is None else scale
    q3 = q3.contiguous()
    if q3.data_ptr() % 16:
        q3 = q3.clone()
    return load_extension().kv4_decode(
        q3, k_cache, v_cache, _index32(block_tables, q.device), _index32(context_lens, q.device),
        int(max_context_len), weights, float(scale)).reshape(q.shape)


def paged_decode_weights(q, k_cache, v_cache, block_tables, context_lens, max_context_len, weights,
                         scale=None, partition_size=None):
    """paged_decode that also adds each token's attention weight to its slot's total.

    weights: fp32 [num_blocks, H_kv, block_size], added to in place: the token's softmax weight,
             summed over the query heads of its kv head. Totals of slots that the sequences do not
             hold stay as they are. A page that several sequences share gets the adds of all.
    The other arguments and the result are paged_decode's; a length above max_context_len is cut
    to it.
    """
    _check_decode(q, k_cache, v_cache)
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must be [num_blocks, H_kv, block_size, D]")
    _check_weights(weights, *k_cache.shape[:3])
    _check_lens(q.shape[0], block_tables, context_lens)
    _check_devices(q, k_cache, v_cache, weights)
    if q.shape[0] == 0 or max_context_len == 0:
        return torch.zeros_like(q)
    q3, kc, vc, bt, lens, max_ctx, scale, partition = _decode_args(
        q, k_cache, v_cache, block_tables, context_lens, max_context_len, scale, partition_size)
    return load_extension().paged_decode_weights(q3, kc, vc, bt, lens, max_ctx, weights, scale,
                                                 partition).reshape(q.shape)


def paged_evict(caches, weights, block_tables, context_lens, max_context_len, new_block_tables, keep,
                recent=0, sinks=0):
    """Cut paged caches to at most `keep` tokens per sequence, by accumulated attention weight.

    caches:   sequence of 1 to 8 tensors [num_blocks, H_kv, block_size, ...] of any type, e.g.
              (k_cache, v_cache) of paged_decode or of paged_decode_kv4; contiguous
    weights:  fp32 [num_blocks, H_kv, block_size], the totals that go by paged_decode_weights
    block_tables, context_lens, max_context_len: the sequences as they are, as in paged_decode
    new_block_tables: [B, new_max_blocks], the pages that take the kept tokens; new_max_blocks *
              block_size >= min(keep, max_context_len). They must not be pages that the sequences
              of the call read or write otherwise; a sequence of at most `keep` tokens may give
              its old pages again and is not moved then.
    recent, sinks: the last and the first tokens, kept whatever their totals

    Per sequence and kv head the first `sinks`, the last `recent` and, of the rest, the tokens
    with the largest totals stay (ties to the lower index, NaN lowest), in their order. Their rows
    of every cache and their totals are copied to the new pages; all else stays as it is, so pages
    shared with other sequences are safe. Returns (new_lens int32 [B], kept int32 [B, H_kv, keep]:
    the kept tokens' old indices, then -1).
    """
    caches = tuple(caches)
    if not 1 <= len(caches) <= 8:
        raise ValueError("caches must be 1 to 8 tensors")
    if weights.dim() != 3:
        raise ValueError("weights must be contiguous fp32 [num_blocks, H_kv, block_size]")
    _check_weights(weights, *weights.shape)
    row_bytes = []
    for c in caches:
        if c.dim() < 3 or c.shape[:3] != weights.shape or not c.is_contiguous():
            raise ValueError("caches must be contiguous [num_blocks, H_kv, block_size, ...]")
        row = c.element_size() * math.prod(c.shape[3:])
        if not 0 < row <= 65536:
            raise ValueError("a cache row must have 1 to 65536 bytes")
        row_bytes.append(row)
    _check_lens(block_tables.shape[0], block_tables, context_lens)
    if new_block_tables.dim() != 2 or new_block_tables.shape[0] != block_tables.shape[0]:
        raise ValueError("new_block_tables must be [B, new_max_blocks]")
    keep, recent, sinks = int(keep), int(recent), int(sinks)
    if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
        raise ValueError("keep must be >= 1, sinks and recent >= 0 and together keep at most")
    _check_devices(weights, *caches)
    dev = weights.device
    if block_tables.shape[0] == 0 or max_context_len == 0:
        i32 = dict(dtype=torch.int32, device=dev)
        return (torch.zeros(block_tables.shape[0], **i32),
                torch.full((block_tables.shape[0], weights.shape[1], keep), -1, **i32))
    return load_extension().paged_evict(
        caches, row_bytes, weights, _index32(block_tables, dev), _index32(context_lens, dev),
        int(max_context_len), _index32(new_block_tables, dev), keep, recent, sinks)
