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

import functools
import math

import torch

from . import (CHUNK, decode_partition, load_extension, _check_decode, _decode_warps_per_sm,
               _sm_count)

_FLOATS = (torch.float16, torch.bfloat16)
_ROW_BYTES = {64: 40, 128: 80}  # head_dim / 2 of codes, head_dim / 8 of scales and lows
_HEAD_DIM = {v: k for k, v in _ROW_BYTES.items()}


def kv4_row_bytes(head_dim):
    """Bytes of one 4-bit row: the last dim of a 4-bit cache (80 at head_dim 128, 40 at 64)."""
    if head_dim not in _ROW_BYTES:
        raise ValueError("head_dim must be 64 or 128")
    return _ROW_BYTES[head_dim]


def _check_kv4_caches(k_cache, v_cache):
    """(num_blocks, H_kv, block_size, head_dim) of a pair of 4-bit caches."""
    shape = k_cache.shape
    if len(shape) != 4 or shape[3] not in _HEAD_DIM or k_cache.dtype != torch.uint8 or \
            v_cache.dtype != torch.uint8:
        raise ValueError("4-bit caches must be uint8 [num_blocks, H_kv, block_size, "
                         "kv4_row_bytes(head_dim)]")
    if v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("4-bit caches must be contiguous")
    nblk, hkv, bs, row = shape
    return nblk, hkv, bs, _HEAD_DIM[row]


def _check_weights(weights, num_blocks, hkv, block_size):
    if weights.dtype != torch.float32 or weights.shape != (num_blocks, hkv, block_size) \
            or not weights.is_contiguous():
        raise ValueError("weights must be contiguous fp32 [num_blocks, H_kv, block_size]")


def _device_of(*tensors):
    """Index of the one CUDA device that the tensors are on."""
    dev = tensors[0].get_device()  # -1: on the CPU
    for t in tensors:
        if t.get_device() != dev or dev < 0:
            if not all(t.is_cuda for t in tensors):
                raise ValueError("tensors must be CUDA tensors")
            raise ValueError("tensors must be on one device")
    return dev


def _check_lens(batch, block_tables, context_lens):
    """max_blocks_per_seq."""
    if block_tables.dim() != 2 or context_lens.dim() != 1:
        raise ValueError("block_tables must be [B, max_blocks], context_lens [B]")
    rows, blocks = block_tables.shape
    if rows != batch or context_lens.shape[0] != batch:
        raise ValueError("block_tables and context_lens must have a row per sequence")
    return blocks


def _index(t, dev, device, dtype=torch.int32):
    """t as a dense tensor of `dtype` on the device: itself where it is that already."""
    if t.dtype == dtype and t.get_device() == dev and t.is_contiguous():
        return t
    return t.to(device=device, dtype=dtype).contiguous()


def _check_slots(slots):
    if slots.dim() != 1 or slots.dtype not in (torch.int64, torch.int32):
        raise ValueError("slots must be an int64 or int32 vector")


def _dense_rows(t):
    """t, or a copy of it where its rows are not 16-byte pieces that the kernel can load."""
    s0, s1, s2 = t.stride()
    if s2 == 1 and s0 % 8 == 0 and s1 % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    # Not contiguous(): a dim of size 1 may have any stride there, and the address stays.
    return t.clone(memory_format=torch.contiguous_format)


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
    shape = k.shape
    if k.dtype not in _FLOATS or v.dtype != k.dtype or len(shape) != 3 or v.shape != shape:
        raise ValueError("k and v must be fp16 or bf16 tensors of one shape [T, H_kv, D]")
    T, hkv, d = shape
    if d not in _ROW_BYTES:
        raise ValueError("head_dim must be 64 or 128")
    nblk, cache_hkv, bs, cache_d = _check_kv4_caches(k_cache, v_cache)
    if (cache_hkv, cache_d) != (hkv, d):
        raise ValueError("k and the cache must have the same kv heads and head_dim")
    _check_slots(slots)
    if slots.shape[0] != T:
        raise ValueError("slots must have one entry per token")
    dev = _device_of(k, v, k_cache, v_cache, slots)
    if weights is not None:
        _check_weights(weights, nblk, hkv, bs)
        _device_of(k, weights)
    if T == 0:
        return
    load_extension().kv4_append(dev, _dense_rows(k), _dense_rows(v), k_cache, v_cache,
                                _index(slots, dev, k.device, torch.int64), weights,
                                (T, hkv, d, bs, nblk))


def paged_read_kv4(k_cache, v_cache, slots, dtype=torch.float16):
    """Values of slots of a 4-bit paged cache: (k, v), each [T, H_kv, D] of `dtype` (fp16 or
    bf16), low + scale * code rounded once (to fp32 first for bf16). A negative slot, or one past the cache (which also
    shows in device_status()), reads as zeros."""
    nblk, hkv, bs, d = _check_kv4_caches(k_cache, v_cache)
    if dtype not in _FLOATS:
        raise ValueError("dtype must be fp16 or bf16")
    _check_slots(slots)
    dev = _device_of(k_cache, v_cache, slots)
    T = slots.shape[0]
    if T == 0:
        return tuple(torch.empty(0, hkv, d, dtype=dtype, device=k_cache.device) for _ in range(2))
    return load_extension().kv4_read(dev, k_cache, v_cache,
                                     _index(slots, dev, k_cache.device, torch.int64), dtype,
                                     (T, hkv, d, bs, nblk))


def paged_decode_kv4(q, k_cache, v_cache, block_tables, context_lens, max_context_len,
                     scale=None, weights=None):
    """Decode attention over a 4-bit paged cache: paged_decode with its arguments, but

    q:            [B, H, D] (or [B, H, 1, D]) fp16 or bf16; H / H_kv any whole number from 1 to 8
    k_cache:      uint8 [num_blocks, H_kv, block_size, kv4_row_bytes(D)] (v_cache the same);
                  block_size even at D = 64
    context_lens: 0 gives a row of zeros; lengths above max_context_len are cut to it
    weights:      optional fp32 [num_blocks, H_kv, block_size]: each token's softmax weight,
                  summed over the query heads of its kv head, is added to its slot's total
    There is no partition size: the context is split over the GPU's warps in equal runs. The
    longest length is the fastest max_context_len, where it is known: rows that it shows to be
    short take one launch (8 sequences of 200 tokens, 8 kv heads, on the device: 5.7 us, and
    8.9 us with 8192 as the bound), and scratch with `weights` goes by it (an fp32 score per
    sequence, head and token up to it, kept until release_workspaces()).
    Softmax weights times V's scales, and V's middles, are rounded to fp16 (attn_b200.h), the
    output once to q's type; all else is fp32. Returns q's shape and type.
    """
    if q.dtype not in _FLOATS:
        raise ValueError("q must be fp16 or bf16")
    q3 = q
    if q.dim() == 4:
        if q.shape[2] != 1:
            raise ValueError("a 4-D decode q must be [B, H, 1, D]")
        q3 = q.reshape(q.shape[0], q.shape[1], q.shape[3])
    elif q.dim() != 3:
        raise ValueError("q must be [B, H, D] (or [B, H, 1, D])")
    B, H, D = q3.shape
    nblk, hkv, bs, d = _check_kv4_caches(k_cache, v_cache)
    if D != d:
        raise ValueError("head_dim must be 64 or 128 and match the cache")
    maxb = _check_lens(B, block_tables, context_lens)
    dev = _device_of(q, k_cache, v_cache)
    if weights is not None:
        _check_weights(weights, nblk, hkv, bs)
        _device_of(q, weights)
    max_context_len = int(max_context_len)
    if B == 0 or max_context_len == 0:
        return torch.zeros_like(q)
    if not q3.is_contiguous() or q3.data_ptr() % 16:
        q3 = q3.clone(memory_format=torch.contiguous_format)
    out = load_extension().kv4_decode(
        dev, q3, k_cache, v_cache, _index(block_tables, dev, q.device),
        _index(context_lens, dev, q.device), weights, (B, H, hkv, D, bs, nblk, maxb),
        max_context_len, 1.0 / math.sqrt(D) if scale is None else float(scale))
    return out if q.dim() == 3 else out.reshape(q.shape)


@functools.lru_cache(maxsize=4096)
def _weights_partition(batch, hkv, max_context_len, dev, heads, head_dim):
    """decode_partition's choice, doubled while that leaves six units per resident warp: fewer
    parts to merge (64 ragged sequences of up to 8192 tokens, 32 query over 8 kv heads, d 128:
    279 us at 256 tokens, 268 at 512, 305 at 1024, which leaves 3.5)."""
    part = decode_partition(batch, hkv, max_context_len, dev, num_heads=heads, head_dim=head_dim)
    units = 6 * _decode_warps_per_sm(heads // hkv, head_dim) * _sm_count(dev)
    while batch * hkv * -(-max_context_len // (2 * part)) >= units:
        part *= 2
    return part


def paged_decode_weights(q, k_cache, v_cache, block_tables, context_lens, max_context_len, weights,
                         scale=None, partition_size=None):
    """paged_decode that also adds each token's attention weight to its slot's total.

    weights: fp32 [num_blocks, H_kv, block_size], added to in place: the token's softmax weight,
             summed over the query heads of its kv head. Totals of slots that the sequences do not
             hold stay as they are. A page that several sequences share gets the adds of all. A
             slot that is given to a new token keeps the old one's total until it is zeroed:
             weights[slots // block_size, :, slots % block_size] = 0, padding's negative
             slots left out (paged_append_kv4 does that for a 4-bit cache).
    The other arguments and the result are paged_decode's; a length above max_context_len is cut
    to it. A sequence whose keys are all NaN gives NaN, where paged_decode gives zeros if it has
    split the sequence. The scratch holds an fp32 score per sequence, head and token up to
    max_context_len and is kept until release_workspaces().
    """
    q3 = _check_decode(q, k_cache, v_cache)
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must be [num_blocks, H_kv, block_size, D]")
    nblk, hkv, bs, D = shape
    B, H = q3.shape[:2]
    _check_weights(weights, nblk, hkv, bs)
    maxb = _check_lens(B, block_tables, context_lens)
    dev = _device_of(q, k_cache, v_cache, weights)
    if B == 0 or max_context_len == 0:
        return torch.zeros_like(q)
    max_context_len = int(max_context_len)
    if partition_size is None:
        partition_size = _weights_partition(B, hkv, max_context_len, dev, H, D)
    partition_size = -(-int(partition_size) // CHUNK) * CHUNK
    out = load_extension().paged_decode_weights(
        dev, q3.contiguous(), k_cache.contiguous(), v_cache.contiguous(),
        _index(block_tables, dev, q.device), _index(context_lens, dev, q.device), weights,
        (B, H, hkv, D, bs, nblk, maxb), max_context_len,
        1.0 / math.sqrt(D) if scale is None else float(scale), partition_size)
    return out if q.dim() == 3 else out.reshape(q.shape)


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
    shape = weights.shape
    if len(shape) != 3:
        raise ValueError("weights must be contiguous fp32 [num_blocks, H_kv, block_size]")
    nblk, hkv, bs = shape
    _check_weights(weights, nblk, hkv, bs)
    row_bytes = []
    for c in caches:
        if c.dim() < 3 or c.shape[:3] != shape or not c.is_contiguous():
            raise ValueError("caches must be contiguous [num_blocks, H_kv, block_size, ...]")
        row = c.element_size() * math.prod(c.shape[3:])
        if not 0 < row <= 65536:
            raise ValueError("a cache row must have 1 to 65536 bytes")
        row_bytes.append(row)
    if block_tables.dim() != 2:
        raise ValueError("block_tables must be [B, max_blocks], context_lens [B]")
    B = block_tables.shape[0]
    maxb = _check_lens(B, block_tables, context_lens)
    if new_block_tables.dim() != 2 or new_block_tables.shape[0] != B:
        raise ValueError("new_block_tables must be [B, new_max_blocks]")
    keep, recent, sinks = int(keep), int(recent), int(sinks)
    if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
        raise ValueError("keep must be >= 1, sinks and recent >= 0 and together keep at most")
    dev, device = _device_of(weights, *caches), weights.device
    max_context_len = int(max_context_len)
    if B == 0 or max_context_len == 0:
        return (torch.zeros(B, dtype=torch.int32, device=device),
                torch.full((B, hkv, keep), -1, dtype=torch.int32, device=device))
    return load_extension().paged_evict(
        dev, caches, row_bytes, weights, _index(block_tables, dev, device),
        _index(context_lens, dev, device), _index(new_block_tables, dev, device),
        (B, hkv, bs, nblk, maxb, new_block_tables.shape[1]), max_context_len, keep, recent, sinks)
