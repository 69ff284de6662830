"""Dense paged KV cache in 8 bits with a scale for each block of tokens and KV head: the operators of a model that is
served without eviction (every token's K and V stay), beside the compact ones of `layers/compact_attention.py`.

The cache of a layer is `k_cache` / `v_cache [blocks, kv_heads, block_size, head_dim]` in float8_e4m3fn (any view of that
shape whose last dimension is contiguous and whose other strides are multiples of 16 bytes, so a
`[blocks, block_size, kv_heads, head_dim]` allocation serves as well, permuted) and `k_scale` / `v_scale
[blocks, kv_heads]` in float32: value = code * scale.  Scales are powers of two between 2^-60 and 2^40, set by
`store_paged_kvcache` from the values it stores; nothing has to be calibrated.  A sequence's blocks are listed in its row
of `block_tables [sequences, columns]` (int32); row r of the sequence is row r % block_size of block
`block_tables[s, r // block_size]`.  One block table serves all layers.

A step, for prompts and for single tokens alike:

    cu_seqlens, slots, positions = build_paged_metadata(new_lens, kv_lens, block_tables, free_blocks, free_count, ...)
    per layer:  store_paged_kvcache(k, v, ..., slots)
                paged_prefill_attention(q, ..., cu_seqlens)   or, with a token per sequence at most,
                paged_decode_attention(q, ..., cu_seqlens_q=cu_seqlens)
    release_paged_blocks(...)   for sequences that ended

The tokens of a step lie one after the other, sequence by sequence, without gaps for sequences that have none.

Every call enqueues on the current stream of its tensors' device and can be captured into a CUDA graph.  There is no CPU
path: tensors must live on a CUDA device.
"""
from __future__ import annotations

from struct import Struct

import torch

from fastdms_b200 import _lib

BLOCK_SIZES = (16, 32, 64, 128)
MAX_DECODE_BATCH = 2048

# The argument blocks of include/fastdms_b200.h; every member is 8 bytes wide.
_METADATA_ARGS = Struct("12P7q")
_STORE_ARGS = Struct("4P12q4P8q")
_ATTN_ARGS = Struct("4P12q8P15qd")
_ROW_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_F8, _I32, _I64, _F32 = torch.float8_e4m3fn, torch.int32, torch.int64, torch.float32


def _device(named: dict) -> int:
    """The CUDA device that all tensors live on."""
    given = {name: t for name, t in named.items() if t is not None}
    _lib.require_cuda(*given.values())
    first = next(iter(given.values())).device
    for name, t in given.items():
        if t.device != first:
            raise ValueError(f"expected {name} on {first}, got {t.device}")
    return first.index


def _on_device(dev: int, fn, *args):
    """Calls a C function with device `dev` current."""
    if torch._C._cuda_getDevice() == dev:
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _launch(fn, args: bytes, dev: int) -> None:
    """Calls a C entry on the current stream of device `dev`."""
    rc = _on_device(dev, fn, args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc)


def _int_vector(t: torch.Tensor, name: str, size: int | None = None) -> None:
    if t.dtype is not _I32 or t.dim() != 1 or not t.is_contiguous() or (size is not None and t.numel() != size):
        shape = "[n]" if size is None else f"[{size}]"
        raise ValueError(f"expected {name} as contiguous int32 {shape}, got {tuple(t.shape)} {t.dtype}")


def _tables(block_tables: torch.Tensor, rows: int) -> tuple[int, int]:
    """Columns and row stride of a block table; one row (or none) may carry any stride."""
    if block_tables.dtype is not _I32 or block_tables.dim() != 2 or block_tables.shape[0] != rows:
        raise ValueError(f"expected block_tables as int32 [{rows}, columns], got {tuple(block_tables.shape)} {block_tables.dtype}")
    cols = block_tables.shape[1]
    stride = block_tables.stride()
    if cols > 1 and stride[1] != 1:
        raise ValueError("block_tables must be contiguous in its last dimension")
    return cols, stride[0] if rows > 1 else cols


def _check_block_size(block_size: int) -> None:
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")


def _cache_shape(k_cache, v_cache, k_scale, v_scale) -> tuple[int, int, int, int]:
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"expected k_cache and v_cache as [blocks, kv_heads, block_size, head_dim], got {tuple(shape)} / {tuple(v_cache.shape)}")
    if k_cache.dtype is not _F8 or v_cache.dtype is not _F8:
        raise ValueError(f"expected float8_e4m3fn caches, got {k_cache.dtype} / {v_cache.dtype}")
    scales = shape[:2]
    if (k_scale.shape != scales or v_scale.shape != scales or k_scale.dtype is not _F32 or v_scale.dtype is not _F32
            or not k_scale.is_contiguous() or not v_scale.is_contiguous()):
        raise ValueError(f"expected k_scale and v_scale as contiguous float32 {tuple(scales)}, got {tuple(k_scale.shape)} {k_scale.dtype} / "
                         f"{tuple(v_scale.shape)} {v_scale.dtype}")
    return shape


def _row_dtype(t: torch.Tensor, name: str) -> int:
    code = _ROW_DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    return code


def build_paged_metadata(
    new_lens: torch.Tensor,
    kv_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_blocks: torch.Tensor,
    free_count: torch.Tensor,
    *,
    block_size: int,
    total_tokens: int,
    kv_lens_out: torch.Tensor | None = None,
    free_count_out: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
    slot_mapping: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Block tables and slot map of a step, from lengths that are on the GPU.

    Sequence i holds `kv_lens[i]` rows and gets `new_lens[i]` more (int32 `[n]`).  The blocks it needs beyond its last one
    are popped from the stack `free_blocks[:free_count]` (int32, `free_count` int32 `[1]`) into its row of `block_tables`,
    sequence by sequence: the result does not depend on timing.  Where the stack runs out, that sequence and the later ones
    that need blocks are not served: no blocks, slots of -1, and `kv_lens` as before (running out raises nothing: compare
    the lengths).  A negative length, one beyond the table's columns, or more tokens than `total_tokens` are not served
    either and raise the device status bit for bad indices.

    `kv_lens` and `free_count` are advanced in place, or left alone where `kv_lens_out` / `free_count_out` are given
    (`kv_lens_out` may be `new_lens`; otherwise they overlap no other argument).
    Returns `cu_seqlens` (int32 `[n + 1]`), `slot_mapping` (int32 `[total_tokens]`, block * block_size + row) and
    `positions` (int64 `[total_tokens]`); buffers given for them are
    filled, and overlap no other argument.  `total_tokens` may exceed the sum of `new_lens`
    (a padded batch): the slots behind it are -1, which the store skips, and the positions 0.  Each sequence has a row of its
    own; free block ids are distinct, and blocks of the cache (`release_paged_blocks` has to know how many those are where the
    stack does not hold them all)."""
    n = kv_lens.numel()
    _int_vector(kv_lens, "kv_lens")
    _int_vector(new_lens, "new_lens", n)
    _int_vector(free_blocks, "free_blocks")
    _int_vector(free_count, "free_count", 1)
    cols, stride = _tables(block_tables, n)
    _check_block_size(block_size)
    total_tokens = int(total_tokens)
    if total_tokens < 0:
        raise ValueError(f"total_tokens must not be negative, got {total_tokens}")
    dev = kv_lens.get_device()
    if (dev < 0 or new_lens.get_device() != dev or block_tables.get_device() != dev or free_blocks.get_device() != dev
            or free_count.get_device() != dev):
        _device(dict(kv_lens=kv_lens, new_lens=new_lens, block_tables=block_tables, free_blocks=free_blocks, free_count=free_count))
    for t, name, size in ((kv_lens_out, "kv_lens_out", n), (free_count_out, "free_count_out", 1), (cu_seqlens, "cu_seqlens", n + 1),
                          (slot_mapping, "slot_mapping", total_tokens)):
        if t is not None:
            _int_vector(t, name, size)
            if t.get_device() != dev:
                _device({"kv_lens": kv_lens, name: t})
    if positions is not None:
        if positions.dtype is not _I64 or positions.shape != (total_tokens,) or not positions.is_contiguous():
            raise ValueError(f"expected positions as contiguous int64 [{total_tokens}], got {tuple(positions.shape)} {positions.dtype}")
        if positions.get_device() != dev:
            _device(dict(kv_lens=kv_lens, positions=positions))
    device = kv_lens.device
    kv_lens_out = kv_lens if kv_lens_out is None else kv_lens_out
    free_count_out = free_count if free_count_out is None else free_count_out
    if cu_seqlens is None:
        cu_seqlens = kv_lens.new_empty(n + 1)
    if slot_mapping is None:
        slot_mapping = kv_lens.new_empty(total_tokens)
    if positions is None:
        positions = kv_lens.new_empty(total_tokens, dtype=_I64)
    need = _lib.lib().fdms_paged_metadata_workspace_bytes(n, total_tokens)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _launch(_lib.lib().fdms_paged_metadata, _METADATA_ARGS.pack(
        new_lens.data_ptr(), kv_lens.data_ptr(), kv_lens_out.data_ptr(), block_tables.data_ptr(), free_blocks.data_ptr(), free_count.data_ptr(),
        free_count_out.data_ptr(), cu_seqlens.data_ptr(), slot_mapping.data_ptr(), positions.data_ptr(), ws.data_ptr() if need else 0,
        _lib.status_word(device).data_ptr(), n, cols, stride, block_size, free_blocks.numel(), total_tokens, need), dev)
    return cu_seqlens, slot_mapping, positions


def release_paged_blocks(
    kv_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_blocks: torch.Tensor,
    free_count: torch.Tensor,
    *,
    block_size: int,
    rows: torch.Tensor | None = None,
    num_blocks: int | None = None,
) -> None:
    """Gives the blocks of the listed rows (int32 indices of `kv_lens` and `block_tables`; all rows without a list) back to
    the stack and empties the rows: table entries -1, length 0.  A row that is listed twice is released once and, like one
    out of range or a block id outside the pool, raises the device status bit for bad indices.

    `num_blocks` is the number of blocks of the cache, whose ids lie below it; without it `free_blocks` has room for all of them.
    A stack that holds only some (a block kept for padding, a range of a shared pool) needs it: ids at or beyond
    `free_blocks.numel()` would be taken for none of the pool's, and their blocks lost."""
    n = kv_lens.numel()
    _int_vector(kv_lens, "kv_lens")
    _int_vector(free_blocks, "free_blocks")
    _int_vector(free_count, "free_count", 1)
    cols, stride = _tables(block_tables, n)
    _check_block_size(block_size)
    if rows is not None:
        _int_vector(rows, "rows")
    num_blocks = free_blocks.numel() if num_blocks is None else int(num_blocks)
    if num_blocks < 0:
        raise ValueError(f"num_blocks must not be negative, got {num_blocks}")
    dev = _device(dict(kv_lens=kv_lens, block_tables=block_tables, free_blocks=free_blocks, free_count=free_count, rows=rows))
    status = _lib.status_word(kv_lens.device)
    with torch.cuda.device(dev):
        rc = _lib.lib().fdms_paged_release_pool(
            _lib.ptr(rows) if rows is not None and rows.numel() else None, n if rows is None else rows.numel(), kv_lens.data_ptr(), n,
            block_tables.data_ptr(), stride, cols, block_size, free_blocks.data_ptr(), free_blocks.numel(), num_blocks,
            free_count.data_ptr(), status.data_ptr(), _lib.stream_ptr(kv_lens.device))
    _lib.check(rc)


def store_paged_kvcache(
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    slot_mapping: torch.Tensor,
) -> None:
    """Quantises `key` / `value [tokens, kv_heads, head_dim]` into the rows `slot_mapping` names (int32 `[tokens]`; negative:
    the token is skipped), in one launch.

    For each block and head that the step writes to, the scale becomes the smallest power of two 2^k with
    |x| <= 448 * 2^k for the rows written, k held in [-60, 40]; where the block holds earlier rows (rows before the first
    one written) it does not fall, and if it grows their codes move to the new scale.  Codes are rounded once, to nearest
    even; values beyond 448 * 2^40 are held at it, a NaN stays one and does not count for the scale.  Rows behind the last
    one written are left as they were.

    The tokens of a block are consecutive, as `build_paged_metadata` lays them out, without skipped ones between them, and no
    block is written by two sequences.  A slot beyond the cache, or in the block of the nearest earlier token that is not
    skipped without following it directly, is skipped and raises the device status bit for bad indices."""
    blocks, heads, block_size, head_dim = _cache_shape(k_cache, v_cache, k_scale, v_scale)
    shape = key.shape
    if len(shape) != 3 or value.shape != shape:
        raise ValueError(f"expected key and value as [tokens, kv_heads, head_dim], got {tuple(shape)} / {tuple(value.shape)}")
    if shape[1] != heads or shape[2] != head_dim:
        raise ValueError(f"expected key as [tokens, {heads}, {head_dim}], got {tuple(shape)}")
    if key.dtype is not value.dtype:
        raise ValueError("key and value must share a dtype")
    dtype = _row_dtype(key, "key")
    _int_vector(slot_mapping, "slot_mapping", shape[0])
    dev = k_cache.get_device()
    if (dev < 0 or key.get_device() != dev or value.get_device() != dev or v_cache.get_device() != dev or k_scale.get_device() != dev
            or v_scale.get_device() != dev or slot_mapping.get_device() != dev):
        _device(dict(k_cache=k_cache, key=key, value=value, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, slot_mapping=slot_mapping))
    _launch(_lib.lib().fdms_paged_store, _STORE_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, heads, block_size, head_dim,
        *k_cache.stride(), *v_cache.stride(), key.data_ptr(), value.data_ptr(), slot_mapping.data_ptr(),
        _lib.status_word(k_cache.device).data_ptr(), shape[0], dtype, *key.stride(), *value.stride()), dev)


def _attention(decode, q, k_cache, v_cache, k_scale, v_scale, block_tables, kv_lens, cu_seqlens_q, scale, out, lse_out, lse_shape):
    """Both attentions."""
    blocks, heads, block_size, head_dim = _cache_shape(k_cache, v_cache, k_scale, v_scale)
    shape = q.shape
    if shape[2] != head_dim:
        raise ValueError(f"cache head_dim {head_dim} does not match q head_dim {shape[2]}")
    tokens, num_q_heads = shape[0], shape[1]
    if num_q_heads == 0 or heads == 0 or num_q_heads % heads != 0 or num_q_heads // heads > 64:
        raise ValueError(f"q_heads={num_q_heads} must be kv_heads={heads} times 1 to 64")
    dtype = _row_dtype(q, "q")
    _int_vector(kv_lens, "kv_lens")
    seqs = kv_lens.numel()
    cols, stride = _tables(block_tables, seqs)
    dev = q.get_device()
    if (dev < 0 or k_cache.get_device() != dev or v_cache.get_device() != dev or k_scale.get_device() != dev or v_scale.get_device() != dev
            or block_tables.get_device() != dev or kv_lens.get_device() != dev or (cu_seqlens_q is not None and cu_seqlens_q.get_device() != dev)):
        _device(dict(q=q, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_tables=block_tables, kv_lens=kv_lens,
                     cu_seqlens_q=cu_seqlens_q))
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype is not q.dtype:
        raise ValueError("out must have q's shape and dtype")
    elif out.get_device() != dev:
        _device(dict(q=q, out=out))
    lse_ptr, lse_stride = 0, (0, 0)
    if lse_out is not None:
        if lse_out.shape != lse_shape or lse_out.dtype is not _F32:
            raise ValueError(f"expected float32 lse_out {tuple(lse_shape)}, got {tuple(lse_out.shape)} {lse_out.dtype}")
        if lse_out.get_device() != dev:
            _device(dict(q=q, lse_out=lse_out))
        lse_ptr, lse_stride = lse_out.data_ptr(), lse_out.stride()
    lib, need, ws = _lib.lib(), 0, None
    if decode:
        need = _on_device(dev, lib.fdms_paged_attn_decode_workspace_bytes, seqs, num_q_heads, heads, head_dim, cols * block_size)
    else:
        need = _on_device(dev, lib.fdms_paged_attn_prefill_workspace_bytes, tokens, seqs, num_q_heads, heads, head_dim, cols * block_size)
    if need > 0:
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    _launch(lib.fdms_paged_attn_decode if decode else lib.fdms_paged_attn_prefill, _ATTN_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, heads, block_size, head_dim,
        *k_cache.stride(), *v_cache.stride(), q.data_ptr(), out.data_ptr(), lse_ptr, block_tables.data_ptr(), kv_lens.data_ptr(),
        0 if cu_seqlens_q is None else cu_seqlens_q.data_ptr(), 0 if ws is None else ws.data_ptr(), _lib.status_word(q.device).data_ptr(),
        tokens, seqs, num_q_heads, dtype, cols, stride, need, *q.stride(), *out.stride(), *lse_stride,
        head_dim ** -0.5 if scale is None else scale), dev)
    return out


def paged_decode_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    scale: float | None = None,
    *,
    cu_seqlens_q: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    lse_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of one token per sequence: `q [batch, q_heads, head_dim]` (post-RoPE) over the first `kv_lens[b]` rows of
    each sequence, the token's own row among them; q head h reads KV head h // (q_heads // kv_heads).  bfloat16 or float16
    queries, head_dim 64 or 128, at most 2048 sequences.  `scale` defaults to head_dim ** -0.5.  A sequence without rows gets
    zeros.  `lse_out` (float32 `[batch, q_heads]`) receives the natural-log log-sum-exp of the scaled scores.  Table
    entries that are needed and name no block of the cache are left out and raise the device status bit for bad indices.

    Without `cu_seqlens_q` row b of q is sequence b's token: every sequence has exactly one in the step.  A step in which some
    sequences have none (`new_lens` of 0: released, or waiting) passes the `cu_seqlens` of `build_paged_metadata` (int32
    `[sequences + 1]`): q, out and `lse_out` are then `[tokens, ...]`, no more tokens than sequences, and sequence b's token is
    row `cu_seqlens_q[b]`.  A sequence without a token takes no part; one with several neither, and raises the device status bit
    for bad indices.  Rows that are no sequence's token (a padded step) are left as they were in `out` and `lse_out`."""
    shape = q.shape
    if len(shape) != 3:
        raise ValueError(f"expected q as [batch, q_heads, head_dim], got {tuple(shape)}")
    batch = kv_lens.numel()
    if cu_seqlens_q is not None:
        _int_vector(cu_seqlens_q, "cu_seqlens_q", batch + 1)
        if shape[0] > batch:
            raise ValueError(f"expected at most {batch} tokens, one per sequence, got {shape[0]}")
    elif batch != shape[0]:
        raise ValueError(f"expected kv_lens as contiguous int32 [{shape[0]}], got {tuple(kv_lens.shape)} {kv_lens.dtype}")
    if batch > MAX_DECODE_BATCH:
        raise RuntimeError(f"at most {MAX_DECODE_BATCH} sequences a call, got {batch}")
    return _attention(True, q, k_cache, v_cache, k_scale, v_scale, block_tables, kv_lens, cu_seqlens_q, scale, out, lse_out, shape[:2])


def paged_prefill_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    scale: float | None = None,
    *,
    out: torch.Tensor | None = None,
    lse_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of a step's tokens `q [tokens, q_heads, head_dim]` (post-RoPE, sequence i's being
    `cu_seqlens_q[i] : cu_seqlens_q[i + 1]`, int32 `[sequences + 1]`) over the cached rows of their sequences, the step's own
    rows stored before the call: with n tokens of a sequence in the step, token i sees its rows 0 .. kv_lens - n + i.  A
    token that sees none gets zeros and a log-sum-exp of -inf.  Tokens behind the last sequence are left as they were in
    `out` and `lse_out` (float32 `[q_heads, tokens]`).  Types, head sizes and table entries as in `paged_decode_attention`."""
    shape = q.shape
    if len(shape) != 3:
        raise ValueError(f"expected q as [tokens, q_heads, head_dim], got {tuple(shape)}")
    _int_vector(cu_seqlens_q, "cu_seqlens_q", kv_lens.numel() + 1)
    return _attention(False, q, k_cache, v_cache, k_scale, v_scale, block_tables, kv_lens, cu_seqlens_q, scale, out, lse_out, (shape[1], shape[0]))
