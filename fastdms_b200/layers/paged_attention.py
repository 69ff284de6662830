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
                paged_prefill_attention(q, ..., cu_seqlens)   or, one token per sequence, paged_decode_attention(q, ...)
    release_paged_blocks(...)   for sequences that ended

Every call enqueues on the current stream of its tensors' device and can be captured into a CUDA graph.  There is no CPU
path: tensors must live on a CUDA device.
"""
from __future__ import annotations

import torch

from fastdms_b200 import _lib

BLOCK_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
MAX_DECODE_BATCH = 2048
MAX_RELEASE_ROWS = 4096


def _same_device(dev: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"expected {name} on {dev}, got {t.device}")


def _int_vector(t: torch.Tensor, name: str, size: int | None = None) -> None:
    if t.dtype != torch.int32 or t.ndim != 1 or not t.is_contiguous() or (size is not None and t.numel() != size):
        shape = "[n]" if size is None else f"[{size}]"
        raise ValueError(f"expected {name} as contiguous int32 {shape}, got {tuple(t.shape)} {t.dtype}")


def _check_tables(block_tables: torch.Tensor, rows: int) -> None:
    if block_tables.ndim != 2 or block_tables.shape[0] != rows or block_tables.dtype != torch.int32:
        raise ValueError(f"expected block_tables as int32 [{rows}, columns], got {tuple(block_tables.shape)} {block_tables.dtype}")
    if block_tables.shape[1] > 1 and block_tables.stride(1) != 1:
        raise ValueError("block_tables must be contiguous in its last dimension")


def _check_block_size(block_size: int) -> None:
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")


def _row_stride(t: torch.Tensor) -> int:
    """Stride of a 2-d tensor's rows, which a tensor of one row (or none) may carry any value for."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_cache(k_cache, v_cache, k_scale, v_scale) -> None:
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"expected k_cache and v_cache as [blocks, kv_heads, block_size, head_dim], got {tuple(k_cache.shape)} / {tuple(v_cache.shape)}")
    if k_cache.dtype != torch.float8_e4m3fn or v_cache.dtype != torch.float8_e4m3fn:
        raise ValueError(f"expected float8_e4m3fn caches, got {k_cache.dtype} / {v_cache.dtype}")
    blocks, heads, block_size, head_dim = k_cache.shape
    _check_block_size(block_size)
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.stride(3) != 1 or any(c.stride(i) % 16 for i in range(3)) or c.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous in its last dimension and aligned to 16 bytes in the others")
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s.shape != (blocks, heads) or s.dtype != torch.float32 or not s.is_contiguous():
            raise ValueError(f"expected {name} as contiguous float32 {(blocks, heads)}, got {tuple(s.shape)} {s.dtype}")


def _check_rows(t: torch.Tensor, name: str) -> None:
    """16-bit rows that the kernels read and write 16 bytes at a time."""
    if t.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    if t.numel() and (t.stride(2) != 1 or t.stride(0) * 2 % 16 or t.stride(1) * 2 % 16 or t.data_ptr() % 16):
        raise ValueError(f"{name} must be contiguous in its last dimension and aligned to 16 bytes in the others")


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

    `kv_lens` and `free_count` are advanced in place, or left alone where `kv_lens_out` / `free_count_out` are given.
    Returns `cu_seqlens` (int32 `[n + 1]`), `slot_mapping` (int32 `[total_tokens]`, block * block_size + row) and
    `positions` (int64 `[total_tokens]`); buffers given for them are filled.  `total_tokens` may exceed the sum of `new_lens`
    (a padded batch): the slots behind it are -1, which the store skips, and the positions 0.  Each sequence has a row of its
    own; free block ids are distinct."""
    n = kv_lens.numel()
    _int_vector(kv_lens, "kv_lens")
    _int_vector(new_lens, "new_lens", n)
    _int_vector(free_blocks, "free_blocks")
    _int_vector(free_count, "free_count", 1)
    _check_tables(block_tables, n)
    _check_block_size(block_size)
    total_tokens = int(total_tokens)
    if total_tokens < 0:
        raise ValueError(f"total_tokens must not be negative, got {total_tokens}")
    _lib.require_cuda(new_lens, kv_lens, block_tables, free_blocks, free_count)
    dev = kv_lens.device
    kv_lens_out = kv_lens if kv_lens_out is None else kv_lens_out
    free_count_out = free_count if free_count_out is None else free_count_out
    _int_vector(kv_lens_out, "kv_lens_out", n)
    _int_vector(free_count_out, "free_count_out", 1)
    if cu_seqlens is None:
        cu_seqlens = torch.empty(n + 1, dtype=torch.int32, device=dev)
    _int_vector(cu_seqlens, "cu_seqlens", n + 1)
    if slot_mapping is None:
        slot_mapping = torch.empty(total_tokens, dtype=torch.int32, device=dev)
    _int_vector(slot_mapping, "slot_mapping", total_tokens)
    if positions is None:
        positions = torch.empty(total_tokens, dtype=torch.int64, device=dev)
    if positions.dtype != torch.int64 or positions.shape != (total_tokens,) or not positions.is_contiguous():
        raise ValueError(f"expected positions as contiguous int64 [{total_tokens}], got {tuple(positions.shape)} {positions.dtype}")
    _same_device(dev, new_lens=new_lens, block_tables=block_tables, free_blocks=free_blocks, free_count=free_count, kv_lens_out=kv_lens_out,
                 free_count_out=free_count_out, cu_seqlens=cu_seqlens, slot_mapping=slot_mapping, positions=positions)
    status = _lib.status_word(dev)
    ws = torch.empty(_lib.lib().fdms_paged_metadata_workspace_bytes(n), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.lib().fdms_paged_metadata(
            new_lens.data_ptr(), kv_lens.data_ptr(), kv_lens_out.data_ptr(), block_tables.data_ptr(), _row_stride(block_tables),
            block_tables.shape[1], block_size, free_blocks.data_ptr(), free_blocks.numel(), free_count.data_ptr(), free_count_out.data_ptr(),
            cu_seqlens.data_ptr(), slot_mapping.data_ptr(), positions.data_ptr(), total_tokens, n, ws.data_ptr(), ws.numel(),
            status.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc)
    return cu_seqlens, slot_mapping, positions


def release_paged_blocks(
    kv_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_blocks: torch.Tensor,
    free_count: torch.Tensor,
    *,
    block_size: int,
    rows: torch.Tensor | None = None,
) -> None:
    """Gives the blocks of the listed rows (int32 indices of `kv_lens` and `block_tables`; all rows without a list) back to
    the stack and empties the rows: table entries -1, length 0.  A row that is listed twice is released once and, like one
    out of range or a block id outside the pool, raises the device status bit for bad indices."""
    n = kv_lens.numel()
    _int_vector(kv_lens, "kv_lens")
    _int_vector(free_blocks, "free_blocks")
    _int_vector(free_count, "free_count", 1)
    _check_tables(block_tables, n)
    _check_block_size(block_size)
    if rows is not None:
        _int_vector(rows, "rows")
    _lib.require_cuda(kv_lens, block_tables, free_blocks, free_count, rows)
    dev = kv_lens.device
    _same_device(dev, block_tables=block_tables, free_blocks=free_blocks, free_count=free_count, rows=rows)
    status = _lib.status_word(dev)
    with torch.cuda.device(dev):
        rc = _lib.lib().fdms_paged_release(
            _lib.ptr(rows) if rows is not None and rows.numel() else None, n if rows is None else rows.numel(), kv_lens.data_ptr(), n,
            block_tables.data_ptr(), _row_stride(block_tables), block_tables.shape[1], block_size, free_blocks.data_ptr(),
            free_blocks.numel(), free_count.data_ptr(), status.data_ptr(), _lib.stream_ptr(dev))
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

    A sequence's tokens are consecutive, as `build_paged_metadata` lays them out, and no block is written by two sequences.
    A slot beyond the cache, or next to a token of its own block that it does not follow, is skipped and raises the device
    status bit for bad indices."""
    if key.ndim != 3 or key.shape != value.shape:
        raise ValueError(f"expected key and value as [tokens, kv_heads, head_dim], got {tuple(key.shape)} / {tuple(value.shape)}")
    if key.dtype != value.dtype:
        raise ValueError("key and value must share a dtype")
    _check_cache(k_cache, v_cache, k_scale, v_scale)
    blocks, heads, block_size, head_dim = k_cache.shape
    tokens = key.shape[0]
    if key.shape[1:] != (heads, head_dim):
        raise ValueError(f"expected key as [tokens, {heads}, {head_dim}], got {tuple(key.shape)}")
    _check_rows(key, "key")
    _check_rows(value, "value")
    _int_vector(slot_mapping, "slot_mapping", tokens)
    _lib.require_cuda(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    dev = k_cache.device
    _same_device(dev, key=key, value=value, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, slot_mapping=slot_mapping)
    status = _lib.status_word(dev)
    with torch.cuda.device(dev):
        rc = _lib.lib().fdms_paged_store(
            key.data_ptr(), value.data_ptr(), _lib.dtype_code(key.dtype), key.stride(0), key.stride(1), value.stride(0), value.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            v_cache.stride(0), v_cache.stride(1), v_cache.stride(2), k_scale.data_ptr(), v_scale.data_ptr(), slot_mapping.data_ptr(),
            tokens, blocks, block_size, heads, head_dim, status.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc)


def _check_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables, kv_lens, out, lse_out, lse_shape) -> torch.device:
    if q.ndim != 3:
        raise ValueError(f"expected q as [tokens, q_heads, head_dim], got {tuple(q.shape)}")
    _check_cache(k_cache, v_cache, k_scale, v_scale)
    heads, head_dim = k_cache.shape[1], k_cache.shape[3]
    if q.shape[2] != head_dim:
        raise ValueError(f"cache head_dim {head_dim} does not match q head_dim {q.shape[2]}")
    if q.shape[1] == 0 or heads == 0 or q.shape[1] % heads != 0 or q.shape[1] // heads > 64:
        raise ValueError(f"q_heads={q.shape[1]} must be kv_heads={heads} times 1 to 64")
    _check_rows(q, "q")
    _int_vector(kv_lens, "kv_lens")
    _check_tables(block_tables, kv_lens.numel())
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have q's shape and dtype")
    _check_rows(out, "out")
    if lse_out is not None and (lse_out.shape != lse_shape or lse_out.dtype != torch.float32):
        raise ValueError(f"expected float32 lse_out {tuple(lse_shape)}, got {tuple(lse_out.shape)} {lse_out.dtype}")
    _lib.require_cuda(q, k_cache, v_cache, k_scale, v_scale, block_tables, kv_lens, out, lse_out)
    _same_device(q.device, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_tables=block_tables, kv_lens=kv_lens,
                 out=out, lse_out=lse_out)
    return q.device


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
    out: torch.Tensor | None = None,
    lse_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of one token per sequence: `q [batch, q_heads, head_dim]` (post-RoPE) over the first `kv_lens[b]` rows of
    each sequence, the token's own row among them; q head h reads KV head h // (q_heads // kv_heads).  bfloat16 or float16
    queries, head_dim 64 or 128, at most 2048 sequences.  `scale` defaults to head_dim ** -0.5.  A sequence without rows gets
    zeros.  `lse_out` (float32 `[batch, q_heads]`) receives the natural-log log-sum-exp of the scaled scores.  Table
    entries that are needed and name no block of the cache are left out and raise the device status bit for bad indices."""
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dev = _check_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables, kv_lens, out, lse_out, q.shape[:2])
    batch, num_q_heads, head_dim = q.shape
    if kv_lens.numel() != batch:
        raise ValueError(f"expected kv_lens [{batch}], got {tuple(kv_lens.shape)}")
    if batch > MAX_DECODE_BATCH:
        raise RuntimeError(f"at most {MAX_DECODE_BATCH} sequences a call, got {batch}")
    if batch == 0:
        return out
    blocks, heads, block_size, _ = k_cache.shape
    status = _lib.status_word(dev)
    with torch.cuda.device(dev):
        need = _lib.lib().fdms_paged_attn_decode_workspace_bytes(batch, num_q_heads, heads, head_dim)
        ws = torch.empty(max(need, 0), dtype=torch.uint8, device=dev)
        rc = _lib.lib().fdms_paged_attn_decode(
            q.data_ptr(), _lib.dtype_code(q.dtype), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2),
            k_scale.data_ptr(), v_scale.data_ptr(), blocks, block_size, block_tables.data_ptr(), _row_stride(block_tables),
            block_tables.shape[1], kv_lens.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), _lib.ptr(lse_out),
            lse_out.stride(0) if lse_out is not None else 0, lse_out.stride(1) if lse_out is not None else 0,
            batch, num_q_heads, heads, head_dim, float(head_dim ** -0.5 if scale is None else scale), ws.data_ptr(), ws.numel(),
            status.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc)
    return out


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
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dev = _check_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables, kv_lens, out, lse_out, (q.shape[1], q.shape[0]))
    tokens, num_q_heads, head_dim = q.shape
    seqs = kv_lens.numel()
    _int_vector(cu_seqlens_q, "cu_seqlens_q", seqs + 1)
    _lib.require_cuda(cu_seqlens_q)
    _same_device(dev, cu_seqlens_q=cu_seqlens_q)
    if tokens == 0 or seqs == 0:
        return out
    blocks, heads, block_size, _ = k_cache.shape
    status = _lib.status_word(dev)
    with torch.cuda.device(dev):
        rc = _lib.lib().fdms_paged_attn_prefill(
            q.data_ptr(), _lib.dtype_code(q.dtype), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2),
            k_scale.data_ptr(), v_scale.data_ptr(), blocks, block_size, block_tables.data_ptr(), _row_stride(block_tables),
            block_tables.shape[1], kv_lens.data_ptr(), cu_seqlens_q.data_ptr(), tokens, out.data_ptr(), out.stride(0), out.stride(1),
            _lib.ptr(lse_out), lse_out.stride(0) if lse_out is not None else 0, lse_out.stride(1) if lse_out is not None else 0,
            seqs, num_q_heads, heads, head_dim, float(head_dim ** -0.5 if scale is None else scale), status.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc)
    return out
