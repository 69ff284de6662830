"""A Llama-style model served from the dense paged cache through `Attention`'s own branch: prompts in chunks, decode steps,
sequences that end and make room.  What every layer gets and gives is checked: the cache's codes and scales exactly, the
attention within the bound of its roundings."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

import paged_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qk_norm,bs", [(False, 16), (True, 32)])
def test_model_on_the_paged_cache(qk_norm, bs):
    from fastdms_b200 import _lib
    from fastdms_b200.layers.paged_attention import build_paged_metadata, release_paged_blocks
    from fastdms_b200.models.registry import build_model
    from fastdms_b200.utils.context import reset_context, set_context
    dev = torch.device("cuda:0")
    _lib.read_device_status(dev)
    cfg = SimpleNamespace(model_type="qwen3" if qk_norm else "llama", hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                          intermediate_size=512, num_hidden_layers=2, vocab_size=512, rms_norm_eps=1e-6, max_position_embeddings=1024,
                          rope_theta=10000.0, hidden_act="silu", tie_word_embeddings=False)
    was = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(dev):
            model = build_model(cfg)
    finally:
        torch.set_default_dtype(was)
    model.to(dev).eval()
    g = torch.Generator(device=dev).manual_seed(3)
    for p in model.parameters():
        p.requires_grad_(False)
        if p.ndim > 1:
            p.data.copy_(torch.randn(p.shape, device=dev, generator=g) * p.shape[-1] ** -0.5)
    seqs, pool, cols = 3, 40, 12
    host, seen = [], []
    for layer in model.attention_modules():
        layer.k_cache, layer.v_cache = (torch.full((pool, 2, bs, 64), 0x7F, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
        layer.k_cache_scale, layer.v_cache_scale = (torch.full((pool, 2), float("nan"), device=dev) for _ in range(2))
        host.append([np.full((pool, 2, bs, 64), 0x7F, np.uint8), np.full((pool, 2, bs, 64), 0x7F, np.uint8), np.full((pool, 2), np.nan),
                     np.full((pool, 2), np.nan)])
        layer.register_forward_hook(lambda m, a, out: seen.append((m.layer_id, *(x.detach().cpu().double().numpy() for x in (*a, out)))))
    i32 = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32).to(dev)
    kv, count, table = i32([0] * seqs), i32([pool]), i32(np.full((seqs, cols), -1))
    free = torch.arange(pool, device=dev, dtype=torch.int32).flip(0).contiguous()
    rng = np.random.default_rng(4)

    @torch.inference_mode()
    def step(new, decode):
        ids = torch.as_tensor(rng.integers(0, 512, sum(new)), device=dev)
        cu, slots, pos = build_paged_metadata(i32(new), kv, table, free, count, block_size=bs, total_tokens=len(ids))
        set_context(not decode, cu_seqlens_q=cu, slot_mapping=slots, context_lens=kv, block_tables=table)
        try:
            logits = model.compute_logits(model(ids, pos))
        finally:
            reset_context()
        assert torch.isfinite(logits.float()).all()
        lens, tab, starts = kv.cpu().numpy(), table.cpu().numpy(), np.concatenate([[0], np.cumsum(new)])
        for layer_id, q, k, v, out in seen:
            codes_k, codes_v, scale_k, scale_v = host[layer_id]
            O.store(k, codes_k, scale_k, slots.cpu().tolist(), bs)
            O.store(v, codes_v, scale_v, slots.cpu().tolist(), bs)
            m = model.attention_modules()[layer_id]
            assert np.array_equal(m.k_cache.view(torch.uint8).cpu().numpy(), codes_k) and np.array_equal(m.v_cache.view(torch.uint8).cpu().numpy(), codes_v)
            assert np.array_equal(m.k_cache_scale.cpu().numpy(), scale_k, equal_nan=True) and np.array_equal(m.v_cache_scale.cpu().numpy(), scale_v, equal_nan=True)
            for s, n in enumerate(new):
                rows = slice(int(starts[s]), int(starts[s + 1]))
                for h in range(4):
                    kk, vv = (O.rows_of(c, f, tab[s], int(lens[s]), h // 2, bs) for c, f in ((codes_k, scale_k), (codes_v, scale_v)))
                    want, _, tol, _ = O.attention(q[rows, h], kk, vv, lens[s] - n + np.arange(n), 64 ** -0.5)
                    assert (np.abs(out[rows, h] - want) <= tol + 2.0 ** -8 * (np.abs(want) + tol)).all()
        assert len(seen) == 2
        seen.clear()

    step([30, 0, 9], decode=False)
    step([11, 21, 1], decode=False)
    for _ in range(3):
        step([1, 1, 1], decode=True)
    release_paged_blocks(kv, table, free, count, block_size=bs, rows=i32([0]))
    step([17, 0, 40], decode=False)
    step([1, 1, 1], decode=True)
    release_paged_blocks(kv, table, free, count, block_size=bs)
    assert sorted(free.tolist()) == list(range(pool)) and int(count) == pool
    assert _lib.read_device_status(dev) == 0


def test_paged_branch_says_what_is_missing():
    from fastdms_b200.layers.attention import Attention
    from fastdms_b200.utils.context import reset_context, set_context
    dev = torch.device("cuda:0")
    att = Attention(4, 64, 0.125, 2)
    q, k = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=dev), torch.zeros((1, 2, 64), dtype=torch.bfloat16, device=dev)
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    try:
        set_context(False, block_tables=table)
        with pytest.raises(RuntimeError, match="k_cache"):
            att(q, k, k)
        att.k_cache = att.v_cache = torch.zeros((1, 2, 16, 64), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        att.k_cache_scale = att.v_cache_scale = torch.ones((1, 2), device=dev)
        with pytest.raises(RuntimeError, match="slot_mapping"):
            att(q, k, k)
        reset_context()
        set_context(False)                       # without tables the branch is not taken
        with pytest.raises(RuntimeError, match="compact KV path"):
            att(q, k, k)
    finally:
        reset_context()
