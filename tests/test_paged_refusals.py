"""What the paged cache's calls refuse, on the CPU: nothing here launches a kernel."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_oracle as O
from fastdms_b200 import _lib
from fastdms_b200.layers import paged_attention as P


def cache(blocks=4, heads=2, bs=16, d=64):
    c = torch.zeros((blocks, heads, bs, d), dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones((blocks, heads))
    return [c, c.view(torch.uint8).clone().view(torch.float8_e4m3fn), s, s.clone()]


def ints(*a):
    return torch.tensor(a, dtype=torch.int32)


def test_calls_need_cuda():
    q, kv, table = torch.zeros((1, 4, 64), dtype=torch.bfloat16), ints(3), torch.zeros((1, 2), dtype=torch.int32)
    k = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.paged_decode_attention(q, *cache(), table, kv)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.paged_prefill_attention(q, *cache(), table, kv, ints(0, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        P.store_paged_kvcache(k, k, *cache(), ints(0))
    with pytest.raises(RuntimeError, match="CUDA"):
        P.build_paged_metadata(ints(1), kv, table, ints(0), ints(1), block_size=16, total_tokens=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.release_paged_blocks(kv, table, ints(0), ints(1), block_size=16)


def _bad(**change):
    a = dict(q=torch.zeros((2, 4, 64), dtype=torch.bfloat16), table=torch.zeros((2, 2), dtype=torch.int32), kv=ints(3, 4), cache=cache())
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros((2, 4, 64))), "bfloat16 or float16"),
    (dict(q=torch.zeros((2, 3, 64), dtype=torch.float16)), "times 1 to 64"),
    (dict(q=torch.zeros((2, 130, 64), dtype=torch.float16)), "times 1 to 64"),
    (dict(q=torch.zeros((2, 0, 64), dtype=torch.float16)), "times 1 to 64"),
    (dict(q=torch.zeros((2, 4, 128), dtype=torch.float16)), "head_dim"),
    (dict(q=torch.zeros((2, 4, 66), dtype=torch.float16)[:, :, 1:65]), "aligned"),
    (dict(q=torch.zeros((2, 64), dtype=torch.float16)), "tokens, q_heads"),
    (dict(kv=torch.tensor([3, 4])), "int32"),
    (dict(kv=ints(3, 0, 4)[::2]), "contiguous"),
    (dict(table=torch.zeros((2, 2))), "int32"),
    (dict(table=torch.zeros((3, 2), dtype=torch.int32)), r"\[2, columns\]"),
    (dict(table=torch.zeros((2, 4), dtype=torch.int32)[:, ::2]), "last dimension"),
    (dict(cache=cache(bs=24)), "block_size"),
    (dict(cache=cache(d=80)), "head_dim"),
    (dict(cache=[c.view(torch.uint8) if c.element_size() == 1 else c for c in cache()]), "float8"),
    (dict(cache=cache()[:3] + [torch.ones((4, 3))]), "v_scale"),
    (dict(cache=cache()[:2] + [torch.ones((2, 4)).t()] + cache()[3:]), "k_scale"),
    (dict(cache=[cache(heads=1)[0]] + cache()[1:]), "kv_heads, block_size"),
])
def test_attention_refuses(change, match):
    a = _bad(**change)
    with pytest.raises(ValueError, match=match):
        P.paged_decode_attention(a["q"], *a["cache"], a["table"], a["kv"])
    with pytest.raises(ValueError, match=match):
        P.paged_prefill_attention(a["q"], *a["cache"], a["table"], a["kv"], ints(0, 1, 2))


def test_attention_refuses_outputs_and_lengths():
    a = _bad()
    args = (a["q"], *a["cache"], a["table"], a["kv"])
    with pytest.raises(ValueError, match="out must"):
        P.paged_decode_attention(*args, out=torch.zeros((2, 4, 64)))
    with pytest.raises(ValueError, match="lse_out"):
        P.paged_decode_attention(*args, lse_out=torch.zeros((4, 2)))
    with pytest.raises(ValueError, match="lse_out"):
        P.paged_prefill_attention(*args, ints(0, 1, 2), lse_out=torch.zeros((2, 4)))
    with pytest.raises(ValueError, match="aligned"):
        P.paged_decode_attention(*args, out=torch.zeros((2, 4, 128), dtype=torch.bfloat16)[:, :, ::2])


def test_store_refuses():
    k = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    for bad, match in [((k, k[:2]), "key and value"), ((k, k.half()), "dtype"), ((k.float(), k.float()), "bfloat16 or float16"),
                       ((k[:, :1], k[:, :1]), "expected key"), ((k[0], k[0]), "key and value")]:
        with pytest.raises(ValueError, match=match):
            P.store_paged_kvcache(*bad, *cache(), ints(0, 1, 2))
    with pytest.raises(ValueError, match="slot_mapping"):
        P.store_paged_kvcache(k, k, *cache(), ints(0, 1))
    with pytest.raises(ValueError, match="slot_mapping"):
        P.store_paged_kvcache(k, k, *cache(), torch.tensor([0, 1, 2]))


def test_tables_refuse():
    kv, table, free, count = ints(1, 2), torch.zeros((2, 4), dtype=torch.int32), ints(0, 1), ints(2)
    ok = dict(block_size=16, total_tokens=3)
    for args, kw, match in [((ints(1), kv, table, free, count), ok, "new_lens"), ((kv, kv, table[:1], free, count), ok, "block_tables"),
                            ((kv, kv, table, free.long(), count), ok, "free_blocks"), ((kv, kv, table, free, ints(1, 2)), ok, "free_count"),
                            ((kv, kv, table, free, count), dict(block_size=8, total_tokens=3), "block_size"),
                            ((kv, kv, table, free, count), dict(block_size=16, total_tokens=-1), "total_tokens")]:
        with pytest.raises(ValueError, match=match):
            P.build_paged_metadata(*args, **kw)
    with pytest.raises(ValueError, match="rows"):
        P.release_paged_blocks(kv, table, free, count, block_size=16, rows=torch.tensor([0]))


def test_c_entries_refuse_without_a_gpu():
    lib = _lib.lib()
    p = 1 << 12
    meta = [p, p, p, p, 4, 4, 16, p, 8, p, p, p, p, p, 4, 2, None, 0, None, None]

    def refused(fn, args, change, code, words):
        a = list(args)
        for i, x in change.items():
            a[i] = x
        assert fn(*a) == code and words in lib.fdms_last_error(), lib.fdms_last_error()

    refused(lib.fdms_paged_metadata, meta, {0: None}, _lib.FDMS_E_ARG, b"null pointer")
    refused(lib.fdms_paged_metadata, meta, {6: 17}, _lib.FDMS_E_ARG, b"block_size")
    refused(lib.fdms_paged_metadata, meta, {4: 3}, _lib.FDMS_E_ARG, b"overlap")
    refused(lib.fdms_paged_metadata, meta, {12: p + 4}, _lib.FDMS_E_ARG, b"aligned")
    refused(lib.fdms_paged_metadata, meta, {14: 1 << 31}, _lib.FDMS_E_CAPACITY, b"31 bits")
    refused(lib.fdms_paged_metadata, meta, {14: 1 << 20}, _lib.FDMS_E_WORKSPACE, b"workspace")
    assert lib.fdms_paged_metadata_workspace_bytes(-1) < 0
    rel = [p, 2, p, 2, p, 4, 4, 16, p, 8, p, None, None]
    refused(lib.fdms_paged_release, rel, {1: 5000}, _lib.FDMS_E_CAPACITY, b"rows a call")
    refused(lib.fdms_paged_release, rel, {0: None, 1: 3}, _lib.FDMS_E_ARG, b"more rows")
    st = [p, p, 1, 128, 64, 128, 64, p, p, 2048, 1024, 64, 2048, 1024, 64, p, p, p, 2, 4, 16, 2, 64, None, None]
    refused(lib.fdms_paged_store, st, {2: 0}, _lib.FDMS_E_DTYPE, b"bf16 or f16")
    refused(lib.fdms_paged_store, st, {22: 96}, _lib.FDMS_E_ARG, b"head_dim")
    refused(lib.fdms_paged_store, st, {3: 129}, _lib.FDMS_E_ARG, b"aligned")
    refused(lib.fdms_paged_store, st, {11: 8}, _lib.FDMS_E_ARG, b"aligned")
    refused(lib.fdms_paged_store, st, {19: 1 << 28}, _lib.FDMS_E_CAPACITY, b"31 bits")
    dec = [p, 1, 256, 64, p, p, 2048, 1024, 64, 2048, 1024, 64, p, p, 4, 16, p, 4, 4, p, p, 256, 64, None, 0, 0, 2, 4, 2, 64, 0.1, p, 1 << 30, None, None]
    refused(lib.fdms_paged_attn_decode, dec, {1: 0}, _lib.FDMS_E_DTYPE, b"bf16 or f16")
    refused(lib.fdms_paged_attn_decode, dec, {27: 5}, _lib.FDMS_E_ARG, b"times 1 to 64")
    refused(lib.fdms_paged_attn_decode, dec, {31: None}, _lib.FDMS_E_ARG, b"null pointer")
    refused(lib.fdms_paged_attn_decode, dec, {26: 2049}, _lib.FDMS_E_CAPACITY, b"2048")
    refused(lib.fdms_paged_attn_decode, dec, {20: p + 2}, _lib.FDMS_E_ARG, b"aligned")
    pre = [p, 1, 256, 64, p, p, 2048, 1024, 64, 2048, 1024, 64, p, p, 4, 16, p, 4, 4, p, p, 9, p, 256, 64, None, 0, 0, 2, 4, 2, 64, 0.1, None, None]
    refused(lib.fdms_paged_attn_prefill, pre, {15: 20}, _lib.FDMS_E_ARG, b"block_size")
    refused(lib.fdms_paged_attn_prefill, pre, {21: -1}, _lib.FDMS_E_ARG, b"negative")
    refused(lib.fdms_paged_attn_prefill, pre, {20: None}, _lib.FDMS_E_ARG, b"null pointer")
    refused(lib.fdms_paged_attn_prefill, pre, {7: 1000}, _lib.FDMS_E_ARG, b"aligned")
    rel[1] = 0
    assert lib.fdms_paged_release(*rel) == _lib.FDMS_OK and lib.fdms_last_error() == b""


def test_plain_statement():
    """The oracle's codes are torch's: every value that is one, values around every border, ties."""
    v = O.VALUES[np.isfinite(O.VALUES)]
    mid = (np.sort(v)[1:] + np.sort(v)[:-1]) / 2
    x = np.concatenate([v, mid, np.nextafter(mid, 1e9), np.nextafter(mid, -1e9), [1e-9, -1e-9, 1000.0, -1e30]])
    x = torch.from_numpy(x).float().clamp(-448, 448)
    assert np.array_equal(O.encode(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert O.scale_of(448.0) == 1.0 and O.scale_of(448.1) == 2.0 and O.scale_of(224.0) == 0.5 and O.scale_of(0.0) == 2.0 ** -60 and O.scale_of(1e30) == 2.0 ** 40
