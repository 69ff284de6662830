"""What the paged cache's calls refuse, on the CPU: nothing here launches a kernel."""
from __future__ import annotations

import re
from pathlib import Path

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
    (dict(q=torch.zeros((2, 64), dtype=torch.float16)), "q_heads, head_dim"),
    (dict(kv=torch.tensor([3, 4])), "int32"),
    (dict(kv=ints(3, 0, 4)[::2]), "contiguous"),
    (dict(table=torch.zeros((2, 2))), "int32"),
    (dict(table=torch.zeros((3, 2), dtype=torch.int32)), r"\[2, columns\]"),
    (dict(table=torch.zeros((2, 4), dtype=torch.int32)[:, ::2]), "last dimension"),
    (dict(cache=[c.view(torch.uint8) if c.element_size() == 1 else c for c in cache()]), "float8"),
    (dict(cache=cache(d=128)), "head_dim"),
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


PTR = 1 << 12
CACHE = dict(k=PTR, v=PTR, ks=PTR, vs=PTR, blocks=4, heads=2, bs=16, d=64, k0=2048, k1=1024, k2=64, k3=1, v0=2048, v1=1024, v2=64, v3=1)
METADATA = dict(new=PTR, kv=PTR, kv_out=PTR, bt=PTR, free=PTR, count=PTR, count_out=PTR, cu=PTR, slots=PTR, pos=PTR, ws=0, status=0, n=2, cols=4,
                stride=4, bs=16, capacity=8, total=4, ws_bytes=0)
STORE = dict(CACHE, key=PTR, value=PTR, slots=PTR, status=0, tokens=2, dtype=1, s0=128, s1=64, s2=1, t0=128, t1=64, t2=1)
ATTN = dict(CACHE, q=PTR, out=PTR, lse=0, bt=PTR, kv=PTR, cu=PTR, ws=PTR, status=0, tokens=2, seqs=2, hq=4, dtype=1, cols=4, stride=4, ws_bytes=1 << 30,
            q0=256, q1=64, q2=1, o0=256, o1=64, o2=1, l0=0, l1=0, scale=0.125)
E, T, C, W = _lib.FDMS_E_ARG, _lib.FDMS_E_DTYPE, _lib.FDMS_E_CAPACITY, _lib.FDMS_E_WORKSPACE


@pytest.mark.parametrize("change,code,words", [
    (dict(new=0), E, b"null pointer"), (dict(pos=0), E, b"null pointer"), (dict(bs=17), E, b"block_size"), (dict(stride=3), E, b"overlap"),
    (dict(n=-1), E, b"negative"), (dict(slots=PTR + 4), E, b"aligned"), (dict(total=1 << 31), C, b"31 bits"), (dict(capacity=1 << 28), C, b"31 bits"),
    (dict(total=1 << 20), W, b"workspace"), (dict(total=1 << 20, ws=PTR + 4, ws_bytes=99), W, b"workspace")])
def test_c_metadata_refuses(change, code, words):
    lib = _lib.lib()
    assert lib.fdms_paged_metadata(P._METADATA_ARGS.pack(*(METADATA | change).values()), None) == code and words in lib.fdms_last_error()
    assert lib.fdms_paged_metadata_workspace_bytes(-1, 4) < 0 and lib.fdms_paged_metadata_workspace_bytes(4, 4) == 0
    assert lib.fdms_paged_metadata(None, None) == E


BAD_CACHE = [(dict(dtype=0), T, b"bf16 or f16"), (dict(d=96), E, b"head_dim"), (dict(bs=24), E, b"block_size"), (dict(heads=0), E, b"no KV heads"),
             (dict(blocks=1 << 28), C, b"31 bits"), (dict(k=0), E, b"null pointer"), (dict(v=PTR + 8), E, b"aligned"), (dict(k2=72), E, b"aligned"),
             (dict(v3=2), E, b"contiguous")]


@pytest.mark.parametrize("change,code,words", BAD_CACHE + [
    (dict(tokens=-1), E, b"negative"), (dict(key=0), E, b"null pointer"), (dict(s0=129), E, b"aligned"), (dict(t2=2), E, b"contiguous"),
    (dict(value=PTR + 2), E, b"aligned")])
def test_c_store_refuses(change, code, words):
    lib = _lib.lib()
    assert lib.fdms_paged_store(P._STORE_ARGS.pack(*(STORE | change).values()), None) == code and words in lib.fdms_last_error()
    assert lib.fdms_paged_store(None, None) == E


BAD_ATTN = BAD_CACHE + [(dict(hq=5), E, b"times 1 to 64"), (dict(hq=130), E, b"times 1 to 64"), (dict(q=0), E, b"null pointer"), (dict(kv=0), E, b"null pointer"),
                        (dict(bt=0), E, b"null pointer"), (dict(out=PTR + 2), E, b"aligned"), (dict(q1=66), E, b"aligned"), (dict(o2=2), E, b"contiguous"),
                        (dict(cols=1 << 28), C, b"31 bits"), (dict(seqs=-1), E, b"negative")]


@pytest.mark.parametrize("change,code,words", BAD_ATTN + [
    (dict(tokens=3), E, b"one token per sequence"), (dict(tokens=2049, seqs=2049), C, b"2048")])
def test_c_decode_refuses(change, code, words):
    lib = _lib.lib()
    assert lib.fdms_paged_attn_decode(P._ATTN_ARGS.pack(*(ATTN | change).values()), None) == code and words in lib.fdms_last_error()
    assert lib.fdms_paged_attn_decode(None, None) == E
    assert lib.fdms_paged_attn_decode_workspace_bytes(2, 3, 2, 64, 64) < 0


@pytest.mark.parametrize("change,code,words", BAD_ATTN + [(dict(cu=0), E, b"null pointer"), (dict(tokens=-1), E, b"negative")])
def test_c_prefill_refuses(change, code, words):
    lib = _lib.lib()
    assert lib.fdms_paged_attn_prefill(P._ATTN_ARGS.pack(*(ATTN | change).values()), None) == code and words in lib.fdms_last_error()
    assert lib.fdms_paged_attn_prefill(None, None) == E


def test_c_release_refuses():
    lib = _lib.lib()
    rel = dict(rows=PTR, listed=2, kv=PTR, n=2, bt=PTR, stride=4, cols=4, bs=16, free=PTR, capacity=8, count=PTR, status=None, stream=None)
    for change, code, words in [(dict(listed=5000), C, b"rows a call"), (dict(rows=None, listed=3), E, b"more rows"), (dict(bs=8), E, b"block_size"),
                                (dict(count=None), E, b"null pointer"), (dict(stride=3), E, b"overlap")]:
        assert lib.fdms_paged_release(*(rel | change).values()) == code and words in lib.fdms_last_error()
    assert lib.fdms_paged_release(*(rel | dict(listed=0)).values()) == _lib.FDMS_OK and lib.fdms_last_error() == b""


def test_layer_refuses_incomplete_contexts():
    from fastdms_b200.layers.attention import Attention
    from fastdms_b200.utils.context import reset_context, set_context
    layer = Attention(4, 64, 0.125, 2)
    q, k = torch.zeros((3, 4, 64), dtype=torch.bfloat16), torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    step = dict(block_tables=torch.zeros((1, 2), dtype=torch.int32), slot_mapping=ints(0, 1, 2), context_lens=ints(3), cu_seqlens_q=ints(0, 3))
    try:
        set_context(True, **step)
        with pytest.raises(RuntimeError, match="k_cache"):
            layer(q, k, k)
        layer.k_cache, layer.v_cache, layer.k_cache_scale, layer.v_cache_scale = cache()
        for missing in ("slot_mapping", "context_lens", "cu_seqlens_q"):
            set_context(True, **(step | {missing: None}))
            with pytest.raises(RuntimeError, match=missing):
                layer(q, k, k)
    finally:
        reset_context()


def test_plain_statement():
    """The oracle's codes are torch's: every value that is one, values around every border, ties."""
    v = O.VALUES[np.isfinite(O.VALUES)]
    mid = (np.sort(v)[1:] + np.sort(v)[:-1]) / 2
    x = np.concatenate([v, mid, np.nextafter(mid, 1e9), np.nextafter(mid, -1e9), [1e-9, -1e-9, 1000.0, -1e30]])
    x = torch.from_numpy(x).float().clamp(-448, 448)
    assert np.array_equal(O.encode(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert O.scale_of(448.0) == 1.0 and O.scale_of(448.1) == 2.0 and O.scale_of(224.0) == 0.5 and O.scale_of(0.0) == 2.0 ** -60 and O.scale_of(1e30) == 2.0 ** 40


def test_decode_refuses_offsets():
    q, kv, table = torch.zeros((2, 4, 64), dtype=torch.bfloat16), ints(3, 4), torch.zeros((2, 2), dtype=torch.int32)
    for cu, match in ((ints(0, 1), "cu_seqlens_q"), (torch.tensor([0, 1, 2]), "cu_seqlens_q"), (ints(0, 9, 1, 9, 2)[::2], "cu_seqlens_q")):
        with pytest.raises(ValueError, match=match):
            P.paged_decode_attention(q, *cache(), table, kv, cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="at most 1 tokens"):
        P.paged_decode_attention(q, *cache(), table[:1], kv[:1], cu_seqlens_q=ints(0, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        P.paged_decode_attention(q[:1], *cache(), table, kv, cu_seqlens_q=ints(0, 0, 1))
    lib = _lib.lib()
    assert lib.fdms_paged_attn_decode(P._ATTN_ARGS.pack(*(ATTN | dict(tokens=1, cu=0)).values()), None) == E and b"one token per sequence" in lib.fdms_last_error()


def test_release_refuses_the_number_of_blocks():
    kv, table, free, count = ints(1, 2), torch.zeros((2, 4), dtype=torch.int32), ints(0, 1), ints(2)
    with pytest.raises(ValueError, match="num_blocks"):
        P.release_paged_blocks(kv, table, free, count, block_size=16, num_blocks=-1)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.release_paged_blocks(kv, table, free, count, block_size=16, num_blocks=9)
    lib = _lib.lib()
    rel = dict(rows=PTR, listed=2, kv=PTR, n=2, bt=PTR, stride=4, cols=4, bs=16, free=PTR, capacity=8, blocks=9, count=PTR, status=None, stream=None)
    for change, code, words in [(dict(blocks=-1), E, b"negative"), (dict(blocks=1 << 28), C, b"31 bits"), (dict(listed=5000), C, b"rows a call")]:
        assert lib.fdms_paged_release_pool(*(rel | change).values()) == code and words in lib.fdms_last_error()


def test_prefill_drains_on_a_barrier_of_its_own():
    """Before the prefill kernel gives its tensor memory back it waits for the products that it issued, also after a wait that ran
    out.  An mbarrier completes a phase with as many arrivals as it was initialised with, and a commit is one: the barrier of
    that wait must take one arrival, from that commit alone, and be waited for in its first phase."""
    src = (Path(__file__).resolve().parent.parent / "fastdms_b200" / "csrc" / "paged_prefill.cu").read_text()
    tail = src[src.index("nothing of this CTA may be in flight"):src.index("tcgen05.dealloc")]
    commits = re.findall(r"tc_commit\(&sh\.(\w+)", tail)
    waits = re.findall(r"bar_\w+\(&sh\.(\w+)(?:\[\w+\])?, (\d)", tail)
    assert len(commits) == 1 and waits == [(commits[0], "0")]
    counts = re.findall(rf"bar_init\(&sh\.{commits[0]}(?:\[\w+\])?, (\w+)\)", src)
    assert counts == ["1"]
    assert len(re.findall(rf"sh\.{commits[0]}\b", src)) == 3                  # its start, the commit and the wait


def test_c_metadata_refuses_lengths_over_later_ones():
    """Beyond one round of the scan, a length written ahead of those still to be read would change them."""
    lib, n = _lib.lib(), 3000
    far = dict(n=n, new=PTR, kv=PTR + 4 * n, total=1 << 20, ws=PTR, ws_bytes=0)        # refused at the latest for its workspace
    for out, code, words in [(PTR + 4, E, b"kv_lens_out"), (PTR + 4 * n - 4, E, b"kv_lens_out"), (PTR + 4 * n + 4, E, b"kv_lens_out"),
                             (PTR, W, b"workspace"), (PTR + 4 * n, W, b"workspace"), (PTR + 8 * n, W, b"workspace")]:
        assert lib.fdms_paged_metadata(P._METADATA_ARGS.pack(*(METADATA | far | dict(kv_out=out)).values()), None) == code and words in lib.fdms_last_error()
    near = far | dict(n=1024, kv=PTR + 4 * n, kv_out=PTR + 4)                # one round reads all lengths before it writes any
    assert lib.fdms_paged_metadata(P._METADATA_ARGS.pack(*(METADATA | near).values()), None) == W


@pytest.mark.parametrize("name", ["k0", "k1", "k2", "v0", "v1", "v2"])
def test_c_calls_refuse_negative_strides(name):
    """Block and row strides are taken as unsigned 32-bit numbers: a negative one would read far behind the cache."""
    lib, bad = _lib.lib(), {name: -2048}
    for fn, args in ((lib.fdms_paged_store, P._STORE_ARGS.pack(*(STORE | bad).values())), (lib.fdms_paged_attn_decode, P._ATTN_ARGS.pack(*(ATTN | bad).values())),
                     (lib.fdms_paged_attn_prefill, P._ATTN_ARGS.pack(*(ATTN | bad).values()))):
        assert fn(args, None) == E and b"negative stride" in lib.fdms_last_error()
