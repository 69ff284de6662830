"""The dense paged cache with block scales on the GPU: tables, store, decode and prefill attention against the plain 64-bit
statement of `paged_oracle`, alone and run together.  Integers, codes and scales are exact; attention is held to the bound
that its roundings give (f16 weights, float32 sums) plus half a step of the output's type."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from fastdms_b200 import _lib
    _lib.lib()
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _status_clean(dev):
    from fastdms_b200 import _lib
    _lib.read_device_status(dev)
    yield
    assert _lib.read_device_status(dev) == 0, "a kernel raised a device status bit"


def raised(dev) -> bool:
    from fastdms_b200 import _lib
    return _lib.read_device_status(dev) == _lib.DEV_BAD_INDEX


def i32(a, dev):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32).to(dev)


def n64(t):
    return t.detach().cpu().double().numpy()


def codes_of(t):
    return t.detach().cpu().contiguous().view(torch.uint8).numpy().copy()


# ---- tables --------------------------------------------------------------------------------------------------------

def _table_state(rng, n, bs, most_new, most_kv, spare, dev, extra_cols=2):
    new = rng.integers(0, most_new + 1, n)
    kv = rng.integers(0, most_kv + 1, n)
    if n > 2:
        new[1], kv[2] = 0, 0
    held, want = -(-kv // bs), -(-(kv + new) // bs)
    pool = int(held.sum() + max(1, int((want - held).sum() * spare)))
    order = rng.permutation(pool)
    table = np.full((n, int(want.max(initial=0)) + extra_cols), -1, np.int64)
    at = 0
    for i in range(n):
        table[i, :held[i]] = order[at:at + held[i]]
        at += held[i]
    free = np.full(pool, -7, np.int64)
    free[:pool - at] = order[at:]
    return new, kv, table, free, pool - at


@pytest.mark.parametrize("n,bs,most_new,most_kv,spare", [
    (1, 16, 1, 0, 1.0), (1, 16, 40, 15, 1.0), (5, 16, 1, 200, 1.0), (33, 32, 1, 96, 1.5), (33, 64, 130, 70, 1.0), (7, 128, 700, 300, 0.5),
    (1024, 16, 3, 60, 0.7), (1500, 16, 2, 33, 1.0), (64, 16, 1000, 40, 0.6), (3, 16, 9000, 0, 1.0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables(dev, n, bs, most_new, most_kv, spare, in_place):
    from fastdms_b200.layers.paged_attention import build_paged_metadata
    rng = np.random.default_rng(n * 7 + bs)
    new, kv, table, free, count = _table_state(rng, n, bs, most_new, most_kv, spare, dev)
    total = int(new.sum()) + 3
    want = O.tables(new, kv, table, free, count, bs, total)
    t_kv, t_count, t_table, t_free = i32(kv, dev), i32([count], dev), i32(table, dev), i32(free, dev)
    outs = {} if in_place else {"kv_lens_out": torch.empty_like(t_kv), "free_count_out": torch.empty_like(t_count)}
    cu, slots, pos = build_paged_metadata(i32(new, dev), t_kv, t_table, t_free, t_count, block_size=bs, total_tokens=total, **outs)
    got_kv, got_count = (t_kv, t_count) if in_place else (outs["kv_lens_out"], outs["free_count_out"])
    assert np.array_equal(cu.cpu().numpy(), want[0])
    assert np.array_equal(got_kv.cpu().numpy(), want[1])
    assert np.array_equal(t_table.cpu().numpy(), want[2])
    assert int(got_count) == want[3]
    assert np.array_equal(slots.cpu().numpy(), want[4])
    assert pos.dtype == torch.int64 and np.array_equal(pos.cpu().numpy(), want[5])
    assert np.array_equal(t_free.cpu().numpy(), free)
    if not in_place:                                                        # the same step again from the same state
        assert np.array_equal(t_kv.cpu().numpy(), kv) and int(t_count) == count
        again = build_paged_metadata(i32(new, dev), t_kv, t_table, t_free, t_count, block_size=bs, total_tokens=total, **outs)
        assert all(torch.equal(a, b) for a, b in zip(again, (cu, slots, pos)))


@pytest.mark.parametrize("total", [0, 1, 5, 20000])
def test_tables_of_no_sequences_or_no_tokens(dev, total):
    from fastdms_b200.layers.paged_attention import build_paged_metadata
    free, count = i32([2, 1, 0], dev), i32([3], dev)
    cu, slots, pos = build_paged_metadata(i32([], dev), i32([], dev), torch.empty((0, 4), dtype=torch.int32, device=dev), free, count,
                                          block_size=16, total_tokens=total)
    assert cu.tolist() == [0] and int(count) == 3 and (slots == -1).all() and (pos == 0).all() and slots.numel() == total
    kv, table = i32([5, 0], dev), i32([[0, -1], [-1, -1]], dev)
    cu, slots, pos = build_paged_metadata(i32([0, 0], dev), kv, table, free, count, block_size=16, total_tokens=total)
    assert cu.tolist() == [0, 0, 0] and kv.tolist() == [5, 0] and table.tolist() == [[0, -1], [-1, -1]] and (slots == -1).all()


@pytest.mark.parametrize("pad", [0, 20000])
def test_tables_leave_out_what_cannot_be(dev, pad):
    from fastdms_b200.layers.paged_attention import build_paged_metadata
    new, kv = [3, -1, 4, 40, 2], [0, 5, -2, 0, 16]                          # good, negative, negative, too wide for the table, good
    table = np.full((5, 2), -1)
    table[4, 0] = 9
    t_kv, t_table, count = i32(kv, dev), i32(table, dev), i32([4], dev)
    cu, slots, pos = build_paged_metadata(i32(new, dev), t_kv, t_table, i32([3, 4, 5, 6, -1], dev), count, block_size=16, total_tokens=49 + pad)
    assert raised(dev)
    assert cu.tolist() == [0, 3, 3, 7, 47, 49] and t_kv.tolist() == [3, 5, -2, 0, 18] and int(count) == 2
    assert t_table.tolist() == [[6, -1], [-1, -1], [-1, -1], [-1, -1], [9, 5]]
    assert slots[:3].tolist() == [96, 97, 98] and (slots[3:47] == -1).all() and slots[47:49].tolist() == [80, 81] and (slots[49:] == -1).all()
    # more tokens than there is room for: what ends beyond it is not served
    t_kv, count = i32([0, 0], dev), i32([4], dev)
    cu, slots, _ = build_paged_metadata(i32([5, 6], dev), t_kv, i32([[-1], [-1]], dev), i32([0, 1, 2, 3], dev), count, block_size=16, total_tokens=10)
    assert raised(dev)
    assert cu.tolist() == [0, 5, 10] and t_kv.tolist() == [5, 0] and int(count) == 3 and (slots[5:] == -1).all()
    # a count beyond the stack's memory serves nobody who needs a block
    t_kv, count = i32([0, 3], dev), i32([9], dev)
    build_paged_metadata(i32([5, 6], dev), t_kv, i32([[-1], [1]], dev), i32([0, 1, 2, 3], dev), count, block_size=16, total_tokens=11)
    assert raised(dev) and t_kv.tolist() == [0, 9]


def test_release(dev):
    from fastdms_b200.layers.paged_attention import build_paged_metadata, release_paged_blocks
    n, bs = 6, 16
    kv, count = i32([0] * n, dev), i32([40], dev)
    table, free = i32(np.full((n, 40), -1), dev), torch.arange(40, device=dev, dtype=torch.int32).flip(0).contiguous()
    build_paged_metadata(i32([1, 16, 17, 0, 200, 33], dev), kv, table, free, count, block_size=bs, total_tokens=267)
    assert int(count) == 40 - (1 + 1 + 2 + 0 + 13 + 3)
    held = table.cpu().numpy().copy()
    before = free[:int(count)].cpu().tolist()
    release_paged_blocks(kv, table, free, count, block_size=bs, rows=i32([4, 0, 3], dev))
    assert kv.tolist() == [0, 16, 17, 0, 0, 33] and int(count) == 40 - 6
    assert free[:int(count)].cpu().tolist() == before + held[4, :13][::-1].tolist() + [held[0, 0]]
    assert (table[4] == -1).all() and (table[0] == -1).all() and np.array_equal(table[5].cpu().numpy(), held[5])
    # admitting a request and releasing it again leaves the stack as it was
    was = free[:int(count)].cpu().tolist()
    build_paged_metadata(i32([0, 0, 0, 100, 0, 0], dev), kv, table, free, count, block_size=bs, total_tokens=100)
    release_paged_blocks(kv, table, free, count, block_size=bs, rows=i32([3], dev))
    assert free[:int(count)].cpu().tolist() == was
    release_paged_blocks(kv, table, free, count, block_size=bs, rows=i32([], dev))
    release_paged_blocks(kv, table, free, count, block_size=bs)
    assert int(count) == 40 and sorted(free.tolist()) == list(range(40)) and (table == -1).all() and (kv == 0).all()


def test_release_leaves_out_what_cannot_be(dev):
    from fastdms_b200.layers.paged_attention import release_paged_blocks
    kv, table = i32([20, 40, -3], dev), i32([[5, 6, -1], [7, 99, 2], [1, 1, 1]], dev)
    free, count = i32([0, -1, -1, -1, -1, -1, -1, -1], dev), i32([1], dev)
    release_paged_blocks(kv, table, free, count, block_size=16, rows=i32([1, 0, 1, 17, -1, 2], dev))
    assert raised(dev)
    assert int(count) == 5 and free[:5].tolist() == [0, 2, 7, 6, 5] and kv.tolist() == [0, 0, 0]
    # a stack without room keeps inside its memory
    kv, table, free, count = i32([40], dev), i32([[0, 1, 2]], dev), i32([0, 1, 2, 9], dev), i32([2], dev)
    release_paged_blocks(kv, table, free[:3], count, block_size=16)
    assert raised(dev) and int(count) == 3 and free.tolist() == [0, 1, 2, 9]


# ---- store ---------------------------------------------------------------------------------------------------------

def make_cache(blocks, heads, bs, d, dev, layout="hnd", fill=0x7F):
    """Caches full of NaN codes and NaN scales (what fresh memory may hold), [blocks, heads, bs, d] in the given layout."""
    out = []
    for _ in range(2):
        if layout == "nhd":
            c = torch.full((blocks, bs, heads, d), fill, dtype=torch.uint8, device=dev).permute(0, 2, 1, 3)
        elif layout == "layers":                                             # one layer of an interleaved allocation
            c = torch.full((blocks, 2, heads, bs, d + 16), fill, dtype=torch.uint8, device=dev)[:, 1, :, :, :d]
        else:
            c = torch.full((blocks, heads, bs, d), fill, dtype=torch.uint8, device=dev)
        out.append(c.view(torch.float8_e4m3fn))
    return (*out, *(torch.full((blocks, heads), float("nan"), device=dev) for _ in range(2)))


def _random_rows(rng, shape, dt, loud=True):
    x = rng.standard_normal(shape) * (2.0 ** rng.integers(-6, 7, shape[:2])[..., None] if loud else 1.0)
    return torch.from_numpy(x).to(DT[dt])


def check_store(kc, vc, ks, vs, want):
    assert np.array_equal(ks.cpu().numpy().astype(np.float64), want[2], equal_nan=True)
    assert np.array_equal(vs.cpu().numpy().astype(np.float64), want[3], equal_nan=True)
    assert np.array_equal(codes_of(kc), want[0]) and np.array_equal(codes_of(vc), want[1])


@pytest.mark.parametrize("d,bs,heads,dt,layout", [
    (64, 16, 2, "bf16", "hnd"), (128, 16, 3, "f16", "nhd"), (64, 32, 1, "f16", "layers"), (128, 32, 8, "bf16", "hnd"), (64, 64, 5, "bf16", "nhd"),
    (128, 128, 2, "bf16", "hnd"), (128, 64, 1, "f16", "layers"), (64, 128, 9, "f16", "hnd")])
def test_store_steps(dev, d, bs, heads, dt, layout):
    """Sequences that grow by ragged steps: fresh blocks, blocks that fill over several steps, scales that grow and stay."""
    from fastdms_b200.layers.paged_attention import store_paged_kvcache
    rng = np.random.default_rng(d + bs + heads)
    n, cols = 5, 8
    blocks = n * cols + 3
    kc, vc, ks, vs = make_cache(blocks, heads, bs, d, dev, layout)
    want = [codes_of(kc), codes_of(vc), np.full((blocks, heads), np.nan), np.full((blocks, heads), np.nan)]
    table = rng.permutation(blocks)[:n * cols].reshape(n, cols)
    kv = np.zeros(n, np.int64)
    for step in ([1, 3, 0, bs, 2 * bs + 5], [1, 1, 1, 1, 1], [bs - 3, 7, 1, bs - 1, 2], [1, 1, 1, 1, 1], [0, 2 * bs, 3, 0, 1]):
        slots = []
        for i, m in enumerate(step):
            slots += [int(table[i, p // bs] * bs + p % bs) for p in range(kv[i], kv[i] + m)]
            kv[i] += m
            slots.append(-1)                                                 # padding between sequences is skipped
        k, v = _random_rows(rng, (len(slots), heads, d), dt), _random_rows(rng, (len(slots), heads, d), dt)
        wide = torch.full((len(slots), heads + 2, 2 * d), float("nan"), dtype=DT[dt])      # k is a view of a wider buffer
        wide[:, 1:1 + heads, d:] = k
        store_paged_kvcache(wide.to(dev)[:, 1:1 + heads, d:], v.to(dev), kc, vc, ks, vs, i32(slots, dev))
        O.store(n64(k), want[0], want[2], slots, bs)
        O.store(n64(v), want[1], want[3], slots, bs)
        check_store(kc, vc, ks, vs, want)


def test_store_of_many_tokens(dev):
    """A prompt batch large enough for several tokens per CTA, with blocks that end inside a CTA's tokens."""
    from fastdms_b200.layers.paged_attention import store_paged_kvcache
    rng = np.random.default_rng(3)
    heads, d, bs = 2, 64, 16
    lens, prior = [4000, 1, 7001, 37, 9000], [3, 15, 0, 16, 8]
    blocks = sum(-(-(a + b) // bs) for a, b in zip(lens, prior))
    order, slots = rng.permutation(blocks), []
    for m, p0 in zip(lens, prior):
        row, order = order[:-(-(m + p0) // bs)], order[-(-(m + p0) // bs):]
        slots += [int(row[p // bs] * bs + p % bs) for p in range(p0, p0 + m)]
    kc, vc, ks, vs = make_cache(blocks, heads, bs, d, dev, fill=0x30)
    ks.fill_(0.25), vs.fill_(2.0 ** -20)
    want = [codes_of(kc), codes_of(vc), np.full((blocks, heads), 0.25), np.full((blocks, heads), 2.0 ** -20)]
    k, v = _random_rows(rng, (len(slots), heads, d), "bf16"), _random_rows(rng, (len(slots), heads, d), "bf16")
    store_paged_kvcache(k.to(dev), v.to(dev), kc, vc, ks, vs, i32(slots, dev))
    O.store(n64(k), want[0], want[2], slots, bs)
    O.store(n64(v), want[1], want[3], slots, bs)
    check_store(kc, vc, ks, vs, want)


def test_store_of_unusual_values(dev):
    from fastdms_b200.layers.paged_attention import store_paged_kvcache
    heads, d, bs = 1, 64, 16
    rows = [[0.0], [-0.0], [448.0], [449.0], [1e-38, -1e-38], [3e38], [float("inf"), 1.0], [float("-inf")], [float("nan"), 2.0], [float("nan")],
            [2.0 ** -60 * 448], [2.0 ** -60 * 450], [2.0 ** 40 * 448], [2.0 ** 41 * 448], [17.0, 19.0, 0.001], [1e-40]]
    x = torch.zeros((len(rows), heads, d), dtype=torch.bfloat16)
    for i, r in enumerate(rows):
        x[i, 0, :len(r)] = torch.tensor(r, dtype=torch.float64).to(torch.bfloat16)
    slots = [i * bs for i in range(len(rows))]
    kc, vc, ks, vs = make_cache(len(rows), heads, bs, d, dev)
    want = [codes_of(kc), codes_of(vc), np.full((len(rows), heads), np.nan), np.full((len(rows), heads), np.nan)]
    store_paged_kvcache(x.to(dev), (-x).to(dev), kc, vc, ks, vs, i32(slots, dev))
    O.store(n64(x), want[0], want[2], slots, bs)
    O.store(n64(-x), want[1], want[3], slots, bs)
    got_nan, want_nan = (codes_of(kc) & 0x7F) == 0x7F, (want[0] & 0x7F) == 0x7F
    assert np.array_equal(got_nan, want_nan) and np.array_equal(np.where(got_nan, 0, codes_of(kc)), np.where(want_nan, 0, want[0]))
    got_nan, want_nan = (codes_of(vc) & 0x7F) == 0x7F, (want[1] & 0x7F) == 0x7F
    assert np.array_equal(got_nan, want_nan) and np.array_equal(np.where(got_nan, 0, codes_of(vc)), np.where(want_nan, 0, want[1]))
    assert np.array_equal(ks.cpu().numpy(), want[2]) and np.array_equal(vs.cpu().numpy(), want[3])


def test_store_leaves_out_what_cannot_be(dev):
    from fastdms_b200.layers.paged_attention import store_paged_kvcache
    heads, d, bs, blocks = 2, 64, 16, 4
    rng = np.random.default_rng(0)
    k = _random_rows(rng, (8, heads, d), "bf16")
    # beyond the cache, the same slot twice, a block written backwards
    slots = [64, 16, 16, 2_000_000_000, 40, 39, -5, 0]
    kc, vc, ks, vs = make_cache(blocks, heads, bs, d, dev)
    ks.fill_(1.0), vs.fill_(1.0)
    want = [codes_of(kc), codes_of(vc), np.ones((blocks, heads)), np.ones((blocks, heads))]
    store_paged_kvcache(k.to(dev), k.to(dev), kc, vc, ks, vs, i32(slots, dev))
    assert raised(dev)
    for i in (0, 1):
        for t in (1, 4, 7):
            O.store(n64(k[t:t + 1]), want[i], want[2 + i], [slots[t]], bs)
    # the token at 40 keeps earlier rows of its block, which are NaN codes here: compare what was written
    got = codes_of(kc)
    for t in (1, 4, 7):
        assert np.array_equal(got[slots[t] // bs, :, slots[t] % bs], want[0][slots[t] // bs, :, slots[t] % bs])
    assert (got[1, :, 1:] == 0x7F).all() and (got[3] == 0x7F).all() and (got[2, :, 9:] == 0x7F).all()
    store_paged_kvcache(k[:0].to(dev), k[:0].to(dev), kc, vc, ks, vs, i32([], dev))
    store_paged_kvcache(k.to(dev), k.to(dev), kc, vc, ks, vs, i32([-1] * 8, dev))
    assert np.array_equal(codes_of(kc), got)


# ---- attention -----------------------------------------------------------------------------------------------------

def build_case(rng, lens, heads, bs, d, dev, layout="hnd", loud=True, spare=5):
    """A filled cache for sequences of the given lengths; everything that no sequence holds is NaN."""
    cols = max(1, -(-max(lens, default=0) // bs))
    need = [-(-m // bs) for m in lens]
    blocks = sum(need) + spare
    order = rng.permutation(blocks)
    table = np.full((len(lens), cols), -1, np.int64)
    codes = [np.full((blocks, heads, bs, d), 0x7F, np.uint8) for _ in range(2)]
    scale = [np.full((blocks, heads), np.nan) for _ in range(2)]
    at = 0
    for i, m in enumerate(lens):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        slots = [int(table[i, p // bs] * bs + p % bs) for p in range(m)]
        for c in range(2):
            if m:
                O.store(rng.standard_normal((m, heads, d)) * (2.0 ** rng.integers(-5, 5) if loud else 1.0), codes[c], scale[c], slots, bs)
    kc, vc, ks, vs = make_cache(blocks, heads, bs, d, dev, layout)
    for t, c in ((kc, codes[0]), (vc, codes[1])):
        t.view(torch.uint8).copy_(torch.from_numpy(c).to(dev))
    ks.copy_(torch.from_numpy(scale[0])), vs.copy_(torch.from_numpy(scale[1]))
    return (kc, vc, ks, vs, i32(table, dev)), (codes, scale, table)


def check_rows(got, got_lse, want, dt):
    out, lse, tol, ltol = want
    half = torch.finfo(DT[dt]).eps / 2
    tiny = torch.finfo(DT[dt]).smallest_normal * half
    assert np.isfinite(got).all()
    assert (np.abs(got - out) <= tol + half * (np.abs(out) + tol) + tiny).all(), np.max(np.abs(got - out) - tol)
    if got_lse is not None:
        empty = np.isneginf(lse)
        assert np.array_equal(np.isneginf(got_lse), empty)
        assert (np.abs(got_lse[~empty] - lse[~empty]) <= ltol[~empty]).all()


DECODE = [
    # lens, kv heads, group, bs, d, dtype, layout
    ([1], 1, 1, 16, 64, "bf16", "hnd"), ([16], 2, 4, 16, 128, "f16", "hnd"), ([17, 0, 15], 2, 8, 16, 64, "f16", "nhd"),
    ([0], 2, 2, 16, 128, "bf16", "hnd"), ([0, 0, 0], 1, 4, 32, 64, "bf16", "hnd"),
    ([201], 8, 4, 16, 128, "f16", "hnd"), ([300, 1, 33, 512], 2, 7, 32, 128, "bf16", "layers"), ([777], 1, 3, 64, 64, "bf16", "nhd"),
    ([129, 128, 127, 1], 4, 5, 128, 128, "f16", "hnd"), ([64] * 40, 2, 2, 16, 64, "bf16", "hnd"), ([2500, 40], 1, 16, 16, 64, "bf16", "hnd"),
    ([600], 1, 12, 64, 128, "f16", "hnd"), ([9000, 3, 0, 1200], 1, 4, 16, 64, "f16", "hnd"), ([100, 90], 1, 64, 16, 64, "bf16", "hnd"),
    # the widest clusters; and, from wide tables, sequences of which many begin and end in one share, next to one that fills many
    ([15000], 2, 3, 16, 128, "bf16", "hnd"), ([15001, 1], 1, 8, 32, 64, "f16", "nhd"),
    ([1] * 30 + [15000, 0] + [40] * 9 + [390, 0, 380, 400, 0], 2, 2, 16, 128, "bf16", "hnd"),
    ([3000, 2] * 10, 2, 4, 64, 64, "f16", "hnd")]


def wide_table(table, bs, rows=70000):
    """The same table with columns for long sequences, which the decode kernel for short ones does not take."""
    wide = torch.full((table.shape[0], rows // bs), -1, dtype=torch.int32, device=table.device)
    wide[:, :table.shape[1]] = table
    return wide


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("lens,heads,group,bs,d,dt,layout", DECODE)
def test_decode(dev, lens, heads, group, bs, d, dt, layout, wide):
    from fastdms_b200.layers.paged_attention import paged_decode_attention
    rng = np.random.default_rng(sum(lens) + heads + group + d)
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, lens, heads, bs, d, dev, layout)
    if wide:
        table = wide_table(table, bs)
    q = _random_rows(rng, (len(lens), heads * group, d), dt, loud=False)
    lse = torch.full((len(lens), heads * group), 7.0, device=dev)
    got = paged_decode_attention(q.to(dev), kc, vc, ks, vs, table, i32(lens, dev), lse_out=lse)
    qn, g, gl = n64(q), n64(got), n64(lse)
    for b, m in enumerate(lens):
        for h in range(heads):
            k, v = (O.rows_of(codes[c], scale[c], tab[b], m, h, bs) for c in range(2))
            r = slice(h * group, (h + 1) * group)
            check_rows(g[b, r], gl[b, r], O.attention(qn[b, r], k, v, [m - 1] * group, d ** -0.5), dt)


def test_decode_of_views_scale_and_buffers(dev):
    """Strided q and out, a wider block table than needed, a scale of its own, an lse laid out the other way, rows of other
    sequences left as they were."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention
    rng = np.random.default_rng(11)
    lens, heads, group, bs, d = [50, 7, 260], 2, 4, 16, 64
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, lens, heads, bs, d, dev)
    wide = torch.full((4, table.shape[1] + 6), 1 << 30, dtype=torch.int32, device=dev)     # never read: beyond the lengths
    wide[:3, :table.shape[1]] = torch.where(table < 0, 1 << 30, table)
    q = _random_rows(rng, (3, heads * group, d), "bf16", loud=False)
    qkv = torch.full((3, heads * group + 4, d), float("nan"), dtype=torch.bfloat16, device=dev)
    qkv[:, :heads * group] = q.to(dev)
    out = torch.full((6, heads * group, 2 * d), 3.0, dtype=torch.bfloat16, device=dev)
    lse = torch.empty((heads * group, 3), device=dev)
    got = paged_decode_attention(qkv[:, :heads * group], kc, vc, ks, vs, wide[:3], i32(lens, dev), 0.3, out=out[::2, :, d:], lse_out=lse.t())
    assert got.data_ptr() == out[::2, :, d:].data_ptr() and (out[1::2] == 3.0).all() and (out[:, :, :d] == 3.0).all()
    for b, m in enumerate(lens):
        for h in range(heads):
            k, v = (O.rows_of(codes[c], scale[c], tab[b], m, h, bs) for c in range(2))
            r = slice(h * group, (h + 1) * group)
            check_rows(n64(got)[b, r], n64(lse.t())[b, r], O.attention(n64(q)[b, r], k, v, [m - 1] * group, 0.3), "bf16")


def _magnitudes(rng, lens, heads, bs, d, dev, exps):
    """Blocks whose scales differ by many powers of two."""
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, lens, heads, bs, d, dev, loud=False)
    for b in np.unique(tab[tab >= 0]):
        for h in range(heads):
            scale[1][b, h] *= 2.0 ** int(rng.choice(exps))
    vs.copy_(torch.from_numpy(scale[1]))
    return (kc, vc, ks, vs, table), (codes, scale, tab)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("exps,dt", [((-50, 0, 40), "bf16"), ((-6, 0, 6), "f16"), ((-30, -29), "bf16")])
def test_blocks_of_very_different_magnitude(dev, exps, dt, wide):
    """V blocks between tiny and huge: the weights stay exact enough for each (a block that matters little in the sum may
    not cost one that matters its digits)."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    rng = np.random.default_rng(5)
    lens, heads, group, bs, d = [400], 2, 4, 16, 64
    (kc, vc, ks, vs, table), (codes, scale, tab) = _magnitudes(rng, lens, heads, bs, d, dev, exps)
    if wide:
        table = wide_table(table, bs)
    q = _random_rows(rng, (1, heads * group, d), dt, loud=False)
    lse, lse2 = torch.empty((1, heads * group), device=dev), torch.empty((heads * group, 1), device=dev)
    dec = paged_decode_attention(q.to(dev), kc, vc, ks, vs, table, i32(lens, dev), lse_out=lse)
    pre = paged_prefill_attention(q.to(dev), kc, vc, ks, vs, table, i32(lens, dev), i32([0, 1], dev), lse_out=lse2)
    for h in range(heads):
        k, v = (O.rows_of(codes[c], scale[c], tab[0], lens[0], h, bs) for c in range(2))
        r = slice(h * group, (h + 1) * group)
        want = O.attention(n64(q)[0, r], k, v, [lens[0] - 1] * group, d ** -0.5)
        check_rows(n64(dec)[0, r], n64(lse)[0, r], want, dt)
        check_rows(n64(pre)[0, r], n64(lse2)[r, 0], want, dt)


def test_queries_of_very_different_magnitude(dev):
    """bf16 queries beyond f16's range, tiny ones, zeros, and one loud channel in a row."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention
    rng = np.random.default_rng(6)
    lens, heads, group, bs, d = [90], 1, 8, 16, 64
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, lens, heads, bs, d, dev, loud=False)
    x = rng.standard_normal((1, 8, d))
    x[0, 0] *= 2.0 ** 100
    x[0, 1] *= 2.0 ** -100
    x[0, 2] = 0
    x[0, 3, 5] = 2.0 ** 12
    x[0, 4] *= 2.0 ** 20
    q = torch.from_numpy(x).to(torch.bfloat16)
    got = n64(paged_decode_attention(q.to(dev), kc, vc, ks, vs, table, i32(lens, dev), 2.0 ** -3))
    k, v = (O.rows_of(codes[c], scale[c], tab[0], lens[0], 0, bs) for c in range(2))
    want = O.attention(n64(q)[0], k, v, [lens[0] - 1] * 8, 2.0 ** -3)
    calm = [1, 2, 3, 5, 6, 7]
    check_rows(got[0, calm], None, tuple(w[calm] for w in want), "bf16")
    # so loud that one key takes all: its row of V
    for r in (0, 4):
        s = k @ n64(q)[0, r]
        assert np.sort(s)[-1] - np.sort(s)[-2] > 2.0 ** 12
        assert (np.abs(got[0, r] - v[s.argmax()]) <= 2.0 ** -8 * np.abs(v[s.argmax()])).all()


@pytest.mark.parametrize("wide", [False, True])
def test_decode_leaves_out_what_cannot_be(dev, wide):
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    rng = np.random.default_rng(8)
    lens, heads, group, bs, d = [70, 40], 1, 2, 16, 64
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, lens, heads, bs, d, dev)
    q = _random_rows(rng, (2, group, d), "bf16", loud=False).to(dev)
    bad = wide_table(table, bs) if wide else table.clone()
    bad[0, 1], bad[0, 3] = -1, kc.shape[0]
    keep = np.r_[0:16, 32:48, 64:70]
    k, v = (O.rows_of(codes[c], scale[c], tab[0], 70, 0, bs)[keep] for c in range(2))
    got = n64(paged_decode_attention(q, kc, vc, ks, vs, bad, i32(lens, dev)))
    assert raised(dev)
    want = O.attention(n64(q)[0], k, v, [len(keep) - 1] * group, d ** -0.5)
    check_rows(got[0], None, want, "bf16")
    pre = n64(paged_prefill_attention(q, kc, vc, ks, vs, bad, i32(lens, dev), i32([0, 1, 2], dev)))
    assert raised(dev)
    check_rows(pre[0], None, want, "bf16")
    # lengths that cannot be: negative ones count as none, too long ones as what the table holds
    got = n64(paged_decode_attention(q, kc, vc, ks, vs, table[:, :3], i32([-4, 1000], dev)))
    assert raised(dev)
    assert (got[0] == 0).all()
    # a table without any usable block gives zeros
    got = paged_decode_attention(q, kc, vc, ks, vs, torch.full_like(table, -1), i32(lens, dev))
    assert raised(dev) and (got == 0).all()
    # a table without columns holds nothing
    got = paged_decode_attention(q, kc, vc, ks, vs, table[:, :0], i32([0, 0], dev))
    assert (got == 0).all()


PREFILL = [
    # (new, kv) per sequence, kv heads, group, bs, d, dtype, layout
    ([(1, 1)], 1, 1, 16, 64, "bf16", "hnd"), ([(77, 77)], 2, 4, 16, 64, "f16", "hnd"), ([(77, 77)], 1, 8, 32, 128, "bf16", "nhd"),
    ([(5, 205), (0, 30), (130, 130), (1, 64)], 2, 4, 16, 128, "f16", "hnd"), ([(33, 300), (64, 64)], 1, 3, 64, 64, "bf16", "layers"),
    ([(200, 456)], 1, 7, 128, 128, "bf16", "hnd"), ([(40, 25), (3, 0), (20, 20)], 2, 2, 16, 64, "bf16", "hnd"),
    ([(17, 17)] * 9, 1, 5, 16, 64, "f16", "nhd"), ([(70, 150)], 1, 64, 16, 64, "bf16", "hnd"), ([(300, 1100)], 1, 1, 16, 128, "bf16", "hnd"),
    ([(31, 31)], 1, 24, 32, 128, "f16", "hnd"), ([(129, 129), (257, 700)], 1, 2, 64, 128, "bf16", "hnd"),
    ([(5, 4100), (2, 1)], 1, 4, 16, 128, "bf16", "hnd"), ([(1, 2500), (70, 2050)], 2, 8, 16, 64, "f16", "nhd")]


def _prefill(dev, rng, seqs, heads, group, bs, d, dt, layout, pad=3):
    case = build_case(rng, [m for _, m in seqs], heads, bs, d, dev, layout)
    cu = np.concatenate([[0], np.cumsum([n for n, _ in seqs])])
    q = _random_rows(rng, (int(cu[-1]) + pad, heads * group, d), dt, loud=False)
    return case, cu, q


def check_prefill(got, lse, q, cu, seqs, host, heads, group, bs, d, dt):
    codes, scale, tab = host
    for i, (n, m) in enumerate(seqs):
        for h in range(heads):
            k, v = (O.rows_of(codes[c], scale[c], tab[i], m, h, bs) for c in range(2))
            for j in range(h * group, (h + 1) * group, max(1, group // 3)):
                rows = slice(int(cu[i]), int(cu[i + 1]))
                want = O.attention(q[rows, j], k, v, m - n + np.arange(n), d ** -0.5)
                check_rows(got[rows, j], None if lse is None else lse[j, rows], want, dt)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("seqs,heads,group,bs,d,dt,layout", PREFILL)
def test_prefill(dev, seqs, heads, group, bs, d, dt, layout, wide):
    """`wide`: a table with columns for long sequences, for which the rows are cut into parts."""
    from fastdms_b200.layers.paged_attention import paged_prefill_attention
    rng = np.random.default_rng(len(seqs) + group + d + bs)
    (dv, host), cu, q = _prefill(dev, rng, seqs, heads, group, bs, d, dt, layout)
    if wide:
        dv = (*dv[:4], wide_table(dv[4], bs))
    out = torch.full(q.shape, 3.0, dtype=DT[dt], device=dev)
    lse = torch.full((heads * group, q.shape[0]), 7.0, device=dev)
    got = paged_prefill_attention(q.to(dev), *dv, i32([m for _, m in seqs], dev), i32(cu, dev), out=out, lse_out=lse)
    assert (got[int(cu[-1]):] == 3.0).all() and (lse[:, int(cu[-1]):] == 7.0).all()        # behind the last sequence
    check_prefill(n64(got), n64(lse), n64(q), cu, seqs, host, heads, group, bs, d, dt)


def test_prefill_of_many_sequences(dev):
    """More sequences than a warp looks at at once, most of them without tokens in the step."""
    from fastdms_b200.layers.paged_attention import paged_prefill_attention
    rng = np.random.default_rng(1)
    seqs = [(0, int(rng.integers(0, 40))) for _ in range(100)]
    for i in (0, 31, 32, 70, 99):
        n = int(rng.integers(1, 50))
        seqs[i] = (n, n + int(rng.integers(0, 30)))
    (dv, host), cu, q = _prefill(dev, rng, seqs, 1, 4, 16, 64, "bf16", "hnd")
    got = paged_prefill_attention(q.to(dev), *dv, i32([m for _, m in seqs], dev), i32(cu, dev))
    check_prefill(n64(got), None, n64(q), cu, seqs, host, 1, 4, 16, 64, "bf16")


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_does_not_see_what_is_masked(dev, d, wide):
    """NaN codes and NaN queries reach exactly the rows that see them."""
    from fastdms_b200.layers.paged_attention import paged_prefill_attention
    rng = np.random.default_rng(d)
    n, heads, group, bs = 150, 1, 2, 16
    (dv, host), cu, q = _prefill(dev, rng, [(n, n)], heads, group, bs, d, "bf16", "hnd", pad=0)
    if wide:
        dv = (*dv[:4], wide_table(dv[4], bs))
    kc, vc, ks, vs, table = dv
    clean = n64(paged_prefill_attention(q.to(dev), *dv, i32([n], dev), i32(cu, dev)))
    v2 = vc.clone()
    key, ch = 83, 5
    v2.view(torch.uint8)[int(table[0, key // bs]), 0, key % bs, ch] = 0xFF
    got = n64(paged_prefill_attention(q.to(dev), kc, v2, ks, vs, table, i32([n], dev), i32(cu, dev)))
    assert np.isnan(got[key:, :, ch]).all()
    rest = np.ones_like(got, dtype=bool)
    rest[key:, :, ch] = False
    assert np.array_equal(got[rest], clean[rest])
    k2 = kc.clone()
    k2.view(torch.uint8)[int(table[0, key // bs]), 0, key % bs, ch] = 0x7F
    got = n64(paged_prefill_attention(q.to(dev), k2, vc, ks, vs, table, i32([n], dev), i32(cu, dev)))
    assert np.isnan(got[key:]).all() and np.array_equal(got[:key], clean[:key])
    q2 = q.clone()
    q2[40, 1, 7] = float("nan")
    got = n64(paged_prefill_attention(q2.to(dev), *dv, i32([n], dev), i32(cu, dev)))
    keep = np.ones((n, group), dtype=bool)
    keep[40, 1] = False
    assert np.isnan(got[40, 1]).all() and np.array_equal(got[keep], clean[keep])


def test_prefill_of_broken_offsets_stays_inside(dev):
    """Offsets that run backwards or beyond the tokens are cut to what there is."""
    from fastdms_b200.layers.paged_attention import paged_prefill_attention
    rng = np.random.default_rng(2)
    seqs = [(20, 20), (30, 30)]
    (dv, host), cu, q = _prefill(dev, rng, seqs, 1, 2, 16, 64, "bf16", "hnd", pad=0)
    for broken in ([0, 20, 5000], [-7, 20, 10], [0, 60, 50]):
        out = paged_prefill_attention(q.to(dev), *dv, i32([20, 30], dev), i32(broken, dev), out=torch.zeros(q.shape, dtype=q.dtype, device=dev))
        assert torch.isfinite(out.float()).all()


def test_attention_refuses_outputs_and_strides(dev):
    from fastdms_b200.layers import paged_attention as P
    kc, vc, ks, vs = make_cache(2, 1, 16, 64, dev)
    q, table, kv = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=dev), i32([[0], [1]], dev), i32([3, 4], dev)
    args = (kc, vc, ks, vs, table, kv)
    for bad, match in [(dict(out=torch.zeros((2, 4, 64), device=dev)), "out must"), (dict(out=torch.zeros_like(q).cpu()), "CUDA"),
                       (dict(lse_out=torch.zeros((4, 3), device=dev)), "lse_out"),
                       (dict(out=torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=dev)[:, :, ::2]), "contiguous")]:
        with pytest.raises((ValueError, RuntimeError), match=match):
            P.paged_decode_attention(q, *args, **bad)
        with pytest.raises((ValueError, RuntimeError), match=match):
            P.paged_prefill_attention(q, *args, i32([0, 1, 2], dev), **bad)
    odd = torch.zeros((2, 4, 66), dtype=torch.bfloat16, device=dev)[:, :, 1:65]
    with pytest.raises(ValueError, match="aligned"):
        P.paged_decode_attention(odd, *args)
    with pytest.raises(ValueError, match="aligned"):
        P.store_paged_kvcache(odd[:, :1], odd[:, :1], kc, vc, ks, vs, i32([0, 16], dev))
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        P.paged_prefill_attention(q, *args, i32([0, 1], dev))
    with pytest.raises(RuntimeError, match="2048"):
        P.paged_decode_attention(q[:1].expand(2049, 4, 64).contiguous(), kc, vc, ks, vs, table[:1].expand(2049, 1).contiguous(), kv[:1].expand(2049).contiguous())
    with pytest.raises(RuntimeError, match="CUDA"):
        P.paged_decode_attention(q, kc, vc, ks.cpu(), vs, table, kv)


# ---- together ------------------------------------------------------------------------------------------------------

class Run:
    """A small server: sequences that are prefilled (in chunks), decode and end, driven through the public calls; beside it
    the same in the plain statement."""

    def __init__(self, dev, seed, n=4, heads=2, group=2, bs=16, d=64, dt="bf16", pool=60, cols=20):
        self.dev, self.rng = dev, np.random.default_rng(seed)
        self.n, self.heads, self.group, self.bs, self.d, self.dt, self.pool = n, heads, group, bs, d, dt, pool
        self.kc, self.vc, self.ks, self.vs = make_cache(pool, heads, bs, d, dev)
        self.kv, self.count = i32([0] * n, dev), i32([pool], dev)
        self.table = i32(np.full((n, cols), -1), dev)
        self.free = torch.arange(pool, device=dev, dtype=torch.int32).flip(0).contiguous()
        self.codes = [codes_of(self.kc), codes_of(self.vc)]
        self.scale = [np.full((pool, heads), np.nan) for _ in range(2)]

    def inputs(self, tokens):
        q = _random_rows(self.rng, (tokens, self.heads * self.group, self.d), self.dt, loud=False)
        k, v = (_random_rows(self.rng, (tokens, self.heads, self.d), self.dt) for _ in range(2))
        return q, k, v

    def call(self, new, q, k, v, decode, total=None):
        from fastdms_b200.layers import paged_attention as P
        cu, slots, pos = P.build_paged_metadata(new, self.kv, self.table, self.free, self.count, block_size=self.bs,
                                                total_tokens=q.shape[0] if total is None else total)
        P.store_paged_kvcache(k, v, self.kc, self.vc, self.ks, self.vs, slots)
        if decode:
            return P.paged_decode_attention(q, self.kc, self.vc, self.ks, self.vs, self.table, self.kv), slots
        return P.paged_prefill_attention(q, self.kc, self.vc, self.ks, self.vs, self.table, self.kv, cu), slots

    def check(self, new, q, k, v, out, slots):
        for c, x in ((0, k), (1, v)):
            O.store(n64(x), self.codes[c], self.scale[c], slots.cpu().tolist(), self.bs)
        check_store(self.kc, self.vc, self.ks, self.vs, (*self.codes, *self.scale))
        cu = np.concatenate([[0], np.cumsum(new)])
        kv, tab = self.kv.cpu().numpy(), self.table.cpu().numpy()
        seqs = [(int(a), int(b)) for a, b in zip(new, kv)]
        check_prefill(n64(out), None, n64(q), cu, seqs, (self.codes, self.scale, tab), self.heads, self.group, self.bs, self.d, self.dt)

    def step(self, new, decode=False):
        q, k, v = self.inputs(sum(new))
        out, slots = self.call(i32(new, self.dev), q.to(self.dev), k.to(self.dev), v.to(self.dev), decode)
        self.check(new, q, k, v, out, slots)


@pytest.mark.parametrize("bs,d,dt", [(16, 64, "bf16"), (32, 128, "f16"), (64, 128, "bf16")])
def test_a_run_of_steps(dev, bs, d, dt):
    from fastdms_b200.layers.paged_attention import release_paged_blocks
    r = Run(dev, bs + d, bs=bs, d=d, dt=dt)
    r.step([30, 5, 0, 17])
    r.step([20, 0, 41, 1])                       # a second chunk, a new prompt, a token
    for _ in range(4):
        r.step([1, 1, 1, 1], decode=True)
    release_paged_blocks(r.kv, r.table, r.free, r.count, block_size=bs, rows=i32([1, 3], dev))
    r.step([0, 9, 0, 50])
    for _ in range(3):
        r.step([1, 1, 1, 1], decode=True)
    release_paged_blocks(r.kv, r.table, r.free, r.count, block_size=bs)
    assert int(r.count) == r.pool and sorted(r.free.tolist()) == list(range(r.pool))


@pytest.mark.parametrize("cols", [20, 1250])
def test_a_captured_step_replays(dev, cols):
    """A decode step captured once advances the sequences at every replay; two captured graphs, replayed in turn, do not
    disturb each other's workspaces."""
    a, b = Run(dev, 1, cols=2500), Run(dev, 2, n=3, bs=32, d=128, dt="f16", cols=cols)
    graphs = []
    for r in (a, b):
        r.step([7 * i + 3 for i in range(r.n)])
        q, k, v = (x.to(dev) for x in r.inputs(r.n))
        new = i32([1] * r.n, dev)
        state = [x.clone() for x in (r.kv, r.count, r.table, r.kc, r.vc, r.ks, r.vs)]
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):                                         # warm-up on the capture's stream, taken back
            r.call(new, q, k, v, True)
        torch.cuda.current_stream(dev).wait_stream(side)
        for x, y in zip((r.kv, r.count, r.table, r.kc, r.vc, r.ks, r.vs), state):
            x.copy_(y)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, slots = r.call(new, q, k, v, True)
        graphs.append((r, g, q, k, v, out, slots, new))               # the graph reads `new` at every replay
    for _ in range(20):
        steps = []
        for r, g, q, k, v, out, slots, _new in graphs:
            hq, hk, hv = r.inputs(r.n)
            q.copy_(hq), k.copy_(hk), v.copy_(hv)
            g.replay()
            steps.append((hq, hk, hv))
        torch.cuda.synchronize(dev)
        for (r, g, q, k, v, out, slots, _new), (hq, hk, hv) in zip(graphs, steps):
            r.check([1] * r.n, hq, hk, hv, out, slots)


@pytest.mark.parametrize("cols", [20, 2500])
def test_two_streams_at_once(dev, cols):
    """Independent steps on two streams, interleaved without any wait between them."""
    runs = [Run(dev, 5, cols=cols), Run(dev, 6, d=128, dt="f16", cols=cols)]
    streams = [torch.cuda.Stream(dev) for _ in runs]
    for r in runs:
        r.step([300, 120, 7, 250])
    torch.cuda.synchronize(dev)
    jobs = []
    for r, s in zip(runs, streams):
        new = i32([1] * r.n, dev)
        ins = [r.inputs(r.n) for _ in range(8)]
        jobs.append((r, s, new, ins, [tuple(x.to(dev) for x in t) for t in ins], []))
    torch.cuda.synchronize(dev)
    for i in range(8):
        for r, s, new, ins, on, got in jobs:
            with torch.cuda.stream(s):
                out, slots = r.call(new, *on[i], True)
                got.append((out, slots, r.kv.clone(), r.table.clone()))
    torch.cuda.synchronize(dev)
    for r, s, new, ins, on, got in jobs:
        last = r.kv, r.table
        for i, (out, slots, kv, table) in enumerate(got):
            for c, x in ((0, ins[i][1]), (1, ins[i][2])):
                O.store(n64(x), r.codes[c], r.scale[c], slots.cpu().tolist(), r.bs)
            cu = np.arange(r.n + 1)
            check_prefill(n64(out), None, n64(ins[i][0]), cu, [(1, int(m)) for m in kv.tolist()], (r.codes, r.scale, table.cpu().numpy()),
                          r.heads, r.group, r.bs, r.d, r.dt)
        assert last[0].tolist() == got[-1][2].tolist()


@pytest.mark.parametrize("wide", [False, True])
def test_decode_and_prefill_agree_with_the_same_bits_twice(dev, wide):
    """The same call gives the same bits again, whatever the order in which CTAs finish."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    g = torch.Generator(device=dev).manual_seed(3)
    bs, heads, group, d, lens = 16, 8, 4, 128, [5000, 17, 900, 12000]
    need = [-(-m // bs) for m in lens]
    kc, vc = (torch.randn((sum(need), heads, bs, d), device=dev, generator=g).to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.exp2(torch.randint(-3, 3, (sum(need), heads), device=dev, generator=g).float()) for _ in range(2))
    table = torch.full((4, max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = torch.arange(at, at + m, device=dev)
        at += m
    q = torch.randn((4, heads * group, d), device=dev, generator=g).to(torch.bfloat16)
    if wide:
        table = wide_table(table, bs)
    first = paged_decode_attention(q, kc, vc, ks, vs, table, i32(lens, dev))
    other = paged_prefill_attention(q, kc, vc, ks, vs, table, i32(lens, dev), i32(range(5), dev))
    for _ in range(5):
        assert torch.equal(paged_decode_attention(q, kc, vc, ks, vs, table, i32(lens, dev)), first)
        assert torch.equal(paged_prefill_attention(q, kc, vc, ks, vs, table, i32(lens, dev), i32(range(5), dev)), other)
    # both compute the same thing: half a step of bf16 each, and 2^-11 of the weights' magnitude
    mag = (first.float().abs() + other.float().abs()).clamp_min(float(vs.max()) * 0.05)
    assert ((first.float() - other.float()).abs() <= mag * 2.0 ** -7).all()


def test_offsets_beyond_32_bits(dev):
    """A pool of more than 2^32 bytes, its last blocks used."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention, store_paged_kvcache
    heads, group, bs, d = 2, 4, 16, 128
    blocks = (1 << 32) // (heads * bs * d) + 8
    kc, vc = (torch.empty((blocks, heads, bs, d), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.ones((blocks, heads), device=dev) for _ in range(2))
    rng = np.random.default_rng(4)
    ids = [blocks - 1, 0, blocks - 3]
    slots = [b * bs + r for b in ids for r in range(bs)][:40]
    k, v = (_random_rows(rng, (40, heads, d), "bf16") for _ in range(2))
    store_paged_kvcache(k.to(dev), v.to(dev), kc, vc, ks, vs, i32(slots, dev))
    small = [np.full((3, heads, bs, d), 0x7F, np.uint8) for _ in range(2)]
    scale = [np.ones((3, heads)) for _ in range(2)]
    for c, x in ((0, k), (1, v)):
        O.store(n64(x), small[c], scale[c], list(range(40)), bs)
    pick = torch.tensor(ids, device=dev)
    assert np.array_equal(kc.view(torch.uint8)[pick].cpu().numpy()[:2], small[0][:2])
    q = _random_rows(rng, (1, heads * group, d), "bf16", loud=False)
    args = (kc, vc, ks, vs, i32([ids], dev), i32([40], dev))
    for got in (paged_decode_attention(q.to(dev), *args), paged_prefill_attention(q.to(dev), *args, i32([0, 1], dev))):
        for h in range(heads):
            a, b = (O.rows_of(small[c], scale[c], [0, 1, 2], 40, h, bs) for c in range(2))
            r = slice(h * group, (h + 1) * group)
            check_rows(n64(got)[0, r], None, O.attention(n64(q)[0, r], a, b, [39] * group, d ** -0.5), "bf16")
