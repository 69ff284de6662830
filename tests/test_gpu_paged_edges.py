"""The dense paged cache at the edges of what its calls allow: weights far below the largest, rows that sit a step out, pools
that are numbered another way, scales that nothing has written.  Beside `test_gpu_paged_attention`, whose helpers it uses."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_oracle as O
from test_gpu_paged_attention import (DT, Run, _random_rows, _status_clean, build_case, check_prefill, check_rows, check_store, codes_of,  # noqa: F401
                                      dev, i32, make_cache, n64, raised, wide_table)

pytestmark = pytest.mark.gpu


def one_sequence(dev, k, v, bs=16):
    """A cache that holds one sequence of one KV head: k, v [rows, d] of values that are e4m3 codes under a scale of 1."""
    rows, d = k.shape
    blocks = -(-rows // bs)
    out = []
    for x in (k, v):
        c = np.zeros((blocks * bs, d), np.uint8)
        c[:rows] = O.encode(x)
        assert np.array_equal(O.VALUES[c[:rows]], x)
        out.append(torch.from_numpy(c.reshape(blocks, 1, bs, d)).to(dev).view(torch.float8_e4m3fn))
    return (*out, torch.ones((blocks, 1), device=dev), torch.ones((blocks, 1), device=dev), torch.arange(blocks, dtype=torch.int32, device=dev)[None])


# ---- weights -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("form,rows,seqs", [("prefill", 131072, 1), ("decode", 2000, 600)])
def test_many_quiet_keys_behind_a_loud_one(dev, form, rows, seqs, dt, wide):
    """One key 17.5 above all others, whose V is zero: what comes out is the sum of weights of 2^-25 each."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    d, scale = 64, 0.125
    k, v = np.zeros((rows, d)), np.full((rows, d), 192.0)
    loud = rows // 2
    k[loud, 0], v[loud] = 8.0, 0.0
    kc, vc, ks, vs, table = one_sequence(dev, k, v)
    q = torch.zeros((seqs, 2, d), dtype=DT[dt])
    q[:, :, 0] = 17.5
    table = table.expand(seqs, table.shape[1])                               # every sequence reads the same blocks
    if wide:
        table = wide_table(table, 16, 200000)
    lens, lse = i32([rows] * seqs, dev), torch.empty((seqs, 2), device=dev)
    if form == "decode":
        got = paged_decode_attention(q.to(dev), kc, vc, ks, vs, table, lens, scale, lse_out=lse)
    else:
        got = paged_prefill_attention(q.to(dev), kc, vc, ks, vs, table, lens, i32([0, 1], dev), scale, lse_out=lse.t())
    want = O.attention_tight(n64(q)[0, :1], k, v, np.ones(rows), [rows - 1], scale, dt == "f16", terms=1)
    for r in (got[0, :1], got[seqs - 1, 1:]):
        check_rows(n64(r), n64(lse)[0, :1], want, dt)
    assert (got == got[0, 0]).all()


@pytest.mark.parametrize("jump", [False, True])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("form", ["prefill", "decode"])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_weights_whose_roundings_add_up(dev, form, dt, wide, jump):
    """Two kinds of keys with V of 1 and -1, all of a kind with the same weight: the roundings of a kind do not cancel while the
    output nearly does, so that an f16 output shows whether a weight's rest has come along.  With `jump` a key in the
    second 32 of a step's half is louder by 2^8 or so, and what is there of the first 32 follows M down."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    d, rows, heads = 64, 200, 32
    k, v = np.zeros((rows, d)), np.ones((rows, d))
    k[::2, 0], k[1::2, 0], v[1::2] = 1.0, 0.9375, -1.0
    if jump:
        k[104, 0], v[104] = 2.5, 0.0
    kc, vc, ks, vs, table = one_sequence(dev, k, v)
    if wide:
        table = wide_table(table, 16)
    q = torch.zeros((1, heads, d), dtype=DT[dt])
    q[0, :, 0] = torch.linspace(3.5, 4.5, heads)
    if form == "decode":
        got = paged_decode_attention(q.to(dev), kc, vc, ks, vs, table, i32([rows], dev), 1.0)
    else:
        got = paged_prefill_attention(q.to(dev), kc, vc, ks, vs, table, i32([rows], dev), i32([0, 1], dev), 1.0)
    check_rows(n64(got)[0], None, O.attention_tight(n64(q)[0], k, v, np.ones(rows), [rows - 1] * heads, 1.0, dt == "f16", terms=1), dt)


# ---- rows that sit a step out --------------------------------------------------------------------------------------

@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d,dt,spare", [(64, "bf16", 0), (128, "f16", 2)])
def test_decode_finds_the_token_of_a_sequence(dev, d, dt, spare, wide):
    """Sequences without a token between others, one of them empty; `spare` rows of q are nobody's."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention
    rng = np.random.default_rng(d)
    heads, group, bs = 2, 4, 16
    lens, new = [40, 333, 0, 7, 90, 0, 1], [1, 0, 1, 1, 0, 0, 1]
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, lens, heads, bs, d, dev)
    if wide:
        table = wide_table(table, bs)
    tokens = sum(new) + spare
    q = _random_rows(rng, (tokens, heads * group, d), dt, loud=False)
    out, lse = torch.full(q.shape, 3.0, dtype=DT[dt], device=dev), torch.full((tokens, heads * group), 7.0, device=dev)
    cu = np.concatenate([[0], np.cumsum(new)])
    got = paged_decode_attention(q.to(dev), kc, vc, ks, vs, table, i32(lens, dev), cu_seqlens_q=i32(cu, dev), out=out, lse_out=lse)
    assert (got[sum(new):] == 3.0).all() and (lse[sum(new):] == 7.0).all()
    for b, m in enumerate(lens):
        if not new[b]:
            continue
        for h in range(heads):
            k, v = (O.rows_of(codes[c], scale[c], tab[b], m, h, bs) for c in range(2))
            r = slice(h * group, (h + 1) * group)
            check_rows(n64(got)[cu[b], r], n64(lse)[cu[b], r], O.attention(n64(q)[cu[b], r], k, v, [m - 1] * group, d ** -0.5), dt)
    # the same bits as the sequences of the tokens by themselves
    have = torch.tensor([b for b in range(len(lens)) if new[b]], device=dev)
    alone = paged_decode_attention(q[:sum(new)].to(dev), kc, vc, ks, vs, table[have].contiguous(), i32(np.asarray(lens)[have.cpu()], dev))
    half = torch.finfo(DT[dt]).eps
    assert ((got[:sum(new)].float() - alone.float()).abs() <= half * alone.float().abs() + half * float(vs.nan_to_num().max())).all()
    # several tokens, or one beyond q: left out, and said
    for broken in ([0, 2, 2, 3, 4, 4, 4, 4], [0, 1, 1, 2, 3, 3, 3, tokens + 1], [-1, 0, 0, 0, 0, 0, 0, 0]):
        out = torch.full(q.shape, 3.0, dtype=DT[dt], device=dev)
        paged_decode_attention(q.to(dev), kc, vc, ks, vs, table, i32(lens, dev), cu_seqlens_q=i32(broken, dev), out=out)
        assert raised(dev)
        held = [a for a, b in zip(broken, broken[1:]) if a >= 0 and b == a + 1 and a < tokens]
        assert all((out[t] == 3.0).all() == (t not in held) for t in range(tokens))
    nobody = paged_decode_attention(q[:0].to(dev), kc, vc, ks, vs, table, i32(lens, dev), cu_seqlens_q=i32([0] * 8, dev))
    assert nobody.shape[0] == 0


@pytest.mark.parametrize("cols", [20, 2500])
def test_a_captured_step_with_rows_that_have_ended(dev, cols):
    """A decode step of four rows, captured once: rows are released, sit steps out and come back between its replays."""
    from fastdms_b200.layers import paged_attention as P
    r = Run(dev, 9, cols=cols)
    r.step([30, 5, 44, 17])
    q, k, v = (x.to(dev) for x in r.inputs(r.n))
    new = i32([1] * r.n, dev)

    def call():
        cu, slots, _ = P.build_paged_metadata(new, r.kv, r.table, r.free, r.count, block_size=r.bs, total_tokens=r.n)
        P.store_paged_kvcache(k, v, r.kc, r.vc, r.ks, r.vs, slots)
        return P.paged_decode_attention(q, r.kc, r.vc, r.ks, r.vs, r.table, r.kv, cu_seqlens_q=cu), slots

    state = [x.clone() for x in (r.kv, r.count, r.table, r.kc, r.vc, r.ks, r.vs)]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream(dev).wait_stream(side)
    for x, y in zip((r.kv, r.count, r.table, r.kc, r.vc, r.ks, r.vs), state):
        x.copy_(y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, slots = call()

    def replay(step):
        new.copy_(i32(step, dev))
        ins = r.inputs(r.n)
        for x, y in zip((q, k, v), ins):
            x.copy_(y)
        g.replay()
        torch.cuda.synchronize(dev)
        r.check(step, *ins, out, slots)

    replay([1, 1, 1, 1])
    P.release_paged_blocks(r.kv, r.table, r.free, r.count, block_size=r.bs, rows=i32([1], dev))
    for _ in range(18):
        replay([1, 0, 1, 1])
    replay([0, 0, 0, 1])
    replay([0, 1, 1, 0])                         # the released row starts again, others wait
    replay([0, 0, 0, 0])
    replay([1, 1, 1, 1])


def test_layer_decodes_with_rows_that_sit_out(dev):
    """`Attention` gives its decode the offsets of the context."""
    from fastdms_b200.layers import paged_attention as P
    from fastdms_b200.layers.attention import Attention
    from fastdms_b200.utils.context import reset_context, set_context
    r = Run(dev, 10)
    r.step([30, 5, 44, 17])
    layer = Attention(r.heads * r.group, r.d, r.d ** -0.5, r.heads)
    layer.k_cache, layer.v_cache, layer.k_cache_scale, layer.v_cache_scale = r.kc, r.vc, r.ks, r.vs
    for new in ([1, 0, 1, 1], [0, 1, 0, 0], [1, 1, 1, 1]):
        q, k, v = r.inputs(sum(new))
        cu, slots, _ = P.build_paged_metadata(i32(new, dev), r.kv, r.table, r.free, r.count, block_size=r.bs, total_tokens=sum(new))
        try:
            set_context(False, cu_seqlens_q=cu, slot_mapping=slots, context_lens=r.kv, block_tables=r.table)
            out = layer(q.to(dev), k.to(dev), v.to(dev))
        finally:
            reset_context()
        r.check(new, q, k, v, out, slots)


# ---- pools whose stack does not hold every block -------------------------------------------------------------------

@pytest.mark.parametrize("first,blocks", [(1, 12), (20, 31)])
def test_release_into_a_stack_of_part_of_the_pool(dev, first, blocks):
    """Blocks below `first` are kept for something else, so that ids reach beyond the stack's length."""
    from fastdms_b200.layers.paged_attention import build_paged_metadata, release_paged_blocks
    n = blocks - first
    free, count = torch.arange(first, blocks, dtype=torch.int32, device=dev), i32([n], dev)
    kv, table = i32([0, 0, 0], dev), i32(np.full((3, 8), -1), dev)
    for _ in range(3):
        build_paged_metadata(i32([40, 16, 70], dev), kv, table, free, count, block_size=16, total_tokens=126)
        assert int(count) == n - 9 and kv.tolist() == [40, 16, 70]
        release_paged_blocks(kv, table, free, count, block_size=16, rows=i32([2, 0], dev), num_blocks=blocks)
        release_paged_blocks(kv, table, free, count, block_size=16, num_blocks=blocks)
        assert int(count) == n and sorted(free.tolist()) == list(range(first, blocks)) and (table == -1).all()
    # an id beyond the pool is no block of it
    kv, table = i32([40], dev), i32([[first, blocks, first + 1]], dev)
    count = i32([n - 2], dev)
    release_paged_blocks(kv, table, free, count, block_size=16, num_blocks=blocks)
    assert raised(dev) and int(count) == n and free[n - 2:].tolist() == [first + 1, first]


# ---- slot maps with gaps -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("gap", [1, 2, 31, 32, 33, 255, 257, 700])
@pytest.mark.parametrize("tokens", [0, 3000])
def test_store_skips_what_returns_to_a_block_after_a_gap(dev, gap, tokens):
    """A block's tokens with skipped ones between them would be two runs in one block, at the same time: the later one is left out
    and said.  Sequences on both sides of such a gap are stored.  `tokens`: a prompt before, with which the kernel takes several
    tokens per CTA and a warp per 16 rows."""
    from fastdms_b200.layers.paged_attention import store_paged_kvcache
    rng = np.random.default_rng(gap + tokens)
    heads, d, bs = 2, 64, 32
    blocks = 8 + -(-tokens // bs)
    prompt = [8 * bs + i for i in range(tokens)]
    skip = [-1] * gap
    for after, lost in (([6, 7], 2), ([5, 6, 7], 3), ([0, 1], 2), ([bs + 3, bs + 4], 0), ([2 * bs, 2 * bs + 1], 0)):
        slots = prompt + [3, 4] + skip + after + [-1] + [3 * bs + 9]
        kc, vc, ks, vs = make_cache(blocks, heads, bs, d, dev, fill=0x30)
        ks.fill_(1.0), vs.fill_(2.0 ** -3)
        want = [codes_of(kc), codes_of(vc), np.full((blocks, heads), 1.0), np.full((blocks, heads), 2.0 ** -3)]
        k, v = _random_rows(rng, (len(slots), heads, d), "bf16"), _random_rows(rng, (len(slots), heads, d), "bf16")
        k[-2 - lost:] *= 16                                                  # louder: the scale would move
        store_paged_kvcache(k.to(dev), v.to(dev), kc, vc, ks, vs, i32(slots, dev))
        assert raised(dev) == (lost > 0)
        kept = list(slots)
        for i in range(lost):
            kept[tokens + 2 + gap + i] = -1
        O.store(n64(k), want[0], want[2], kept, bs)
        O.store(n64(v), want[1], want[3], kept, bs)
        check_store(kc, vc, ks, vs, want)


# ---- scales that the store did not write ---------------------------------------------------------------------------

@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d,dt", [(64, "bf16"), (128, "f16")])
def test_scales_of_zero_and_nan(dev, d, dt, wide):
    """A block whose V scale is 0 holds values of 0, which count in the softmax, whatever its codes are; one of NaN makes NaN of the
    rows that see it.  Decode and prefill say the same."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    rng = np.random.default_rng(d)
    heads, group, bs, rows = 2, 4, 16, 300
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, [rows], heads, bs, d, dev, loud=False)
    if wide:
        table = wide_table(table, bs)
    q = _random_rows(rng, (1, heads * group, d), dt, loud=False)

    def both(t, head, lens=rows):
        args = (q.to(dev), kc, vc, ks, t, table, i32([lens], dev))
        got = [paged_decode_attention(*args), paged_prefill_attention(*args, i32([0, 1], dev))]
        return [n64(x)[0, head * group:(head + 1) * group] for x in got]

    for zeros in ([0], [3, 4, 9], list(range(19))):
        now = scale[1].copy()
        now[tab[0, zeros], 1] = 0.0
        t = torch.from_numpy(now).float().to(dev)
        k, v = (O.rows_of(codes[c], s, tab[0], rows, 1, bs) for c, s in ((0, scale[0]), (1, now)))
        r = slice(group, 2 * group)
        # a code of 448 at a scale of 2^-60 in place of 0
        out, lse, tol, ltol = O.attention(n64(q)[0, r], k, v, [rows - 1] * group, d ** -0.5)
        for got in both(t, 1):
            check_rows(got, None, (out, lse, tol + 448 * 2.0 ** -60, ltol), dt)
    t = vs.clone()
    t[int(tab[0, 5]), 0] = float("nan")
    for got, other in zip(both(t, 0), both(t, 1)):
        assert np.isnan(got).all() and np.isfinite(other).all()
    for got in both(t, 0, 80):                   # its rows lie behind the last
        assert np.isfinite(got).all()
    # a prompt: the rows before the block's do not see it
    n, first = 250, int(5 * bs)
    q = _random_rows(rng, (n, heads * group, d), dt, loud=False)
    for at in (table, table[:, :-(-rows // bs)]):
        clean, got = (n64(paged_prefill_attention(q.to(dev), kc, vc, ks, x, at, i32([n], dev), i32([0, n], dev))) for x in (vs, t))
        assert np.isnan(got[first:, :group]).all() and np.array_equal(got[:first], clean[:first]) and np.array_equal(got[:, group:], clean[:, group:])


# ---- sizes ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("pages", [(1 << 30) + 5, (1 << 31) - 1 - 2048 * 24])
def test_decode_of_tables_for_very_many_rows(dev, pages):
    """The pages that the tables may hold are counted in 31 bits: 2048 sequences of which two hold rows, all with the same wide row."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention
    rng = np.random.default_rng(3)
    seqs, bs, d, rows = 2048, 16, 64, 900
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, [rows], 1, bs, d, dev)
    cols = pages // seqs
    wide = torch.full((1, cols), -1, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    lens = [0] * seqs
    lens[3], lens[2047] = rows, 70
    q = _random_rows(rng, (seqs, 2, d), "bf16", loud=False)
    got = n64(paged_decode_attention(q.to(dev), kc, vc, ks, vs, wide.expand(seqs, cols), i32(lens, dev)))
    for b in (3, 2047):
        k, v = (O.rows_of(codes[c], scale[c], tab[0], lens[b], 0, bs) for c in range(2))
        check_rows(got[b], None, O.attention(n64(q)[b], k, v, [lens[b] - 1] * 2, d ** -0.5), "bf16")
    got[[3, 2047]] = 0
    assert (got == 0).all()
    with pytest.raises(RuntimeError, match="too many rows"):
        cols = ((1 << 31) - 1) // seqs + 1
        wide = torch.full((1, cols), -1, dtype=torch.int32, device=dev)
        paged_decode_attention(q.to(dev), kc, vc, ks, vs, wide.expand(seqs, cols), i32([0] * seqs, dev))


# ---- queries -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("power", [122, 114, 100, -100, -125])
def test_queries_at_the_ends_of_bfloat16(dev, power, wide):
    """Queries near bf16's largest and smallest numbers, with a scale that brings the scores back."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    rng = np.random.default_rng(power + 200)
    heads, group, bs, d, rows = 1, 8, 16, 64, 90
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, [rows], heads, bs, d, dev, loud=False)
    if wide:
        table = wide_table(table, bs)
    x = np.clip(rng.standard_normal((1, heads * group, d)), -1.9, 1.9)
    q = torch.from_numpy(x * 2.0 ** power).to(torch.bfloat16)
    small = q.abs().double() < 2.0 ** -126                                   # what bf16 holds as a subnormal counts as 0
    q = torch.where(small, torch.zeros_like(q), q)
    back = 2.0 ** (-3 - power)
    args = (q.to(dev), kc, vc, ks, vs, table, i32([rows], dev))
    k, v = (O.rows_of(codes[c], scale[c], tab[0], rows, 0, bs) for c in range(2))
    want = O.attention(n64(q)[0], k, v, [rows - 1] * group, back)
    for got in (paged_decode_attention(*args, back), paged_prefill_attention(*args, i32([0, 1], dev), back)):
        check_rows(n64(got)[0], None, want, "bf16")


@pytest.mark.parametrize("form,seqs", [("decode", 600), ("prefill", 1)])
def test_scores_whose_steps_are_coarse(dev, form, seqs):
    """Scores of 2^24 to 2^29 times log2(e): what lies between two neighbouring float32 numbers there is the room that the weights
    have, so that M and the bound of a weight are rounded themselves.  No weight may leave f16 for it."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    d, rows, heads = 64, 300, 24
    k, v = np.zeros((rows, d)), np.ones((rows, d))
    k[:, 0] = k[:, 2] = 1.0
    k[200, 1], v[200] = 1.0, 2.0                                             # ahead of the keys before it by a few such steps
    kc, vc, ks, vs, table = one_sequence(dev, k, v)
    for dt in ("bf16", "f16"):
        q = torch.zeros((1, heads, d), dtype=torch.float64)
        for h in range(heads):
            q[0, h, 0] = 2.0 ** (24 + h % 6)
            q[0, h, 1] = 2.0 ** (1 + h // 6) * (1 + (h % 2) / 2)
            q[0, h, 2] = 2.0 ** (1 + h % 5)
        scale = float(np.log(2.0))
        if dt == "f16":                                                      # the same scores from queries that f16 holds
            q, scale = q * 2.0 ** -15, scale * 2.0 ** 15
        q = q.to(DT[dt])
        assert (q[0, :, 0] > 0).all() and torch.isfinite(q.float()).all()
        args = (q.to(dev).expand(seqs, heads, d).contiguous(), kc, vc, ks, vs, table.expand(seqs, table.shape[1]), i32([rows] * seqs, dev))
        lse = torch.empty((seqs, heads), device=dev)
        if form == "decode":
            got = paged_decode_attention(*args, scale, lse_out=lse)
        else:
            got = paged_prefill_attention(*args, i32([0, 1], dev), scale, lse_out=lse.t())
        assert torch.isfinite(got.float()).all() and torch.isfinite(lse).all()
        assert (got >= 1.0).all() and (got <= 2.0).all()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d,dt,power", [(64, "bf16", 28), (128, "bf16", 40), (64, "bf16", 100), (128, "f16", 13)])
def test_scores_beyond_float32s_whole_numbers(dev, d, dt, power, wide):
    """Scores so loud that one key takes all: its row of V comes out, from decode and from prefill, of tokens that see it and of
    tokens that do not; rows of ordinary queries between them give the bits that they give alone."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    rng = np.random.default_rng(power)
    heads, group, bs, rows, n = 1, 8, 16, 700, 40
    (kc, vc, ks, vs, table), (codes, scale, tab) = build_case(rng, [rows], heads, bs, d, dev, loud=False)
    if wide:
        table = wide_table(table, bs)
    x = rng.standard_normal((n, group, d))
    calm = torch.from_numpy(x).to(DT[dt])
    x[:, ::2] *= 2.0 ** power
    q = torch.from_numpy(x).to(DT[dt])
    mul = 2.0 ** 15 if dt == "f16" else 1.0
    k, v = (O.rows_of(codes[c], scale[c], tab[0], rows, 0, bs) for c in range(2))
    args = (kc, vc, ks, vs, table, i32([rows], dev))
    lse = torch.empty((group, n), device=dev)
    pre = n64(paged_prefill_attention(q.to(dev), *args, i32([0, n], dev), mul, lse_out=lse))
    dec = n64(paged_decode_attention(q[-1:].to(dev), *args, mul))
    if mul == 1.0:
        ref = n64(paged_prefill_attention(calm.to(dev), *args, i32([0, n], dev), mul))
        assert np.array_equal(pre[:, 1::2], ref[:, 1::2])
    half, checked = torch.finfo(DT[dt]).eps / 2, 0
    for i in range(n):
        for h in range(0, group, 2):
            s = k[:rows - n + i + 1] @ n64(q)[i, h] * mul
            top = np.sort(s)[-2:]
            mag = (np.abs(k) @ np.abs(n64(q)[i, h])).max() * mul
            if top[1] - top[0] <= 64 + mag * (d + 8) * 2.0 ** -22:          # nearer than the scores' own roundings
                continue
            want = v[s.argmax()]
            checked += 1
            for got in (pre[i, h], dec[0, h])[:2 if i == n - 1 else 1]:
                assert (np.abs(got - want) <= half * np.abs(want)).all()
            assert abs(float(lse[h, i]) - top[1]) <= mag * (d + 8) * 2.0 ** -22
    assert checked > n


# ---- caches --------------------------------------------------------------------------------------------------------

def test_a_cache_without_blocks(dev):
    """Rows that no block can hold are left out and said, by both forms; without rows nothing is wrong."""
    from fastdms_b200.layers.paged_attention import paged_decode_attention, paged_prefill_attention
    cache = make_cache(0, 1, 16, 64, dev)
    q = torch.ones((2, 4, 64), dtype=torch.bfloat16, device=dev)
    for cols in (2, 5000):
        table = torch.zeros((2, cols), dtype=torch.int32, device=dev)
        for lens in ([0, 0], [3, 0]):
            assert (paged_decode_attention(q, *cache, table, i32(lens, dev)) == 0).all()
            assert raised(dev) == any(lens)
            assert (paged_prefill_attention(q, *cache, table, i32(lens, dev), i32([0, 1, 2], dev)) == 0).all()
            assert raised(dev) == any(lens)


# ---- prefill beside itself -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("cols", [20, 2500])
def test_prefill_on_two_streams_and_captured(dev, cols):
    """Prompt steps of two servers on two streams without any wait between them, eager and from graphs; with wide tables the rows are
    cut into parts, whose workspaces must not meet."""
    runs = [Run(dev, 21, cols=cols, pool=90), Run(dev, 22, d=128, dt="f16", cols=cols, pool=90)]
    streams = [torch.cuda.Stream(dev) for _ in runs]
    step = [9, 0, 40, 3]
    for r in runs:
        r.step([60, 120, 7, 100])
    jobs = []
    for r, s in zip(runs, streams):
        ins = [r.inputs(sum(step)) for _ in range(3)]
        jobs.append((r, s, i32(step, dev), ins, [tuple(x.to(dev) for x in t) for t in ins], []))
    torch.cuda.synchronize(dev)
    for i in range(3):
        for r, s, new, ins, on, got in jobs:
            with torch.cuda.stream(s):
                got.append(r.call(new, *on[i], False))
                got[-1] += tuple(x.clone() for x in (r.kv, r.table))
    torch.cuda.synchronize(dev)
    for r, s, new, ins, on, got in jobs:
        cu = np.concatenate([[0], np.cumsum(step)])
        for (q, k, v), (out, slots, kv, table) in zip(ins, got):
            for c, x in ((0, k), (1, v)):
                O.store(n64(x), r.codes[c], r.scale[c], slots.cpu().tolist(), r.bs)
            check_prefill(n64(out), None, n64(q), cu, [(a, int(m)) for a, m in zip(step, kv.tolist())], (r.codes, r.scale, table.cpu().numpy()),
                          r.heads, r.group, r.bs, r.d, r.dt)
    graphs = []
    for r, s, new, ins, on, got in jobs:
        g, live = torch.cuda.CUDAGraph(), [x.clone() for x in on[0]]
        with torch.cuda.graph(g, stream=s):
            out, slots = r.call(new, *live, False)
        graphs.append((r, s, g, new, live, out, slots))
    for _ in range(2):
        fed = []
        for r, s, g, new, live, out, slots in graphs:
            ins = r.inputs(sum(step))
            for x, y in zip(live, ins):
                x.copy_(y)
            fed.append(ins)
        torch.cuda.synchronize(dev)
        for r, s, g, new, live, out, slots in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize(dev)
        for (r, s, g, new, live, out, slots), ins in zip(graphs, fed):
            r.check(step, *ins, out, slots)
