"""The dense paged cache at the edges of what its calls allow: weights far below the largest, rows that sit a step out, pools
that are numbered another way, scales that nothing has written.  Beside `test_gpu_paged_attention`, whose helpers it uses."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_oracle as O
from test_gpu_paged_attention import (DT, Run, _random_rows, _status_clean, build_case, check_rows, check_store, codes_of, dev, i32, make_cache,  # noqa: F401
                                      n64, raised, wide_table)

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
