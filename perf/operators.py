"""What is measured of the block-scaled paged KV cache: its tables, its store and the attention that reads it.

The cache holds K and V in e4m3, `[blocks, kv_heads, block_size, head_dim]`, with one float32 scale (a power of two)
for each block and KV head; a sequence's blocks are listed in its row of a block table.  Four operators:

  tables   block tables, slot map and positions of a step, from the requests' lengths and a stack of free blocks
  store    K and V rows of a step into the cache, with the scales of the blocks that they fall into
  decode   attention of one new token of every sequence over its cached rows
  prefill  causal attention of a step's prompt tokens over their sequence's cached rows

`run` computes them in plain torch operations, or, where `own` is true, by the framework's entry points.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
SCALE_EXP_MIN, SCALE_EXP_MAX = -60, 40          # a block's scale is 2^k with k in this range
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one decode step of a full server: a token for each of 256 requests, every 16th opens a block
        {"name": "tables: decode 256", "op": "tables", "requests": 256, "new": 1, "prior": 8192, "block": 16, "spare": 1.0},
        # admission of waiting prompts at once; the pool ends before the queue does
        {"name": "tables: admit 64 prompts", "op": "tables", "requests": 64, "new": 32768, "prior": 0, "block": 32, "spare": 0.8},
        # the next prompt chunks of a few requests whose earlier chunks are stored
        {"name": "tables: chunks of 9", "op": "tables", "requests": 9, "new": 2048, "prior": 5000, "block": 64, "spare": 1.2},
        # append of a small decode batch (8 KV heads of 64), where the launch is what counts
        {"name": "store: append 8", "op": "store", "seqs": 8, "new": 1, "prior": 1291, "kv_heads": 8, "head_dim": 64, "block": 16, "dtype": "bf16"},
        # append of a large decode batch
        {"name": "store: append 256", "op": "store", "seqs": 256, "new": 1, "prior": 700, "kv_heads": 8, "head_dim": 128, "block": 32, "dtype": "f16"},
        # prompts of a prefill step, ragged, some of them later chunks that begin inside a block
        {"name": "store: prompts 16k", "op": "store", "seqs": 6, "new": 5500, "prior": 777, "kv_heads": 8, "head_dim": 128, "block": 16, "dtype": "bf16"},
        # a single short conversation: latency
        {"name": "decode: 1 x 201", "op": "decode", "seqs": 1, "kv": 201, "ragged": False, "kv_heads": 8, "group": 4, "head_dim": 128, "block": 16, "dtype": "f16"},
        # eight sequences after 8 K prompts, heads of 64: the headline's batch without eviction
        {"name": "decode: 8 x 8192", "op": "decode", "seqs": 8, "kv": 8192, "ragged": False, "kv_heads": 8, "group": 4, "head_dim": 64, "block": 16, "dtype": "bf16"},
        # mixed traffic: lengths from one token to long ones
        {"name": "decode: 64 ragged", "op": "decode", "seqs": 64, "kv": 16384, "ragged": True, "kv_heads": 8, "group": 4, "head_dim": 128, "block": 32, "dtype": "bf16"},
        # one short prompt
        {"name": "prefill: 77 tokens", "op": "prefill", "seqs": 1, "new": 77, "prior": 0, "ragged": False, "kv_heads": 8, "group": 4, "head_dim": 64, "block": 16, "dtype": "f16"},
        # a chunk of a long prompt over what is stored of it
        {"name": "prefill: chunk over 14k", "op": "prefill", "seqs": 1, "new": 2048, "prior": 14336, "ragged": False, "kv_heads": 8, "group": 4, "head_dim": 128, "block": 16, "dtype": "bf16"},
        # prompts of a step, ragged, with cached beginnings
        {"name": "prefill: 7 ragged", "op": "prefill", "seqs": 7, "new": 3001, "prior": 900, "ragged": True, "kv_heads": 8, "group": 4, "head_dim": 64, "block": 64, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "store", "decode", "prefill"])
    block = rng.choice([16, 16, 32, 64, 128])
    if op == "tables":
        step = rng.random() < 0.5
        return {"op": op, "requests": _log(rng, 1, 1024) if step else _log(rng, 1, 64), "new": 1 if step else _log(rng, 2, 16384),
                "prior": _log(rng, 1, 16384) if step or rng.random() < 0.5 else 0, "block": block, "spare": rng.choice([0.6, 1.0, 1.5])}
    heads = {"kv_heads": rng.choice([1, 2, 4, 8]), "head_dim": rng.choice([64, 128]), "block": block, "dtype": rng.choice(["bf16", "f16"])}
    if op == "store":
        step = rng.random() < 0.5
        return {"op": op, "seqs": _log(rng, 1, 256) if step else _log(rng, 1, 6), "new": 1 if step else _log(rng, 2, 5000), "prior": _log(rng, 1, 1500), **heads}
    heads["group"] = rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "decode":
        seqs = _log(rng, 1, 128)
        return {"op": op, "seqs": seqs, "kv": _log(rng, 1, min(131072, 400000 // seqs)), "ragged": rng.random() < 0.5, **heads}
    seqs = _log(rng, 1, 8)
    new = _log(rng, 1, 2048 if seqs == 1 else 3000)
    return {"op": op, "seqs": seqs, "new": new, "prior": _log(rng, 1, min(8192, 12_000_000 // (seqs * new))) if rng.random() < 0.6 else 0, "ragged": rng.random() < 0.5, **heads}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _lens(g, n, most, ragged, least=0):
    """n lengths up to `most`; ragged ones are spread evenly from `least` on, in an order of the seed's."""
    if not ragged or n == 1:
        return torch.full((n,), most, dtype=torch.int64, device="cuda")
    spread = least + torch.arange(n, device="cuda") * (most - least) // (n - 1)
    return spread[torch.randperm(n, generator=g, device="cuda")]


def _pow2_scale(amax):
    """The smallest power of two 2^k with amax <= 448 * 2^k, k held in its range."""
    m, e = torch.frexp(amax)
    k = e - torch.where(m <= 0.875, 9, 8)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, k, SCALE_EXP_MIN).clamp(SCALE_EXP_MIN, SCALE_EXP_MAX))


def _pool(g, blocks, case):
    """A cache of `blocks` filled blocks, whose magnitude differs from block to block and head to head."""
    h, b, d = case["kv_heads"], case["block"], case["head_dim"]
    loud = torch.exp2(torch.randint(-2, 2, (blocks, h, 1, 1), generator=g, device="cuda").float())
    x = torch.randn((blocks, h, b, d), generator=g, device="cuda") * loud
    s = _pow2_scale(x.abs().amax(dim=(2, 3)))
    return (x / s[:, :, None, None]).to(torch.float8_e4m3fn), s


def _tables(g, need, blocks):
    """Block tables of sequences that hold `need` blocks each, out of a shuffled pool."""
    cols = torch.arange(int(max(1, need.max())), device="cuda")
    order = torch.randperm(blocks, generator=g, device="cuda")
    first = torch.cumsum(need, 0) - need
    at = (first[:, None] + cols[None, :]).clamp(max=blocks - 1)
    return torch.where(cols[None, :] < need[:, None], order[at], -1).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, block = case["op"], case["block"]
    s = {"op": op, "block": block}
    if op == "tables":
        n = case["requests"]
        new = torch.ones(n, dtype=torch.int64, device="cuda") if case["new"] == 1 else _lens(g, n, case["new"], n > 1)
        prior = _lens(g, n, case["prior"], n > 1) if case["prior"] else torch.zeros(n, dtype=torch.int64, device="cuda")
        held, want = -(-prior // block), -(-(prior + new) // block)
        total, spare = int(new.sum()), int((want - held).sum() * case["spare"])
        blocks = int(held.sum()) + max(spare, 1)
        cols = -(-(case["new"] + case["prior"]) // block) + 3
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        first = torch.cumsum(held, 0) - held
        c = torch.arange(cols, device="cuda")
        tables = torch.where(c[None, :] < held[:, None], order[(first[:, None] + c[None, :]).clamp(max=blocks - 1)], -1).to(torch.int32)
        used = int(held.sum())
        free = torch.full((blocks,), -1, dtype=torch.int32, device="cuda")
        free[: blocks - used] = order[used:]
        s |= {"new": new.to(torch.int32), "kv": prior.to(torch.int32), "tables": tables.contiguous(), "free": free,
              "count": torch.tensor([blocks - used], dtype=torch.int32, device="cuda"), "total": total + 5}
        # the state after the step goes to buffers of its own, so that a step can be taken again from the same state
        return s | {"kv_out": torch.empty_like(s["kv"]), "count_out": torch.empty_like(s["count"])}
    n, h, d, dt = case["seqs"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    if op == "store":
        new = torch.ones(n, dtype=torch.int64, device="cuda") if case["new"] == 1 else _lens(g, n, case["new"], n > 1)
        prior = _lens(g, n, case["prior"], n > 1)
        need = -(-(prior + new) // block)
        blocks = int((prior // block + new // block).sum()) + 2 * n        # the same for every seed
        tables = _tables(g, need, blocks)
        (kc, ks), (vc, vs) = _pool(g, blocks, case), _pool(g, blocks, case)
        cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
        t = torch.arange(int(cu[-1]), device="cuda")
        seq = torch.searchsorted(cu[1:], t, right=True)
        pos = prior[seq] + t - cu[seq]
        slots = (tables[seq, pos // block].to(torch.int64) * block + pos % block).to(torch.int32)
        # the step's rows: a few tokens are much louder than the others, so that some scales have to grow
        loud = torch.where(torch.rand((t.numel(), h, 1), generator=g, device="cuda") < 0.05, 6.0, 1.0)
        k = (torch.randn((t.numel(), h, d), generator=g, device="cuda") * loud).to(dt)
        v = (torch.randn((t.numel(), h, d), generator=g, device="cuda") * loud).to(dt)
        return s | {"k": k, "v": v, "slots": slots, "kc": kc, "vc": vc, "ks": ks, "vs": vs}
    group = case["group"]
    if op == "decode":
        kv = _lens(g, n, case["kv"], case["ragged"], 1 if case["kv"] > 0 else 0)
        new = torch.ones(n, dtype=torch.int64, device="cuda")
    else:
        new = _lens(g, n, case["new"], case["ragged"])
        prior = _lens(g, n, case["prior"], case["ragged"]) if case["prior"] else torch.zeros(n, dtype=torch.int64, device="cuda")
        kv = prior + new
    need = -(-kv // block)
    blocks = int(need.sum()) + 4
    tables = _tables(g, need, blocks)
    (kc, ks), (vc, vs) = _pool(g, blocks, case), _pool(g, blocks, case)
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    q = torch.randn((int(cu[-1]), h * group, d), generator=g, device="cuda").to(dt)
    return s | {"q": q, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "tables": tables, "kv": kv.to(torch.int32), "cu": cu.to(torch.int32),
                "max_new": case["new"] if op == "prefill" else 1, "max_kv": tables.shape[1] * block}


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _plain_tables(s):
    b, new, kv, tables = s["block"], s["new"].long(), s["kv"].long(), s["tables"]
    n, cols = tables.shape
    held = (kv + b - 1) // b
    need = (kv + new + b - 1) // b - held
    end = torch.cumsum(need, 0)
    served = (need == 0) | (end <= s["count"].long())
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    c = torch.arange(cols, device=tables.device)[None, :]
    j = c - held[:, None]
    src = (s["count"].long() - 1 - (end - need))[:, None] - j
    opens = served[:, None] & (j >= 0) & (j < need[:, None])
    tables.copy_(torch.where(opens, s["free"][src.clamp(0, s["free"].numel() - 1)], tables))
    t = torch.arange(s["total"], device=tables.device)
    at = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    seq = at.clamp(max=n - 1)
    pos = kv[seq] + t - cu[seq]
    slot = tables[seq, (pos // b).clamp(max=cols - 1)].long() * b + pos % b
    slot = torch.where((at < n) & served[seq], slot, -1).to(torch.int32)
    pos = torch.where(at < n, pos, 0)
    taken = torch.where(served, need, 0).sum()
    s["kv_out"].copy_(kv + torch.where(served, new, 0))
    s["count_out"].copy_(s["count"] - taken)
    return {"cu_seqlens": cu.to(torch.int32), "kv_lens": s["kv_out"], "free_count": s["count_out"],
            "block_tables": tables, "slot_mapping": slot, "positions": pos}


def _plain_store_one(x, cache, scale, slots, b):
    blk, off = slots.long() // b, slots.long() % b
    amax = x.float().abs().amax(dim=2)                                       # [tokens, heads]
    blocks, h = scale.shape
    peak = torch.zeros((blocks, h), device=x.device).scatter_reduce(0, blk[:, None].expand(-1, h), amax, "amax")
    first = torch.full((blocks,), b, dtype=torch.int64, device=x.device).scatter_reduce(0, blk, off, "amin")
    grown = _pow2_scale(peak[blk])                                           # of the blocks that the tokens fall into
    old, before = scale[blk], first[blk]
    now = torch.where(before[:, None] > 0, torch.maximum(old, grown), grown)
    rows = cache[blk].float()                                                # [tokens, heads, block, dim]
    moved = (rows * (old / now)[:, :, None, None]).to(torch.float8_e4m3fn)
    keep = torch.arange(b, device=x.device)[None, None, :, None] < before[:, None, None, None]
    cache.view(torch.uint8)[blk] = torch.where(keep, moved.view(torch.uint8), cache.view(torch.uint8)[blk])
    rows = (x.float() / now[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    cache.view(torch.uint8).permute(0, 2, 1, 3)[blk, off] = rows.view(torch.uint8)
    scale[blk] = now


def _plain_store(s):
    _plain_store_one(s["k"], s["kc"], s["ks"], s["slots"], s["block"])
    _plain_store_one(s["v"], s["vc"], s["vs"], s["slots"], s["block"])
    return {"k_cache": s["kc"], "v_cache": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _rows(cache, scale, tables):
    """The cached rows of every sequence, padded to the longest: [seqs, heads, rows, dim] in float32."""
    t = tables.long().clamp(min=0)
    x = cache[t].float() * scale[t][..., None, None]                        # [seqs, columns, heads, block, dim]
    n, c, h, b, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(n, h, c * b, d)


def _plain_attention(s, decode):
    q, kv, cu, m = s["q"], s["kv"].long(), s["cu"].long(), s["max_new"]
    n, hq, d = kv.numel(), q.shape[1], q.shape[2]
    k, v = _rows(s["kc"], s["ks"], s["tables"]), _rows(s["vc"], s["vs"], s["tables"])
    h, g = k.shape[1], hq // k.shape[1]
    new = cu[1:] - cu[:-1]
    i = torch.arange(m, device=q.device)
    at = (cu[:-1, None] + i[None, :]).clamp(max=q.shape[0] - 1)              # [seqs, longest step]
    x = q[at].float().reshape(n, m, h, g, d).permute(0, 2, 3, 1, 4).reshape(n, h, g * m, d)
    score = torch.matmul(x, k.transpose(2, 3)).mul_(d ** -0.5).view(n, h, g, m, -1)
    sees = kv[:, None] - new[:, None] + i[None, :]                           # the last row that a token sees
    hidden = torch.arange(k.shape[2], device=q.device)[None, None, :] > sees[:, :, None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = score.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p.view(n, h, g * m, -1), v).view(n, h, g, m, d) / total.clamp(min=1e-30)
    lse = (top + total.log()).squeeze(-1)
    if decode:
        return {"out": out.reshape(n, hq, d).to(q.dtype), "lse": lse.reshape(n, hq)}
    tok = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
    j = tok - cu[seq]
    return {"out": out.permute(0, 3, 1, 2, 4)[seq, j].reshape(-1, hq, d).to(q.dtype), "lse": lse.permute(0, 3, 1, 2)[seq, j].reshape(-1, hq).t().contiguous()}


def run(s):
    if own:
        from fastdms_b200.layers import paged_attention as P
        if s["op"] == "tables":
            cu, slots, pos = P.build_paged_metadata(s["new"], s["kv"], s["tables"], s["free"], s["count"], block_size=s["block"],
                                                    total_tokens=s["total"], kv_lens_out=s["kv_out"], free_count_out=s["count_out"])
            return {"cu_seqlens": cu, "kv_lens": s["kv_out"], "free_count": s["count_out"], "block_tables": s["tables"], "slot_mapping": slots, "positions": pos}
        if s["op"] == "store":
            P.store_paged_kvcache(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
            return {"k_cache": s["kc"], "v_cache": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}
        if s["op"] == "decode":
            lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=s["q"].device)
            out = P.paged_decode_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["tables"], s["kv"], lse_out=lse)
            return {"out": out, "lse": lse}
        lse = torch.empty((s["q"].shape[1], s["q"].shape[0]), dtype=torch.float32, device=s["q"].device)
        out = P.paged_prefill_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["tables"], s["kv"], s["cu"], lse_out=lse)
        return {"out": out, "lse": lse}
    if s["op"] == "tables":
        return _plain_tables(s)
    if s["op"] == "store":
        return _plain_store(s)
    return _plain_attention(s, s["op"] == "decode")


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def _mean_len(most, ragged, least=0):
    return (most + least) / 2 if ragged else most


def work(case):
    """Bytes read once and written once, and operations; ragged lengths count with their mean."""
    op, b = case["op"], case["block"]
    if op == "tables":
        n = case["requests"]
        new = 1 if case["new"] == 1 else _mean_len(case["new"], n > 1)
        total = n * new
        return {"bytes": 4 * (5 * n + 3) + total * 12 + 8 * total / b, "flops": 0}
    n, h, d = case["seqs"], case["kv_heads"], case["head_dim"]
    if op == "store":
        new = 1 if case["new"] == 1 else _mean_len(case["new"], n > 1)
        total = n * new
        # the rows in 16 bits and out in 8, slots, scales; rows before the first of a partly filled block only move where a scale grows
        return {"bytes": total * (4 + h * d * 2 * 3) + (total / b + n) * h * 2 * 8, "flops": total * h * d * 4}
    hq = h * case["group"]
    if op == "decode":
        kv = _mean_len(case["kv"], case["ragged"] and n > 1, 1)
        rows, pairs, tokens = n * kv, n * kv, n
    else:
        new, prior = _mean_len(case["new"], case["ragged"] and n > 1), _mean_len(case["prior"], case["ragged"] and n > 1)
        rows, tokens = n * (prior + new), n * new
        pairs = n * (new * prior + new * (new + 1) / 2)
    return {"bytes": rows * h * d * 2 + rows / b * (h * 8 + 4) + tokens * hq * (4 * d + 4), "flops": 4 * pairs * hq * d}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _e4m3_of(x):
    """Nearest e4m3 value of float64 numbers, ties to even, held at +-448: steps of 2^(e-3), of 2^-9 below 2^-6."""
    m, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_store(x, cache, scale, slots, b):
    """Block by block: the loudest value sets the scale, which never falls while a block fills."""
    cache, scale = cache.double(), scale.double()
    slots = slots.long()
    x = x.double()
    starts = torch.ones_like(slots, dtype=torch.bool)
    starts[1:] = (slots[1:] % b == 0) | (slots[1:] != slots[:-1] + 1)
    run = torch.cumsum(starts, 0) - 1                                       # which run of one block a token is in
    count = int(run[-1]) + 1
    first = slots[starts]
    blk, before = first // b, first % b
    peak = x.new_zeros((count, x.shape[1])).index_reduce_(0, run, x.abs().amax(dim=2), "amax")
    k = torch.ceil(torch.log2(peak / E4M3_MAX))                              # log2 may be off by a rounding: put right below
    k = torch.where(peak > E4M3_MAX * torch.exp2(k), k + 1, k)
    k = torch.where(peak <= E4M3_MAX * torch.exp2(k - 1), k - 1, k)
    now = torch.exp2(torch.where(peak > 0, k, float(SCALE_EXP_MIN)).clamp(SCALE_EXP_MIN, SCALE_EXP_MAX))
    now = torch.where(before[:, None] > 0, torch.maximum(now, scale[blk]), now)
    for lo in range(0, count, 4096):
        c = slice(lo, lo + 4096)
        again = _e4m3_of(cache[blk[c]] * scale[blk[c]][:, :, None, None] / now[c][:, :, None, None])
        old = torch.arange(b, device=x.device)[None, None, :, None] < before[c][:, None, None, None]
        cache[blk[c]] = torch.where(old, again, cache[blk[c]])
    cache[slots // b, :, slots % b] = _e4m3_of(x / now[run][:, :, None])
    scale[blk] = now
    return cache, scale


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] == "store":
        kc, ks = _exact_store(s["k"], s["kc"], s["ks"], s["slots"], s["block"])
        vc, vs = _exact_store(s["v"], s["vc"], s["vs"], s["slots"], s["block"])
        return {"k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs}
    q, d, decode = s["q"].double(), case["head_dim"], case["op"] == "decode"
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for i, (rows, lo, hi) in enumerate(zip(s["kv"].tolist(), s["cu"].tolist(), s["cu"].tolist()[1:])):
        ids = s["tables"][i, : -(-rows // s["block"])].long()
        for h in range(case["kv_heads"]):
            k, v = ((c[ids, h].double() * f[ids, h].double()[:, None, None]).reshape(-1, d)[:rows] for c, f in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            for j in range(h * case["group"], (h + 1) * case["group"]):
                for a in range(lo, hi, 2048):                               # query tokens, in parts that fit
                    z = min(a + 2048, hi)
                    score = q[a:z, j] @ k.t() / math.sqrt(d)
                    last = torch.arange(a, z, device=q.device) - hi + rows
                    score[torch.arange(rows, device=q.device)[None, :] > last[:, None]] = -math.inf
                    lse[a:z, j] = torch.logsumexp(score, 1)
                    seen = last >= 0
                    out[a:z, j][seen] = torch.softmax(score[seen], 1) @ v
    return {"out": out, "lse": lse if decode else lse.t().contiguous()}
