"""Plain 64-bit statement of the block-scaled paged cache's operators (numpy), for the tests."""
from __future__ import annotations

import math

import numpy as np

EXP_MIN, EXP_MAX, E4M3_MAX = -60, 40, 448.0


def decode_table() -> np.ndarray:
    """Value of every e4m3 code."""
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[c] = math.nan if (c & 0x7F) == 0x7F else v
        if c & 0x80:
            out[c] = -out[c]
    return out


VALUES = decode_table()


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest code of float64 values, ties to even, held at +-448; the sign of zero is kept."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), E4M3_MAX)
    with np.errstate(invalid="ignore"):
        e = np.maximum(np.frexp(a)[1] - 1, -6)
        r = np.rint(np.nan_to_num(a) / 2.0 ** (e - 3.0)) * 2.0 ** (e - 3.0)
        e = np.maximum(np.frexp(r)[1] - 1, -6)
        m = r / 2.0 ** (e - 3.0)                                      # 8 .. 15, below 8 for subnormals
        code = np.where(m < 8, m, (e + 7) * 8 + (m - 8)).astype(np.int64)
    code = np.where(np.isnan(x), 0x7F, code) | np.where(np.signbit(x), 0x80, 0)
    return code.astype(np.uint8)


def scale_of(amax: float) -> float:
    if not amax > 0:
        return 2.0 ** EXP_MIN
    k = EXP_MIN
    while k < EXP_MAX and amax > E4M3_MAX * 2.0 ** k:
        k += 1
    return 2.0 ** k


def store(x, codes, scale, slots, block_size):
    """Stores x [tokens, heads, dim] (float64) into codes [blocks, heads, bs, dim] (uint8) / scale [blocks, heads], in place."""
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % block_size:
            n += 1
        b, off = slots[t] // block_size, slots[t] % block_size
        for h in range(x.shape[1]):
            rows = x[t:t + n, h]
            mag = np.abs(rows)
            s = scale_of(float(np.max(mag[~np.isnan(mag)], initial=0.0)))
            if off and scale[b, h] > s:
                s = float(scale[b, h])
            if off and scale[b, h] < s:
                codes[b, h, :off] = encode(VALUES[codes[b, h, :off]] * (float(scale[b, h]) / s))
            codes[b, h, off:off + n] = encode(rows / s)
            scale[b, h] = s
        t += n


def tables(new, kv, table, free, count, block_size, total):
    """One step: (cu, kv_out, table_out, count_out, slots, positions), sequence by sequence."""
    table, kv_out = table.copy(), kv.copy()
    slots, pos = np.full(total, -1, np.int64), np.zeros(total, np.int64)
    cu, left, dry = [0], int(count), False
    for i in range(len(new)):
        held, want = -(-kv[i] // block_size), -(-(kv[i] + new[i]) // block_size)
        need = want - held
        ok = need == 0 or (not dry and need <= left)
        if need and not ok:
            dry = True
        if ok:
            for j in range(need):
                left -= 1
                table[i, held + j] = free[left]
            kv_out[i] = kv[i] + new[i]
        for j in range(new[i]):
            p = kv[i] + j
            pos[cu[-1] + j] = p
            if ok:
                slots[cu[-1] + j] = table[i, p // block_size] * block_size + p % block_size
        cu.append(cu[-1] + int(new[i]))
    return np.array(cu), kv_out, table, left, slots, pos


def rows_of(codes, scale, table_row, n, head, block_size):
    """The first n cached rows of a sequence, [n, dim] in float64."""
    ids = np.asarray(table_row[: -(-n // block_size)], np.int64)
    x = VALUES[codes[ids, head]] * scale[ids, head].astype(np.float64)[:, None, None]
    return x.reshape(-1, codes.shape[3])[:n]


def attention(q, k, v, last, scale):
    """Softmax attention of rows q [n, dim] over k, v [rows, dim], row i seeing keys 0 .. last[i]; with it the bound that the
    kernels' roundings give for each output (before its own), and that of the log-sum-exp."""
    n, d = q.shape
    out, lse = np.zeros((n, d)), np.full(n, -np.inf)
    tol, ltol = np.zeros((n, d)), np.zeros(n)
    for i in range(n):
        m = int(last[i]) + 1
        if m <= 0:
            continue
        s = (k[:m] @ q[i]) * scale
        top = s.max()
        p = np.exp(s - top)
        w = p / p.sum()
        out[i] = w @ v[:m]
        lse[i] = top + math.log(p.sum())
        # a score: float32 products added in any order and truncated (2^-23 a step), then one multiply-add in the exponent
        mag = float((np.abs(k[:m]) @ np.abs(q[i])).max()) * abs(scale)
        ds = mag * (d + 4) * 2.0 ** -23 + (np.abs(s).max() * 1.45 + 64) * 2.0 ** -23
        # a weight: half a step of f16 (2^-11), or of its subnormals (2^-25 of weights that are 1 at the top); the sums
        tol[i] = (np.abs(v[:m]).T @ w) * (2.0 ** -11 + 2 * ds + m * 2.0 ** -24) + m * 2.0 ** -25 * np.abs(v[:m]).max() * 2
        ltol[i] = ds + m * 2.0 ** -24 + (abs(lse[i]) + 64) * 2.0 ** -23
    return out, lse, tol, ltol


def attention_tight(q, k, v, vs, last, scale, f16, terms=None):
    """As `attention`, with what the type leaves of a weight and what every key's own V makes of it.  `vs [rows]` are the
    scales of the keys' blocks; `terms`: products of a score that are not zero.

    A weight is an f16 value, or for f16 outputs two of them: 2^-11 or 2^-22 of it, or 2^-25 where f16 has no finer steps (three
    times: the value, the rest, a change of M).  The weights 2^(x + log2 vs - M) of a row sum to 2^6 at least (prefill; 2^7 in
    decode), so that 3 * 2^-25 is 3 * 2^-31 of the sum of w_j vs_j at most; a key's term is that times v_j / vs_j."""
    n, d = q.shape
    out, lse = np.zeros((n, d)), np.full(n, -np.inf)
    tol, ltol = np.zeros((n, d)), np.zeros(n)
    for i in range(n):
        m = int(last[i]) + 1
        if m <= 0:
            continue
        s = (k[:m] @ q[i]) * scale
        top = s.max()
        p = np.exp(s - top)
        w = p / p.sum()
        out[i] = w @ v[:m]
        lse[i] = top + math.log(p.sum())
        mag = float((np.abs(k[:m]) @ np.abs(q[i])).max()) * abs(scale)
        ds = mag * ((d if terms is None else terms) + 4) * 2.0 ** -23 + (np.abs(s).max() * 1.45 + 64) * 2.0 ** -23
        tol[i] = (np.abs(v[:m]).T @ w) * ((2.0 ** -22 if f16 else 2.0 ** -11) + 2 * ds + m * 2.0 ** -24)
        tol[i] += 3 * 2.0 ** -31 * (w * vs[:m]).sum() * (np.abs(v[:m]) / vs[:m, None]).sum(0)
        ltol[i] = ds + m * 2.0 ** -24 + (abs(lse[i]) + 64) * 2.0 ** -23
    return out, lse, tol, ltol
