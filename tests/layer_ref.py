"""64-bit references of the attention layer's calls, in numpy."""
from __future__ import annotations

import numpy as np

TYPES = {"f16": 1, "q4_0": 2, "q5_0": 6, "q8_0": 8}
SIZE = {"f16": 64, "q4_0": 18, "q5_0": 22, "q8_0": 34}


def row_values(raw, kind):
    """[n, row bytes] ggml rows as [n, width] float64."""
    n = raw.shape[0]
    if kind == "f16":
        return np.ascontiguousarray(raw).view(np.float16).astype(np.float64)
    b = raw.reshape(n, -1, SIZE[kind])
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    if kind == "q8_0":
        c = np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64)
    else:
        low, high = b[..., -16:] & 15, b[..., -16:] >> 4
        c = np.concatenate([low, high], -1).astype(np.float64)
        if kind == "q5_0":
            bits = np.unpackbits(np.ascontiguousarray(b[..., 2:6]), axis=-1, bitorder="little")
            c = c + 16.0 * bits - 16.0
        else:
            c = c - 8.0
    with np.errstate(invalid="ignore"):
        return (c * d).reshape(n, -1)


def quantize(x, kind):
    """float32 rows as ggml bytes (quantize_row_*_ref: 32-bit arithmetic, roundf)."""
    f32 = np.float32
    n = x.shape[0]
    if kind == "f16":
        return np.ascontiguousarray(x.astype(np.float16)).view(np.uint8)
    x = np.ascontiguousarray(x, f32).reshape(n, -1, 32)
    a = np.abs(x)
    top = a.max(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        if kind == "q8_0":
            d = top / f32(127)
            y = x * np.where(d != 0, f32(1) / d, f32(0))
            whole = np.trunc(y)
            code = whole + np.where(np.abs(y - whole) >= 0.5, np.sign(y), f32(0))
            parts = [code.astype(np.int8).view(np.uint8)]
        else:
            mid = 8 if kind == "q4_0" else 16
            d = np.take_along_axis(x, a.argmax(-1)[..., None], -1) / f32(-mid)
            c = np.trunc(x * np.where(d != 0, f32(1) / d, f32(0)) + f32(mid + 0.5)).astype(np.int64)
            c = np.minimum(c, 2 * mid - 1)
            parts = [((c[..., :16] & 15) | ((c[..., 16:] & 15) << 4)).astype(np.uint8)]
            if kind == "q5_0":
                parts.insert(0, np.packbits((c >> 4).astype(np.uint8), axis=-1, bitorder="little"))
    return np.concatenate([np.ascontiguousarray(d.astype(np.float16)).view(np.uint8)] + parts, -1).reshape(n, -1)


def attend(q, k_rows, v_rows, kinds, n_head_kv, T, n_slots, table, q_start, kv_len, scale, causal, out):
    """(out, tolerance scale): out float64 with the rows of every request filled
    in; weight[r, h, d] = sum_j p_j |v_jd| / sum_j p_j, and peak[r, h, d] the
    largest |v| a row sees."""
    rows, hq, D = q.shape
    G = hq // n_head_kv
    out = out.astype(np.float64).copy()
    spread, peak = np.zeros_like(out), np.zeros_like(out)
    kall, vall = row_values(k_rows, kinds[0]), row_values(v_rows, kinds[1])
    for s in range(len(kv_len)):
        lo, hi = int(q_start[s]), int(q_start[s + 1])
        n, kv = hi - lo, max(0, int(kv_len[s]))
        j = np.arange(min(kv, table.shape[1] * T))
        slot = table[s, j // T].astype(np.int64) if j.size else j
        seen_page = (slot >= 0) & (slot < n_slots)
        cell = np.where(seen_page, slot * T + j % T, 0)
        for i in range(n):
            r = lo + i
            if r < 0 or r >= rows:
                continue
            see = seen_page & (j <= kv - n + i) if causal else seen_page
            c = cell[see]
            for h in range(hq):
                at = slice(h // G * D, h // G * D + D)
                if c.size == 0:
                    out[r, h] = 0.0
                    continue
                x = kall[c, at] @ q[r, h].astype(np.float64) * scale
                p = np.exp(x - x.max())
                out[r, h] = p @ vall[c, at] / p.sum()
                spread[r, h] = p @ np.abs(vall[c, at]) / p.sum()
                peak[r, h] = np.abs(vall[c, at]).max(0)
    return out, spread, peak


def map_batch(past, new, free, T, table, n_rows):
    """The documented rules, request by request."""
    table = table.copy()
    B, cols = table.shape
    start, kv_len, cells, pos, seq = [0], [], np.full(n_rows, -1, np.int64), np.zeros(n_rows, np.int32), np.full(n_rows, -1, np.int32)
    asked = taken = idle = tokens = row = 0
    for i in range(B):
        p, n = int(past[i]), int(new[i])
        rows = max(n, 0)
        held, blocks = -(-p // T), -(-(p + n) // T)
        good = p >= 0 and n >= 0 and blocks <= cols and row + rows <= n_rows and p + n < 2 ** 31
        need = blocks - held if good else 0
        asked += need
        runs = good and (need == 0 or asked <= len(free))
        if runs:
            table[i, held:blocks] = free[asked - need:asked]
            taken += need
            tokens += n
        idle += not runs
        kv_len.append(p + n if runs else 0)
        for t in range(min(rows, n_rows - row)):
            pos[row + t] = (p + t) & 0x7fffffff if p >= 0 else p + t
            seq[row + t] = i
            if runs and table[i, (p + t) // T] >= 0:
                cells[row + t] = int(table[i, (p + t) // T]) * T + (p + t) % T
        row = min(row + rows, n_rows)
        start.append(row)
    return dict(table=table, q_start=np.array(start, np.int32), kv_len=np.array(kv_len, np.int32), cells=cells, pos=pos,
                seq=seq, info=np.array([taken, row, idle, tokens], np.int32))
