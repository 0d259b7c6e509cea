"""The attention layer around a quantized KV window, operator by operator: the
cases that are timed, their plain forms in elementary torch operations, and the
calls of this repository's own kernels for the same work.

Four kinds of pass (the "kind" of a case):

  map   the step's block tables and cell map from the requests' lengths:
        kvm.map_batch
  rope  RMS norm of every query and key head with the position rotation:
        kvm.qk_norm_rope
  rows  K and V rows quantized into the cells of the window and read back as
        values: kvm.write_rows, kvm.read_rows
  attn  attention of the step's queries over the quantized window:
        kvm.attend

A window (cache) is ggml rows: token t of slot s is the row s*T + t ("cell") of
n_head_kv*head_dim values, in blocks of 32 values: F16, Q8_0 (f16 scale, 32
int8), Q5_0 (f16 scale, 32 high bits, 16 bytes of low nibbles) or Q4_0 (f16
scale, 16 bytes; byte j holds values j and j + 16).
"""
import os
import random
import sys

import torch

own = False

TYPES = {"f16": 1, "q4_0": 2, "q5_0": 6, "q8_0": 8}
BLOCK_BYTES = {"f16": 64, "q4_0": 18, "q5_0": 22, "q8_0": 34}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DTYPE_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
WORK_BYTES = 32 << 20          # kvm.attend's workspace


def _kvm():
    package = os.path.join(os.getcwd(), "kvmem-llama.cpp_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kvm
    return kvm


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # one decode step of 64 sessions: the smallest call, all latency
        dict(name="map_decode_64", kind="map", n_seq=64, tokens=128, past_max=49152, new_max=1, pad=0),
        # a prefill step: 512 requests of ragged prompts, a padded batch
        dict(name="map_prefill_512", kind="map", n_seq=512, tokens=128, past_max=16384, new_max=1024, pad=1000),
        # decode of 64 sessions, 24 query and 4 KV heads of 256
        dict(name="rope_decode_64", kind="rope", n=64, hq=24, hkv=4, d=256, rot=64, dtype="bf16", pos_max=1 << 20),
        # one large prefill batch of the same layer
        dict(name="rope_prefill_8192", kind="rope", n=8192, hq=24, hkv=4, d=256, rot=256, dtype="bf16", pos_max=1 << 18),
        # the decode step's rows into 4-bit windows and back
        dict(name="rows_decode_64", kind="rows", n=64, hkv=4, d=256, tokens=128, slots=96, tk="q4_0", tv="q4_0",
             dtype="bf16", back="f16", skipped=3),
        # a prefill batch into the mixed q8_0 / q4_0 window
        dict(name="rows_prefill_8191", kind="rows", n=8191, hkv=4, d=256, tokens=128, slots=512, tk="q8_0", tv="q4_0",
             dtype="f16", back="bf16", skipped=0),
        # one agent session decoding over a full 32768-token window
        dict(name="attn_decode_1x32768", kind="attn", n_seq=1, kv_max=32768, new_max=1, even=True, hkv=4, group=6, d=256,
             tokens=128, tk="q4_0", tv="q4_0", dtype="bf16", causal=True, refused=False, pad=0),
        # the smallest attention call: two short requests
        dict(name="attn_decode_2x333", kind="attn", n_seq=2, kv_max=333, new_max=1, even=False, hkv=2, group=3, d=128,
             tokens=32, tk="q4_0", tv="q4_0", dtype="f16", causal=True, refused=False, pad=0),
        # a full decode batch with ragged windows
        dict(name="attn_decode_32x32768", kind="attn", n_seq=32, kv_max=32768, new_max=1, even=False, hkv=4, group=6, d=256,
             tokens=128, tk="q4_0", tv="q4_0", dtype="bf16", causal=True, refused=True, pad=0),
        # the mixed-precision recipe: q8_0 keys, q4_0 values
        dict(name="attn_decode_q8q4_16", kind="attn", n_seq=16, kv_max=20001, new_max=1, even=False, hkv=4, group=6, d=256,
             tokens=128, tk="q8_0", tv="q4_0", dtype="f16", causal=True, refused=False, pad=0),
        # drafted tokens verified four at a time in eight sessions
        dict(name="attn_verify_8x4", kind="attn", n_seq=8, kv_max=16385, new_max=4, even=False, hkv=4, group=6, d=256,
             tokens=128, tk="q4_0", tv="q4_0", dtype="bf16", causal=True, refused=False, pad=5),
        # a 2048-token prompt chunk behind a full window
        dict(name="attn_prefill_2048", kind="attn", n_seq=1, kv_max=34816, new_max=2048, even=True, hkv=4, group=6, d=256,
             tokens=128, tk="q4_0", tv="q4_0", dtype="bf16", causal=True, refused=False, pad=0),
    ]


def _log(rng, low, high):
    """A whole number, spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["map", "rope", "rows", "attn", "attn", "attn"])
    if kind == "map":
        n_seq, new_max = _log(rng, 1, 2048), rng.choice([1, _log(rng, 1, 1024)])
        new_max = max(1, min(new_max, 262144 // n_seq))
        return dict(kind="map", n_seq=n_seq, tokens=rng.choice([16, 32, 48, 64, 100, 128, 256]), past_max=_log(rng, 1, 49152),
                    new_max=new_max, pad=rng.choice([0, 1, _log(rng, 1, 1000)]))
    if kind == "rope":
        d = rng.choice([64, 80, 96, 128, 192, 256])
        hkv = rng.randint(1, 8)
        return dict(kind="rope", n=_log(rng, 1, 4096), hq=hkv * rng.randint(1, 6), hkv=hkv, d=d, rot=16 * rng.randint(1, d // 16),
                    dtype=rng.choice(["f32", "f16", "bf16"]), pos_max=_log(rng, 1, 1 << 20))
    types = rng.choice([("q4_0", "q4_0"), ("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q5_0", "q5_0"), ("q8_0", "q8_0"), ("f16", "f16"),
                        (rng.choice(list(TYPES)), rng.choice(list(TYPES)))])
    if kind == "rows":
        n, tokens = _log(rng, 1, 8000), rng.choice([16, 32, 48, 100, 128])
        return dict(kind="rows", n=n, hkv=rng.randint(1, 4), d=rng.choice([64, 128, 256]), tokens=tokens,
                    slots=-(-n // tokens) + rng.randint(0, 9), tk=types[0], tv=types[1], dtype=rng.choice(["f32", "f16", "bf16"]),
                    back=rng.choice(["f16", "bf16"]), skipped=rng.choice([0, min(n - 1, rng.randint(0, 7))]))
    d, hkv, group = rng.choice([64, 128, 256]), rng.randint(1, 4), rng.randint(1, 8)
    new_max = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 1024)])
    n_seq = _log(rng, 1, 32) if new_max <= 8 else _log(rng, 1, 6)
    most = (1 << 20) // n_seq if new_max == 1 else (24 * 2048 * 32768) // (n_seq * hkv * group * new_max)
    kv_max = _log(rng, new_max, max(new_max, min(32768, most)))
    return dict(kind="attn", n_seq=n_seq, kv_max=kv_max, new_max=new_max, even=rng.random() < 0.3, hkv=hkv, group=group, d=d,
                tokens=rng.choice([16, 32, 48, 64, 100, 128]), tk=types[0], tv=types[1], dtype=rng.choice(["f16", "bf16"]),
                causal=rng.random() < 0.8, refused=n_seq > 2 and rng.random() < 0.3, pad=rng.choice([0, 0, rng.randint(1, 9)]))


def _lengths(case):
    """(past, new) of every request, by the case alone: ragged, the largest among them."""
    r = random.Random(17 * case["n_seq"] + case["new_max"])
    new = [case["new_max"]] + [r.randint(0 if case["new_max"] > 1 else 1, case["new_max"]) for _ in range(case["n_seq"] - 1)]
    past = [case["past_max"]] + [r.randint(0, case["past_max"]) for _ in range(case["n_seq"] - 1)]
    return list(zip(past, new))


def _kv_lengths(case):
    """(kv_len, new) of every request of an attention case; a refused one has kv_len 0."""
    r = random.Random(29 * case["n_seq"] + case["kv_max"])
    got = [(case["kv_max"], case["new_max"])]
    for i in range(1, case["n_seq"]):
        new = case["new_max"] if case["even"] else r.randint(1, case["new_max"])
        kv = case["kv_max"] if case["even"] else r.randint(new, max(new, case["kv_max"]))
        got.append((0 if case["refused"] and i == 1 else kv, new))
    return got


# ----------------------------------------------------------------- inputs --

def _activations(shape, dtype, g):
    """N(0, 1) with one channel in a hundred 20 times as large, as activations have them."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    big = torch.rand(shape[-1], generator=g, device="cuda") < 0.01
    return (x * torch.where(big, 20.0, 1.0)).to(dtype)


def _cache(cells, width, kind, g):
    """Rows of N(0, 1) values in the window's format, [cells, row bytes]."""
    out = torch.empty((cells, width // 32 * BLOCK_BYTES[kind]), dtype=torch.uint8, device="cuda")
    for at in range(0, cells, 65536):
        n = min(65536, cells - at)
        out[at:at + n] = _to_rows(_activations((n, width), torch.float32, g), kind)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    kind = case["kind"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if kind == "map":
        lengths = _lengths(case)
        r.shuffle(lengths)
        past, new = [p for p, _ in lengths], [n for _, n in lengths]
        T, B, rows = case["tokens"], case["n_seq"], sum(new) + case["pad"]
        held = [-(-p // T) for p in past]
        needs = sum(-(-(p + n) // T) - h for p, n, h in zip(past, new, held))
        cols = -(-(case["past_max"] + case["new_max"]) // T)
        slots = list(range(sum(held) + needs + 1))
        r.shuffle(slots)
        table = torch.full((B, cols), -1, dtype=torch.int32)
        at = 0
        for i, h in enumerate(held):
            table[i, :h] = torch.tensor(slots[at:at + h], dtype=torch.int32)
            at += h
        # a pool with room for nine in ten of the new blocks: the rest has to wait, as in a full server
        free = slots[at:at + max(1, needs - needs // 10)]
        return dict(kind=kind, past=ints(past), new=ints(new), table=table.cuda(), free=ints(free), tokens=T,
                    q_start=ints([0] * (B + 1)), kv_len=ints([0] * B), cells=torch.zeros(rows, dtype=torch.int64, device="cuda"),
                    pos=ints([0] * rows), seq=ints([0] * rows), info=ints([0] * 4))
    if kind == "rope":
        n, d, dt = case["n"], case["d"], DTYPES[case["dtype"]]
        # q and k as the projection leaves them: side by side in one tensor
        qkv = _activations((n, case["hq"] + 2 * case["hkv"], d), dt, g)
        half = case["rot"] // 2
        return dict(kind=kind, q=qkv[:, :case["hq"]], k=qkv[:, case["hq"]:case["hq"] + case["hkv"]], eps=1e-6,
                    qw=1.0 + 0.2 * torch.randn(d, generator=g, device="cuda"), kw=1.0 + 0.2 * torch.randn(d, generator=g, device="cuda"),
                    freqs=(1e6 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda(),
                    pos=torch.randint(0, case["pos_max"], (n,), generator=g, device="cuda", dtype=torch.int32),
                    q_out=torch.empty((n, case["hq"], d), dtype=dt, device="cuda"),
                    k_out=torch.empty((n, case["hkv"], d), dtype=dt, device="cuda"))
    T, width = case["tokens"], case["hkv"] * case["d"]
    if kind == "rows":
        n, slots = case["n"], case["slots"]
        cells = torch.randperm(slots * T, generator=g, device="cuda")[:n]
        cells[n - case["skipped"]:] = -1
        made = {w: torch.zeros((slots * T, width // 32 * BLOCK_BYTES[case["t" + w]]), dtype=torch.uint8, device="cuda") for w in "kv"}
        rows = {w: _activations((n, case["hkv"], case["d"]), DTYPES[case["dtype"]], g) for w in "kv"}
        back = {w: torch.empty((n, case["hkv"], case["d"]), dtype=DTYPES[case["back"]], device="cuda") for w in "kv"}
        return dict(kind=kind, case=case, cells=cells, cache=made, rows=rows, back=back)
    lengths = _kv_lengths(case)
    r.shuffle(lengths)
    blocks = [-(-k // T) for k, _ in lengths]
    slots = list(range(sum(blocks) + 3))
    r.shuffle(slots)
    table = torch.full((case["n_seq"], max(1, max(blocks))), -1, dtype=torch.int32)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = torch.tensor(slots[at:at + b], dtype=torch.int32)
        at += b
    start = [0]
    for _, n in lengths:
        start.append(start[-1] + n)
    rows, hq, dt = start[-1] + case["pad"], case["hkv"] * case["group"], DTYPES[case["dtype"]]
    return dict(kind=kind, case=case, kc=_cache(len(slots) * T, width, case["tk"], g), vc=_cache(len(slots) * T, width, case["tv"], g),
                slots=len(slots), table=table.cuda(), q_start=ints(start), kv_len=ints([k for k, _ in lengths]),
                q=torch.randn((rows, hq, case["d"]), generator=g, device="cuda").to(dt),
                out=torch.zeros((rows, hq, case["d"]), dtype=dt, device="cuda"), scale=case["d"] ** -0.5,
                work=torch.empty(WORK_BYTES, dtype=torch.uint8, device="cuda"))


# ------------------------------------------------------------ plain forms --

def _half_bytes(x):
    return x.contiguous().view(torch.uint8)


def _to_rows(x, kind):
    """[n, width] values as [n, row bytes] ggml rows, in 32 bits as ggml computes them."""
    n = x.shape[0]
    if kind == "f16":
        return _half_bytes(x.to(torch.float16))
    x = x.float().reshape(n, -1, 32)
    if kind == "q8_0":
        d = x.abs().amax(-1, keepdim=True) / 127.0
        y = x * torch.where(d != 0, 1.0 / d, 0.0)
        t = torch.trunc(y)
        code = t + torch.where((y - t).abs() >= 0.5, torch.sign(y), 0.0)
        return torch.cat([_half_bytes(d.half()), _half_bytes(code.to(torch.int8))], -1).reshape(n, -1)
    top, middle = (15, 8.0) if kind == "q4_0" else (31, 16.0)
    a = x.abs()
    first = (a == a.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
    d = x.gather(-1, first) / -middle
    code = torch.trunc(x * torch.where(d != 0, 1.0 / d, 0.0) + (middle + 0.5)).clamp(max=top).to(torch.int64)
    low, high = code[..., :16], code[..., 16:]
    nibbles = ((low & 15) | ((high & 15) << 4)).to(torch.uint8)
    if kind == "q4_0":
        return torch.cat([_half_bytes(d.half()), nibbles], -1).reshape(n, -1)
    bit = 1 << torch.arange(32, device=x.device)
    fifth = ((code >> 4) * bit).sum(-1, keepdim=True).to(torch.int32)
    fifth = torch.where(fifth > 0x7fffffff, fifth - (1 << 32), fifth).to(torch.int32)
    return torch.cat([_half_bytes(d.half()), _half_bytes(fifth), nibbles], -1).reshape(n, -1)


def _values(raw, kind):
    """[..., row bytes] ggml rows as [..., width] float32 values."""
    lead = raw.shape[:-1]
    if kind == "f16":
        return raw.contiguous().view(torch.float16).float()
    raw = raw.reshape(*lead, -1, BLOCK_BYTES[kind])
    d = raw[..., :2].contiguous().view(torch.float16).float()
    if kind == "q8_0":
        return (d * raw[..., 2:].contiguous().view(torch.int8).float()).reshape(*lead, -1)
    nibbles = raw[..., -16:]
    code = torch.cat([nibbles & 15, nibbles >> 4], -1)
    if kind == "q4_0":
        return (d * (code.float() - 8.0)).reshape(*lead, -1)
    fifth = raw[..., 2:6].contiguous().view(torch.int32)
    high = (fifth >> torch.arange(32, dtype=torch.int32, device=raw.device)) & 1
    return (d * (code.float() + 16.0 * high.float() - 16.0)).reshape(*lead, -1)


def _map_plain(s):
    past, new, T, table, free = s["past"].long(), s["new"].long(), s["tokens"], s["table"], s["free"].long()
    B, rows = past.numel(), s["cells"].numel()
    held, total = (past + T - 1) // T, (past + new + T - 1) // T
    end = torch.cumsum(total - held, 0)
    admitted = (total == held) | (end <= free.numel())
    first = end - (total - held)                       # place of a request's first new block in the free list
    col = torch.arange(table.shape[1], device=past.device)
    fresh = (col >= held[:, None]) & (col < total[:, None]) & admitted[:, None]
    place = (first[:, None] + col - held[:, None]).clamp(0, free.numel() - 1)
    table = torch.where(fresh, free[place].int(), table)
    start = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    row = torch.arange(rows, device=past.device)
    seq = torch.searchsorted(start, row, right=True) - 1
    there = row < start[-1]
    seq = torch.where(there, seq, 0)
    pos = past[seq] + row - start[seq]
    ok = there & admitted[seq]
    slot = table[seq, torch.where(ok, pos // T, 0)].long()
    taken = (torch.where(admitted, total - held, 0)).sum()
    info = torch.stack([taken, start[-1], (~admitted).sum(), torch.where(admitted, new, 0).sum()]).int()
    return dict(table=table, q_start=start.int(), kv_len=torch.where(admitted, past + new, 0).int(),
                cells=torch.where(ok, slot * T + pos % T, -1), pos=torch.where(there, pos, 0).int(),
                seq=torch.where(there, seq, -1).int(), info=info)


def _rope_plain(x, weight, eps, freqs, pos):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * weight
    angle = pos.double()[:, None, None] * freqs.double()
    cos, sin, half = torch.cos(angle).float(), torch.sin(angle).float(), freqs.numel()
    a, b = y[..., :half], y[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1).to(x.dtype)


def _rows_plain(s):
    case, cells = s["case"], s["cells"]
    got = []
    there = cells >= 0
    at = torch.where(there, cells, 0)
    for w in "kv":
        kind, x = case["t" + w], s["rows"][w]
        raw = _to_rows(x.reshape(x.shape[0], -1), kind)
        cache = s["cache"][w]
        kept = cache.shape[0]
        full = torch.cat([cache, cache[:1]])           # the last row takes what is skipped
        full[torch.where(there, cells, kept)] = raw
        back = _values(full[at], kind).reshape(x.shape)
        got.append(torch.where(there[:, None, None], back, 0.0).to(DTYPES[case["back"]]))
    return got


def _attend_plain(s):
    case, q, kv_len, start = s["case"], s["q"], s["kv_len"].long(), s["q_start"].long()
    T, hkv, d, G, B = case["tokens"], case["hkv"], case["d"], case["group"], kv_len.numel()
    keys, news = case["kv_max"], case["new_max"]
    j = torch.arange(keys, device=q.device)
    i = torch.arange(news, device=q.device)
    held = j < kv_len[:, None]
    cell = torch.where(held, s["table"].long()[:, j // T] * T + j % T, 0)
    k = _values(s["kc"][cell], case["tk"]).reshape(B, keys, hkv, d).permute(0, 2, 3, 1)
    v = _values(s["vc"][cell], case["tv"]).reshape(B, keys, hkv, d).transpose(1, 2)
    new = start[1:] - start[:-1]
    real = i < new[:, None]
    row = torch.where(real, start[:-1, None] + i, 0)
    x = q[row].float().reshape(B, news, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * news, d)
    score = torch.matmul(x, k).reshape(B, hkv, G, news, keys) * s["scale"]
    seen = held[:, None, :]
    if case["causal"]:
        seen = seen & (j < (kv_len[:, None] - new[:, None] + i + 1)[..., None])
    seen = seen[:, None, None]
    score = score.masked_fill(~seen, -float("inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -float("inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.reshape(B, hkv, G * news, keys), v).reshape(B, hkv, G, news, d)
    y = torch.where(total > 0, y / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, news, hkv * G, d)
    out = torch.cat([s["out"], s["out"][:1]])          # the last row takes the padded ones
    out[torch.where(real, start[:-1, None] + i, q.shape[0])] = y.to(q.dtype)
    return out[:-1]


# ------------------------------------------------------------------- runs --

def run(state):
    s, kind = state, state["kind"]
    if kind == "map":
        if own:
            _kvm().map_batch(s["past"], s["new"], s["free"], s["tokens"], s["table"], s["q_start"], s["kv_len"], s["cells"],
                             s["pos"], s["seq"], s["info"])
            return {x: s[x] for x in ("table", "q_start", "kv_len", "cells", "pos", "seq", "info")}
        return _map_plain(s)
    if kind == "rope":
        if own:
            _kvm().qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["eps"], s["freqs"], s["pos"], s["q_out"], s["k_out"])
            return [s["q_out"], s["k_out"]]
        return [_rope_plain(s["q"], s["qw"], s["eps"], s["freqs"], s["pos"]),
                _rope_plain(s["k"], s["kw"], s["eps"], s["freqs"], s["pos"])]
    case = s["case"]
    if kind == "rows":
        if own:
            kvm = _kvm()
            cache = kvm.Cache(s["cache"]["k"], s["cache"]["v"], TYPES[case["tk"]], TYPES[case["tv"]], case["hkv"], case["d"],
                              case["tokens"], case["slots"])
            kvm.write_rows(cache, s["cells"], s["rows"]["k"], s["rows"]["v"])
            kvm.read_rows(cache, s["cells"], s["back"]["k"], s["back"]["v"])
            return [s["back"]["k"], s["back"]["v"]]
        return _rows_plain(s)
    if own:
        kvm = _kvm()
        cache = kvm.Cache(s["kc"], s["vc"], TYPES[case["tk"]], TYPES[case["tv"]], case["hkv"], case["d"], case["tokens"], s["slots"])
        kvm.attend(cache, s["q"], s["q_start"], s["kv_len"], s["table"], s["out"], s["work"], scale=s["scale"],
                   causal=case["causal"], max_new=case["new_max"])
        return s["out"]
    return _attend_plain(s)


# ------------------------------------------------------------------- work --

def work(case):
    kind = case["kind"]
    if kind == "map":
        lengths, T = _lengths(case), case["tokens"]
        fresh = sum(-(-(p + n) // T) - -(-p // T) for p, n in lengths)
        rows = sum(n for _, n in lengths) + case["pad"]
        return {"bytes": 16.0 * len(lengths) + 8.0 * fresh + 16.0 * rows, "flops": 0.0}
    if kind == "rope":
        values = case["n"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 2.0 * DTYPE_BYTES[case["dtype"]] * values + 4.0 * case["n"] + 8.0 * case["d"], "flops": 8.0 * values}
    width = case["hkv"] * case["d"]
    row = {w: width // 32 * BLOCK_BYTES[case["t" + w]] for w in "kv"}
    if kind == "rows":
        n = case["n"]
        return {"bytes": n * (16.0 + 2 * width * (DTYPE_BYTES[case["dtype"]] + DTYPE_BYTES[case["back"]]) + 2 * (row["k"] + row["v"])),
                "flops": 8.0 * n * width}
    lengths, hq, d = _kv_lengths(case), case["hkv"] * case["group"], case["d"]
    pairs = sum(sum(max(0, min(kv, kv - n + i + 1)) if case["causal"] else kv for i in range(n)) for kv, n in lengths)
    return {"bytes": sum(kv for kv, _ in lengths) * float(row["k"] + row["v"]) + 4.0 * hq * d * sum(n for _, n in lengths),
            "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------- 64-bit definition --

def _decode64(raw, kind):
    """ggml rows as float64 values, block by block of 32."""
    if kind == "f16":
        return raw.contiguous().view(torch.float16).double()
    size, n = BLOCK_BYTES[kind], raw.shape[0]
    byte = raw.reshape(-1, size).to(torch.int64)
    d = raw.reshape(-1, size)[:, 0:2].contiguous().view(torch.float16).double()
    value = torch.empty((byte.shape[0], 32), dtype=torch.float64, device=raw.device)
    for e in range(32):
        if kind == "q8_0":
            b = byte[:, 2 + e]
            code = b - 256 * (b > 127)
        else:
            at = size - 16 + e % 16
            code = (byte[:, at] // (1 if e < 16 else 16)) % 16
            if kind == "q5_0":
                code = code + 16 * ((byte[:, 2 + e // 8] // (1 << (e % 8))) % 2) - 16
            else:
                code = code - 8
        value[:, e] = code.double() * d[:, 0]
    return value.reshape(n, -1)


def _rounded64(x, kind):
    """The values that ggml's rows stand for, quantized in 64 bits."""
    if kind == "f16":
        return x.half().double()
    b = x.double().reshape(x.shape[0], -1, 32)
    at = b.abs().argmax(-1, keepdim=True)
    size = b.abs().gather(-1, at)
    if kind == "q8_0":
        d = size / 127
        y = torch.where(d > 0, b / d, 0.0)
        code = torch.sign(y) * torch.floor(y.abs() + 0.5)
    else:
        half = 8 if kind == "q4_0" else 16
        d = torch.gather(b, -1, at) / -half
        code = torch.where(d != 0, torch.floor(b / d + half + 0.5), torch.tensor(float(half), device=b.device, dtype=torch.float64))
        code = torch.clamp(code, max=2 * half - 1) - half
    return (code * d.half().double()).reshape(x.shape[0], -1)


def exact(case, seed):
    kind = case["kind"]
    if kind == "map":
        return None
    s = prepare(case, seed)
    if kind == "rope":
        got = []
        half = case["rot"] // 2
        turn = torch.polar(torch.ones((case["n"], 1, half), dtype=torch.float64, device="cuda"),
                           (s["pos"].double().outer(s["freqs"].double()))[:, None, :])
        for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
            x = x.double()
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["d"] + s["eps"]) * w.double()
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
            got.append(torch.cat([z.real, z.imag, x[..., 2 * half:]], -1))
        return got
    if kind == "rows":
        got = []
        for w in "kv":
            x = s["rows"][w]
            y = _rounded64(x.reshape(x.shape[0], -1), case["t" + w]).reshape(x.shape)
            y[s["cells"] < 0] = 0.0
            got.append(y)
        return got
    out = s["out"].double()
    T, G, d = case["tokens"], case["group"], case["d"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    for b, kv in enumerate(lens):
        lo, n = starts[b], starts[b + 1] - starts[b]
        if kv == 0 or n == 0:
            continue
        cells = (s["table"][b, :-(-kv // T)].long()[:, None] * T + torch.arange(T, device="cuda")).reshape(-1)[:kv]
        k, v = _decode64(s["kc"][cells], case["tk"]), _decode64(s["vc"][cells], case["tv"])
        hidden = None
        if case["causal"]:
            hidden = torch.ones((n, kv), dtype=torch.bool, device="cuda").triu(kv - n + 1)
        for h in range(case["hkv"] * G):
            at = slice(h // G * d, h // G * d + d)
            score = s["q"][lo:lo + n, h].double() @ k[:, at].T * s["scale"]
            if hidden is not None:
                score = score.masked_fill(hidden, -float("inf"))
            weight = torch.nan_to_num(torch.softmax(score, -1))
            out[lo:lo + n, h] = weight @ v[:, at]
    return out
