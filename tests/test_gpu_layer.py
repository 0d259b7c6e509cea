"""The attention layer's calls on the device against 64-bit references:
kvm_map_batch, kvm_qk_norm_rope, kvm_write_rows / kvm_read_rows, kvm_attend, and
a run of them behind a reselection step."""
import numpy as np
import pytest

import layer_ref as ref

pytestmark = pytest.mark.gpu
TYPES = ref.TYPES
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}     # half a step, relative


def dt(torch, name):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


# ---------------------------------------------------------------- map_batch --

def run_map(kvm, past, new, free, T, table, n_rows, stride=None):
    import torch
    i = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    B, cols = table.shape
    wide = torch.full((B, stride or cols), -77, dtype=torch.int32, device="cuda")
    wide[:, :cols] = i(table)
    out = dict(q_start=i([9] * (B + 1)), kv_len=i([9] * B), cells=torch.full((n_rows,), 9, dtype=torch.int64, device="cuda"),
               pos=i([9] * n_rows), seq=i([9] * n_rows), info=i([9] * 4))
    kvm.map_batch(i(past), i(new), i(free), T, wide[:, :cols], *out.values())
    got = {k: v.cpu().numpy() for k, v in out.items()}
    got["table"] = wide[:, :cols].cpu().numpy()
    assert (wide[:, cols:] == -77).all()
    return got


def check_map(kvm, past, new, free, T, table, n_rows, **kw):
    want = ref.map_batch(past, new, free, T, table, n_rows)
    got = run_map(kvm, past, new, free, T, table, n_rows, **kw)
    for k, v in want.items():
        assert np.array_equal(got[k], v), k


@pytest.mark.parametrize("B, T, past_max, new_max, pad, short", [
    (1, 128, 0, 1, 0, 0), (1, 1, 7, 9, 2, 0), (3, 16, 100, 1, 0, 1), (64, 128, 49152, 1, 5, 3), (513, 100, 999, 40, 77, 20),
    (600, 48, 300, 3, 0, 0), (4096, 16, 64, 2, 1, 100), (7, 256, 5000, 4000, 33, 4)])
def test_map_batch(kvm_lib, B, T, past_max, new_max, pad, short):
    rng = np.random.default_rng(B * 131 + T)
    past, new = rng.integers(0, past_max + 1, B), rng.integers(0, new_max + 1, B)
    held, blocks = -(-past // T), -(-(past + new) // T)
    cols = int(blocks.max()) + 2
    ids = rng.permutation(int(blocks.sum()) + 50).astype(np.int32)
    table, at = np.full((B, cols), -1, np.int32), 0
    for i in range(B):
        table[i, :held[i]] = ids[at:at + held[i]]
        at += held[i]
    free = ids[at:at + max(0, int((blocks - held).sum()) - short)]
    check_map(kvm_lib, past, new, free, T, table, int(new.sum()) + pad, stride=cols + 3)


def test_map_batch_refuses_bad_requests(kvm_lib):
    T, cols = 16, 4
    past = [5, -1, 30, 64, 10, 0, 2 ** 31 - 8]
    new = [3, 4, 40, 1, -2, 20, 100]      # fits, negative, too long, too long, negative, fits, overflow
    table = np.full((7, cols), -1, np.int32)
    table[0, 0] = 3
    want = ref.map_batch(past, new, np.array([7, 8, 9], np.int32), T, table, 300)
    got = run_map(kvm_lib, past, new, [7, 8, 9], T, table, 300)
    for k in ("table", "q_start", "kv_len", "cells", "seq", "info"):
        assert np.array_equal(got[k], want[k]), k
    assert got["info"][2] == 5 and got["kv_len"].tolist() == [8, 0, 0, 0, 0, 20, 0]


@pytest.mark.parametrize("n_rows", [0, 1, 7, 12, 13])
def test_map_batch_rows_past_the_end(kvm_lib, n_rows):
    """Requests whose rows end past n_rows are refused and q_start stays there."""
    table = np.arange(12, dtype=np.int32).reshape(4, 3)
    check_map(kvm_lib, [4, 0, 9, 1], [1, 6, 0, 5], np.arange(100, 112, dtype=np.int32), 4, table, n_rows)


def test_map_batch_waiting_requests_and_held_holes(kvm_lib):
    """Behind the first request that does not fit only those that need no slot
    run; a held entry of -1 gives cell -1; no free slot at all is fine."""
    table = np.array([[0, 1], [2, -1], [3, -1], [-1, 5]], np.int32)
    check_map(kvm_lib, [8, 4, 3, 5], [1, 4, 1, 2], np.zeros(0, np.int32), 4, np.pad(table, ((0, 0), (0, 2)), constant_values=-1), 8)
    check_map(kvm_lib, [8, 4, 3, 5], [1, 9, 1, 2], np.array([40, 41], np.int32), 4,
              np.pad(table, ((0, 0), (0, 2)), constant_values=-1), 20)


# -------------------------------------------------------------------- rope --

def rope_ref(x, w, eps, freqs, pos):
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if w is not None:
        y = y * w
    h = len(freqs)
    a = (pos.astype(np.float64)[:, None] * freqs.astype(np.float64))[:, None, :]
    c, s = np.cos(a), np.sin(a)
    u, v = y[..., :h], y[..., h:2 * h]
    size = np.abs(y)
    size[..., :h] = size[..., h:2 * h] = np.abs(u) + np.abs(v)
    return np.concatenate([u * c - v * s, v * c + u * s, y[..., 2 * h:]], -1), size


def check_rope(kvm, torch, q, k, qw, kw, eps, freqs, pos, q_out, k_out, dtype):
    qn, kn = (x.detach().float().cpu().numpy() for x in (q, k))
    n = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    kvm.qk_norm_rope(q, k, qw, kw, eps, freqs, pos, q_out, k_out)
    for x, w, out in ((qn, qw, q_out), (kn, kw, k_out)):
        want, size = rope_ref(x, n(w), eps, n(freqs) if freqs is not None else np.zeros(0), n(pos) if pos is not None else np.zeros(x.shape[0]))
        got = out.float().cpu().numpy().astype(np.float64)
        # F32: a sum of d squares is off by at most d half steps, halved by the
        # root; root, products, cos and sin and the two products' sum add 12 more
        d = x.shape[-1]
        tol = size * (d / 2 + 12) * 2.0 ** -24 + (np.abs(want) * HALF[dtype] if dtype != "f32" else 0) + 1e-30
        if dtype == "f16":
            tol = tol + 2.0 ** -25        # half a step of the subnormals
        assert (np.abs(got - want) <= tol).all(), np.abs((got - want) / tol).max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, hq, hkv, d, rot", [(1, 1, 1, 16, 16), (5, 6, 2, 128, 128), (3, 24, 4, 256, 64), (33, 7, 1, 80, 32),
                                                (2, 3, 3, 96, 96), (4, 2, 1, 512, 512), (9, 5, 5, 64, 0), (2, 40, 8, 192, 176)])
def test_qk_norm_rope(kvm_lib, dtype, n, hq, hkv, d, rot):
    import torch
    g = torch.Generator(device="cuda").manual_seed(n * 7 + d)
    T = dt(torch, dtype)
    qkv = torch.randn((n, hq + 2 * hkv, d), generator=g, device="cuda").to(T)
    qw, kw = (1 + 0.3 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    freqs = torch.tensor((1e6 ** -np.linspace(0, 1, max(1, rot // 2)))[:rot // 2], dtype=torch.float32, device="cuda")
    pos = torch.randint(0, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
    check_rope(kvm_lib, torch, qkv[:, :hq], qkv[:, hq:hq + hkv], qw, kw, 1e-6, freqs if rot else None, pos if rot else None,
               torch.full((n, hq, d), 9.0, dtype=T, device="cuda"), torch.full((n, hkv, d), 9.0, dtype=T, device="cuda"), dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_qk_norm_rope_strides_far_positions_and_in_place(kvm_lib, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    T, n, d = dt(torch, dtype), 6, 64
    pos = torch.tensor([2 ** 31 - 1, -(2 ** 31) + 1, 0, 1, 123456789, -7], dtype=torch.int32, device="cuda")
    freqs = torch.tensor([1.0, 0.7, 0.3, 1e-3, 1e-6, 3.0, 2.0, 0.0], dtype=torch.float32, device="cuda")
    w = torch.randn(d, generator=g, device="cuda")
    # dims apart, heads interleaved, an odd offset
    q = torch.randn((d, n, 5), generator=g, device="cuda").to(T).permute(1, 2, 0)
    k = torch.randn((n, 3, d + 3), generator=g, device="cuda").to(T)[:, 1:, 1:d + 1]
    qo = torch.zeros((n, d, 5), dtype=T, device="cuda").transpose(1, 2)
    ko = torch.zeros((n, 2, 2 * d), dtype=T, device="cuda")[:, :, ::2]
    check_rope(kvm_lib, torch, q, k, w, None, 1e-5, freqs, pos, qo, ko, dtype)
    q2, k2 = q.contiguous(), k.contiguous()
    check_rope(kvm_lib, torch, q2, k2, w, None, 1e-5, freqs, pos, q2, k2, dtype)      # in place
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    q3 = torch.zeros_like(q2)
    kvm_lib.qk_norm_rope(q, None, w, None, 1e-5, freqs, pos, q3, None)
    assert torch.equal(q3, q2)


def test_qk_norm_rope_zero_rows_and_heads(kvm_lib):
    """A head of zeros stays zero (eps keeps the root finite); NaN stays in its head."""
    import torch
    q = torch.zeros((2, 2, 64), device="cuda", dtype=torch.bfloat16)
    q[1, 0, 3] = float("nan")
    out = torch.full_like(q, 9.0)
    kvm_lib.qk_norm_rope(q, None, None, None, 1e-6, None, None, out, None)
    assert (out[0] == 0).all() and (out[1, 1] == 0).all() and out[1, 0].isnan().all()
    kvm_lib.qk_norm_rope(q[:0], None, None, None, 1e-6, None, None, out[:0], None)


# -------------------------------------------------------------------- rows --

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tk, tv", [("q4_0", "q4_0"), ("q8_0", "q5_0"), ("f16", "q8_0"), ("q5_0", "f16")])
@pytest.mark.parametrize("n, h, d, T", [(1, 1, 32, 1), (37, 2, 128, 32), (130, 4, 256, 100), (9, 3, 96, 16)])
def test_rows_in_and_out(kvm_lib, oracle, dtype, tk, tv, n, h, d, T):
    import torch
    rng = np.random.default_rng(n * 3 + d)
    D, slots, w = dt(torch, dtype), n // T + 3, h * d
    x = {}
    for name in "kv":
        v = rng.standard_normal((n, h, d)).astype(np.float32) * np.where(rng.random(d) < 0.03, 20, 1).astype(np.float32)
        v[0, 0, :32] = 0.0                                   # a block of zeros
        v[n // 2, 0, :32] = np.where(np.arange(32) % 2, -1.5, 1.5)     # ties of both signs: the first decides
        x[name] = torch.from_numpy(v).to(D).cuda()
    cells = rng.permutation(slots * T)[:n].astype(np.int64)
    if n > 5:
        cells[[1, 4, 5]] = [-1, slots * T, 2 ** 40]          # skipped
    ok = (cells >= 0) & (cells < slots * T)
    raw = {s: torch.full((slots * T, w // 32 * ref.SIZE[t]), 0xA5, dtype=torch.uint8, device="cuda") for s, t in (("k", tk), ("v", tv))}
    cache = kvm_lib.Cache(raw["k"], raw["v"], TYPES[tk], TYPES[tv], h, d, T, slots)
    at = torch.from_numpy(cells).cuda()
    kvm_lib.write_rows(cache, at, x["k"], x["v"])
    for s, t in (("k", tk), ("v", tv)):
        wide = x[s].float().cpu().numpy().reshape(n, w)
        want = np.full(raw[s].shape, 0xA5, np.uint8)
        want[cells[ok]] = ref.quantize(wide, t)[ok]
        assert np.array_equal(raw[s].cpu().numpy(), want)
        if dtype == "f16" and t != "f16":
            assert np.array_equal(want[cells[ok]], oracle.quantize_rows_f16(TYPES[t], x[s].cpu().numpy().reshape(n, w))[ok])
    for back in ("f32", "f16", "bf16"):
        out = {s: torch.full((n, h, d), 9.0, dtype=dt(torch, back), device="cuda") for s in "kv"}
        kvm_lib.read_rows(cache, at, out["k"], out["v"])
        for s, t in (("k", tk), ("v", tv)):
            values = np.zeros((n, w))
            values[ok] = ref.row_values(raw[s].cpu().numpy()[cells[ok]], t)
            want = torch.from_numpy(values.astype(np.float32)).to(dt(torch, back)).reshape(n, h, d)
            assert torch.equal(out[s].cpu(), want)


def test_rows_strides_and_one_side(kvm_lib):
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    n, h, d, T, slots = 21, 2, 64, 8, 4
    raw = [torch.full((slots * T, h * d // 32 * 18), 7, dtype=torch.uint8, device="cuda") for _ in "kv"]
    cache = kvm_lib.Cache(raw[0], raw[1], 2, 2, h, d, T, slots)
    cells = torch.randperm(slots * T, generator=g, device="cuda")[:n]
    x = torch.randn((d, h, n), generator=g, device="cuda", dtype=torch.float32).permute(2, 1, 0)
    kvm_lib.write_rows(cache, cells, x, None)
    assert (raw[1] == 7).all()
    want = ref.quantize(x.contiguous().cpu().numpy().reshape(n, -1), "q4_0")
    assert np.array_equal(raw[0][cells].cpu().numpy(), want)
    kvm_lib.write_rows(cache, cells, None, x.contiguous())
    assert torch.equal(raw[1][cells], raw[0][cells])
    out = torch.full((n, d + 1, h), 9.0, device="cuda", dtype=torch.float32)
    view = out[:, 1:].transpose(1, 2)
    kvm_lib.read_rows(cache, cells, None, view)
    assert (out[:, 0] == 9).all()
    assert np.array_equal(view.cpu().numpy().reshape(n, -1), ref.row_values(want, "q4_0").astype(np.float32))


# ------------------------------------------------------------------ attend --

class Window:
    """A cache of random rows with a permuted table, and the call on it."""

    def __init__(self, kvm, torch, seed, kinds, hkv, D, T, lens, cols=None, spare=2, scale_v=None, base=0):
        self.kvm, self.torch, self.kinds, self.hkv, self.D, self.T, self.lens = kvm, torch, kinds, hkv, D, T, lens
        rng = np.random.default_rng(seed)
        self.rng = rng
        blocks = [-(-max(0, n) // T) for n in lens]
        self.slots = sum(blocks) + spare
        ids = rng.permutation(self.slots)
        self.table = np.full((len(lens), cols or max(1, max(blocks))), -1, np.int32)
        at = 0
        for i, b in enumerate(blocks):
            self.table[i, :b] = ids[at:at + b][:self.table.shape[1]]
            at += b
        self.raw = []
        for side, kind in enumerate(kinds):
            x = rng.standard_normal((self.slots * T, hkv * D)).astype(np.float32)
            if side and scale_v is not None:
                x *= scale_v(rng, x.shape[0])[:, None].astype(np.float32)
            self.raw.append(ref.quantize(x, kind))
        self.base = base
        self.dev = []
        for r in self.raw:
            buf = torch.zeros(r.size + 64, dtype=torch.uint8, device="cuda")
            buf[base:base + r.size] = torch.from_numpy(r.reshape(-1)).cuda()
            self.dev.append(buf[base:base + r.size])
        self.cache = kvm.Cache(self.dev[0], self.dev[1], TYPES[kinds[0]], TYPES[kinds[1]], hkv, D, T, self.slots)

    def put(self, side, rows):
        self.raw[side] = rows
        self.dev[side].copy_(self.torch.from_numpy(np.ascontiguousarray(rows).reshape(-1)).cuda())

    def cell(self, s, j):
        return int(self.table[s, j // self.T]) * self.T + j % self.T

    def run(self, q, q_start, causal=True, out=None, scale=None, max_new=1, work=None, kv_len=None, stream=None, table=None):
        torch = self.torch
        scale = self.D ** -0.5 if scale is None else scale
        i = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        out = torch.zeros_like(q) if out is None else out
        work = torch.empty(self.kvm.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda") if work is None else work
        self.kvm.attend(self.cache, q, i(q_start), i(self.lens if kv_len is None else kv_len),
                        i(self.table if table is None else table), out, work, scale=scale, causal=causal, max_new=max_new, stream=stream)
        return out

    def check(self, q, q_start, causal=True, scale=None, max_new=1, out=None, kv_len=None):
        scale = self.D ** -0.5 if scale is None else scale
        before = None if out is None else out.float().cpu().numpy()
        got = self.run(q, q_start, causal, out, scale, max_new, kv_len=kv_len)
        qn = q.float().cpu().numpy()
        kv = self.lens if kv_len is None else kv_len
        want, spread, peak = ref.attend(qn, self.raw[0], self.raw[1], self.kinds, self.hkv, self.T, self.slots, self.table,
                                        q_start, kv, scale, causal, np.zeros(q.shape) if before is None else before)
        check_attend(got.float().cpu().numpy(), want, spread, peak, qn, ref.row_values(self.raw[0], self.kinds[0]), scale,
                     max([1] + [int(x) for x in kv]), str(got.dtype).endswith("bfloat16"))
        return got


def check_attend(got, want, spread, peak, q, k, scale, keys, bf16):
    """Two roundings of a weight to F16 (2^-11 each) and one of a dequantized V or
    K value where the kernel makes them; the score's F32 sum of D products and
    the K rounding move every weight by at most `ds`; weights below 2^-39 of the
    largest vanish; the output's own half step."""
    D = q.shape[-1]
    with np.errstate(invalid="ignore"):
        k = np.abs(np.where(np.isfinite(k), k, 0.0)).max()
        ds = abs(scale) * np.abs(q).max() * k * (np.sqrt(D) * 2.0 ** -11 + D * 2.0 ** -23)
    tol = spread * (3 * 2.0 ** -11 + 2 * ds) + keys * 2.0 ** -39 * peak + np.abs(want) * (2.0 ** -8 if bf16 else 2.0 ** -11) + 2.0 ** -25
    assert np.isfinite(want).all()
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


def queries(torch, rng, rows, hq, D, dtype):
    return torch.from_numpy(rng.standard_normal((rows, hq, D)).astype(np.float32)).to(dt(torch, dtype)).cuda()


KINDS = [("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q5_0", "q5_0"), ("f16", "f16"), ("q4_0", "f16"), ("f16", "q8_0"), ("q8_0", "q5_0")]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kinds", KINDS)
def test_attend_decode(kvm_lib, D, kinds):
    """One token a request, at the lengths around a step, a warp's and a CTA's share."""
    import torch
    lens = [1, 0, 15, 16, 17, 127, 128, 129, 500]
    w = Window(kvm_lib, torch, D, kinds, 2, D, 32, lens)
    q = queries(torch, w.rng, len(lens), 6, D, "bf16" if D == 128 else "f16")
    got = w.check(q, range(len(lens) + 1))
    assert (got[1] == 0).all()


@pytest.mark.parametrize("hkv, group, T, new, dtype", [(1, 1, 16, 1, "f16"), (3, 8, 100, 1, "bf16"), (2, 9, 48, 1, "f16"), (4, 6, 128, 4, "bf16"),
                                                       (1, 5, 1, 3, "f16"), (2, 2, 16, 40, "bf16"), (1, 7, 64, 133, "f16"), (1, 64, 32, 2, "bf16")])
@pytest.mark.parametrize("causal", [True, False])
def test_attend_rows(kvm_lib, hkv, group, T, new, dtype, causal):
    """Row tiles from one row to many, head groups, block sizes, both masks."""
    import torch
    lens = [new + 211, new, 300 + new, new + 1]
    news = [new, new, max(1, new // 2), 0]
    w = Window(kvm_lib, torch, group * 10 + new, ("q4_0", "q4_0"), hkv, 128, T, lens)
    start = np.concatenate([[0], np.cumsum(news)])
    q = queries(torch, w.rng, int(start[-1]), hkv * group, 128, dtype)
    w.check(q, start, causal, max_new=new)


@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q5_0", "q8_0"), ("f16", "f16"), ("f16", "q5_0")])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_prompt_types(kvm_lib, kinds, D):
    import torch
    w = Window(kvm_lib, torch, D + 1, kinds, 2, D, 48, [333, 70])
    q = queries(torch, w.rng, 200 + 70, 6, D, "bf16")
    w.check(q, [0, 200, 270], True, max_new=200)


@pytest.mark.parametrize("D, group, news, lens", [(64, 8, [500, 410, 300], [700, 410, 900]), (256, 6, [260, 17], [5000, 3001])])
def test_attend_prompt_items_of_every_cut(kvm_lib, D, group, news, lens):
    """Several items a CTA, and items that several CTAs share."""
    import torch
    w = Window(kvm_lib, torch, D, ("q4_0", "q4_0"), 4, D, 32, lens)
    start = np.concatenate([[0], np.cumsum(news)])
    q = queries(torch, w.rng, int(start[-1]), 4 * group, D, "bf16")
    got = w.run(q, start, True, max_new=max(news))
    rows = np.unique(np.concatenate([[0, 1, start[1] - 1, start[1], start[-1] - 1], w.rng.integers(0, start[-1], 40)]))
    for r in rows:                        # each row as a request of its own that sees what it saw
        s = int(np.searchsorted(start, r, side="right")) - 1
        seen = lens[s] - news[s] + int(r - start[s]) + 1
        want, spread, peak = ref.attend(q[r:r + 1].float().cpu().numpy(), w.raw[0], w.raw[1], w.kinds, 4, 32, w.slots,
                                        w.table[s:s + 1], [0, 1], [seen], D ** -0.5, True, np.zeros((1, 4 * group, D)))
        check_attend(got[r:r + 1].float().cpu().numpy(), want, spread, peak, q[r:r + 1].float().cpu().numpy(),
                     ref.row_values(w.raw[0], "q4_0"), D ** -0.5, seen, True)
    for _ in range(3):
        assert torch.equal(w.run(q, start, True, max_new=max(news)), got)


def test_attend_long_window(kvm_lib):
    """Many splits of one window, and the same bits on every run."""
    import torch
    w = Window(kvm_lib, torch, 1, ("q4_0", "q4_0"), 1, 256, 128, [20011])
    q = queries(torch, w.rng, 1, 6, 256, "bf16")
    a = w.check(q, [0, 1])
    for _ in range(3):
        assert torch.equal(w.run(q, [0, 1]), a)


def test_attend_many_requests(kvm_lib):
    """More requests than a CTA has threads, most of them short, some empty."""
    import torch
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(0, 60, 700)]
    news = [int(x) for x in rng.integers(0, 3, 700)]
    w = Window(kvm_lib, torch, 8, ("q4_0", "q4_0"), 1, 64, 16, lens)
    start = np.concatenate([[0], np.cumsum(news)])
    w.check(queries(torch, w.rng, int(start[-1]), 4, 64, "f16"), start, max_new=2)


@pytest.mark.parametrize("new", [5, 40])
def test_attend_rows_without_keys(kvm_lib, new):
    """kv_len < new: the first rows see nothing and are 0."""
    import torch
    w = Window(kvm_lib, torch, new, ("q4_0", "q4_0"), 2, 128, 16, [3, 64])
    q = queries(torch, w.rng, 2 * new, 4, 128, "f16")
    got = w.check(q, [0, new, 2 * new], True, max_new=new)
    assert (got[:new - 3] == 0).all() and not (got[new - 3] == 0).all()


@pytest.mark.parametrize("new", [2, 37])
def test_attend_rows_of_no_request_stay(kvm_lib, new):
    import torch
    w = Window(kvm_lib, torch, new, ("q4_0", "q4_0"), 1, 64, 16, [50, 60])
    q = queries(torch, w.rng, 2 * new + 6, 3, 64, "bf16")
    out = torch.full_like(q, 7.0)
    w.check(q, [2, 2 + new, 2 + 2 * new], True, max_new=new, out=out)
    assert (out[:2] == 7).all() and (out[2 + 2 * new:] == 7).all()
    # rows past the end and before the start are skipped
    out = torch.full_like(q, 7.0)
    w.run(q, [-3, 1, 4 * new + 9], out=out, max_new=new)
    assert (out[:1] == 7).all()


@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q8_0"), ("f16", "f16"), ("q5_0", "q5_0")])
@pytest.mark.parametrize("new, D", [(1, 128), (3, 256), (60, 64)])
def test_attend_hidden_rows_hold_anything(kvm_lib, kinds, new, D):
    """Cells behind a request's end, other requests' blocks and, for the causal
    rows, later keys may hold infinities and NaN."""
    import torch
    w = Window(kvm_lib, torch, new, kinds, 2, D, 32, [90, 75])
    q = queries(torch, w.rng, new, 4, D, "f16")
    start = [0, new, new]
    clean = w.check(q, start, True, max_new=new).clone()
    for side in (0, 1):
        raw = w.raw[side].copy()
        seen = {w.cell(0, j) for j in range(90)}
        for c in range(raw.shape[0]):
            if c not in seen:
                raw[c].view(np.uint8)[:] = 0xFF          # every half is NaN
        w.put(side, raw)
    assert torch.equal(w.run(q, start, True, max_new=new), clean)
    if new == 1:
        return
    # the last key, seen by the last row alone, is infinite in K and V
    for side in (0, 1):
        raw = w.raw[side].copy()
        c = w.cell(0, 89)
        raw[c, 0:2] = np.array([0x00, 0x7C], np.uint8)
        raw[c, -2:] = np.array([0x00, 0x7C], np.uint8)
        if kinds[side] == "f16":
            raw[c].view(np.float16)[:] = np.inf
        w.put(side, raw)
    got = w.run(q, start, True, max_new=new)
    # the infinite key may sit in a step that is summed in another way: compare
    # with the definition, not bit by bit
    assert torch.isfinite(got[:new - 1]).all()
    assert torch.allclose(got[:new - 1].float(), clean[:new - 1].float(), rtol=2.0 ** -9, atol=2.0 ** -9)


def test_attend_bad_table_entries_are_not_seen(kvm_lib):
    import torch
    w = Window(kvm_lib, torch, 3, ("q4_0", "q4_0"), 2, 128, 16, [100, 64, 40])
    w.table[0, 2], w.table[0, 5], w.table[1, 0], w.table[2, :] = -1, w.slots, 2 ** 31 - 1, -5
    for new in (1, 30):
        q = queries(torch, w.rng, 3 * new, 4, 128, "bf16")
        got = w.check(q, [0, new, 2 * new, 3 * new], True, max_new=new)
        assert (got[2 * new:] == 0).all()


def test_attend_lengths_past_the_table(kvm_lib):
    """Keys beyond the table's columns are not seen; a negative length sees none."""
    import torch
    w = Window(kvm_lib, torch, 4, ("q4_0", "q4_0"), 1, 64, 16, [64, 48], cols=4)
    for new in (1, 20):
        q = queries(torch, w.rng, 2 * new, 2, 64, "f16")
        w.check(q, [0, new, 2 * new], True, max_new=new, kv_len=[80, 2 ** 31 - 1])
        got = w.check(q, [0, new, 2 * new], True, max_new=new, kv_len=[-5, 30])
        assert (got[:new] == 0).all()


@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q5_0")])
@pytest.mark.parametrize("new", [1, 50])
def test_attend_value_scales_of_every_size(kvm_lib, kinds, new):
    """V rows from 1e-6 to 1e4: small ones first, so that the running scale grows."""
    import torch
    w = Window(kvm_lib, torch, 9, kinds, 1, 128, 16, [400], scale_v=lambda r, n: 10.0 ** r.uniform(-6, 4, n))
    w.check(queries(torch, w.rng, new, 4, 128, "f16"), [0, new], True, scale=0.05, max_new=new)
    w2 = Window(kvm_lib, torch, 10, kinds, 1, 64, 16, [300], scale_v=lambda r, n: np.full(n, 3e-6))
    q = queries(torch, w2.rng, new, 2, 64, "bf16")
    got = w2.run(q, [0, new], True, max_new=new).float().cpu().numpy()
    want, spread, _ = ref.attend(q.float().cpu().numpy(), w2.raw[0], w2.raw[1], kinds, 1, 16, w2.slots, w2.table, [0, new], [300],
                                 64 ** -0.5, True, np.zeros(q.shape))
    assert (np.abs(got - want) <= 0.02 * spread + 2.0 ** -8 * np.abs(want)).all()


@pytest.mark.parametrize("new", [1, 40])
def test_attend_queries_of_every_size(kvm_lib, new):
    """Query rows from 1e-30 to 1e30 (BF16) with the scale that brings them back,
    zero rows, and a NaN row that stays alone."""
    import torch
    w = Window(kvm_lib, torch, 2, ("q4_0", "q4_0"), 1, 128, 32, [170])
    base = queries(torch, w.rng, new, 4, 128, "bf16")
    want = w.check(base, [0, new], True, max_new=new)
    for e in (-90, 90):
        q = (base.float() * 2.0 ** e).to(torch.bfloat16)
        got = w.run(q, [0, new], True, scale=128 ** -0.5 * 2.0 ** -e, max_new=new)
        assert torch.equal(got, want)
    q = base.clone()
    q[0, 1] = 0
    q[0, 2, 5] = float("nan")
    got = w.run(q, [0, new], True, max_new=new)
    assert got[0, 2].isnan().all() and torch.equal(got[0, 0], want[0, 0]) and torch.equal(got[0, 3], want[0, 3])
    assert torch.isfinite(got[0, 1]).all()


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30])
@pytest.mark.parametrize("new", [1, 40])
def test_attend_scales(kvm_lib, new, scale):
    """A scale of 0 is a mean over the seen keys; a negative one turns the order."""
    import torch
    w = Window(kvm_lib, torch, 2, ("q4_0", "q5_0"), 1, 128, 32, [170])
    w.check(queries(torch, w.rng, new, 4, 128, "bf16"), [0, new], True, scale=scale, max_new=new)


@pytest.mark.parametrize("base", [0, 4, 16])
@pytest.mark.parametrize("new", [1, 30])
def test_attend_strides_and_alignment(kvm_lib, base, new):
    import torch
    w = Window(kvm_lib, torch, 6, ("q4_0", "q8_0"), 2, 128, 32, [150, 77], base=base)
    q = queries(torch, w.rng, 2 * new, 6, 128, "f16")
    want = w.check(q, [0, new, 2 * new], True, max_new=new)
    odd = torch.zeros((128, 6, 2 * new + 1), dtype=q.dtype, device="cuda").permute(2, 1, 0)[1:]
    odd.copy_(q)
    out = torch.full((2 * new, 6, 129), 7.0, dtype=q.dtype, device="cuda")
    got = w.run(odd, [0, new, 2 * new], True, out=out[:, :, 1:], max_new=new)
    assert torch.equal(got, want) and (out[:, :, 0] == 7).all()
    wide = torch.full((2, 9), -3, dtype=torch.int32, device="cuda")
    wide[:, :w.table.shape[1]] = torch.tensor(w.table, device="cuda")
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out2 = torch.zeros_like(q)
    kvm_lib.attend(w.cache, q, i([0, new, 2 * new]), i(w.lens), wide[:, :w.table.shape[1]], out2,
                   torch.empty(kvm_lib.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda"), scale=128 ** -0.5, max_new=new)
    assert torch.equal(out2, want)


@pytest.mark.parametrize("max_new", [0, 1, 7, 1000])
def test_attend_max_new_is_only_a_hint(kvm_lib, max_new):
    import torch
    w = Window(kvm_lib, torch, 12, ("q4_0", "q4_0"), 2, 128, 16, [260, 20, 300])
    q = queries(torch, w.rng, 100 + 1 + 9, 4, 128, "f16")
    w.check(q, [0, 100, 101, 110], True, max_new=max_new)


def test_attend_captured_and_replayed(kvm_lib):
    """One graph for every step: the lengths, table and queries change under it."""
    import torch
    w = Window(kvm_lib, torch, 21, ("q4_0", "q4_0"), 2, 128, 32, [400, 120, 3])
    i = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    for news in ([1, 1, 1], [33, 2, 3]):
        start = np.concatenate([[0], np.cumsum(news)])
        q = queries(torch, w.rng, int(start[-1]), 6, 128, "bf16")
        out, work = torch.zeros_like(q), torch.empty(kvm_lib.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda")
        qs, kv, table = i(start), i([1, 1, 1]), i(w.table)
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            kvm_lib.attend(w.cache, q, qs, kv, table, out, work, scale=0.1, max_new=max(news))
            graph.capture_begin()
            kvm_lib.attend(w.cache, q, qs, kv, table, out, work, scale=0.1, max_new=max(news))
            graph.capture_end()
        torch.cuda.current_stream().wait_stream(side)
        for lens in ([400, 120, 3], [64, 119, 3], [0, 33, 1]):
            kv.copy_(i(lens))
            q.copy_(queries(torch, w.rng, int(start[-1]), 6, 128, "bf16"))
            work.fill_(0xFF)
            graph.replay()
            want = w.run(q, start, scale=0.1, max_new=max(news), kv_len=lens)
            assert torch.equal(out, want)


def test_attend_two_streams(kvm_lib):
    """Calls on two streams with a workspace each, many times."""
    import torch
    w = Window(kvm_lib, torch, 31, ("q4_0", "q4_0"), 2, 128, 32, [3000, 900])
    q = queries(torch, w.rng, 2, 6, 128, "f16")
    want = w.run(q, [0, 1, 2])
    i = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    qs, kv, table = i([0, 1, 2]), i(w.lens), i(w.table)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.zeros_like(q) for _ in range(20)] for _ in streams]
    works = [torch.empty(kvm_lib.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for n in range(20):
        for s, o, wk in zip(streams, outs, works):
            kvm_lib.attend(w.cache, q, qs, kv, table, o[n], wk, scale=128 ** -0.5, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for side in outs for o in side)


# -------------------------------------------------------------- the binding --

def test_binding_refuses_what_does_not_fit(kvm_lib):
    import torch
    kvm = kvm_lib
    w = Window(kvm, torch, 1, ("q4_0", "q4_0"), 1, 64, 16, [32])
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q, work = queries(torch, w.rng, 1, 2, 64, "f16"), torch.empty(kvm.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda")
    good = dict(q=q, q_start=i([0, 1]), kv_len=i([32]), table=i(w.table), out=torch.empty_like(q), work=work, scale=0.1)
    kvm.attend(w.cache, **good)
    for name, bad in (("q", q.float()), ("q", q.cpu()), ("q", q[0]), ("q_start", i([0])), ("q_start", i([0, 1]).long()),
                      ("kv_len", i([32]).cpu()), ("table", i(w.table).t()[:1].t().repeat(2, 1)), ("table", i(w.table).long()),
                      ("out", torch.empty_like(q)[:, :1]), ("work", work[:100]), ("work", work.cpu()), ("q_start", i([0, 5, 1])[::2])):
        with pytest.raises(kvm.KvmError) as e:
            kvm.attend(w.cache, **{**good, name: bad})
        assert e.value.status == kvm.KVM_EINVAL
    for args in ((2, 2, 1, 64, 16, 1000), (3, 2, 1, 64, 16, 1), (2, 2, 1, 40, 16, 1), (2, 2, 1, 64, 0, 1)):
        with pytest.raises(kvm.KvmError):
            kvm.Cache(w.dev[0], w.dev[1], *args)
    host = torch.zeros(64, dtype=torch.uint8)
    with pytest.raises(kvm.KvmError):
        kvm.Cache(host, host, 2, 2, 1, 64, 1, 1)


def test_host_pointers_are_refused(kvm_lib):
    """The C entry points look at the first pointer: host memory is EINVAL."""
    import ctypes as C

    import torch
    kvm = kvm_lib
    host = torch.zeros(4096, dtype=torch.uint8).pin_memory().data_ptr()
    m = kvm._BatchMap(host, host, host, host, 8, 8, 4, 16, 128, 64, 0, host, host, host, host, host, host)
    assert kvm.lib().kvm_map_batch(None, C.byref(m)) == kvm.KVM_EINVAL
    assert b"not a device pointer" in kvm.lib().kvm_last_error(None)


# --------------------------------------------------------------- a whole run --

@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q4_0")])
def test_layer_behind_a_reselection_step(kvm_lib, kinds):
    """score -> select -> diff -> stage-in fill the window; then, twice, the step's
    cell map, norm and rotation, the new rows into the window and the attention
    over it, a prompt chunk first and one token after; the last output against the
    definition over the window's bytes."""
    import torch
    from kvm_testlib import Shape, make_query, make_rig
    kvm = kvm_lib
    sh = Shape(n_layer=1, n_blocks=40, block_tokens=32, n_head_kv=2, head_dim=128, n_head_q=6, budget_blocks=8, gen_blocks=4,
               type_k=TYPES[kinds[0]], type_v=TYPES[kinds[1]])
    rig = make_rig(sh, seed=4)
    q0, count = make_query(sh, np.random.default_rng(5))
    rig.sess.set_query(q0, count)
    rig.sess.step(rig.src, rig.k_bases(), rig.v_bases())
    plan = rig.sess.plan()
    T, H, D, held = 32, 2, 128, int(plan["total_window_tokens"])
    slots = rig.sess.n_slots
    cache = kvm.Cache(rig.win_k, rig.win_v, sh.type_k, sh.type_v, H, D, T, slots)
    i = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    table = np.full((1, slots), -1, np.int32)
    table[0, :len(plan["selected"])] = np.arange(len(plan["selected"]))       # slot i holds selected[i]
    table, free = i(table), i(np.arange(len(plan["selected"]), slots))
    freqs = torch.tensor(1e4 ** -np.linspace(0, 1, 32), dtype=torch.float32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(6)
    work = torch.empty(kvm.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda")
    for new in (45, 1):
        q, k, v = (torch.randn((new, h, D), generator=g, device="cuda").to(torch.bfloat16) for h in (6, H, H))
        qs, kv, cells, pos, seq, info = i([0, 0]), i([0]), torch.empty(new, dtype=torch.int64, device="cuda"), i([0] * new), i([0] * new), i([0] * 4)
        kvm.map_batch(i([held]), i([new]), free, T, table, qs, kv, cells, pos, seq, info)
        taken = int(info[0])
        if new == 45:                     # what register_append gives the model's own tokens
            rig.sess.register_append(new, resident=True)
        free = free[taken:]
        held += new
        kvm.qk_norm_rope(q, k, None, None, 1e-6, freqs, pos + 1000, q, k)
        kvm.write_rows(cache, cells, k, v)
        out = torch.zeros_like(q)
        kvm.attend(cache, q, qs, kv, table, out, work, scale=D ** -0.5, max_new=new)
        back = torch.empty_like(k)
        kvm.read_rows(cache, cells, back, None)
        assert int(info[2]) == 0 and int(kv[0]) == held
        assert (back.float() - k.float()).abs().max() < k.float().abs().max() / 5
        raw = [w.cpu().numpy().reshape(slots * T, -1) for w in (rig.win_k, rig.win_v)]
        want, spread, peak = ref.attend(q.float().cpu().numpy(), raw[0], raw[1], kinds, H, T, slots, table.cpu().numpy(), [0, new],
                                        [held], D ** -0.5, True, np.zeros(q.shape))
        check_attend(out.float().cpu().numpy(), want, spread, peak, q.float().cpu().numpy(), ref.row_values(raw[0], kinds[0]),
                     D ** -0.5, held, True)
    rig.sess.close()
