"""Attention over values of every size, against the definition in 64 bits with a
tolerance from each row's own |q|.|k|: blocks whose values leave F16's range, in
keys that some rows see and others do not, in every kernel."""
import numpy as np
import pytest

import layer_ref as ref
from test_gpu_layer import Window, queries

pytestmark = pytest.mark.gpu


def reference(w, q, start, lens, scale, causal=True, rows=None):
    """(want, spread, peak, ds) of the rows of q: the definition, sum p |v| / sum p, the
    largest |v| a row sees, and the most that an F16 rounding of K (2^-11) and an F32 sum
    of D products move one of the row's scores."""
    n, hq, D = q.shape
    G = hq // w.hkv
    k, v = (ref.row_values(r, t) for r, t in zip(w.raw, w.kinds))
    want, spread, peak = (np.zeros((n, hq, D)) for _ in range(3))
    ds = np.zeros((n, hq, 1))
    for s in range(len(lens)):
        lo, hi, kv = int(start[s]), int(start[s + 1]), int(lens[s])
        j = np.arange(kv)
        cell = w.table[s, j // w.T].astype(np.int64) * w.T + j % w.T
        for r in range(lo, hi):
            if rows is not None and r not in rows:
                continue
            c = cell[:max(0, kv - (hi - lo) + (r - lo) + 1)] if causal else cell
            if c.size == 0:
                continue
            for h in range(hq):
                at = slice(h // G * D, h // G * D + D)
                x = k[c, at] @ q[r, h] * scale
                p = np.exp(x - x.max())
                p /= p.sum()
                want[r, h], spread[r, h] = p @ v[c, at], p @ np.abs(v[c, at])
                peak[r, h] = np.abs(v[c, at]).max(0)
                # the same bound for keys that weigh nothing would hide the others' errors
                near = p > 1e-9
                ds[r, h] = abs(scale) * (np.abs(k[c, at][near]) @ np.abs(q[r, h])).max() * (2.0 ** -11 + D * 2.0 ** -23)
    return want, spread, peak, ds


def agree(got, want, spread, peak, ds, keys):
    """Two roundings of a weight to F16 and one of a V value (2^-11 each), a score moved by
    ds in numerator and denominator, one rounding more for an item that several CTAs share,
    weights below 2^-31 of the largest lost, the output's half step."""
    half = 2.0 ** -8 if str(got.dtype).endswith("bfloat16") else 2.0 ** -11
    tol = spread * (4 * 2.0 ** -11 + 2 * ds) + keys * 2.0 ** -31 * 2.0 ** -11 * peak + np.abs(want) * half
    if half == 2.0 ** -11:
        tol = tol + 2.0 ** -25          # half a step of F16's subnormals
    error = np.abs(got.float().cpu().numpy().astype(np.float64) - want)
    assert (error <= tol).all(), np.nanmax(np.where(error <= tol, 0, error / np.maximum(tol, 1e-300)))


def rewrite(w, side, change):
    """The window's rows of one side after `change`(values [cells, width])."""
    w.put(side, ref.quantize(change(ref.row_values(w.raw[side], w.kinds[side])).astype(np.float32), w.kinds[side]))


# ---------------------------------------------- values beyond F16, not seen by all --

SHAPES = [(64, 2, 40), (128, 4, 20), (128, 4, 70), (256, 6, 12), (256, 6, 50)]      # head size, group, rows: single CTAs and pairs


@pytest.mark.parametrize("kinds", [("q8_0", "q8_0"), ("q4_0", "q4_0"), ("f16", "q8_0"), ("q8_0", "q5_0"), ("q5_0", "q4_0")])
@pytest.mark.parametrize("D, group, new", SHAPES)
def test_a_value_beyond_f16_stays_with_the_rows_that_see_it(kvm_lib, kinds, D, group, new):
    """The last key's V is 1e5, finite in its block's scale and codes: rows that do not see it
    are as without it, the last one is the definition's."""
    import torch
    keys = 210
    w = Window(kvm_lib, torch, D + new, kinds, 1, D, 32, [keys])
    q = queries(torch, w.rng, new, group, D, "bf16")
    clean = w.run(q, [0, new], True, max_new=new)

    def change(v):
        v[w.cell(0, keys - 1)] = 1e5 * np.where(np.arange(D) % 3, 1.0, -0.7)
        return v
    rewrite(w, 1, change)
    got = w.run(q, [0, new], True, max_new=new)
    assert torch.isfinite(got).all()
    assert torch.allclose(got[:new - 1].float(), clean[:new - 1].float(), rtol=2.0 ** -8, atol=2.0 ** -9)
    agree(got, *reference(w, q.float().cpu().numpy(), [0, new], [keys], D ** -0.5), keys)


# ------------------------------------------- items that several CTAs share --

@pytest.mark.parametrize("kinds", [("q8_0", "q8_0"), ("q4_0", "q4_0")])
@pytest.mark.parametrize("D, group, new", [(64, 1, 20), (128, 2, 70), (256, 6, 25)])
@pytest.mark.parametrize("size", [1e-5, 2e5])
def test_outputs_of_every_size_from_shared_items(kvm_lib, kinds, D, group, new, size):
    """One request over a window that many CTAs share: means far below and far above F16's
    range keep their bits on the way through the workspace."""
    import torch
    keys = 1500
    w = Window(kvm_lib, torch, D + new, kinds, 1, D, 32, [keys])
    # every dim has a mean of its own size beside the noise, the last 32 dims a thirtieth
    rewrite(w, 1, lambda v: (v * 0.1 + 1.0) * size * np.where(np.arange(D) >= D - 32, 0.03, 1.0))
    q = queries(torch, w.rng, new, group, D, "bf16")
    got = w.run(q, [0, new], True, max_new=new)
    seen = list(range(0, new, 7))
    want = reference(w, q.float().cpu().numpy(), [0, new], [keys], D ** -0.5, rows=seen)
    agree(got[seen], *(x[seen] for x in want), keys)


# ------------------------------------------------------------ keys beyond F16 --

@pytest.mark.parametrize("kinds", [("q8_0", "q8_0"), ("q4_0", "q4_0"), ("q5_0", "f16"), ("q8_0", "q4_0")])
@pytest.mark.parametrize("D, group, new", SHAPES + [(128, 4, 1), (64, 2, 6)])
@pytest.mark.parametrize("T", [32, 24])
def test_keys_beyond_f16(kvm_lib, kinds, D, group, new, T):
    """Some keys' first block is of 1e5 where the queries are of 1e-5: finite scores, the
    definition's, whatever kernel takes the request."""
    import torch
    keys = 210
    w = Window(kvm_lib, torch, D + new, kinds, 1, D, T, [keys])
    big = [w.cell(0, j) for j in (0, 17, 63, 64, 100, 127, 128, 129, 200, keys - 1) if j < keys]

    def change(k):
        k[big, :32] *= 1e5
        return k
    rewrite(w, 0, change)
    q = queries(torch, w.rng, new, group, D, "bf16")
    q[..., :32] *= 1e-5
    results = [w.run(q, [0, new], True, max_new=m) for m in (1, new, 1000)]
    want = reference(w, q.float().cpu().numpy(), [0, new], [keys], D ** -0.5)
    for got in results:
        agree(got, *want, keys)


# ------------------------------------------- what ran on the SM before a call --

def test_f16_decode_does_not_see_what_ran_before(kvm_lib):
    """F16 rows of 256 dims come in steps of 16 keys.  The same bits whether another kernel
    left ones or zeros in shared memory, with an infinite value whose weight underflows."""
    import torch
    n, keys = 160, 300
    w = Window(kvm_lib, torch, 7, ("f16", "f16"), 1, 256, 32, [keys] * n)
    for side, (scale, value) in enumerate(((0.1, -30.0), (1.0, np.inf))):
        raw = (w.raw[side].view(np.float16) * np.float16(scale)).astype(np.float16)
        for s in range(n):
            raw[w.cell(s, 5)] = value
        w.put(side, raw.view(np.uint8))
    q = torch.ones((n, 4, 256), dtype=torch.float16, device="cuda")
    before = Window(kvm_lib, torch, 8, ("q4_0", "q4_0"), 1, 256, 32, [4000])
    rows = queries(torch, before.rng, 1200, 8, 256, "f16")
    got = []
    for byte in (0xFF, 0):
        for side in (0, 1):
            before.put(side, np.full_like(before.raw[side], byte))
        before.run(rows, [0, 1200], max_new=1200)
        got.append(w.run(q, range(n + 1)))
    assert torch.equal(got[0].view(torch.int16), got[1].view(torch.int16))


# ------------------------------------- value blocks of very different sizes --

@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q8_0"), ("f16", "q5_0")])
@pytest.mark.parametrize("D, group, new", [(64, 2, 1), (128, 6, 1), (256, 6, 1), (128, 12, 1), (256, 6, 20)])
@pytest.mark.parametrize("apart", [14, 20, 26])
def test_value_blocks_of_very_different_sizes(kvm_lib, kinds, D, group, new, apart):
    """Every other block of 32 dims is 2^-apart of its neighbours: each dim keeps its own
    relative accuracy."""
    import torch
    keys = 260
    w = Window(kvm_lib, torch, D + new, kinds, 1, D, 32, [keys, 90])
    rewrite(w, 1, lambda v: v * np.where(np.arange(D) // 32 % 2, 2.0 ** (6 - apart), 2.0 ** 6))
    q = queries(torch, w.rng, 2 * new, group, D, "bf16")
    got = w.run(q, [0, new, 2 * new], True, max_new=new)
    agree(got, *reference(w, q.float().cpu().numpy(), [0, new, 2 * new], [keys, 90], D ** -0.5), keys)


# --------------------------------------- row tiles of different fill behind one another --

@pytest.mark.parametrize("kinds", [("q8_0", "q5_0"), ("q4_0", "f16")])
def test_short_row_tiles_behind_full_ones(kvm_lib, kinds):
    """A CTA's next row tile may fill two of its four pairs of warps while the others still
    store the last one, which V blocks beyond F16 make long: every row as the definition
    has it, and the same bits on every run."""
    import torch
    news, lens = [66, 44, 109, 65, 34, 71, 97, 92], [94, 61, 110, 81, 33, 69, 113, 91]
    w = Window(kvm_lib, torch, 3, kinds, 4, 128, 32, lens)

    def change(v):
        v[np.random.default_rng(0).random(v.shape[0]) < 0.05] *= 6e4 if kinds[1] == "f16" else 75000.0
        return np.clip(v, -6e4, 6e4) if kinds[1] == "f16" else np.clip(v, -4e5, 4e5)
    rewrite(w, 1, change)
    if kinds[1] == "f16":                      # infinities are what F16 rows have to add apart
        raw = w.raw[1].copy()
        raw.view(np.float16)[w.cell(2, 3)] = np.inf
        w.put(1, raw)
    start = np.concatenate([[0], np.cumsum(news)])
    q = queries(torch, w.rng, int(start[-1]), 48, 128, "bf16")
    got = w.run(q, start, True, max_new=7)
    for _ in range(5):
        assert torch.equal(w.run(q, start, True, max_new=7).view(torch.int16), got.view(torch.int16))
    with np.errstate(invalid="ignore"):
        want = reference(w, q.float().cpu().numpy(), start, lens, 128 ** -0.5, rows=range(0, int(start[-1]), 5))
    pick = [r for r in range(0, int(start[-1]), 5) if not (start[2] <= r < start[3] and kinds[1] == "f16")]
    agree(got[pick], *(x[pick] for x in want), max(lens))
