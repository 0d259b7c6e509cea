"""Where the attention kernels cut their work: every key counted once in every row, by
values that mark their key.  One key lost, doubled or seen too much fails each of these."""
import numpy as np
import pytest

import layer_ref as ref
from test_gpu_layer import Window, queries
from test_gpu_layer_range import agree, reference

pytestmark = pytest.mark.gpu

# head size, KV heads, group, rows and keys of the requests, tokens a block
FEW = [(256, 4, 6, [1], [20011], 128),                          # one window over every CTA, four KV heads a CTA
       (256, 1, 6, [1], [20011], 128),
       (128, 2, 3, [1] * 4, [9001, 333, 17, 4000], 32),
       (128, 4, 12, [1] * 9, [3000, 1, 777, 2048, 15, 16, 17, 4001, 640], 32),      # row tiles of 16
       (64, 2, 4, [2, 1, 2], [5000, 4, 999], 24),               # blocks that end inside a step
       (64, 4, 2, [1] * 70, [50 + 3 * i for i in range(70)], 16)]       # short windows, nothing cut
MANY = [(64, 4, 8, [500, 410, 300], [700, 410, 900], 32),       # single CTAs: several items a CTA
        (64, 1, 3, [70, 9], [6001, 64], 24),
        (256, 4, 6, [260, 17], [5000, 3001], 32),               # pairs: items of several pairs
        (128, 2, 4, [100, 20, 70], [400, 3000, 100], 24),
        (256, 2, 6, [4] * 8, [1000 + 77 * i for i in range(8)], 128)]   # drafts


def setup(kvm, torch, kinds, D, hkv, group, news, lens, T):
    w = Window(kvm, torch, D + len(lens), kinds, hkv, D, T, lens)
    start = np.concatenate([[0], np.cumsum(news)])
    return w, start, queries(torch, w.rng, int(start[-1]), hkv * group, D, "f16")


def mark(w, side, values):
    """Rows of one side: values(request, key numbers) [keys, width], zeros elsewhere."""
    x = np.zeros((w.raw[side].shape[0], w.hkv * w.D), np.float32)
    for s, n in enumerate(w.lens):
        j = np.arange(n)
        x[w.table[s, j // w.T].astype(np.int64) * w.T + j % w.T] = values(s, j)
    w.put(side, ref.quantize(x, w.kinds[side]))


@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q8_0"), ("q5_0", "f16"), ("f16", "q5_0")])
@pytest.mark.parametrize("D, hkv, group, news, lens, T", FEW + MANY)
@pytest.mark.parametrize("causal", [True, False])
def test_every_key_counts_once(kvm_lib, kinds, D, hkv, group, news, lens, T, causal):
    """A scale of 0 gives every key the same weight; key j of KV head h holds one value, in dim
    (2 h + 1) j mod D.  Each dim is its keys' number over all keys': F32 sums of exact
    products, one rounding on the way through the workspace and one of the output."""
    import torch
    w, start, q = setup(kvm_lib, torch, kinds, D, hkv, group, news, lens, T)
    unit = 127.0 if kinds[1] == "q8_0" else 128.0              # exact in a block of zeros and this

    def values(s, j):
        x = np.zeros((j.size, hkv, D), np.float32)
        for h in range(hkv):
            x[np.arange(j.size), h, (2 * h + 1) * j % D] = unit
        return x.reshape(j.size, -1)
    mark(w, 1, values)
    got = w.run(q, start, causal, scale=0.0, max_new=max(news)).float().cpu().numpy().astype(np.float64)
    for s, (new, keys) in enumerate(zip(news, lens)):
        seen = np.clip(keys - new + 1 + np.arange(new), 0, keys) if causal else np.full(new, keys)
        for h in range(hkv):
            dim = (2 * h + 1) * np.arange(keys) % D
            count = np.zeros((keys + 1, D))
            count[1:] = np.cumsum(np.eye(D)[dim], 0)
            want = unit * count[seen] / np.maximum(seen, 1)[:, None]
            tol = want * (2 * 2.0 ** -11 + 2.0 ** -16)
            # one key more or less moves its dim by more than that
            assert (unit / np.maximum(seen, 1)[:, None] > 2 * tol + 2.0 ** -24).all()
            part = got[start[s]:start[s + 1], h * group:(h + 1) * group]
            assert (np.abs(part - want[:, None]) <= (tol + 2.0 ** -25)[:, None]).all(), (s, h)


@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("f16", "q8_0"), ("q4_0", "f16")])
@pytest.mark.parametrize("D, hkv, group, news, lens, T", [
    (64, 2, 4, [2, 1, 2], [1500, 4, 999], 24), (128, 4, 3, [3, 5, 1, 2], [1901, 333, 17, 700], 32), (256, 1, 6, [4] * 4, [1999, 80, 257, 1024], 128),
    (64, 4, 8, [500, 410, 300], [700, 410, 900], 32), (256, 2, 6, [260, 17], [1500, 1001], 32), (128, 2, 4, [100, 20, 70], [400, 1900, 100], 24)])
def test_every_row_ends_at_its_last_key(kvm_lib, kinds, D, hkv, group, news, lens, T):
    """Key j scores 20 above key j - 1, so a row is the value of the last key it sees: K is j + 1
    in every dim, exact in these types, and V marks j in one dim of D."""
    import torch
    w, start, q = setup(kvm_lib, torch, kinds, D, hkv, group, news, lens, T)
    q = torch.ones_like(q)
    mark(w, 0, lambda s, j: np.repeat(j[:, None] + 1.0, hkv * D, 1))
    unit = 127.0 if kinds[1] == "q8_0" else 128.0
    mark(w, 1, lambda s, j: np.tile(unit * np.eye(D)[j % D], (1, hkv)))
    got = w.run(q, start, True, scale=20.0 / D, max_new=max(news)).float().cpu().numpy()
    for s, (new, keys) in enumerate(zip(news, lens)):
        last = keys - new + np.arange(new)
        want = np.where(last[:, None] >= 0, unit * np.eye(D)[last % D], 0.0)
        assert (np.abs(got[start[s]:start[s + 1]] - want[:, None]) <= unit * 2.0 ** -10).all(), s


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q5_0", "q5_0"), ("f16", "f16"), ("q4_0", "f16"), ("f16", "q8_0")])
def test_few_rows_round_no_key(kvm_lib, kinds, D):
    """The few-row kernel takes K's codes and scales as they are: scores as an F32 sum gives them."""
    import torch
    w = Window(kvm_lib, torch, D, kinds, 2, D, 32, [500, 1, 33, 190])
    q = queries(torch, w.rng, 4, 6, D, "f16") * 4
    got = w.run(q, range(5))
    want, spread, peak, ds = reference(w, q.float().cpu().numpy(), range(5), w.lens, D ** -0.5)
    agree(got, want, spread, peak, ds * (D * 2.0 ** -23) / (2.0 ** -11 + D * 2.0 ** -23), 500)
