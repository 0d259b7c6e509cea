"""Attention of requests with many query rows: what the pairs of CTAs (over 128
rows a KV head) and the single ones do with hidden and infinite values, odd
alignment, requests of every size behind one another, capture and streams."""
import numpy as np
import pytest

from test_gpu_layer import Window, queries

pytestmark = pytest.mark.gpu


def ints(torch, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q8_0"), ("q5_0", "q4_0"), ("f16", "q4_0")])
@pytest.mark.parametrize("D, T", [(128, 16), (256, 32), (128, 24)])
def test_long_requests_and_hidden_rows(kvm_lib, kinds, D, T):
    """Other blocks' rows may be NaN; an infinite key and value that only the last
    row sees stays with it."""
    import torch
    new, keys = 70, 333
    w = Window(kvm_lib, torch, D + T, kinds, 2, D, T, [keys, 75])
    q = queries(torch, w.rng, new, 8, D, "f16")
    start = [0, new, new]
    clean = w.check(q, start, True, max_new=new).clone()
    for side in (0, 1):
        raw = w.raw[side].copy()
        seen = {w.cell(0, j) for j in range(keys)}
        for c in range(raw.shape[0]):
            if c not in seen:
                raw[c].view(np.uint8)[:] = 0xFF
        w.put(side, raw)
    assert torch.equal(w.run(q, start, True, max_new=new), clean)
    for side in (0, 1):
        raw = w.raw[side].copy()
        c = w.cell(0, keys - 1)
        raw[c, 0:2] = np.array([0x00, 0x7C], np.uint8)
        raw[c, -2:] = np.array([0x00, 0x7C], np.uint8)
        if kinds[side] == "f16":
            raw[c].view(np.float16)[:] = np.inf
        w.put(side, raw)
    got = w.run(q, start, True, max_new=new)
    assert torch.isfinite(got[:new - 1]).all() and not torch.isfinite(got[new - 1]).all()
    assert torch.allclose(got[:new - 1].float(), clean[:new - 1].float(), rtol=2.0 ** -9, atol=2.0 ** -9)


@pytest.mark.parametrize("D", [128, 256])
def test_long_requests_see_an_infinite_value(kvm_lib, D):
    """A V block whose scale is infinite, seen by every row: its dims are infinite or
    NaN in every row, the others as without it."""
    import torch
    new, keys = 40, 200
    w = Window(kvm_lib, torch, 5, ("q4_0", "q4_0"), 1, D, 32, [keys])
    q = queries(torch, w.rng, new, 6, D, "bf16")
    clean = w.run(q, [0, new], False, max_new=new)
    raw = w.raw[1].copy()
    for block in (1, D // 32 - 1):                    # one in each CTA's half
        raw[w.cell(0, 9), 18 * block:18 * block + 2] = np.array([0x00, 0x7C], np.uint8)
    w.put(1, raw)
    got = w.run(q, [0, new], False, max_new=new)
    hit = torch.zeros(D, dtype=torch.bool, device="cuda")
    for block in (1, D // 32 - 1):
        hit[32 * block:32 * block + 32] = True
    assert not torch.isfinite(got[..., hit]).any()
    assert torch.equal(got[..., ~hit], clean[..., ~hit])


@pytest.mark.parametrize("base", [0, 4])
@pytest.mark.parametrize("D", [128, 256])
def test_long_requests_strides_and_alignment(kvm_lib, base, D):
    import torch
    new = 33
    w = Window(kvm_lib, torch, 6, ("q4_0", "q8_0"), 2, D, 32, [150, 77], base=base)
    q = queries(torch, w.rng, 2 * new, 10, D, "f16")
    start = [0, new, 2 * new]
    want = w.check(q, start, True, max_new=new)
    odd = torch.zeros((D, 10, 2 * new + 1), dtype=q.dtype, device="cuda").permute(2, 1, 0)[1:]
    odd.copy_(q)
    out = torch.full((2 * new, 10, D + 1), 7.0, dtype=q.dtype, device="cuda")
    got = w.run(odd, start, True, out=out[:, :, 1:], max_new=new)
    assert torch.equal(got, want) and (out[:, :, 0] == 7).all()


@pytest.mark.parametrize("D, hkv, group, most", [(64, 1, 1, 130), (128, 2, 3, 43), (128, 1, 4, 60), (256, 1, 6, 22), (128, 1, 4, 32), (256, 1, 3, 42)])
def test_requests_of_every_size_behind_one_another(kvm_lib, D, hkv, group, most):
    """Row tiles with one to four pairs of warps in use, in every order, with and
    without keys, on every CTA: more requests than SMs and threads."""
    import torch
    rng = np.random.default_rng(D + most)
    news = [int(x) for x in rng.integers(0, most + 1, 600)]
    lens = [int(rng.integers(0, 2 * n + 40)) if i % 7 else 0 for i, n in enumerate(news)]
    w = Window(kvm_lib, torch, 8, ("q4_0", "q4_0"), hkv, D, 16, lens)
    start = np.concatenate([[0], np.cumsum(news)])
    q = queries(torch, w.rng, int(start[-1]), hkv * group, D, "f16")
    first = w.check(q, start, True, max_new=most)
    assert torch.equal(w.run(q, start, True, max_new=most), first)


def test_long_requests_captured_and_replayed(kvm_lib):
    import torch
    w = Window(kvm_lib, torch, 21, ("q4_0", "q4_0"), 2, 128, 32, [700, 420, 90])
    start = [0, 100, 150, 160]
    q = queries(torch, w.rng, 160, 6, 128, "bf16")
    out, work = torch.zeros_like(q), torch.empty(kvm_lib.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda")
    qs, kv, table = ints(torch, start), ints(torch, [1, 1, 1]), ints(torch, w.table)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kvm_lib.attend(w.cache, q, qs, kv, table, out, work, scale=0.1, max_new=100)
        graph.capture_begin()
        kvm_lib.attend(w.cache, q, qs, kv, table, out, work, scale=0.1, max_new=100)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for lens in ([700, 420, 90], [64, 419, 3], [0, 33, 1]):
        kv.copy_(ints(torch, lens))
        q.copy_(queries(torch, w.rng, 160, 6, 128, "bf16"))
        work.fill_(0xFF)
        graph.replay()
        assert torch.equal(out, w.run(q, start, scale=0.1, max_new=100, kv_len=lens))


def test_long_requests_on_two_streams(kvm_lib):
    import torch
    w = Window(kvm_lib, torch, 31, ("q4_0", "q4_0"), 2, 128, 32, [3000, 900])
    q = queries(torch, w.rng, 300, 6, 128, "f16")
    start = [0, 200, 300]
    want = w.run(q, start, max_new=200)
    qs, kv, table = ints(torch, start), ints(torch, w.lens), ints(torch, w.table)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.zeros_like(q) for _ in range(6)] for _ in streams]
    works = [torch.empty(kvm_lib.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for n in range(6):
        for s, o, wk in zip(streams, outs, works):
            kvm_lib.attend(w.cache, q, qs, kv, table, o[n], wk, scale=128 ** -0.5, max_new=200, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for side in outs for o in side)


@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q5_0")])
def test_long_requests_values_and_queries_of_every_size(kvm_lib, kinds):
    import torch
    new = 50
    w = Window(kvm_lib, torch, 9, kinds, 1, 128, 16, [400], scale_v=lambda r, n: 10.0 ** r.uniform(-6, 3.5, n))
    q = queries(torch, w.rng, new, 8, 128, "bf16")
    want = w.check(q, [0, new], True, scale=0.05, max_new=new)
    for e in (-90, 90):
        scaled = (q.float() * 2.0 ** e).to(torch.bfloat16)
        assert torch.equal(w.run(scaled, [0, new], True, scale=0.05 * 2.0 ** -e, max_new=new), want)


def test_rows_that_share_a_cell_leave_the_others(kvm_lib):
    """Two rows for one cell: its content is undefined, every other cell is right."""
    import torch
    n, width, T = 40, 256, 16
    g = torch.Generator().manual_seed(3)
    x = torch.randn((n, 2, 128), generator=g).half().cuda()
    rows = torch.zeros(64 * 144, dtype=torch.uint8, device="cuda")
    once = torch.zeros_like(rows)
    cells = torch.arange(n, dtype=torch.int64, device="cuda") + 5
    kvm_lib.write_rows(kvm_lib.Cache(once, once.clone(), kvm_lib.TYPE_Q4_0, kvm_lib.TYPE_Q4_0, 2, 128, T, 4), cells, x, None)
    cells[7] = cells[31]
    kvm_lib.write_rows(kvm_lib.Cache(rows, rows.clone(), kvm_lib.TYPE_Q4_0, kvm_lib.TYPE_Q4_0, 2, 128, T, 4), cells, x, None)
    keep = [c for c in range(64) if c not in (12, 36)]
    assert torch.equal(rows.view(64, 144)[keep], once.view(64, 144)[keep])
    assert not rows.view(64, 144)[12].any()


@pytest.mark.parametrize("T", [128, 24])
def test_cells_past_four_gigabytes(kvm_lib, T):
    """The last blocks of a cache of 4.6 GB a side: rows in, rows out and attention
    are those of a small cache with the same rows."""
    import torch
    h, d, keys = 4, 256, 300
    blocks = -(-keys // T)
    slots = 4_300_000 // T
    row = h * d // 32 * 34
    far = [torch.zeros(slots * T * row, dtype=torch.uint8, device="cuda") for _ in "kv"]
    near = [torch.zeros(blocks * T * row, dtype=torch.uint8, device="cuda") for _ in "kv"]
    g = torch.Generator().manual_seed(T)
    k, v = ((torch.randn((keys, h, d), generator=g)).half().cuda() for _ in "kv")
    outs = []
    for bufs, n in ((far, slots), (near, blocks)):
        cache = kvm_lib.Cache(bufs[0], bufs[1], kvm_lib.TYPE_Q8_0, kvm_lib.TYPE_Q8_0, h, d, T, n)
        table = ints(torch, [[n - 1 - b for b in range(blocks)]])
        cells = torch.tensor([(n - 1 - j // T) * T + j % T for j in range(keys)], dtype=torch.int64, device="cuda")
        kvm_lib.write_rows(cache, cells, k, v)
        back = [torch.zeros_like(k) for _ in "kv"]
        kvm_lib.read_rows(cache, cells, *back)
        outs.append(back)
        for new in (1, 7, 60):
            q = torch.randn((new, 3 * h, d), generator=torch.Generator().manual_seed(new)).half().cuda()
            out = torch.zeros_like(q)
            kvm_lib.attend(cache, q, ints(torch, [0, new]), ints(torch, [keys]), table, out,
                           torch.empty(kvm_lib.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda"), scale=d ** -0.5, max_new=new)
            outs[-1].append(out)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert outs[0][2].any() and (outs[0][0].float() - k.float()).abs().max() < 0.05


@pytest.mark.parametrize("D, new", [(64, 1), (64, 20), (128, 130)])
def test_lengths_up_to_the_last_key_number(kvm_lib, D, new):
    """A table of 2^31 keys of which two blocks hold any, the second at its very end:
    key numbers stay inside 32 bits, and keys from 2^31 - 65536 on are not seen."""
    import layer_ref as ref
    import torch
    T, cols = 4096, 524288
    w = Window(kvm_lib, torch, D, ("q4_0", "q4_0"), 1, D, T, [2 * T], spare=1)
    table = np.full((1, cols), -1, np.int32)
    table[0, 0], table[0, cols - 17], table[0, cols - 16:] = 0, 1, 2      # 17 blocks are 65536 + T keys
    q = queries(torch, w.rng, new, 1, D, "f16")
    got = w.run(q, [0, new], False, max_new=new, kv_len=[2 ** 31 - 1], table=table).float().cpu().numpy()
    near = np.array([[0, 1]], np.int32)
    w.table = near
    same = w.check(q, [0, new], False, max_new=new, kv_len=[2 * T]).float().cpu().numpy()
    # both sum the same keys, in other places: each is off by what the check allows
    _, spread, _ = ref.attend(q.float().cpu().numpy(), w.raw[0], w.raw[1], w.kinds, 1, T, w.slots, near, [0, new], [2 * T],
                              D ** -0.5, False, np.zeros(q.shape))
    assert (np.abs(got - same) <= spread * 2.0 ** -8 + np.abs(same) * 2.0 ** -10 + 2.0 ** -24).all()


@pytest.mark.parametrize("kinds", [("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q5_0", "q5_0"), ("f16", "f16")])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B, group, new", [(12, 6, 2), (3, 6, 4), (2, 3, 8)])
def test_drafts_of_few_and_many_requests(kvm_lib, kinds, D, B, group, new):
    """9 to 24 rows a KV head, in row tiles of 16 (many requests) and of 8 (few)."""
    import torch
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(new, 700, B)]
    w = Window(kvm_lib, torch, 40 + B, kinds, 2, D, 32, lens)
    start = [new * i for i in range(B + 1)]
    w.check(queries(torch, w.rng, new * B, 2 * group, D, "bf16"), start, True, max_new=new)
