"""Bounded waits of the attention kernels: rows that never arrive (a box that the test
flags leave unloaded) end in NaN where they were needed, never in a wrong value, and the
next call is right.  Nothing faults; each case waits for some seconds."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_layer import Window, queries

pytestmark = pytest.mark.gpu


def call(kvm, torch, w, q, start, max_new, flags):
    ints = [torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda") for v in (w.table, start, w.lens)]
    out, work = torch.zeros_like(q), torch.empty(kvm.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda")
    n, hq, D = q.shape
    t = {torch.float16: kvm.TYPE_F16, torch.bfloat16: kvm.TYPE_BF16}[q.dtype]
    rows = [kvm.Rows(x.data_ptr(), t, hq, D, 0, 2, 2 * D, 2 * D * hq) for x in (q, out)]
    cols = w.table.shape[1]
    batch = kvm._AttendBatch(ints[0].data_ptr(), cols, cols, len(w.lens), ints[1].data_ptr(), ints[2].data_ptr(), n, max_new,
                             kvm.ATTEND_CAUSAL | flags, D ** -0.5)
    st = kvm.lib().kvm_attend(torch.cuda.current_stream().cuda_stream, C.byref(w.cache), C.byref(batch), C.byref(rows[0]),
                              C.byref(rows[1]), work.data_ptr(), work.numel())
    assert st == kvm.KVM_OK
    torch.cuda.synchronize()
    return out


def check(kvm, torch, w, q, start, max_new, side):
    clean = call(kvm, torch, w, q, start, max_new, 0)
    assert torch.isfinite(clean).all()
    got = call(kvm, torch, w, q, start, max_new, kvm.ATTEND_TEST_SKIP_K if side == "k" else kvm.ATTEND_TEST_SKIP_V)
    lost = got.isnan()
    assert torch.equal(lost.all(-1), lost.any(-1))              # a row and head as a whole ...
    assert torch.equal(got[~lost], clean[~lost])                # ... or as it should be
    # the first row tile of the first request and KV head is what the flag names
    group = q.shape[1] // w.hkv
    first = min(int(start[1]), 8 // group or 1)
    assert lost[:first, :min(group, 8)].all()
    assert torch.equal(call(kvm, torch, w, q, start, max_new, 0), clean)
    return lost


@pytest.mark.parametrize("side, kinds, D, hkv, group, news, lens", [
    ("k", ("q4_0", "q4_0"), 128, 2, 6, [1] * 3, [300, 80, 700]),         # whole windows: a KV head a CTA, nothing cut
    ("v", ("q8_0", "q5_0"), 256, 4, 6, [1] * 2, [9000, 20000]),          # windows that many CTAs share
    ("k", ("f16", "q8_0"), 128, 4, 12, [1] * 9, [5000] * 9),             # row tiles of 16
    ("v", ("q4_0", "f16"), 64, 4, 3, [2, 5, 1], [200, 4000, 64]),        # several rows a request
    ("k", ("q4_0", "q4_0"), 128, 2, 4, [20, 9, 31], [300, 2000, 100]),   # single CTAs, items of many CTAs
    ("v", ("q8_0", "q4_0"), 64, 4, 8, [90, 40], [300, 90]),              # more than one piece a CTA
    ("k", ("q4_0", "q4_0"), 128, 2, 4, [100, 20, 70], [400, 3000, 100]), # pairs: the first CTA's keys,
    ("v", ("q8_0", "q4_0"), 256, 1, 6, [80], [5000])])                   # the second one's values
def test_rows_that_never_arrive(kvm_lib, side, kinds, D, hkv, group, news, lens):
    import torch
    w = Window(kvm_lib, torch, D + len(lens), kinds, hkv, D, 32, lens)
    start = np.concatenate([[0], np.cumsum(news)])
    q = queries(torch, w.rng, int(start[-1]), hkv * group, D, "f16")
    check(kvm_lib, torch, w, q, start, max(news) if max(news) > 8 else 1, side)
