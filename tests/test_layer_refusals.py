"""Refusals of the attention layer's calls (kvm_map_batch, kvm_qk_norm_rope,
kvm_write_rows, kvm_read_rows, kvm_attend): every bad argument is KVM_EINVAL
with a reason, before any device work.  The addresses are never used, so this
runs without a GPU."""
import ctypes as C

import pytest

import kvm

P = 0x100000                      # an aligned address that nothing reads
WORK = kvm.ATTEND_WORK_BYTES


def rows(heads=8, dim=128, type_=kvm.TYPE_F16, data=P, es=2, **kw):
    r = kvm.Rows(data, type_, heads, dim, 0, es, dim * es, heads * dim * es)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def cache(**kw):
    c = kvm._Cache(P, P, kvm.TYPE_Q4_0, kvm.TYPE_Q4_0, 2, 128, 128, 16)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def refused(st, word):
    assert st == kvm.KVM_EINVAL
    assert word in kvm.lib().kvm_last_error(None).decode()


def batch_map(**kw):
    m = kvm._BatchMap(P, P, P, P, 8, 8, 4, 16, 128, 64, 0, P, P, P, P, P, P)
    for k, v in kw.items():
        setattr(m, k, v)
    return m


@pytest.mark.parametrize("change, word", [
    (dict(n_seq=0), "requests"), (dict(n_seq=4097), "requests"), (dict(block_tokens=0), "block_tokens"),
    (dict(table_stride=7), "table_stride"), (dict(d_past=None), "null"), (dict(d_free=None), "null"),
    (dict(d_cells=None), "null"), (dict(d_info=None), "null"), (dict(d_table=None), "null"),
    (dict(n_rows=1 << 31), "2^31"), (dict(d_cells=P + 4), "aligned"), (dict(d_pos=P + 2), "aligned")])
def test_map_batch(change, word):
    refused(kvm.lib().kvm_map_batch(None, C.byref(batch_map(**change))), word)


def test_map_batch_null():
    refused(kvm.lib().kvm_map_batch(None, None), "null")


def rope(n=4, q=None, k=None, qo=None, ko=None, eps=1e-6, n_rot=64, freqs=P, pos=P, qw=P):
    b = lambda r: None if r is None else C.byref(r)  # noqa: E731
    return kvm.lib().kvm_qk_norm_rope(None, n, b(q or rows()), b(k or rows(2)), qw, P, eps, freqs, n_rot, pos,
                                      b(qo or rows()), b(ko or rows(2)))


@pytest.mark.parametrize("args, word", [
    (dict(q=rows(dim=120), qo=rows(dim=120)), "head_dim"), (dict(q=rows(dim=528), qo=rows(dim=528)), "head_dim"),
    (dict(n_rot=24), "n_rot"), (dict(n_rot=144), "n_rot"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(freqs=None), "freqs"), (dict(pos=None), "pos"), (dict(qw=P + 2), "aligned"),
    (dict(q=rows(type_=kvm.TYPE_Q8_0)), "type"), (dict(qo=rows(type_=kvm.TYPE_BF16)), "one type"),
    (dict(k=rows(2, type_=kvm.TYPE_BF16)), "one type"), (dict(k=rows(2, dim=64)), "heads of"),
    (dict(qo=rows(9)), "heads of"), (dict(q=rows(data=P + 1)), "multiples"), (dict(q=rows(nb_head=129)), "multiples"),
    (dict(q=rows(data=None)), "null"), (dict(q=rows(0), qo=rows(0)), "heads")])
def test_qk_norm_rope(args, word):
    refused(rope(**args), word)


def test_qk_norm_rope_k_without_output():
    st = kvm.lib().kvm_qk_norm_rope(None, 4, C.byref(rows()), C.byref(rows(2)), P, P, 1e-6, P, 64, P, C.byref(rows()), None)
    refused(st, "together")


@pytest.mark.parametrize("name", ["kvm_write_rows", "kvm_read_rows"])
@pytest.mark.parametrize("args, word", [
    (dict(c=cache(type_k=3)), "types"), (dict(c=cache(type_v=kvm.TYPE_F32)), "types"), (dict(c=cache(d_v=None)), "null"),
    (dict(c=cache(head_dim=48)), "multiple of 32"), (dict(c=cache(n_head_kv=0)), "KV heads"),
    (dict(c=cache(n_head_kv=65)), "KV heads"), (dict(c=cache(n_slots=0)), "n_slots"),
    (dict(c=cache(n_slots=1 << 24)), "n_slots"), (dict(c=cache(d_k=P + 2)), "4-byte"), (dict(cells=None), "cells"),
    (dict(cells=P + 4), "cells"), (dict(k=None, v=None), "neither"), (dict(k=rows(3)), "heads of"),
    (dict(v=rows(2, type_=kvm.TYPE_F32, es=4)), "one type"), (dict(k=rows(2, type_=kvm.TYPE_Q4_0)), "type")])
def test_rows(name, args, word):
    a = dict(c=cache(), cells=P, k=rows(2), v=rows(2))
    a.update(args)
    b = lambda r: None if r is None else C.byref(r)  # noqa: E731
    refused(getattr(kvm.lib(), name)(None, C.byref(a["c"]), 4, a["cells"], b(a["k"]), b(a["v"])), word)


def attend(c=None, q=None, out=None, work=P, work_bytes=WORK, **kw):
    bt = kvm._AttendBatch(P, 8, 8, 4, P, P, 4, 1, 1, 0.125)
    for k, v in kw.items():
        setattr(bt, k, v)
    return kvm.lib().kvm_attend(None, C.byref(c or cache()), C.byref(bt), C.byref(q or rows()), C.byref(out or rows()),
                                work, work_bytes)


@pytest.mark.parametrize("args, word", [
    (dict(c=cache(head_dim=96)), "64, 128 or 256"), (dict(q=rows(7), out=rows(7)), "multiple of"),
    (dict(q=rows(type_=kvm.TYPE_F32, es=4)), "F16 or BF16"), (dict(out=rows(type_=kvm.TYPE_F32, es=4)), "F16 or BF16"),
    (dict(out=rows(4)), "heads of"), (dict(flags=2), "flags"), (dict(scale=float("inf")), "finite"),
    (dict(scale=float("nan")), "finite"), (dict(table_stride=7), "table_stride"), (dict(d_table=None), "null"),
    (dict(d_q_start=None), "null"), (dict(d_kv_len=None), "null"), (dict(d_kv_len=P + 2), "4-byte"),
    (dict(work=None), "workspace"), (dict(work_bytes=WORK - 1), "workspace"), (dict(work=P + 8), "workspace"),
    (dict(n_seq=65536), "65535"), (dict(n_rows=1 << 30, ), "too many"), (dict(c=cache(d_v=P + 1)), "4-byte"),
    (dict(q=rows(data=P + 1)), "multiples")])
def test_attend(args, word):
    refused(attend(**args), word)


def test_calls_with_no_rows_do_nothing():
    L = kvm.lib()
    assert attend(n_seq=0) == kvm.KVM_OK and attend(n_rows=0) == kvm.KVM_OK
    assert rope(n=0) == kvm.KVM_OK
    for fn in (L.kvm_write_rows, L.kvm_read_rows):
        assert fn(None, C.byref(cache()), 0, None, C.byref(rows(2)), None) == kvm.KVM_OK


def test_packed_structs_match_ctypes():
    """The binding packs its structs by format strings: the same bytes as ctypes'."""
    r = (0x1122334455667788, 30, 7, 128, 0, 2, 256, 1 << 40)
    assert kvm._PACK_ROWS(*r) == bytes(kvm.Rows(*r))
    m = tuple(range(3, 20))
    assert kvm._PACK_MAP(*m) == bytes(kvm._BatchMap(*m))
    b = (1, 2, 3, 4, 5, 6, 7, 8, 9, 0.25)
    assert kvm._PACK_ATTEND(*b) == bytes(kvm._AttendBatch(*b))


def test_struct_layouts_match_c(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "layout.c"
    fields = {"kvm_cache": kvm._Cache, "kvm_batch_map": kvm._BatchMap, "kvm_attend_batch": kvm._AttendBatch}
    lines = [f'printf("{n} %zu\\n", sizeof({n}));' + "".join(
        f'printf("{n}.{f[0]} %zu\\n", offsetof({n}, {f[0]}));' for f in c._fields_) for n, c in fields.items()]
    lines.append('printf("work %zu\\n", (size_t) KVM_ATTEND_WORK_BYTES);')
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "kvm.h"\nint main(void) {' + "\n".join(lines) + "return 0;}")
    exe = tmp_path / "layout"
    r = subprocess.run([os.environ.get("CC", "gcc"), "-I", os.path.join(root, "include"), str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    if r.returncode != 0:
        pytest.skip("no C compiler: " + r.stderr[:200])
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n") if x)
    for n, c in fields.items():
        assert int(got[n]) == C.sizeof(c)
        for f in c._fields_:
            assert int(got[f"{n}.{f[0]}"]) == getattr(c, f[0]).offset
    assert int(got["work"]) == kvm.ATTEND_WORK_BYTES
