"""The binding packs its arguments itself: numbers that do not fit their field are refused
like any other bad argument."""
import pytest

from test_gpu_layer import Window, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [dict(max_new=-1), dict(max_new=1 << 32), dict(scale=1e39), dict(max_new=1.5), dict(scale=None)])
def test_attend_refuses_numbers_that_do_not_fit(kvm_lib, bad):
    import torch
    kvm = kvm_lib
    w = Window(kvm, torch, 1, ("q4_0", "q4_0"), 1, 64, 16, [32])
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = queries(torch, w.rng, 1, 2, 64, "f16")
    args = dict(q=q, q_start=i([0, 1]), kv_len=i([32]), table=i(w.table), out=torch.empty_like(q),
                work=torch.empty(kvm.ATTEND_WORK_BYTES, dtype=torch.uint8, device="cuda"), scale=0.1)
    kvm.attend(w.cache, **args)
    with pytest.raises(kvm.KvmError) as e:
        kvm.attend(w.cache, **{**args, **bad})
    assert e.value.status == kvm.KVM_EINVAL


@pytest.mark.parametrize("tokens", [-1, 1 << 32, 2.5, None])
def test_map_batch_refuses_numbers_that_do_not_fit(kvm_lib, tokens):
    import torch
    kvm = kvm_lib
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(kvm.KvmError) as e:
        kvm.map_batch(i([0]), i([1]), i([0]), tokens, i([[-1]]), i([0, 0]), i([0]), torch.zeros(1, dtype=torch.int64, device="cuda"), i([0]),
                      i([0]), i([0] * 4))
    assert e.value.status == kvm.KVM_EINVAL
