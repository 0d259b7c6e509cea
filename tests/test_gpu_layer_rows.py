"""kvm_write_rows on blocks at the edges of the quantizers: zeros of both signs, infinities
and NaN give the bytes of kvm_quantize_rows, and those of zeros the oracle's."""
import numpy as np
import pytest

import layer_ref as ref

pytestmark = pytest.mark.gpu


def blocks():
    """[n, 32] float16 blocks."""
    z = np.zeros((12, 32), np.float16)
    z[1] = -0.0                                # the first value -0
    z[2, 0] = -0.0                             # ... and the others +0
    z[3, 1:] = -0.0
    z[4, 5], z[4, 9] = -0.0, 2.0 ** -24        # the smallest value
    z[5, 0], z[5, 31] = -0.0, -2.0 ** -24
    z[6, 0], z[6, 3], z[6, 17] = -0.0, 1.5, -1.5
    z[7], z[7, 3] = 1.0, np.inf
    z[8], z[8, 3] = -1.0, np.nan
    z[9] = np.nan
    z[10], z[10, 0], z[10, 1] = 2.0, -np.inf, np.inf
    z[11] = 65504.0
    return z


@pytest.mark.parametrize("dtype", ["f16", "f32", "bf16"])
@pytest.mark.parametrize("kind", ["q4_0", "q5_0", "q8_0"])
def test_write_rows_zeros_and_specials(kvm_lib, oracle, kind, dtype):
    import torch
    kvm, t, size = kvm_lib, ref.TYPES[kind], ref.SIZE[kind]
    x = blocks()
    if dtype == "bf16":
        x = x[[0, 1, 2, 3, 6, 7, 8, 9, 10]]    # those that BF16 holds
    n = len(x)
    rows = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    want = torch.zeros((n, size), dtype=torch.uint8, device="cuda")
    kvm.quantize_rows(t, rows, n, 32, want)
    for width in (1, 2):                       # a block a row (single blocks), and two
        m = n // width * width
        raw = torch.zeros((m, size), dtype=torch.uint8, device="cuda")
        cache = kvm.Cache(raw, raw.clone(), t, t, width, 32, 1, m // width)
        act = rows[:m].to({"f16": torch.float16, "f32": torch.float32, "bf16": torch.bfloat16}[dtype]).reshape(m // width, width, 32)
        kvm.write_rows(cache, torch.arange(m // width, device="cuda"), act, None)
        assert torch.equal(raw, want[:m])
        zero = [i for i in range(m) if not x[i].any()]
        assert len(zero) == 4
        assert np.array_equal(raw.cpu().numpy()[zero], oracle.quantize_rows_f16(t, x[zero]))
