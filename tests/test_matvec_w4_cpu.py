"""Products with 4-bit weights: what is refused before anything reaches a GPU."""
import ctypes as C

import pytest
import torch


def call(pkg, n=32, k=256, group=64, E=1, dtype=0, gated=0, zeros=None, by_token=0, plan=None, rows=1):
    err = C.create_string_buffer(256)
    w = pkg._lib.W4(None, None, zeros, E, n, k, group)
    rc = pkg._lib.load().moe_fp8_b200_matvec_w4(None, 0, by_token, C.byref(w), gated, None, 0, dtype,
                                                None if plan is None else C.byref(plan), rows, None, err, 256)
    return rc, err.value.decode()


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=2), "bf16 or fp16"), (dict(group=16), "group"), (dict(group=256), "group"), (dict(k=96), "multiple"),
    (dict(k=0), "multiple"), (dict(k=8256), "8192"), (dict(n=24), "multiple of 16"), (dict(n=0), "multiple of 16"),
    (dict(n=(1 << 20) + 16), "2^20"), (dict(E=0), "num_experts"), (dict(E=1025), "num_experts"), (dict(E=2), "plan"),
    (dict(by_token=1), "plan"), (dict(rows=-1), "num_rows"), (dict(rows=(1 << 21) + 1), "rows are more"),
    (dict(rows=1 << 21, n=1 << 20), "too many"), (dict(k=192, gated=1, zeros=16), "even number of groups")])
def test_sizes(pkg, bad, text):
    rc, msg = call(pkg, **bad)
    assert rc == pkg._lib.ERR_INVALID_ARGUMENT and text in msg, msg


def test_plan_of_other_experts_and_null_weights(pkg):
    rc, msg = call(pkg, E=4, plan=pkg._lib.Plan(1, 1, 3, 1, None, None, None, None))
    assert rc == pkg._lib.ERR_INVALID_ARGUMENT and "3 experts" in msg
    rc, msg = call(pkg, E=3, plan=pkg._lib.Plan(-1, 1, 3, 1, None, None, None, None))
    assert rc == pkg._lib.ERR_INVALID_ARGUMENT and "out of range" in msg
    assert pkg._lib.load().moe_fp8_b200_matvec_w4(None, 0, 0, None, 0, None, 0, 0, None, 1, None, None, 0) == \
        pkg._lib.ERR_INVALID_ARGUMENT
    assert call(pkg, rows=0)[0] == pkg._lib.OK
    assert C.sizeof(pkg._lib.W4) == 3 * 8 + 4 * 4


def test_host_tensors(pkg):
    with pytest.raises(ValueError, match="CUDA"):
        pkg.matvec_w4(torch.zeros(1, 32, dtype=torch.bfloat16), torch.zeros(16, 16, dtype=torch.uint8),
                      torch.zeros(16, 1, dtype=torch.bfloat16))
