"""Sort, dispatch and combine: what is refused before anything reaches a GPU, and the sizes of a plan."""
import ctypes as C

import pytest
import torch


def plan_struct(pkg, T=4, K=2, E=8, align=1):
    return pkg._lib.Plan(T, K, E, align, None, None, None, None)


@pytest.mark.parametrize("T,K,E,align,rows", [
    (1, 1, 1, 1, 1), (1, 8, 256, 1, 8), (1, 8, 256, 128, 1024), (5, 3, 2, 1, 15), (5, 3, 2, 8, 32), (5, 3, 2, 7, 28),
    (12288, 8, 256, 128, 12288 * 8 + 256 * 128 - 256), (0, 8, 256, 128, 0), (16384, 8, 32, 1, 131072)])
def test_plan_rows(pkg, T, K, E, align, rows):
    want = T * K + min(E, T * K) * (align - 1)
    want = -(-want // align) * align
    assert pkg.plan_rows(T, K, E, align) == want
    if align in (1, 8, 128) and T != 12288:
        assert want == rows


@pytest.mark.parametrize("T,K,E,align", [(-1, 8, 256, 1), (1, 0, 256, 1), (1, 17, 256, 1), (1, 8, 0, 1), (1, 8, 1025, 1),
                                         (1, 8, 256, 0), (1, 8, 256, 1025), (2**28, 8, 256, 1), (2**31 - 1, 1, 256, 1)])
def test_plan_sizes_out_of_range(pkg, T, K, E, align):
    with pytest.raises(ValueError):
        pkg.plan_rows(T, K, E, align)
    lib = pkg._lib.load()
    err = C.create_string_buffer(256)
    p = plan_struct(pkg, T, K, E, align)
    assert lib.moe_fp8_b200_sort_tokens(None, 32, 0, C.byref(p), None, err, 256) == pkg._lib.ERR_INVALID_ARGUMENT
    assert b"out of range" in err.value


def test_null_plan_and_no_buffer_for_the_text(pkg):
    lib = pkg._lib.load()
    for rc in (lib.moe_fp8_b200_sort_tokens(None, 32, 0, None, None, None, 0),
               lib.moe_fp8_b200_dispatch_rows(None, 0, None, 0, 0, 1, None, 0, None, None, 0),
               lib.moe_fp8_b200_sort_and_dispatch(None, 32, 0, None, 0, None, 0, 0, 1, None, 0, None, None, 0),
               lib.moe_fp8_b200_combine_rows(None, 0, None, None, 0, 0, 1, None, None, None, 0),
               lib.moe_fp8_b200_combine_rows_backward(None, 0, None, 0, None, None, 0, None, 0, 1, None, 0, None, None, 0)):
        assert rc == pkg._lib.ERR_INVALID_ARGUMENT


def test_python_refuses_host_tensors_and_wrong_types(pkg):
    ids = torch.zeros(4, 2, dtype=torch.int32)
    x = torch.zeros(4, 16)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.sort_tokens(ids, 8)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.sort_and_dispatch(x, ids, 8)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.ExpertPlan(ids, ids.view(-1), torch.zeros(9, dtype=torch.int32), torch.zeros(8, dtype=torch.int32))
    for call in (lambda: pkg.dispatch(x, None), lambda: pkg.combine(x, x, None), lambda: pkg.dispatch_backward(x, None),
                 lambda: pkg.combine_backward(x, x, x, None), lambda: pkg.sort_tokens([[1]], 8)):
        with pytest.raises(TypeError):
            call()


def test_binding_matches_the_header(pkg):
    import re
    from pathlib import Path
    txt = (Path(__file__).resolve().parent.parent / "include" / "moe_fp8_b200.h").read_text()
    L = pkg._lib
    for name in ("BF16", "FP16", "FP32"):
        assert int(re.search(rf"MOE_FP8_B200_{name} = (\d+)", txt).group(1)) == getattr(L, name)
    for name in ("PLAN_MAX_TOP_K", "PLAN_MAX_EXPERTS"):
        assert int(re.search(rf"MOE_FP8_B200_{name} (\d+)", txt).group(1)) == getattr(L, name)
    assert C.sizeof(L.Plan) == 4 * 4 + 4 * 8


@pytest.mark.parametrize("a,b", [(a, b) for a in range(4) for b in range(4) if a != b])
def test_plan_arrays_that_share_memory(pkg, a, b):
    """Refused before a pointer is looked at: the addresses belong to nothing."""
    T, K, E, align = 4, 2, 8, 1
    size = [4 * T * K, 4 * pkg.plan_rows(T, K, E, align), 4 * (E + 1), 4 * E]
    at = [4096, 8192, 12288, 16384]
    at[b] = at[a] + size[a] - 4   # the last element of a is the first of b
    lib, err = pkg._lib.load(), C.create_string_buffer(256)
    p = pkg._lib.Plan(T, K, E, align, *at)
    assert lib.moe_fp8_b200_sort_tokens(1 << 20, 32, 0, C.byref(p), None, err, 256) == pkg._lib.ERR_INVALID_ARGUMENT
    assert b"share memory" in err.value


@pytest.mark.parametrize("at", range(4))
@pytest.mark.parametrize("wrap", [1 << 32, -(1 << 32), 1 << 64])
def test_plan_sizes_beyond_32_bits(pkg, at, wrap):
    sizes = [5, 8, 16, 4]
    sizes[at] += wrap   # cut to 32 bits, a size that is allowed
    with pytest.raises(ValueError, match="no plan"):
        pkg.plan_rows(*sizes)


@pytest.mark.parametrize("at", range(4))
def test_plan_sizes_that_are_no_whole_numbers(pkg, at):
    sizes = [5, 8, 16, 4]
    rows = pkg.plan_rows(*sizes)
    sizes[at] += 0.5
    with pytest.raises(ValueError, match=f"no plan.*{sizes[at]}"):
        pkg.plan_rows(*sizes)
    sizes[at] -= 0.5   # the whole number, as a float
    assert pkg.plan_rows(*sizes) == rows
