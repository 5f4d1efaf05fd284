"""Products with 4-bit weights (B200) against 64 bits, and the operators around the experts as a decode step runs them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def make_weights(lead, N, K, group, dtype, zeros, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(*lead, N, K // group, generator=g, device="cuda") * 0.02 + 1e-3).to(dtype)
    z = torch.randint(0, 16, (*lead, N, K // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return codes, scales, z


def decoded(codes, scales, zeros):
    q = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).double()
    group = q.shape[-1] // scales.shape[-1]
    q = q.unflatten(-1, (-1, group))
    return ((q - (8 if zeros is None else zeros.double()[..., None])) * scales.double()[..., None]).flatten(-2)


def expect(x, w, gated):
    """(result, bound) in 64 bits, before the rounding to x's type.

    A product code * x is exact.  The sum: two matrix instructions of 16 products each per 32 columns, each addition off by
    at most a step of fp32 of the terms' magnitude so far; then one product with the scale and one fused addition per 32
    columns, of which a warp adds up at most 16, and at most 16 warps' sums.  By integers the sum is exact but x is not: its
    31-bit numbers are off by up to half of 2^-30 of the power of two above the row's largest value."""
    y, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    err = (34 * 2.0 ** -23 + (2 * 16 + 16) * 2.0 ** -24) * mag
    err = err + 2.0 ** -31 * 2 * x.double().abs().amax(1, keepdim=True) * w.abs().sum(1)[None, :]
    if not gated:
        return y, err
    n = w.shape[0] // 2
    lin, gate, el, eg = y[:, :n], y[:, n:], err[:, :n], err[:, n:]
    silu = gate * torch.sigmoid(gate)
    # |silu'| <= 1.1; the exponential's argument is rounded to fp32 and it has a few units of error, then three operations
    bound = 1.1 * eg * (lin.abs() + el) + silu.abs() * el + (silu * lin).abs() * (gate.abs() + 8) * 2.0 ** -22
    return silu * lin, bound


def close(got, want, bound, dtype):
    u = torch.finfo(dtype).eps / 2
    lost = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133
    return bool(((got.double() - want).abs() <= u * want.abs() + (1 + u) * bound + lost).all())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,group", [
    (1, 16, 32, 32), (1, 7168, 2048, 128), (3, 48, 64, 32), (8, 4096, 7168, 128), (9, 160, 1024, 64), (17, 2048, 96, 32),
    (64, 1040, 2304, 128), (5, 32, 8192, 32), (2, 272, 8192, 64), (40, 64, 4096, 128), (1, 64, 6080, 32), (7, 336, 4160, 64)])
def test_one_matrix(pkg, M, N, K, group, dtype, zeros, gated):
    codes, scales, z = make_weights((), N, K, group, dtype, zeros, M + N + K)
    x = torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    if gated and zeros and (K // group) % 2:
        with pytest.raises(pkg.MoeError, match="even number of groups"):
            pkg.matvec_w4(x, codes, scales, zeros=z, gated=True)
        return
    got = pkg.matvec_w4(x, codes, scales, zeros=z, gated=gated)
    want, bound = expect(x, decoded(codes, scales, z), gated)
    assert got.shape == want.shape and close(got, want, bound, dtype)


def test_every_code_and_zero_point(pkg):
    """One row of weights per (code, zero point), one column of x at a time: exact results."""
    K, group = 128, 32
    for dtype in DTYPES:
        codes = torch.zeros(256, K, dtype=torch.uint8)
        zeros = torch.zeros(256, K // group, dtype=torch.uint8)
        for r in range(256):
            codes[r] = r % 16
            zeros[r] = r // 16
        packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).cuda()
        scales = (2.0 ** torch.arange(-4, 0)).expand(256, 4).to(dtype).cuda().contiguous()
        x = torch.zeros(K, K, dtype=dtype, device="cuda")
        x.diagonal().fill_(3.0)
        got = pkg.matvec_w4(x, packed, scales, zeros=zeros.cuda())
        want = 3.0 * decoded(packed, scales, zeros.cuda()).t()
        assert torch.equal(got.double(), want)
        got = pkg.matvec_w4(x, packed, scales)
        assert torch.equal(got.double(), 3.0 * decoded(packed, scales, None).t())


def routed(T, K, experts, seed, skew=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    score = torch.randn(T, experts, generator=g, device="cuda") - skew * torch.arange(experts, device="cuda")
    return score.topk(K, dim=1).indices


@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T,top_k,experts,first,E,align,N,K,group,zeros,dtype,skew", [
    (1, 8, 256, 0, 256, 1, 64, 512, 128, False, torch.bfloat16, 0.0),
    (1, 1, 4, 2, 2, 16, 32, 64, 32, True, torch.float16, 0.0),
    (16, 8, 64, 32, 32, 128, 96, 1024, 64, True, torch.bfloat16, 0.0),
    (64, 8, 16, 0, 16, 1, 416, 2048, 128, False, torch.float16, 0.0),
    (33, 4, 8, 0, 8, 8, 4096, 4096, 32, True, torch.bfloat16, 1.0),
    (200, 2, 700, 0, 700, 1, 16, 256, 128, False, torch.bfloat16, 0.01),
    (24, 3, 5, 1, 3, 1, 2048, 7168, 128, False, torch.bfloat16, 0.0)])
def test_experts_rows(pkg, T, top_k, experts, first, E, align, N, K, group, zeros, dtype, skew, by_token, gated):
    plan = pkg.sort_tokens(routed(T, top_k, experts, T, skew), E, first_expert=first, align=align)
    codes, scales, z = make_weights((E,), N, K, group, dtype, zeros, T + N)
    rows = T if by_token else plan.capacity
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(dtype)
    out = torch.full((plan.capacity, N // 2 if gated else N), 7.0, dtype=dtype, device="cuda")
    assert pkg.matvec_w4(x, codes, scales, zeros=z, plan=plan, by_token=by_token, gated=gated, out=out) is out
    live = plan.row_pair >= 0
    assert bool((out[~live] == 7).all()), "rows without a pair are the caller's"
    offset, count = plan.expert_offset.tolist(), plan.expert_count.tolist()
    assert int(live.sum()) == sum(count)
    for e in range(E):
        if count[e]:
            r = slice(offset[e], offset[e] + count[e])
            xe = x[plan.row_pair[r].long() // top_k] if by_token else x[r]
            want, bound = expect(xe, decoded(codes[e], scales[e], None if z is None else z[e]), gated)
            assert close(out[r], want, bound, dtype), e


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(pkg, dtype):
    M, N, K, group = 11, 96, 1024, 64
    codes, scales, z = make_weights((), N, K, group, dtype, True, 5)
    base = torch.randn(M, K + 40, device="cuda").to(dtype)
    w = decoded(codes, scales, z)
    for x in (base[:, 8:8 + K], base[:, 3:3 + K], base[:1, :K].expand(M, K), base.view(-1)[1:1 + M * K].view(M, K)):
        out = torch.full((M, N + 5), 7.0, dtype=dtype, device="cuda")
        pkg.matvec_w4(x, codes, scales, zeros=z, out=out[:, 2:2 + N])
        want, bound = expect(x, w, False)
        assert close(out[:, 2:2 + N], want, bound, dtype)
        assert bool((out[:, :2] == 7).all()) and bool((out[:, 2 + N:] == 7).all())


def test_infinities_and_nan_stay_in_their_row(pkg):
    M, N, K = 10, 64, 256
    codes, scales, _ = make_weights((), N, K, 64, torch.bfloat16, False, 9)
    x = torch.randn(M, K, device="cuda").to(torch.bfloat16)
    x[2, 7], x[9, 100] = float("inf"), float("nan")
    got = pkg.matvec_w4(x, codes, scales)
    rows = torch.isfinite(got).all(1).tolist()
    assert rows == [r not in (2, 9) for r in range(M)]
    w = decoded(codes, scales, None)
    hit = w[:, 7]
    assert torch.equal(got[2][hit != 0].double(), torch.sign(hit[hit != 0]) * float("inf")) and got[2][hit == 0].isnan().all()
    assert got[9].isnan().all()


@pytest.mark.parametrize("M", [1, 2, 3, 4, 6])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_of_any_magnitude(pkg, M, zeros):
    """Outliers, rows of zeros, subnormal rows, rows near the end of the range, single values."""
    N, K = 64, 2048
    for dtype, scales_of in ((torch.bfloat16, (1.0, 2.0 ** -130, 2.0 ** -100, 2.0 ** 112, 0.0)),
                             (torch.float16, (1.0, 2.0 ** -22, 2.0 ** -14, 2.0 ** 6, 0.0))):
        codes, scales, z = make_weights((), N, K, 128, dtype, zeros, M)
        w = decoded(codes, scales, z)
        for scale in scales_of:
            x = torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(M), device="cuda").double()
            x[0, 5] *= 2.0 ** 10          # an outlier
            x[-1, :1024] *= 2.0 ** -9     # a warp's columns are not another one's
            x = (x * scale).to(dtype)
            want, bound = expect(x, w, False)
            assert close(pkg.matvec_w4(x, codes, scales, zeros=z), want, bound, dtype), (dtype, scale)
        x = torch.zeros(M, K, dtype=dtype, device="cuda")
        x[:, 77] = torch.finfo(dtype).max
        x[:, 78] = torch.finfo(dtype).smallest_normal
        small = (scales.double() * 2.0 ** -9).to(dtype)   # rounded in fp16, where it is subnormal
        got = pkg.matvec_w4(x, codes, small, zeros=z)
        want, bound = expect(x, decoded(codes, small, z), False)
        assert close(got, want, bound, dtype)


def test_a_gate_far_from_zero(pkg):
    """silu at the ends: exp overflows or vanishes, the product does not."""
    K = 64
    codes = torch.full((32, K // 2), 0x99, dtype=torch.uint8, device="cuda")   # every weight 1
    scales = torch.ones(32, 1, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(4, K, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = torch.tensor([-300.0, 300.0, -88.0, 0.0])
    got = pkg.matvec_w4(x, codes, scales, gated=True)
    assert bool((got[0] == 0).all()) and bool((got[1] == 90112).all()) and bool((got[2].abs() < 1e-30).all())
    assert bool((got[3] == 0).all())


def test_a_decode_step(pkg):
    """Routing, sort, both products, combine, as a decode step of a layer with 4-bit experts runs them: eager on another
    stream, and captured and replayed with other contents."""
    T, hidden, inter, E, first, group = 6, 7168, 2048, 32, 64, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    w1 = make_weights((E,), 2 * inter, hidden, group, torch.bfloat16, False, 1)
    w2 = make_weights((E,), hidden, inter, group, torch.bfloat16, False, 2)
    logits = torch.randn(T, 256, generator=g, device="cuda")
    bias = torch.zeros(256, dtype=torch.bfloat16, device="cuda")
    bias[first:first + E] = 0.5    # enough pairs here
    x = (torch.randn(T, hidden, generator=g, device="cuda") * 0.05).to(torch.bfloat16)
    idx = torch.empty(T, 8, dtype=torch.int32, device="cuda")
    weight = torch.empty(T, 8, device="cuda")
    counts = torch.empty(256, dtype=torch.int32, device="cuda")
    plan = pkg.ExpertPlan.empty(T, 8, E)
    act = torch.zeros(plan.capacity, inter, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(plan.capacity, hidden, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(T, hidden, dtype=torch.bfloat16, device="cuda")
    lib = pkg._lib.load()

    def step():
        rc = lib.moe_fp8_b200_route_noalloc(logits.data_ptr(), bias.data_ptr(), T, 0, 256, 2.5, 0, idx.data_ptr(),
                                            weight.data_ptr(), counts.data_ptr(), torch.cuda.current_stream().cuda_stream,
                                            None, 0)
        assert rc == 0
        pkg.sort_tokens(idx, E, first_expert=first, plan=plan)
        pkg.matvec_w4(x, w1[0], w1[1], plan=plan, by_token=True, gated=True, out=act)
        pkg.matvec_w4(act, w2[0], w2[1], plan=plan, out=y)
        pkg.combine(y, weight, plan, out=out)

    def check():
        torch.cuda.synchronize()
        e = idx.long() - first
        live = (e >= 0) & (e < E)
        assert int(live.sum()) >= T
        assert torch.equal(live, plan.pair_row >= 0)
        for t in range(T):
            want, mag = torch.zeros(hidden, dtype=torch.float64, device="cuda"), 0.0
            for k in range(8):
                if not live[t, k]:
                    continue
                r, ek = int(plan.pair_row[t, k]), int(e[t, k])
                a, bound = expect(x[t:t + 1], decoded(w1[0][ek], w1[1][ek], None), True)
                assert close(act[r:r + 1], a, bound, torch.bfloat16)
                # from the rounded activations on: each step by itself
                v, bound = expect(act[r:r + 1], decoded(w2[0][ek], w2[1][ek], None), False)
                assert close(y[r:r + 1], v, bound, torch.bfloat16)
                want += weight[t, k].double() * y[r].double()
                mag = mag + (weight[t, k].double() * y[r].double()).abs()
            # eight fused multiply-adds in fp32, then bf16: it keeps 8 significant bits, the last of them worth 2^-7 of the
            # leading one, so that a rounding is off by at most 2^-8 of the value (0.0397 as bf16 is a multiple of 2^-12:
            # off by up to 2^-13 = 1.22e-4 > 2^-9 * 0.0397)
            assert bool(((out[t].double() - want).abs() <= 2.0 ** -8 * want.abs() + 9 * 2.0 ** -24 * mag + 2.0 ** -133).all())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (11, 12):
        g.manual_seed(seed)
        logits.copy_(torch.randn(T, 256, generator=g, device="cuda"))
        x.copy_(torch.randn(T, hidden, generator=g, device="cuda") * 0.05)
        graph.replay()
        check()


def test_a_plan_of_nonsense_reads_and_writes_nothing_outside(pkg):
    """Offsets and counts that no sort gives: rows outside the matrices, experts on top of one another."""
    T, K, E, N, C = 40, 2, 8, 32, 128
    codes, scales, _ = make_weights((E,), N, C, 64, torch.bfloat16, False, 3)
    for by_token in (False, True):
        plan = pkg.sort_tokens(routed(T, K, E, 5), E)
        plan.expert_offset[2], plan.expert_count[2] = -5, 3
        plan.expert_offset[3], plan.expert_count[3] = plan.capacity + 7, 2
        plan.expert_count[4] = 2**31 - 1
        plan.row_pair[:4] = torch.tensor([-1, 2**31 - 1, -2**31, T * K], dtype=torch.int32, device="cuda")
        x = torch.randn(T if by_token else plan.capacity, C, device="cuda").to(torch.bfloat16)
        guard = torch.full((plan.capacity + 64, N), 3.0, dtype=torch.bfloat16, device="cuda")
        pkg.matvec_w4(x, codes, scales, plan=plan, by_token=by_token, out=guard[32:32 + plan.capacity])
        plan.expert_offset.fill_(0)
        plan.expert_count.fill_(2**31 - 1)
        pkg.matvec_w4(x, codes, scales, plan=plan, by_token=by_token, out=guard[32:32 + plan.capacity])
        torch.cuda.synchronize()
        assert bool((guard[:32] == 3).all()) and bool((guard[32 + plan.capacity:] == 3).all())


def test_refusals(pkg):
    M, N, K, group = 4, 32, 256, 64
    codes, scales, z = make_weights((), N, K, group, torch.bfloat16, True, 1)
    x = torch.randn(M, K, device="cuda").to(torch.bfloat16)
    out = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    plan = pkg.sort_tokens(routed(M, 1, 2, 1), 2)
    wide = torch.zeros(16, 16 * 17, dtype=torch.uint8, device="cuda")
    for call, error in (
            (lambda: pkg.matvec_w4(x.float(), codes, scales), TypeError),
            (lambda: pkg.matvec_w4(x.half(), codes, scales), TypeError),
            (lambda: pkg.matvec_w4(x, codes.view(torch.int8), scales), TypeError),
            (lambda: pkg.matvec_w4(x, codes[:, 1:], scales), ValueError),
            (lambda: pkg.matvec_w4(x[:, :-2], codes, scales), ValueError),
            (lambda: pkg.matvec_w4(x, codes[None], scales[None]), ValueError),
            (lambda: pkg.matvec_w4(x, codes, scales, plan=plan), ValueError),
            (lambda: pkg.matvec_w4(x, codes, scales, by_token=True), ValueError),
            (lambda: pkg.matvec_w4(x, codes, scales, zeros=z[:-1]), ValueError),
            (lambda: pkg.matvec_w4(x, codes, scales, zeros=z.to(torch.int8)), TypeError),
            (lambda: pkg.matvec_w4(x, codes, scales, out=out[:-1]), ValueError),
            (lambda: pkg.matvec_w4(x, codes, scales, gated=True, out=out), ValueError),
            (lambda: pkg.matvec_w4(x.cpu(), codes, scales), ValueError),
            (lambda: pkg.matvec_w4(x.clone().requires_grad_(), codes, scales), ValueError),
            (lambda: pkg.matvec_w4(x, codes[:24], scales[:24]), pkg.MoeError),             # n
            (lambda: pkg.matvec_w4(x, codes, scales[:, :1].contiguous()), pkg.MoeError),   # group 256
            (lambda: pkg.matvec_w4(x, codes, scales, out=out[:1].expand(M, N)), pkg.MoeError),
            (lambda: pkg.matvec_w4(torch.zeros(1, 8224, dtype=torch.bfloat16, device="cuda"),
                                   torch.zeros(16, 4112, dtype=torch.uint8, device="cuda"),
                                   torch.zeros(16, 257, dtype=torch.bfloat16, device="cuda")), pkg.MoeError),
            (lambda: pkg.matvec_w4(x[:, :32].contiguous(), wide.view(-1)[8:8 + 256].view(16, 16),
                                   torch.zeros(16, 1, dtype=torch.bfloat16, device="cuda")), pkg.MoeError)):
        with pytest.raises(error):
            call()
    assert pkg.matvec_w4(x[:0], codes, scales).shape == (0, N)


def test_out_over_the_plan(pkg):
    T, K, E, N, cols = 3, 2, 4, 16, 64
    ids = torch.randint(0, E, (T, K), generator=torch.Generator().manual_seed(2)).int().cuda()
    codes = torch.zeros(E, N, cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.ones(E, N, 2, dtype=torch.bfloat16, device="cuda")
    x = torch.ones(T, cols, dtype=torch.bfloat16, device="cuda")
    for field, size in (("row_pair", T * K), ("expert_offset", E + 1), ("expert_count", E)):
        memory = torch.zeros(T * K * N // 2, dtype=torch.int32, device="cuda")
        arrays = dict(pair_row=(T, K), row_pair=(T * K,), expert_offset=(E + 1,), expert_count=(E,))
        arrays = {k: torch.empty(v, dtype=torch.int32, device="cuda") for k, v in arrays.items()}
        arrays[field] = memory[:size]
        plan = pkg.sort_tokens(ids, E, plan=pkg.ExpertPlan(**arrays))
        with pytest.raises(pkg.MoeError, match=f"out and {field} share memory"):
            pkg.matvec_w4(x, codes, scales, plan=plan, by_token=True, out=memory.view(torch.bfloat16).view(T * K, N))


def test_sizes_beyond_32_bits(pkg):
    x = torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda")
    codes = torch.zeros(16, 32, dtype=torch.uint8, device="cuda")
    scales = torch.ones(16, 2, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="too many"):
        pkg.matvec_w4(x.expand((1 << 32) + 1, 64), codes, scales)
    with pytest.raises(ValueError, match="too many"):
        pkg.matvec_w4(x, torch.empty((1 << 32) + 16, 32, dtype=torch.uint8, device="meta"),
                      torch.empty((1 << 32) + 16, 2, dtype=torch.bfloat16, device="meta"))


def test_products_of_several_threads(pkg):
    """Calls that need different amounts of shared memory of one kernel: what one sets for its launch holds for the other's."""
    import ctypes as C
    from test_gpu_expert_rows import calls_of_threads
    N = 64

    def make(K):
        codes, scales, _ = make_weights((), N, K, 128, torch.bfloat16, False, K)
        x, out = torch.ones(1, K, dtype=torch.bfloat16, device="cuda"), torch.empty(1, N, dtype=torch.bfloat16, device="cuda")
        w = pkg._lib.W4(codes.data_ptr(), scales.data_ptr(), None, 1, N, K, 128)

        def check():
            want, bound = expect(x, decoded(codes, scales, None), False)
            assert close(out, want, bound, torch.bfloat16)

        return (pkg._lib.load().moe_fp8_b200_matvec_w4, (x.data_ptr(), K, 0, C.byref(w), 0, out.data_ptr(), N, 0, None, 1), check)

    assert not calls_of_threads(pkg, make, (2048, 256))


@pytest.mark.parametrize("by_token", [False, True])
def test_out_over_any_array_of_the_plan(pkg, by_token):
    T, K, E, N, cols = 3, 2, 4, 16, 64
    ids = torch.randint(0, E, (T, K), generator=torch.Generator().manual_seed(2)).int().cuda()
    codes = torch.zeros(E, N, cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.ones(E, N, 2, dtype=torch.bfloat16, device="cuda")
    x = torch.ones(T if by_token else T * K, cols, dtype=torch.bfloat16, device="cuda")
    shapes = dict(pair_row=(T, K), row_pair=(T * K,), expert_offset=(E + 1,), expert_count=(E,))
    for field, shape in shapes.items():
        memory = torch.zeros(T * K * N // 2, dtype=torch.int32, device="cuda")
        arrays = {k: torch.empty(v, dtype=torch.int32, device="cuda") for k, v in shapes.items()}
        arrays[field] = memory[:torch.Size(shape).numel()].view(shape)
        plan = pkg.sort_tokens(ids, E, plan=pkg.ExpertPlan(**arrays))
        kept = arrays[field].clone()
        with pytest.raises(pkg.MoeError, match=f"out and {field} share memory"):
            pkg.matvec_w4(x, codes, scales, plan=plan, by_token=by_token, out=memory.view(torch.bfloat16).view(T * K, N))
        assert torch.equal(arrays[field], kept)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 6])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_scales_of_any_magnitude(pkg, M, zeros, group):
    """bf16 scales near either end of fp32's range, with x that brings the results back into it.  A product with a scale is held
    to half of fp32's smallest step, 2^-150; in front of it stands at most 2^14 times the power of two above the largest x, and at
    most K / 32 products of each of four bytes, each byte worth 2^-8 of the next one, meet in a result."""
    N, K = 64, 2048
    for shift_x, shift_s in ((-60, 105), (-100, 125), (-125, 120), (0, 100), (0, -100), (60, -115), (100, -125), (118, -126)):
        codes, scales, z = make_weights((), N, K, group, torch.bfloat16, zeros, M)
        scales = (scales.double() * 2.0 ** shift_s).bfloat16()
        x = torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(M), device="cuda").double()
        x = (x * 2.0 ** shift_x).bfloat16()
        want, bound = expect(x, decoded(codes, scales, z), False)
        assert bool(torch.isfinite(want.bfloat16()).all())
        bound = bound + 1.01 * K / 32 * 2.0 ** -150 * 2.0 ** 14 * 2 * x.double().abs().amax(1, keepdim=True)
        got = pkg.matvec_w4(x, codes, scales, zeros=z)
        assert close(got, want, bound, torch.bfloat16), (shift_x, shift_s)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 6])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_an_outlier_that_meets_no_weight(pkg, M, zeros, dtype):
    """A large x whose weights are zero takes nothing away from the small ones: sums of exact products in fp32."""
    N, K, group, at = 64, 2048, 128, 77
    codes, scales, z = make_weights((), N, K, group, dtype, zeros, M)
    codes[:32, at // 2] = codes[:32, at // 2] & 15 | ((z[:32, at // group] if zeros else 8) << 4)   # an odd column: the upper half
    large, small = (2.0 ** 30, 2.0 ** -6) if dtype == torch.bfloat16 else (2.0 ** 15, 2.0 ** -17)
    x = (torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(M), device="cuda") * small).to(dtype)
    x[0, at] = large
    x[M - 1, at] = -large
    w = decoded(codes, scales, z)
    assert not w[:32, at].any() and bool(w[32:, at].any())
    got = pkg.matvec_w4(x, codes, scales, zeros=z)
    want, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    # as in expect, without its term for an inexact x
    assert close(got, want, (34 * 2.0 ** -23 + (2 * 16 + 16) * 2.0 ** -24) * mag, dtype)


@pytest.mark.parametrize("M", [1, 2, 3, 4])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_small_value_under_a_large_one_is_exact(pkg, M, zeros, dtype):
    """One column of weight one, the others zero: the result is that column of x, however far it lies below the largest value."""
    N, K = 16, 64
    mid = 5 if zeros else 8
    codes = torch.full((N, K // 2), mid * 17, dtype=torch.uint8, device="cuda")
    codes[:, 20] = mid + 1 | mid << 4   # column 40
    z = torch.full((N, 1), mid, dtype=torch.uint8, device="cuda") if zeros else None
    scales = torch.ones(N, 1, dtype=dtype, device="cuda")
    info, top = torch.finfo(dtype), 2.0 ** (100 if dtype == torch.bfloat16 else 15)
    for k in range(1, 42 if dtype == torch.bfloat16 else 39):
        small = (1 + info.eps) * top * 2.0 ** -k   # all of its bits, fewer where fp16 is subnormal
        x = torch.zeros(M, K, dtype=dtype, device="cuda")
        x[:, 7], x[M - 1, 40] = -top, small
        want = torch.zeros(M, N, dtype=dtype, device="cuda")
        want[M - 1] = x[M - 1, 40]
        assert bool(want[M - 1].any())
        assert torch.equal(pkg.matvec_w4(x, codes, scales, zeros=z), want), k


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,group", [(3, 48, 3104, 32), (2, 32, 3104, 32), (9, 32, 4096, 32), (4, 64, 2080, 32), (5, 48, 2112, 64),
                                         (1, 80, 3968, 128)])
def test_eight_warps_per_tile(pkg, M, N, K, group, dtype, zeros, gated):
    """2048 < K <= 4096, with rows that are no multiple of 256 columns and odd numbers of 32-column blocks."""
    codes, scales, z = make_weights((), N, K, group, dtype, zeros, M + N + K)
    x = torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    if gated and zeros and (K // group) % 2:
        with pytest.raises(pkg.MoeError, match="even number of groups"):
            pkg.matvec_w4(x, codes, scales, zeros=z, gated=True)
        return
    got = pkg.matvec_w4(x, codes, scales, zeros=z, gated=gated)
    want, bound = expect(x, decoded(codes, scales, z), gated)
    assert got.shape == want.shape and close(got, want, bound, dtype)
