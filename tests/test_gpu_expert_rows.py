"""Tokens sorted by expert and back (B200): the plan against a loop over the pairs, the copy bit for bit, the weighted sum
and the gradients against 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def plan_by_loop(ids, E, first, align, capacity):
    T, K = ids.shape
    mine = [[] for _ in range(E)]
    for pair, e in enumerate(ids.reshape(-1).tolist()):
        if first <= e < first + E:
            mine[e - first].append(pair)
    pair_row, row_pair, offset = np.full(T * K, -1, np.int32), np.full(capacity, -1, np.int32), [0]
    for pairs in mine:
        for i, pair in enumerate(pairs):
            pair_row[pair], row_pair[offset[-1] + i] = offset[-1] + i, pair
        offset.append(offset[-1] + -(-len(pairs) // align) * align)
    return pair_row.reshape(T, K), row_pair, np.array(offset, np.int32), np.array([len(m) for m in mine], np.int32)


def some_ids(T, K, experts, seed, dtype=torch.int32, kind="distinct"):
    g = torch.Generator().manual_seed(seed)
    if kind == "distinct":
        score = torch.randn(T, experts, generator=g)
        if experts < K:
            return torch.randint(0, experts, (T, K), generator=g).to(dtype).cuda()
        return score.topk(K, dim=1).indices.to(dtype).cuda()
    if kind == "one":        # every pair the same expert
        return torch.full((T, K), experts // 2, dtype=dtype).cuda()
    if kind == "none":       # no pair in range
        return torch.full((T, K), -1, dtype=dtype).cuda()
    ids = torch.randint(-3, experts + 3, (T, K), generator=g)   # "any": repeats, out of range on both sides
    return ids.to(dtype).cuda()


def check_plan(pkg, plan, ids, E, first, align):
    want = plan_by_loop(ids.cpu(), E, first, align, pkg.plan_rows(*ids.shape, E, align))
    for name, w in zip(("pair_row", "row_pair", "expert_offset", "expert_count"), want):
        assert np.array_equal(getattr(plan, name).cpu().numpy(), w), name
    return want


def fresh_plan(pkg, T, K, E, align):
    plan = pkg.ExpertPlan.empty(T, K, E, align)
    for t in (plan.pair_row, plan.row_pair, plan.expert_offset, plan.expert_count):
        t.fill_(1 << 30)   # every entry must be written
    return plan


@pytest.mark.parametrize("kind", ["distinct", "any", "one", "none"])
@pytest.mark.parametrize("T,K,experts,first,E,align", [
    (1, 8, 256, 0, 256, 1), (1, 1, 1, 0, 1, 1), (7, 2, 8, 2, 3, 4), (57, 8, 256, 96, 32, 128), (128, 8, 256, 0, 256, 1),
    (129, 8, 256, 64, 128, 16), (300, 6, 64, 0, 64, 7), (515, 16, 1024, 0, 1024, 1), (1000, 8, 256, 0, 256, 128),
    (4099, 5, 160, 32, 100, 1), (12288, 8, 256, 0, 256, 128), (20000, 8, 256, 224, 32, 8)])
def test_plan(pkg, kind, T, K, experts, first, E, align):
    for dtype in (torch.int32, torch.int64):
        ids = some_ids(T, K, experts, T + K, dtype, kind)
        plan = pkg.sort_tokens(ids, E, first_expert=first, align=align, plan=fresh_plan(pkg, T, K, E, align))
        check_plan(pkg, plan, ids, E, first, align)


def test_ids_at_the_ends_of_64_bits(pkg):
    lim = torch.iinfo(torch.int64)
    ids = torch.tensor([[lim.min, lim.max], [-1, 5], [5 + 2**32, 6]], device="cuda")
    plan = pkg.sort_tokens(ids, 4, first_expert=4, plan=fresh_plan(pkg, 3, 2, 4, 1))
    check_plan(pkg, plan, ids, 4, 4, 1)


def test_no_tokens(pkg):
    ids = torch.zeros(0, 8, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 64, device="cuda")
    rows, plan = pkg.sort_and_dispatch(x, ids, 16, align=8)
    assert rows.shape == (0, 64) and plan.expert_offset.tolist() == [0] * 17 and plan.expert_count.tolist() == [0] * 16
    w = torch.zeros(0, 8, device="cuda")
    assert pkg.combine(rows, w, plan).shape == (0, 64)
    assert pkg.dispatch_backward(rows, plan).shape == (0, 64)
    dy, dw = pkg.combine_backward(x, rows, w, plan)
    assert dy.shape == (0, 64) and dw.shape == (0, 8)


def wide(rows, cols, dtype, layout, seed):
    """A random matrix as a view: contiguous, columns of a wider one, off a 16-byte boundary, or one row for all."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    full = torch.randn(rows, cols + 24, generator=g, device="cuda").to(dtype)
    if layout == "plain":
        return full[:, :cols].contiguous()
    if layout == "columns":
        return full[:, 8:8 + cols]
    if layout == "odd":
        return full[:, 3:3 + cols]
    return full[:1, :cols].expand(rows, cols)


SIZES = [(1, 8, 256, 0, 256, 1, 7168), (3, 2, 4, 1, 2, 4, 1), (57, 8, 256, 96, 32, 1, 7168), (129, 8, 256, 0, 256, 16, 1001),
         (33, 16, 64, 0, 64, 8, 40), (500, 6, 64, 16, 32, 128, 264), (2049, 1, 8, 0, 8, 1, 16), (260, 12, 300, 0, 300, 3, 4100)]


@pytest.mark.parametrize("layout", ["plain", "columns", "odd", "broadcast"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,experts,first,E,align,H", SIZES)
def test_dispatch(pkg, T, K, experts, first, E, align, H, dtype, layout):
    ids = some_ids(T, K, experts, 5 * T + H, kind="distinct" if T % 2 else "any")
    x = wide(T, H, dtype, layout, 3)
    cap = pkg.plan_rows(T, K, E, align)
    rows = wide(cap, H, dtype, "plain" if layout == "broadcast" else layout, 4)
    before = rows.clone()
    got, plan = pkg.sort_and_dispatch(x, ids, E, first_expert=first, align=align, rows=rows)
    assert got is rows
    _, row_pair, offset, _ = check_plan(pkg, plan, ids, E, first, align)
    pair = torch.from_numpy(row_pair).cuda().long()
    want = torch.where((pair >= 0)[:, None], x[(pair.clamp(min=0) // K)], torch.zeros((), dtype=dtype, device="cuda"))
    end = int(offset[-1])
    assert torch.equal(rows[:end], want[:end])
    assert torch.equal(rows[end:], before[end:]), "rows behind the last expert are the caller's"
    # the two calls apart, and new matrices: zeros behind the last expert
    new = pkg.dispatch(x, pkg.sort_tokens(ids, E, first_expert=first, align=align))
    assert torch.equal(new[:end], want[:end]) and not new[end:].any()
    new, _ = pkg.sort_and_dispatch(x, ids, E, first_expert=first, align=align)
    assert torch.equal(new[:end], want[:end]) and not new[end:].any()


def rows_in_64(values, pair_row):
    at = pair_row.long()
    return torch.where((at >= 0)[..., None], values[at.clamp(min=0)].double(), 0.0)


def smallest(dtype):
    """Half of the smallest subnormal step: what a rounding loses below the normal range."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134


@pytest.mark.parametrize("layout", ["plain", "columns", "odd", "broadcast"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,experts,first,E,align,H", SIZES)
def test_combine_and_gradients(pkg, T, K, experts, first, E, align, H, dtype, layout):
    ids = some_ids(T, K, experts, 7 * T + H, kind="distinct" if T % 2 else "any")
    plan = pkg.sort_tokens(ids, E, first_expert=first, align=align)
    cap = plan.capacity
    y = wide(cap, H, dtype, layout, 5)
    if layout != "broadcast":
        y.masked_fill_((plan.row_pair < 0)[:, None], float("nan"))   # padding and unused rows are not read
    w = torch.rand(T, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    u, lost = half_step(dtype), smallest(dtype)
    # K fused multiply-adds in fp32, one rounding to the type
    terms = rows_in_64(y, plan.pair_row) * w.double()[..., None]
    want, mag = terms.sum(1), terms.abs().sum(1)
    out = wide(T, H, dtype, "plain" if layout == "broadcast" else layout, 7)
    assert pkg.combine(y, w, plan, out=out) is out
    bound = u * want.abs() + (1 + u) * K * 2.0 ** -24 * mag + lost
    assert bool(((out.double() - want).abs() <= bound).all())
    assert torch.equal(pkg.combine(y, w, plan), out)
    # dispatch's gradient: the same without weights
    terms = rows_in_64(y, plan.pair_row)
    want, mag = terms.sum(1), terms.abs().sum(1)
    got = pkg.dispatch_backward(y, plan)
    assert bool(((got.double() - want).abs() <= u * want.abs() + (1 + u) * K * 2.0 ** -24 * mag + lost).all())
    # combine's gradients: one product in fp32, rounded to the type; a sum of H products, at most H / 32 + 32 of them one after
    # the other in a lane, then five additions over the warp and eight over the warps of a row
    g = wide(T, H, dtype, layout, 8)
    dy = wide(cap, H, dtype, "plain" if layout == "broadcast" else layout, 9)
    before = dy.clone()
    dy2, dw = pkg.combine_backward(g, y, w, plan, grad_y=dy)
    assert dy2 is dy
    end = int(plan.expert_offset[-1])
    pair = plan.row_pair.long()
    live = pair >= 0
    want = torch.where(live[:, None], g[(pair.clamp(min=0) // K)].double() * w.view(-1)[pair.clamp(min=0)].double()[:, None], 0.0)
    assert bool(((dy.double() - want).abs()[:end] <= ((1 + 2.0 ** -24) * u + 2.0 ** -24) * want.abs()[:end] + lost).all())
    assert torch.equal(dy[end:].nan_to_num(), before[end:].nan_to_num())
    prod = rows_in_64(y, plan.pair_row) * g.double()[:, None, :]
    want, mag = prod.sum(-1), prod.abs().sum(-1)
    assert bool(((dw.double() - want).abs() <= (H / 32 + 32 + 13) * 2.0 ** -24 * mag + 2.0 ** -140).all())
    assert not dw[plan.pair_row < 0].any()
    # each alone, in new matrices
    dy3, none = pkg.combine_backward(g, y, w, plan, need_weights=False)
    assert none is None and torch.equal(dy3[:end], dy[:end]) and not dy3[end:].any()
    none, dw3 = pkg.combine_backward(g, y, w, plan, need_y=False)
    assert none is None and torch.equal(dw3, dw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_stay_in_their_token(pkg, dtype):
    T, K, E, H = 9, 4, 16, 48
    ids = some_ids(T, K, E, 1)
    plan = pkg.sort_tokens(ids, E)
    w = torch.rand(T, K, device="cuda")
    w[3, 1] = 0.0
    y = torch.randn(plan.capacity, H, device="cuda").to(dtype)
    y[plan.pair_row[3, 1], 5] = float("inf")      # 0 * inf = NaN, as in the formula
    y[plan.pair_row[4, 0], 6] = float("-inf")
    y[plan.pair_row[5, 2], 7] = float("nan")
    out = pkg.combine(y, w, plan)
    bad = ~torch.isfinite(out)
    assert bad.nonzero().tolist() == [[3, 5], [4, 6], [5, 7]]
    assert out[4, 6] == float("-inf") and out[3, 5].isnan() and out[5, 7].isnan()
    top = torch.finfo(dtype).max
    y.fill_(top)
    w.fill_(1.0)
    out = pkg.combine(y, w, plan)
    if dtype != torch.float32:   # a sum beyond the type's range is infinite, as the rounding says
        assert bool(torch.isinf(out).all())


def test_a_plan_with_rows_out_of_range_reads_and_writes_nothing_there(pkg):
    T, K, E, H = 40, 4, 8, 64
    ids = some_ids(T, K, E, 2)
    plan = pkg.sort_tokens(ids, E, align=8)
    plan.pair_row[0, 0], plan.pair_row[1, 1], plan.pair_row[2, 2] = plan.capacity, -7, 2**31 - 1
    good = plan.pair_row.clone()
    good[0, 0] = good[1, 1] = good[2, 2] = -1
    x = torch.randn(T, H, device="cuda")
    guard = torch.full((plan.capacity + 64, H), 3.0, device="cuda")
    pkg.dispatch(x, plan, rows=guard[32:32 + plan.capacity])
    assert bool((guard[:32] == 3).all()) and bool((guard[32 + plan.capacity:] == 3).all())
    y, w = torch.randn(plan.capacity, H, device="cuda"), torch.rand(T, K, device="cuda")
    want = (rows_in_64(y, good) * w.double()[..., None]).sum(1)
    assert torch.allclose(pkg.combine(y, w, plan).double(), want, rtol=1e-5, atol=1e-6)
    plan.expert_offset[-1] = 2**31 - 1
    plan.expert_offset[3] = -2**31
    dy, _ = pkg.combine_backward(x, y, w, plan, grad_y=guard[32:32 + plan.capacity])
    torch.cuda.synchronize()
    assert bool((guard[:32] == 3).all()) and bool((guard[32 + plan.capacity:] == 3).all())


@pytest.mark.parametrize("align", [1, 8])
def test_autograd_against_the_formula_and_differences(pkg, align):
    T, K, experts, first, E, H = 23, 3, 16, 4, 8, 20
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = some_ids(T, K, experts, 11)
    x = torch.randn(T, H, generator=g, device="cuda", requires_grad=True)
    w = torch.rand(T, K, generator=g, device="cuda", requires_grad=True)
    scale = torch.randn(E, H, generator=g, device="cuda", requires_grad=True)   # the experts: y = row * scale[e]
    up = torch.randn(T, H, generator=g, device="cuda")

    def forward(x, w, scale):
        rows, plan = pkg.sort_and_dispatch(x, ids, E, first_expert=first, align=align)
        at = torch.arange(plan.capacity, device="cuda")
        e = (torch.searchsorted(plan.expert_offset.long(), at, right=True) - 1).clamp(max=E - 1)
        return pkg.combine(rows * scale[e], w, plan)

    def loss(x, w, scale):
        return (forward(x, w, scale) * up).sum()

    loss(x, w, scale).backward()
    x64, w64, s64 = (t.detach().double().requires_grad_() for t in (x, w, scale))
    e = ids.long() - first
    live = (e >= 0) & (e < E)
    y64 = x64[:, None, :] * s64[e.clamp(0, E - 1)] * live[..., None]
    ((y64 * w64[..., None]).sum(1) * up.double()).sum().backward()
    for got, want in ((x.grad, x64.grad), (w.grad, w64.grad), (scale.grad, s64.grad)):
        # a few tens of fp32 roundings of sums whose terms are of the size of their result or a few times it
        assert float((got.double() - want).norm() / want.norm()) < 64 * 2.0 ** -24
    with torch.no_grad():
        # the loss is linear in each argument: differences are exact up to the rounding of two sums of T * H terms
        for t, grad in ((x, x.grad), (w, w.grad)):
            d = torch.randn(t.shape, generator=g, device="cuda")
            plus = [(v + 0.5 * d) if v is t else v for v in (x, w, scale)]
            minus = [(v - 0.5 * d) if v is t else v for v in (x, w, scale)]
            step = (forward(*plus).double() * up.double()).sum() - (forward(*minus).double() * up.double()).sum()
            size = (forward(*plus).double() * up.double()).abs().sum()
            assert abs(float(step - (grad.double() * d.double()).sum())) < 64 * 2.0 ** -24 * float(size)


def test_autograd_of_parts(pkg):
    """Only what needs a gradient gets one; a broadcast gradient and a broadcast input work; results passed in are refused."""
    T, K, E, H = 12, 2, 4, 32
    ids = some_ids(T, K, E, 3)
    plan = pkg.sort_tokens(ids, E)
    one = torch.randn(1, H, device="cuda", requires_grad=True)
    rows = pkg.dispatch(one.expand(T, H), plan)
    rows.sum().backward()
    assert torch.equal(one.grad, torch.full_like(one, T * K))
    y = torch.randn(plan.capacity, H, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(T, K, device="cuda", requires_grad=True)
    pkg.combine(y, w, plan).sum().backward()
    want = rows_in_64(y, plan.pair_row).sum(-1)
    assert torch.allclose(w.grad.double(), want, rtol=1e-5, atol=1e-4)
    with pytest.raises(ValueError, match="rows cannot be given"):
        pkg.dispatch(one.expand(T, H), plan, rows=torch.empty(plan.capacity, H, device="cuda"))
    with pytest.raises(ValueError, match="out cannot be given"):
        pkg.combine(y, w, plan, out=torch.empty(T, H, device="cuda", dtype=torch.bfloat16))


def test_graph_replays_see_new_contents(pkg):
    T, K, E, H, align = 300, 4, 32, 512, 16
    ids = some_ids(T, K, E, 21)
    x = torch.randn(T, H, device="cuda").to(torch.bfloat16)
    w = torch.rand(T, K, device="cuda")
    up = torch.randn(T, H, device="cuda").to(torch.bfloat16)
    cap = pkg.plan_rows(T, K, E, align)
    plan, rows = pkg.ExpertPlan.empty(T, K, E, align), torch.zeros(cap, H, device="cuda", dtype=torch.bfloat16)
    out, dy, dx = torch.empty_like(x), torch.zeros_like(rows), torch.empty_like(x)
    dw = torch.empty_like(w)

    def step():
        pkg.sort_and_dispatch(x, ids, E, align=align, plan=plan, rows=rows)
        pkg.combine(rows, w, plan, out=out)
        pkg.combine_backward(up, rows, w, plan, grad_y=dy, grad_weights=dw)
        pkg.dispatch_backward(dy, plan, out=dx)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (22, 23):
        ids.copy_(some_ids(T, K, E, seed))
        x.copy_(torch.randn(T, H, device="cuda"))
        w.copy_(torch.rand(T, K, device="cuda"))
        rows.zero_(), dy.zero_()
        graph.replay()
        got = [t.clone() for t in (plan.row_pair, rows, out, dy, dw, dx)]
        rows.zero_(), dy.zero_()
        step()
        for a, b in zip(got, (plan.row_pair, rows, out, dy, dw, dx)):
            assert torch.equal(a, b)
        check_plan(pkg, plan, ids, E, 0, align)


def test_autograd_in_a_graph(pkg):
    """Forward and backward captured together, after warm-up on a side stream, replayed with other contents."""
    T, K, E, H = 50, 4, 16, 96
    ids = some_ids(T, K, E, 41)
    x = torch.randn(T, H, device="cuda", requires_grad=True)
    w = torch.rand(T, K, device="cuda", requires_grad=True)
    up = torch.randn(T, H, device="cuda")

    def step():
        rows, plan = pkg.sort_and_dispatch(x, ids, E)
        (pkg.combine(rows * 2.0, w, plan) * up).sum().backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            x.grad = w.grad = None
            step()
    torch.cuda.current_stream().wait_stream(side)
    x.grad = w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    with torch.no_grad():
        x.copy_(torch.randn(T, H, device="cuda"))
        w.copy_(torch.rand(T, K, device="cuda"))
        ids.copy_(some_ids(T, K, E, 42))
    graph.replay()
    torch.cuda.synchronize()
    # every pair has a row: out = sum of the weights times 2x
    want_x = 2.0 * up.double() * w.detach().double().sum(1, keepdim=True)
    want_w = (2.0 * up.double() * x.detach().double()).sum(1, keepdim=True).expand(T, K)
    # a product, K additions and two more products in fp32; a sum of H products against the sum of their magnitudes
    assert bool(((x.grad.double() - want_x).abs() <= (K + 4) * 2.0 ** -24 * want_x.abs()).all())
    mag = (2.0 * up.double() * x.detach().double()).abs().sum(1, keepdim=True)
    assert bool(((w.grad.double() - want_w).abs() <= (H / 32 + 32 + 13 + 2) * 2.0 ** -24 * mag).all())


def test_a_plan_filled_anew_before_the_backward_pass(pkg):
    T, K, E, H = 8, 2, 4, 16
    plan = pkg.ExpertPlan.empty(T, K, E)
    x = torch.randn(T, H, device="cuda", requires_grad=True)
    rows, _ = pkg.sort_and_dispatch(x, some_ids(T, K, E, 1), E, plan=plan)
    pkg.sort_tokens(some_ids(T, K, E, 2), E, plan=plan)
    with pytest.raises(RuntimeError, match="filled anew"):
        rows.sum().backward()


def test_another_stream(pkg):
    T, K, E, H = 2000, 8, 64, 1024
    ids = some_ids(T, K, E, 31)
    x = torch.randn(T, H, device="cuda")
    want, plan = pkg.sort_and_dispatch(x, ids, E)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, plan2 = pkg.sort_and_dispatch(x, ids, E)
        back = pkg.dispatch_backward(got, plan2)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(plan.pair_row, plan2.pair_row)
    assert torch.equal(back, pkg.dispatch_backward(want, plan))


def test_refusals_on_the_gpu(pkg):
    T, K, E, H = 6, 2, 4, 16
    ids = some_ids(T, K, E, 1)
    plan = pkg.sort_tokens(ids, E)
    x = torch.randn(T, H, device="cuda")
    w = torch.rand(T, K, device="cuda")
    y = pkg.dispatch(x, plan)
    for call, error in (
            (lambda: pkg.sort_tokens(ids.float(), E), TypeError), (lambda: pkg.sort_tokens(ids.view(-1), E), ValueError),
            (lambda: pkg.sort_tokens(ids.t(), E), ValueError), (lambda: pkg.sort_tokens(ids, 0), ValueError),
            (lambda: pkg.sort_tokens(ids, E + 1, plan=plan), ValueError),
            (lambda: pkg.sort_tokens(ids, E, align=2, plan=plan), ValueError),
            (lambda: pkg.dispatch(x.double(), plan), TypeError), (lambda: pkg.dispatch(x[:-1], plan), ValueError),
            (lambda: pkg.dispatch(x.cpu(), plan), ValueError),
            (lambda: pkg.dispatch(torch.randn(H, T, device="cuda").t(), plan), ValueError),
            (lambda: pkg.dispatch(x, plan, rows=y[:-1]), ValueError),
            (lambda: pkg.dispatch(x, plan, rows=y.half()), TypeError),
            (lambda: pkg.dispatch(x, plan, rows=y[:1].expand(plan.capacity, H)), pkg.MoeError),
            (lambda: pkg.combine(y, w.half(), plan), TypeError), (lambda: pkg.combine(y, w[:, :1], plan), ValueError),
            (lambda: pkg.combine(y, w, plan, out=y[:T]), pkg.MoeError),
            (lambda: pkg.dispatch_backward(y[:-1], plan), ValueError),
            (lambda: pkg.combine_backward(x, y, w, plan, grad_y=y), pkg.MoeError),
            (lambda: pkg.combine_backward(x, y, w, plan, grad_weights=w), pkg.MoeError)):
        with pytest.raises(error):
            call()
    # columns of one wider matrix are apart
    both = torch.zeros(plan.capacity, 2 * H, device="cuda")
    both[:, :H] = y
    dy, _ = pkg.combine_backward(x, both[:, :H], w, plan, grad_y=both[:, H:])
    assert torch.equal(dy, pkg.combine_backward(x, y, w, plan)[0])
    # managed by the C entry: host memory where device memory is due
    import ctypes as C
    err = C.create_string_buffer(256)
    rc = pkg._lib.load().moe_fp8_b200_sort_tokens(ids.cpu().data_ptr(), 32, 0, plan._c, None, err, 256)
    assert rc == pkg._lib.ERR_INVALID_ARGUMENT and b"current CUDA device" in err.value
    rc = pkg._lib.load().moe_fp8_b200_sort_tokens(ids.data_ptr(), 16, 0, plan._c, None, err, 256)
    assert rc == pkg._lib.ERR_INVALID_ARGUMENT and b"id_bits" in err.value


@pytest.mark.parametrize("T", [4, 700])   # sorted and copied by one kernel, by two
def test_plan_and_tensors_that_share_memory(pkg, T):
    """Ids that the plan would be written over, and results that would be written over the plan."""
    K, E, H = 2, 8, 64
    ids = some_ids(T, K, E, 1)
    plan = pkg.sort_tokens(ids, E)
    want = [t.clone() for t in (plan.pair_row, plan.row_pair, plan.expert_offset, plan.expert_count)]
    x = torch.randn(T, H, device="cuda")
    rows = pkg.dispatch(x, plan)
    w = torch.rand(T, K, device="cuda")
    over_ids = pkg.ExpertPlan(ids, *(torch.empty_like(t) for t in (plan.row_pair, plan.expert_offset, plan.expert_count)))
    by_row = pkg.ExpertPlan(torch.empty_like(ids), ids.view(-1), torch.empty_like(plan.expert_offset),
                            torch.empty_like(plan.expert_count))
    kept = ids.clone()
    for p in (over_ids, by_row):
        with pytest.raises(pkg.MoeError, match="topk_idx and the plan"):
            pkg.sort_tokens(ids, E, plan=p)
        with pytest.raises(pkg.MoeError, match="topk_idx and the plan"):
            pkg.sort_and_dispatch(x, ids, E, plan=p)
    # a plan within the memory of the results
    memory = torch.zeros(T * K * H, device="cuda")
    inside = pkg.ExpertPlan(memory[:T * K].view(torch.int32).view(T, K), torch.empty_like(plan.row_pair),
                            torch.empty_like(plan.expert_offset), torch.empty_like(plan.expert_count))
    pkg.sort_tokens(ids, E, plan=inside)
    whole = memory.view(T * K, H)
    for call in (lambda: pkg.dispatch(x, inside, rows=whole), lambda: pkg.sort_and_dispatch(x, ids, E, plan=inside, rows=whole),
                 lambda: pkg.sort_and_dispatch(whole[:T], ids, E, plan=inside),
                 lambda: pkg.combine(rows, w, inside, out=whole[:T]), lambda: pkg.dispatch_backward(rows, inside, out=whole[:T]),
                 lambda: pkg.combine_backward(x, rows, w, inside, grad_y=whole),
                 lambda: pkg.combine_backward(x, rows, w, inside, grad_weights=memory[:T * K].view(T, K))):
        with pytest.raises(pkg.MoeError, match="share memory"):
            call()
    assert torch.equal(ids, kept) and torch.equal(inside.pair_row, want[0])
    with pytest.raises(pkg.MoeError, match="rows and topk_idx share memory"):
        mem = torch.zeros(T * K, H, device="cuda")
        mine = mem.view(-1)[:T * K].view(torch.int32).view(T, K)
        pkg.sort_and_dispatch(x, mine, E, rows=mem)


def test_numbers_that_pass_their_bits(pkg):
    ids = some_ids(4, 2, 8, 1)
    x = torch.randn(4, 16, device="cuda")
    for wrong in (dict(num_experts=8 + (1 << 32)), dict(num_experts=8, align=1 + (1 << 32)),
                  dict(num_experts=8, first_expert=1 << 64), dict(num_experts=8, first_expert=-(1 << 63) - 1)):
        with pytest.raises(ValueError):
            pkg.sort_tokens(ids, **wrong)
        with pytest.raises(ValueError):
            pkg.sort_and_dispatch(x, ids, **wrong)
    plan = pkg.sort_tokens(ids, 8)
    wide = torch.empty(4, (1 << 32) + 16, device="meta")
    for call in (lambda: pkg.dispatch(wide, plan), lambda: pkg.sort_and_dispatch(wide, ids, 8),
                 lambda: pkg.dispatch_backward(wide, plan), lambda: pkg.combine(wide, torch.rand(4, 2, device="cuda"), plan)):
        with pytest.raises(ValueError, match="columns"):
            call()


def test_given_results_and_autograd(pkg):
    """A tensor that a backward pass keeps, written again as a result, is noticed; results with a gradient are refused."""
    T, K, E, H, cols = 6, 2, 8, 16, 64
    ids = some_ids(T, K, E, 3)
    plan = pkg.sort_tokens(ids, E)
    x, w = torch.randn(T, H, device="cuda"), torch.rand(T, K, device="cuda")
    y, dw = torch.randn(T * K, H, device="cuda"), torch.empty(T, K, device="cuda")
    ones = torch.ones(T, H, device="cuda", requires_grad=True)
    half = torch.randn(T * K, cols, device="cuda").bfloat16()
    codes, scales = torch.zeros(16, cols // 2, dtype=torch.uint8, device="cuda"), torch.ones(16, 2, device="cuda").bfloat16()
    out, rows = torch.empty(T, H, device="cuda"), torch.empty(T * K, H, device="cuda")
    narrow = torch.empty(T * K, 16, device="cuda").bfloat16()
    for given, call in ((rows, lambda t: pkg.dispatch(x, plan, rows=t)), (rows, lambda t: pkg.sort_and_dispatch(x, ids, E, rows=t)),
                        (out, lambda t: pkg.combine(y, w, plan, out=t)), (out, lambda t: pkg.dispatch_backward(y, plan, out=t)),
                        (rows, lambda t: pkg.combine_backward(x, y, w, plan, grad_y=t)),
                        (dw, lambda t: pkg.combine_backward(x, y, w, plan, grad_weights=t)),
                        (narrow, lambda t: pkg.matvec_w4(half, codes, scales, out=t))):
        factor = torch.ones_like(given, requires_grad=True)
        given.zero_()
        loss = (factor * given).float().sum()
        call(given)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        leaf = given.clone().requires_grad_()
        with pytest.raises(ValueError, match="requires a gradient"):
            call(leaf)
        with torch.no_grad():
            call(leaf)
        with torch.inference_mode():
            call(torch.empty_like(given))
    # a leaf of the forward pass next to given rows: refused before the plan is filled
    filled = plan._filled
    with pytest.raises(ValueError, match="rows cannot be given"):
        pkg.sort_and_dispatch(ones, ids, E, plan=plan, rows=rows)
    assert plan._filled == filled


def test_what_is_no_tensor(pkg):
    ids = some_ids(4, 2, 8, 1)
    plan = pkg.sort_tokens(ids, 8)
    y, w = torch.randn(8, 16, device="cuda"), torch.rand(4, 2, device="cuda")
    filled = plan._filled
    for call in (lambda: pkg.combine(y, None, plan), lambda: pkg.combine(y.clone().requires_grad_(), None, plan),
                 lambda: pkg.combine(None, w, plan), lambda: pkg.dispatch([[1.0]], plan), lambda: pkg.dispatch_backward(None, plan),
                 lambda: pkg.sort_and_dispatch(None, ids, 8, plan=plan), lambda: pkg.combine_backward(None, y, w, plan),
                 lambda: pkg.combine_backward(y[:4], y, None, plan), lambda: pkg.combine_backward(y[:4], None, w, plan),
                 lambda: pkg.combine(y, w, plan, out=3)):
        with pytest.raises(TypeError):
            call()
    assert plan._filled == filled


def calls_of_threads(pkg, make, sizes, rounds=6000, threads_per_size=3):
    """Errors of C calls that several threads make at once, each with a stream and tensors of its own.  make(size): the entry point,
    its arguments, and a check of the results."""
    import ctypes as C
    import threading
    failed, start = [], threading.Barrier(len(sizes) * threads_per_size)

    def calls(size):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                fn, args, check = make(size)
                stream, err = torch.cuda.current_stream().cuda_stream, C.create_string_buffer(256)
                torch.cuda.synchronize()
                start.wait()
                failed.extend(err.value for _ in range(rounds) if fn(*args, stream, err, 256) != pkg._lib.OK)
                check()
        except BaseException as e:
            failed.append(e)
            start.abort()

    threads = [threading.Thread(target=calls, args=(size,)) for size in sizes for _ in range(threads_per_size)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return failed


def test_sorts_of_several_threads(pkg):
    """Calls that need different amounts of shared memory of one kernel: what one sets for its launch holds for the other's."""
    T, K = 400, 8

    def make(E):
        ids = some_ids(T, K, E, E)
        plan = fresh_plan(pkg, T, K, E, 1)
        return (pkg._lib.load().moe_fp8_b200_sort_tokens, (ids.data_ptr(), 32, 0, plan._c), lambda: check_plan(pkg, plan, ids, E, 0, 1))

    assert not calls_of_threads(pkg, make, (1024, 400))


def test_a_plan_filled_through_another_object(pkg):
    """Two plans over the same four tensors, and writes to the arrays themselves: the backward pass notices all of them."""
    T, K, E, H = 8, 2, 4, 16

    def forward(plan, which):
        x = torch.randn(T, H, device="cuda", requires_grad=True)
        if which == "dispatch":
            return pkg.sort_and_dispatch(x, some_ids(T, K, E, 1), E, plan=plan)[0]
        pkg.sort_tokens(some_ids(T, K, E, 1), E, plan=plan)
        return pkg.combine(torch.randn(T * K, H, device="cuda", requires_grad=True), torch.rand(T, K, device="cuda"), plan)

    for which in ("dispatch", "combine"):
        plan = pkg.ExpertPlan.empty(T, K, E)
        arrays = (plan.pair_row, plan.row_pair, plan.expert_offset, plan.expert_count)
        other, ids = pkg.ExpertPlan(*arrays), some_ids(T, K, E, 2)
        views = pkg.ExpertPlan(*(t.view(t.shape) for t in arrays))
        x = torch.randn(T, H, device="cuda")
        for refill in (lambda: pkg.sort_tokens(ids, E, plan=other), lambda: pkg.sort_and_dispatch(x, ids, E, plan=other),
                       lambda: pkg.sort_and_dispatch(x, ids, E, plan=other, rows=torch.empty(T * K, H, device="cuda")),
                       lambda: pkg.sort_tokens(ids, E, plan=views), lambda: plan.pair_row.fill_(-1)):
            out = forward(plan, which)
            refill()
            with pytest.raises(RuntimeError, match="filled anew"):
                out.sum().backward()
        forward(plan, which).sum().backward()


def test_a_callers_graph_learns_that_the_plan_was_filled(pkg):
    """A node outside this package that kept one of the plan's arrays raises too."""
    T, K, E, H = 8, 2, 4, 16
    plan = pkg.ExpertPlan.empty(T, K, E)
    y = torch.randn(T * K, H, device="cuda", requires_grad=True)
    factor = torch.randn(E + 1, device="cuda", requires_grad=True)
    for use in (lambda: y.index_select(0, plan.pair_row.view(-1)), lambda: y.index_select(0, plan.row_pair),
                lambda: factor * plan.expert_offset, lambda: factor[:E] * plan.expert_count):
        pkg.sort_tokens(some_ids(T, K, E, 1), E, plan=plan)
        loss = use().sum()
        pkg.sort_tokens(some_ids(T, K, E, 2), E, plan=plan)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("kind", ["one buffer", "inference"])
def test_plans_whose_versions_say_nothing(pkg, kind):
    """Pieces of one buffer, which share its version, and tensors of the inference mode, which have none: a plan filled next to this
    one is no obstacle, and this one's own refill changes no gradient."""
    T, K, E, H = 9, 2, 5, 16
    sizes = (T * K, T * K, E + 1, E)
    if kind == "one buffer":
        pieces = torch.empty(2 * sum(sizes), dtype=torch.int32, device="cuda").split(sizes + sizes)
    else:
        with torch.inference_mode():
            pieces = [torch.empty(n, dtype=torch.int32, device="cuda") for n in sizes + sizes]
    plans = [pkg.ExpertPlan(p[0].view(T, K), *p[1:]) for p in (pieces[:4], pieces[4:])]
    seeds, xs, ys, ws, losses = (1, 2), [], [], [], []
    up, upr = torch.randn(T, H, device="cuda"), torch.randn(T * K, H, device="cuda")
    for plan, seed in zip(plans, seeds):
        xs.append(torch.randn(T, H, device="cuda", requires_grad=True))
        ys.append(torch.randn(T * K, H, device="cuda", requires_grad=True))
        ws.append(torch.rand(T, K, device="cuda", requires_grad=True))
        rows, _ = pkg.sort_and_dispatch(xs[-1], some_ids(T, K, E + 2, seed), E, first_expert=1, plan=plan)
        losses.append((rows * upr).sum() + (pkg.combine(ys[-1], ws[-1], plan) * up).sum())
    pkg.sort_tokens(some_ids(T, K, E + 2, 3), E, first_expert=1, plan=plans[1])
    for i, seed in enumerate(seeds):
        losses[i].backward()
        plan = pkg.sort_tokens(some_ids(T, K, E + 2, seed), E, first_expert=1)
        dy, dw = pkg.combine_backward(up, ys[i].detach(), ws[i].detach(), plan)
        assert torch.equal(xs[i].grad, pkg.dispatch_backward(upr, plan))
        assert torch.equal(ys[i].grad, dy) and torch.equal(ws[i].grad, dw)


def test_a_plan_is_read_only(pkg):
    plan = pkg.sort_tokens(some_ids(6, 2, 8, 4), 8)
    for name in ("pair_row", "row_pair", "expert_offset", "expert_count", "align", "num_tokens", "top_k", "num_experts", "capacity",
                 "device", "index"):
        value = getattr(plan, name)
        with pytest.raises(AttributeError):
            setattr(plan, name, value)


def test_forward_mode_tangents_are_refused(pkg):
    """What would come back without its tangent raises, as it does where the input wants a gradient too."""
    import torch.autograd.forward_ad as fwd
    T, K, E, H = 6, 2, 8, 16
    ids = some_ids(T, K, E, 4)
    plan = pkg.sort_tokens(ids, E)
    x, w = torch.randn(T, H, device="cuda"), torch.rand(T, K, device="cuda")
    y = torch.randn(T * K, H, device="cuda")
    half = torch.randn(T, 64, device="cuda").bfloat16()
    codes, scales = torch.zeros(16, 32, dtype=torch.uint8, device="cuda"), torch.ones(16, 2, device="cuda").bfloat16()
    calls = (("x", x, lambda t: pkg.dispatch(t, plan)), ("x", x, lambda t: pkg.sort_and_dispatch(t, ids, E, plan=plan)),
             ("y", y, lambda t: pkg.combine(t, w, plan)), ("weights", w, lambda t: pkg.combine(y, t, plan)),
             ("grad_rows", y, lambda t: pkg.dispatch_backward(t, plan)),
             ("grad_out", x, lambda t: pkg.combine_backward(t, y, w, plan)), ("y", y, lambda t: pkg.combine_backward(x, t, w, plan)),
             ("weights", w, lambda t: pkg.combine_backward(x, y, t, plan)),
             ("x", half, lambda t: pkg.matvec_w4(t, codes, scales)), ("scales", scales, lambda t: pkg.matvec_w4(half, codes, t)),
             # given results would keep a tangent of what they held before
             ("rows", y, lambda t: pkg.dispatch(x, plan, rows=t)), ("out", x.clone(), lambda t: pkg.combine(y, w, plan, out=t)),
             ("grad_y", y.clone(), lambda t: pkg.combine_backward(x, y, w, plan, grad_y=t)))
    filled = plan._filled
    with fwd.dual_level():
        for name, t, call in calls:
            with pytest.raises(NotImplementedError, match=f"{name}.*forward mode"):
                call(fwd.make_dual(t, torch.ones_like(t)))
            assert plan._filled == filled
            with pytest.raises(NotImplementedError):
                call(fwd.make_dual(t.clone().requires_grad_(), torch.ones_like(t)))
            call(t)   # no tangent: as ever
            filled = plan._filled


def test_gradient_calls_on_tensors_that_want_a_gradient(pkg):
    """dispatch_backward and combine_backward have no gradient of their own: they refuse instead of leaving the graph."""
    T, K, E, H = 6, 2, 8, 16
    plan = pkg.sort_tokens(some_ids(T, K, E, 4), E)
    x, w, y = torch.randn(T, H, device="cuda"), torch.rand(T, K, device="cuda"), torch.randn(T * K, H, device="cuda")
    for t, call in ((y, lambda t: pkg.dispatch_backward(t, plan)), (x, lambda t: pkg.combine_backward(t, y, w, plan)),
                    (y, lambda t: pkg.combine_backward(x, t, w, plan)), (w, lambda t: pkg.combine_backward(x, y, t, plan))):
        leaf = t.clone().requires_grad_()
        with pytest.raises(ValueError, match="has no gradient"):
            call(leaf)
        with torch.no_grad():
            call(leaf)
        call(t)


def test_combine_keeps_only_what_its_gradients_read(pkg):
    """The gradient of y does not read y, that of the weights does not read the weights: either may be written after the pass."""
    T, K, E, H = 7, 2, 4, 24
    plan = pkg.sort_tokens(some_ids(T, K, E + 1, 5), E)
    y0, w0, up = torch.randn(T * K, H, device="cuda"), torch.rand(T, K, device="cuda"), torch.randn(T, H, device="cuda")
    dy, dw = pkg.combine_backward(up, y0, w0, plan)
    leaf = y0.clone().requires_grad_()
    y = leaf * 1.0
    out = pkg.combine(y, w0, plan)
    y.add_(1.0)
    out.backward(up)
    assert torch.equal(leaf.grad, dy)
    leaf = w0.clone().requires_grad_()
    w = leaf * 1.0
    out = pkg.combine(y0, w, plan)
    w.add_(1.0)
    out.backward(up)
    assert torch.equal(leaf.grad, dw)
    # both wanted: both are read
    for which in range(2):
        y, w = y0.clone().requires_grad_() * 1.0, w0.clone().requires_grad_() * 1.0
        out = pkg.combine(y, w, plan)
        (y, w)[which].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward(up)
    # as plain calls
    got, none = pkg.combine_backward(up, None, w0, plan, need_weights=False)
    assert none is None and torch.equal(got, dy)
    none, got = pkg.combine_backward(up, y0, None, plan, need_y=False)
    assert none is None and torch.equal(got, dw)
    for y, w, need_y, need_weights in ((None, w0, True, True), (None, w0, False, True), (y0, None, True, True), (y0, None, True, False)):
        with pytest.raises(TypeError):
            pkg.combine_backward(up, y, w, plan, need_y=need_y, need_weights=need_weights)
    assert pkg.combine_backward(up, None, None, plan, need_y=False, need_weights=False) == (None, None)


def test_first_experts_at_the_end_of_64_bits(pkg):
    """An id is compared as a number: the experts behind the last 64-bit id are refused, they do not begin again at the first."""
    lim = torch.iinfo(torch.int64)
    ids = torch.tensor([[lim.min, lim.max], [lim.min + 2, lim.max - 2]], device="cuda")
    x = torch.randn(2, 16, device="cuda")
    for first, E in ((lim.max, 2), (lim.max - 2, 4)):
        with pytest.raises(ValueError, match="64"):
            pkg.sort_tokens(ids, E, first_expert=first)
        with pytest.raises(ValueError, match="64"):
            pkg.sort_and_dispatch(x, ids, E, first_expert=first)
    for first, E in ((lim.max, 1), (lim.max - 3, 4), (lim.min, 4)):
        check_plan(pkg, pkg.sort_tokens(ids, E, first_expert=first, plan=fresh_plan(pkg, 2, 2, E, 1)), ids, E, first, 1)
    # the C entry by itself
    import ctypes as C
    lib, err = pkg._lib.load(), C.create_string_buffer(256)
    plan = fresh_plan(pkg, 2, 2, 4, 1)
    rc = lib.moe_fp8_b200_sort_tokens(ids.data_ptr(), 64, lim.max - 2, plan._c, None, err, 256)
    assert rc == pkg._lib.ERR_INVALID_ARGUMENT and b"64-bit ids" in err.value


def test_sizes_from_numpy(pkg):
    ids = some_ids(4, 2, 8, 1)
    want = pkg.sort_tokens(ids, 8, align=4)
    got = pkg.sort_tokens(ids, np.int64(8), first_expert=np.int32(0), align=np.int64(4))
    assert torch.equal(got.row_pair, want.row_pair)
    got = pkg.sort_tokens(ids, np.int32(8), first_expert=np.int64(0), align=np.int32(4), plan=pkg.ExpertPlan.empty(4, 2, 8, 4))
    assert torch.equal(got.row_pair, want.row_pair)


def test_sizes_that_are_no_whole_numbers(pkg):
    ids = some_ids(4, 2, 8, 1)
    x = torch.randn(4, 16, device="cuda")
    for wrong in (dict(num_experts=8.5), dict(num_experts=8, align=1.5)):
        with pytest.raises(ValueError, match="no plan"):
            pkg.sort_tokens(ids, **wrong)
        with pytest.raises(ValueError, match="no plan"):
            pkg.sort_and_dispatch(x, ids, **wrong)
    plan = pkg.sort_tokens(ids, 8)
    before = plan.pair_row.clone()
    for call in (lambda: pkg.sort_tokens(ids + 1, 8, first_expert=0.5, plan=plan),
                 lambda: pkg.sort_and_dispatch(x, ids + 1, 8, first_expert=0.5, plan=plan)):
        with pytest.raises(TypeError):
            call()
    assert torch.equal(plan.pair_row, before)
    with pytest.raises(ValueError, match="align 1.5"):
        pkg.ExpertPlan.empty(4, 2, 8, 1.5)
    same = pkg.sort_tokens(ids, np.int64(8), first_expert=np.int32(0), align=np.int64(1))
    assert torch.equal(same.pair_row, before)
    assert torch.equal(pkg.sort_tokens(ids, 8.0, align=1.0).pair_row, before)
