"""Performance cases of the operators around the experts: tokens sorted by expert and copied to packed rows, the
experts' rows back at their tokens with the routing weights applied, the gradients of both, and the experts' products
with 4-bit weights for small batches.

A case is a dict of plain values.  `op` names the operator; the fields it uses:

  "dispatch"       expert ids [T, top_k] -> the plan (pair_row, row_pair, expert_offset, expert_count) and the packed
                   rows of x [T, hidden]; pairs whose expert is not in [first, first + local) have no row
  "combine"        packed rows y and weights [T, top_k] -> out[t] = sum over the token's rows of weight * row
  "dispatch_grad"  gradient of the packed rows -> gradient of x: the plain sum over a token's rows
  "combine_grad"   gradient of out -> gradients of y and of the weights
  "matvec"         y = W_e x for the rows of each expert, W_e [n, k] in 4-bit codes with one scale (and, with `zeros`,
                   one zero point) per `group` input columns; `gated`: W_e holds n/2 linear and n/2 gated rows and the
                   result is silu(gated) * linear; `by_token`: x holds one row per token instead of packed rows;
                   local == 0: one matrix [n, k] for all rows, no plan

  tokens T, hidden, top_k, experts (of the router), first / local (experts held here), align (rows of an expert
  rounded up to it, the rest zero), dtype of the rows ("bf16", "fp16", "fp32"), ids ("int32", "int64"), skew (a few
  popular experts), k, n, group, zeros, gated, by_token
"""
from __future__ import annotations

import math
import zlib

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IDS = {"int32": torch.int32, "int64": torch.int64}
RSF = 2.5   # the router's scaling of the weights


def _case(op, name=None, **kw):
    c = dict(op=op, tokens=1, hidden=7168, top_k=8, experts=256, first=0, local=256, align=1, dtype="bf16", ids="int32",
             skew=False)
    if op == "matvec":
        c.update(k=7168, n=4096, group=128, zeros=False, gated=False, by_token=False)
        del c["hidden"]
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one decode token, all experts on this GPU: latency
        _case("dispatch", "dispatch_t1"),
        # the headline batch laid out for a grouped GEMM with 128-row tiles, ids as torch.topk gives them
        _case("dispatch", "dispatch_t12288_align128", tokens=12288, align=128, ids="int64"),
        # a decode batch on one shard of an eight-GPU job: half of the tokens have no row here
        _case("combine", "combine_t57_shard", tokens=57, first=96, local=32),
        # the longest batch with a skewed router, half of the experts
        _case("combine", "combine_t16384_e128_skew", tokens=16384, first=64, local=128, skew=True),
        # backward of an odd training micro-batch in fp16, narrower model
        _case("dispatch_grad", "dispatch_grad_t901_fp16", tokens=901, hidden=4096, dtype="fp16"),
        # backward in fp32 of a model with six experts per token, half of them here
        _case("dispatch_grad", "dispatch_grad_t4099_fp32", tokens=4099, hidden=2048, top_k=6, first=128, local=128,
              dtype="fp32", ids="int64"),
        # rows that end off a 16-byte boundary
        _case("combine_grad", "combine_grad_t129_h1001", tokens=129, hidden=1001, align=16),
        # backward of the headline batch, all experts on this GPU
        _case("combine_grad", "combine_grad_t12288", tokens=12288),
        # one decode token through a single matrix: the smallest product
        _case("matvec", "matvec_dense_t1", tokens=1, local=0, k=2048, n=7168),
        # one decode token, all experts here: eight experts' gate and up weights stream
        _case("matvec", "matvec_gated_t1_e256", tokens=1, gated=True, by_token=True),
        # a small fp16 decode batch on one shard, fine groups with zero points, another intermediate size
        _case("matvec", "matvec_gated_t16_g32_fp16", tokens=16, first=160, local=32, n=2 * 1920, group=32, zeros=True,
              gated=True, by_token=True, dtype="fp16"),
        # the second product of a decode batch of 64 on a quarter of the experts
        _case("matvec", "matvec_t64_e64_g64", tokens=64, first=64, local=64, k=2048, n=7168, group=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("dispatch", "combine", "dispatch_grad", "combine_grad", "matvec", "matvec"))
    experts = rng.choice((256, 256, 128, 64))
    local = rng.choice([e for e in (32, 64, 128, 256) if e <= experts])
    top_k = rng.choice((8, 8, 6, 4, 2, 1))
    c = _case(op, experts=experts, first=32 * rng.randrange((experts - local) // 32 + 1), local=local, top_k=top_k,
              ids=rng.choice(("int32", "int64")), skew=rng.random() < 0.25)
    if op == "matvec":
        c["group"] = rng.choice((128, 128, 64, 32))
        wide = rng.choice((7168, 4096, 2048, 2 * c["group"] * rng.randint(1, 4096 // c["group"])))
        c.update(tokens=_log_int(rng, 1, 64), k=wide, n=rng.choice((2048, 4096, 7168, 16 * rng.randint(1, 448))),
                 zeros=rng.random() < 0.4, gated=rng.random() < 0.5, by_token=rng.random() < 0.5,
                 dtype=rng.choice(("bf16", "bf16", "fp16")))
        if rng.random() < 0.25:
            c.update(local=0, by_token=False)
        if max(c["local"], 1) * c["n"] * c["k"] > 64 * 7168 * 2048:
            c["tokens"] = min(c["tokens"], 8 // top_k)
        return c
    c.update(dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), align=rng.choice((1, 1, 8, 128)),
             hidden=rng.choice((7168, 7168, 4096, 2048, rng.randint(64, 4096))))
    size = 4 if c["dtype"] == "fp32" else 2
    most = 12288 * 8 * 7168 * 2 // (top_k * c["hidden"] * size)
    c["tokens"] = _log_int(rng, 1, min(16384, most))
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _capacity(c):
    """Rows that any choice of experts fits into: every pair, and the rounding of each expert that has one."""
    pairs, experts, align = c["tokens"] * c["top_k"], c["local"], c["align"]
    most = pairs + min(experts, pairs) * (align - 1)
    return -(-most // align) * align


def _generator(seed, *what):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr((int(seed),) + what).encode()))
    return g


def _routing(c, seed):
    """Distinct expert ids of each token and their weights, as a sigmoid router gives them."""
    g = _generator(seed, "routing")
    score = torch.randn(c["tokens"], c["experts"], generator=g, device="cuda")
    if c["skew"]:
        rank = torch.randperm(c["experts"], generator=g, device="cuda") + 1
        score -= 1.5 * torch.log(rank.float())[None, :]
    top, ids = score.topk(c["top_k"], dim=1)
    prob = torch.sigmoid(top)
    return ids.to(IDS[c["ids"]]).contiguous(), (prob / prob.sum(1, keepdim=True) * RSF).contiguous()


def _sorted(c, ids):
    """The plan from elementary operations: rows by expert, within an expert by token."""
    T, K, E, align, cap = c["tokens"], c["top_k"], c["local"], c["align"], _capacity(c)
    expert = ids.reshape(-1).long() - c["first"]
    expert = torch.where((expert >= 0) & (expert < E), expert, E)
    order = torch.argsort(expert, stable=True)
    by = expert[order]
    count = torch.zeros(E + 1, dtype=torch.long, device=ids.device).scatter_add_(0, expert, torch.ones_like(expert))
    padded = torch.div(count + align - 1, align, rounding_mode="floor") * align
    start = torch.cumsum(count, 0) - count
    offset = torch.cumsum(padded, 0) - padded
    row = offset[by] + torch.arange(T * K, device=ids.device) - start[by]
    row = torch.where(by < E, row, cap)
    row_pair = torch.full((cap + 1,), -1, dtype=torch.int32, device=ids.device)
    row_pair.scatter_(0, row, order.to(torch.int32))
    pair_row = torch.empty(T * K, dtype=torch.int32, device=ids.device)
    pair_row.scatter_(0, order, torch.where(by < E, row, -1).to(torch.int32))
    return dict(pair_row=pair_row.view(T, K), row_pair=row_pair[:cap],
                expert_offset=offset.to(torch.int32), expert_count=count[:E].to(torch.int32))


def _weights(c, seed):
    """Codes as a quantiser leaves normal weights (the largest of a group near the end of the range), two per byte with
    the even column in the low half, one scale per group, and zero points off the middle."""
    E, n, k, group = max(c["local"], 1), c["n"], c["k"], c["group"]
    g = _generator(seed, "weights")
    codes = torch.empty(E, n, k // 2, dtype=torch.uint8, device="cuda")
    zeros = torch.randint(6, 11, (E, n, k // group), generator=g, device="cuda", dtype=torch.uint8) if c["zeros"] else None
    for e in range(E):
        q = torch.randn(n, k, generator=g, device="cuda") * 2.7
        mid = zeros[e].repeat_interleave(group, dim=1).float() if c["zeros"] else 8.0
        q = (q.round_() + mid).clamp_(0, 15).to(torch.uint8)
        codes[e] = q[:, 0::2] | (q[:, 1::2] << 4)
    scales = torch.randn(E, n, k // group, generator=g, device="cuda").mul_(0.25).exp_().mul_(0.0075)
    scales = scales.to(DTYPES[c["dtype"]])
    if c["local"] == 0:
        return codes[0], scales[0], None if zeros is None else zeros[0]
    return codes, scales, zeros


def _normal(seed, what, dtype, *shape):
    return torch.randn(*shape, generator=_generator(seed, what), device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    s = dict(case=c)
    if c["op"] == "matvec":
        s["codes"], s["scales"], s["zeros"] = _weights(c, seed)
        rows = c["tokens"]
        if c["local"] > 0:
            ids, _ = _routing(c, seed)
            s["plan"] = _sorted(c, ids)
            rows = _capacity(c)
        s["x"] = _normal(seed, "x", dt, c["tokens"] if c["by_token"] else rows, c["k"])
        s["out"] = torch.zeros(rows, c["n"] // 2 if c["gated"] else c["n"], dtype=dt, device="cuda")
        return s
    T, H, cap = c["tokens"], c["hidden"], _capacity(c)
    ids, weights = _routing(c, seed)
    if c["op"] == "dispatch":
        s.update(ids=ids, x=_normal(seed, "x", dt, T, H), rows=torch.zeros(cap, H, dtype=dt, device="cuda"))
        s["buffers"] = dict(pair_row=torch.empty(T, c["top_k"], dtype=torch.int32, device="cuda"),
                            row_pair=torch.empty(cap, dtype=torch.int32, device="cuda"),
                            expert_offset=torch.empty(c["local"] + 1, dtype=torch.int32, device="cuda"),
                            expert_count=torch.empty(c["local"], dtype=torch.int32, device="cuda"))
        return s
    s["plan"] = _sorted(c, ids)
    if c["op"] == "combine":
        s.update(y=_normal(seed, "y", dt, cap, H), weights=weights, out=torch.empty(T, H, dtype=dt, device="cuda"))
    elif c["op"] == "dispatch_grad":
        s.update(grad_rows=_normal(seed, "grad_rows", dt, cap, H), out=torch.empty(T, H, dtype=dt, device="cuda"))
    else:
        s.update(y=_normal(seed, "y", dt, cap, H), weights=weights, grad_out=_normal(seed, "grad_out", dt, T, H),
                 grad_y=torch.zeros(cap, H, dtype=dt, device="cuda"),
                 grad_weights=torch.empty(T, c["top_k"], dtype=torch.float32, device="cuda"))
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _package():
    import __graft_entry__ as entry
    return entry.load_package()


def _plan(moe, c, tensors):
    return moe.ExpertPlan(tensors["pair_row"], tensors["row_pair"], tensors["expert_offset"], tensors["expert_count"],
                          align=c["align"])


def _run_own(s):
    moe, c = _package(), s["case"]
    if c["op"] == "dispatch":
        rows, plan = moe.sort_and_dispatch(s["x"], s["ids"], c["local"], first_expert=c["first"], align=c["align"],
                                           plan=_plan(moe, c, s["buffers"]), rows=s["rows"])
        return dict(rows=rows, pair_row=plan.pair_row, row_pair=plan.row_pair, expert_offset=plan.expert_offset,
                    expert_count=plan.expert_count)
    if c["op"] == "combine":
        return moe.combine(s["y"], s["weights"], _plan(moe, c, s["plan"]), out=s["out"])
    if c["op"] == "dispatch_grad":
        return moe.dispatch_backward(s["grad_rows"], _plan(moe, c, s["plan"]), out=s["out"])
    if c["op"] == "combine_grad":
        grad_y, grad_weights = moe.combine_backward(s["grad_out"], s["y"], s["weights"], _plan(moe, c, s["plan"]),
                                                    grad_y=s["grad_y"], grad_weights=s["grad_weights"])
        return dict(grad_y=grad_y, grad_weights=grad_weights)
    plan = _plan(moe, c, s["plan"]) if c["local"] > 0 else None
    return moe.matvec_w4(s["x"], s["codes"], s["scales"], zeros=s["zeros"], plan=plan, gated=c["gated"],
                         by_token=c["by_token"], out=s["out"])


def _rows_of(values, pair_row):
    """values[pair_row] in 32 bits, zeros where a pair has no row: [T, K, H]."""
    at = pair_row.long()
    return torch.where((at >= 0)[..., None], values[at.clamp(min=0)].float(), 0.0)


def _decoded(codes, scales, zeros):
    """The weights' values in 32 bits: [..., n, k]."""
    q = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float()
    group = q.shape[-1] // scales.shape[-1]
    q = q.unflatten(-1, (-1, group))
    mid = 8.0 if zeros is None else zeros.float()[..., None]
    return ((q - mid) * scales.float()[..., None]).flatten(-2)


def _activated(c, y):
    if not c["gated"]:
        return y
    linear, gate = y[..., :c["n"] // 2], y[..., c["n"] // 2:]
    return gate / (1.0 + torch.exp(-gate)) * linear


def _matvec_plain(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    if c["local"] == 0:
        w = _decoded(s["codes"], s["scales"], s["zeros"])
        return _activated(c, s["x"].float() @ w.t()).to(dt)
    p, T, K, E = s["plan"], c["tokens"], c["top_k"], c["local"]
    cap = _capacity(c)
    at = torch.arange(cap, device="cuda")
    pair = p["row_pair"].long()
    live = pair >= 0
    expert = (torch.searchsorted(p["expert_offset"].long(), at, right=True) - 1).clamp(max=E - 1)
    x = (s["x"][torch.div(pair.clamp(min=0), K, rounding_mode="floor")] if c["by_token"] else s["x"]).float()
    if cap <= E:
        # fewer rows than experts: each row's own weights
        zeros = None if s["zeros"] is None else s["zeros"][expert]
        w = _decoded(s["codes"][expert], s["scales"][expert], zeros)
        y = (w @ x[:, :, None])[:, :, 0]
    else:
        # every expert's rows side by side; an expert has at most one row per token
        slot = (at - p["expert_offset"].long()[expert]).clamp(max=T)
        to = torch.where(live, expert * T + slot, E * T)
        spread = torch.zeros(E * T + 1, c["k"], device="cuda").index_copy_(0, to, x)
        w = _decoded(s["codes"], s["scales"], s["zeros"])
        y = torch.bmm(spread[:E * T].view(E, T, -1), w.transpose(1, 2)).flatten(0, 1)[to.clamp(max=E * T - 1)]
    return torch.where(live[:, None], _activated(c, y), 0.0).to(dt)


def run(state):
    if own:
        return _run_own(state)
    s, c = state, state["case"]
    dt = DTYPES[c["dtype"]]
    if c["op"] == "dispatch":
        plan = _sorted(c, s["ids"])
        pair = plan["row_pair"].long()
        token = torch.div(pair.clamp(min=0), c["top_k"], rounding_mode="floor")
        rows = torch.where((pair >= 0)[:, None], s["x"][token], torch.zeros((), dtype=dt, device="cuda"))
        return dict(rows=rows, **plan)
    if c["op"] == "combine":
        return (_rows_of(s["y"], s["plan"]["pair_row"]) * s["weights"][..., None]).sum(1).to(dt)
    if c["op"] == "dispatch_grad":
        return _rows_of(s["grad_rows"], s["plan"]["pair_row"]).sum(1).to(dt)
    if c["op"] == "combine_grad":
        pair = s["plan"]["row_pair"].long()
        token = torch.div(pair.clamp(min=0), c["top_k"], rounding_mode="floor")
        scaled = s["grad_out"][token].float() * s["weights"].flatten()[pair.clamp(min=0)][:, None]
        grad_y = torch.where((pair >= 0)[:, None], scaled, 0.0).to(dt)
        grad_weights = (_rows_of(s["y"], s["plan"]["pair_row"]) * s["grad_out"].float()[:, None, :]).sum(-1)
        return dict(grad_y=grad_y, grad_weights=grad_weights)
    return _matvec_plain(s)


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "matvec":
        return _matvec_exact(s)
    T, K, H, cap = c["tokens"], c["top_k"], c["hidden"], _capacity(c)
    if c["op"] == "dispatch":
        ids = s["ids"].cpu().reshape(-1).tolist()
        mine = [[] for _ in range(c["local"])]
        for pair, e in enumerate(ids):
            if 0 <= e - c["first"] < c["local"]:
                mine[e - c["first"]].append(pair)
        pair_row, row_pair, offset = [-1] * (T * K), [-1] * cap, [0]
        for pairs in mine:
            for i, pair in enumerate(pairs):
                pair_row[pair], row_pair[offset[-1] + i] = offset[-1] + i, pair
            offset.append(offset[-1] + -(-len(pairs) // c["align"]) * c["align"])
        rows = torch.zeros(cap, H, dtype=torch.float64, device="cuda")
        used = [r for r in range(cap) if row_pair[r] >= 0]
        rows[used] = s["x"].double()[[row_pair[r] // K for r in used]]
        whole = dict(pair_row=torch.tensor(pair_row).view(T, K), row_pair=torch.tensor(row_pair),
                     expert_offset=torch.tensor(offset), expert_count=torch.tensor([len(m) for m in mine]))
        return dict(rows=rows, **{name: v.to(torch.int32) for name, v in whole.items()})
    at = s["plan"]["pair_row"].long()
    if c["op"] in ("combine", "dispatch_grad"):
        src = s["y"] if c["op"] == "combine" else s["grad_rows"]
        out = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        for k in range(K):
            live = (at[:, k] >= 0).nonzero()[:, 0]
            part = src[at[live, k]].double()
            out[live] += part * s["weights"][live, k, None].double() if c["op"] == "combine" else part
        return out
    grad_y = torch.zeros(cap, H, dtype=torch.float64, device="cuda")
    grad_weights = torch.zeros(T, K, dtype=torch.float64, device="cuda")
    g = s["grad_out"].double()
    for k in range(K):
        live = (at[:, k] >= 0).nonzero()[:, 0]
        grad_y[at[live, k]] = g[live] * s["weights"][live, k, None].double()
        grad_weights[live, k] = (g[live] * s["y"][at[live, k]].double()).sum(-1)
    return dict(grad_y=grad_y, grad_weights=grad_weights)


def _matvec_exact(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]

    def product(codes, scales, zeros, x):
        w = torch.empty(n, k, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
        w = w.view(n, k // group, group)
        w -= 8 if zeros is None else zeros.double()[:, :, None]
        w *= scales.double()[:, :, None]
        y = x.double() @ w.view(n, k).t()
        return y[:, n // 2:] * torch.sigmoid(y[:, n // 2:]) * y[:, :n // 2] if c["gated"] else y

    if c["local"] == 0:
        return product(s["codes"], s["scales"], s["zeros"], s["x"])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    first, count = s["plan"]["expert_offset"].tolist(), s["plan"]["expert_count"].tolist()
    for e in range(c["local"]):
        if count[e] == 0:
            continue
        r = slice(first[e], first[e] + count[e])
        x = s["x"][s["plan"]["row_pair"][r].long() // c["top_k"]] if c["by_token"] else s["x"][r]
        out[r] = product(s["codes"][e], s["scales"][e], None if s["zeros"] is None else s["zeros"][e], x)
    return out


# ------------------------------------------------------------------------------------------------ what it costs
def _routed(c):
    """Expected (rows, tokens with a row, experts with a row) by the routing's distribution: a few samples of it, more
    of them the fewer tokens there are."""
    g = torch.Generator()
    g.manual_seed(12)
    samples = max(2, 512 // c["tokens"])
    total = [0.0, 0.0, 0.0]
    for _ in range(samples):
        score = torch.randn(c["tokens"], c["experts"], generator=g)
        if c["skew"]:
            score -= 1.5 * torch.log((torch.randperm(c["experts"], generator=g) + 1).float())[None, :]
        ids = score.topk(c["top_k"], dim=1).indices - c["first"]
        mine = (ids >= 0) & (ids < c["local"])
        for i, v in enumerate((mine.sum(), mine.any(1).sum(), ids[mine].unique().numel())):
            total[i] += float(v) / samples
    return total


def work(case):
    """What one pass cannot do without: every value it needs read once, every result written once."""
    c = case
    T, size = c["tokens"], 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "matvec":
        rows, _, experts = (T, T, 1) if c["local"] == 0 else _routed(c)
        per = c["n"] * c["k"] / 2 + c["n"] * (c["k"] // c["group"]) * (3 if c["zeros"] else 2)
        outs = c["n"] // 2 if c["gated"] else c["n"]
        return {"bytes": float(experts * per + min(T if c["by_token"] else rows, rows) * c["k"] * size + rows * outs * size),
                "flops": float(2 * rows * c["n"] * c["k"])}
    rows, live, _ = _routed(c)
    H, pairs = c["hidden"], T * c["top_k"]
    if c["op"] == "dispatch":
        ids = pairs * (4 if c["ids"] == "int32" else 8)
        return {"bytes": float(ids + 4 * pairs + 4 * _capacity(c) + 8 * c["local"] + (live + rows) * H * size), "flops": 0.0}
    if c["op"] == "combine":
        return {"bytes": float((rows + T) * H * size + 8 * pairs), "flops": float(2 * rows * H)}
    if c["op"] == "dispatch_grad":
        return {"bytes": float((rows + T) * H * size + 4 * pairs), "flops": float(rows * H)}
    return {"bytes": float((2 * rows + live) * H * size + 12 * pairs), "flops": float(3 * rows * H)}
