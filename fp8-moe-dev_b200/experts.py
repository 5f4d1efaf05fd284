"""The operators around a caller's own experts, on top of the C ABI: tokens sorted by expert and copied to packed rows,
the experts' rows back at their tokens with the routing weights applied, and the gradients of both.

    plan = sort_tokens(topk_idx, num_experts)              # which packed row every (token, expert) pair has
    rows = dispatch(x, plan)                               # [plan.capacity, hidden], grouped by expert
    y = ...                                                # the experts' results, row by row
    out = combine(y, topk_weights, plan)                   # [T, hidden]

`sort_and_dispatch` is the first two in one call.  `dispatch` and `combine` take part in autograd, in reverse mode;
`dispatch_backward` and `combine_backward` are their gradients as plain calls.  Tensors with a tangent of forward mode are
refused everywhere.  A plan written to after a forward pass is refused by its backward pass.  Results go to the tensors passed
for them, or to new ones.
Everything runs on the current stream of the tensors' device, returns without synchronising and may be captured into a
graph.  (A captured backward pass follows torch's own rule: no other graph of the same leaves may be alive, since the nodes that
accumulate their gradients belong to the stream that made them.  The `_backward` functions have no such rule.)  `matvec_w4`
is the experts' product of a decode batch with 4-bit weights.  The counterparts
inside the reference's layer are kernel/moe_fp8.cu:1064-1115 (permute) and :2254-2323 (combine).
"""
from __future__ import annotations

import ctypes as C
import operator
import threading
from typing import Optional, Tuple

import torch

from . import _lib
from .op import MoeError

_ROW_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}
_ID_BITS = {torch.int32: 32, torch.int64: 64}
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_forward_ad = torch.autograd.forward_ad
_MAX_COLUMNS = 1 << 24
_SMALL = 1 << 20   # tokens up to which a plan's size needs no word from the library, first experts that need no closer look


class _Text(threading.local):
    """A thread's buffer for error messages."""

    def __init__(self):
        self.buffer = C.create_string_buffer(256)


_text = _Text()


def _call(fn, index, *args):
    """fn(*args, stream, err, err_len) with GPU `index` current."""
    err = _text.buffer
    if index == _current_device():
        rc = fn(*args, _raw_stream(index), err, 256)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index), err, 256)
    if rc != _lib.OK:
        raise MoeError(rc, err.value.decode())


# The checks are written out and compare GPU indices, not device objects: small calls are bound by the host's time.
def _on_gpu(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    index = t.get_device()
    if index < 0 or not t.is_cuda:
        raise ValueError(f"{name} must live on a CUDA device, got {t.device}")
    return index


def _wrong(name, t, dtype, shape, index):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_cuda or t.get_device() != index:
        raise ValueError(f"{name} must live on cuda:{index}, got {t.device}")
    raise ValueError(f"{name} must be contiguous")


def _packed(name, t, dtype, shape, index):
    """The address of a contiguous tensor."""
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or not t.is_cuda
            or t.get_device() != index):
        _wrong(name, t, dtype, shape, index)
    return t.data_ptr()


def _matrix(name, t, rows, columns, dtype, index):
    """A [rows, columns] matrix whose rows are contiguous, at any stride: its address and stride."""
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != (rows, columns) or not t.is_cuda
            or t.get_device() != index):
        _wrong(name, t, dtype, (rows, columns), index)
    stride, column = t.stride()
    if column != 1 and columns > 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous")
    return t.data_ptr(), stride


def _row_type(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    kind = _ROW_TYPES.get(t.dtype)
    if kind is None:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.dim() != 2 or not 1 <= t.shape[1] <= _MAX_COLUMNS:
        raise ValueError(f"{name} must be a matrix of 1 .. {_MAX_COLUMNS} columns, got shape {tuple(t.shape)}")
    return kind


# Tangents of forward-mode differentiation go with tensors that want no gradient.  A result without one would say that it is zero.
def _no_tangents(**tensors):
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has a tangent, and there is no derivative in forward mode here")


def _result(name, t):
    if _forward_ad._current_level >= 0:
        _no_tangents(**{name: t})
    if isinstance(t, torch.Tensor) and _wants_grad(t):
        raise ValueError(f"{name} requires a gradient: give a tensor that does not, or call under torch.no_grad()")


# autograd learns that a given tensor, or an array of a plan, was written: a backward pass that saved it raises instead of reading the
# new contents
_written = torch._C._increment_version


def plan_rows(num_tokens: int, top_k: int, num_experts: int, align: int = 1) -> int:
    """Rows that any choice of experts fits into: what `rows` of a dispatch must hold."""
    given = num_tokens, top_k, num_experts, align
    if (type(num_tokens) is type(top_k) is type(num_experts) is type(align) is int and 0 <= num_tokens <= _SMALL
            and 1 <= top_k <= _lib.PLAN_MAX_TOP_K and 1 <= num_experts <= _lib.PLAN_MAX_EXPERTS and 1 <= align <= 1024):
        pairs = num_tokens * top_k
        return (pairs + min(num_experts, pairs) * (align - 1) + align - 1) // align * align
    whole = int(num_tokens), int(top_k), int(num_experts), int(align)
    # what passes 32 bits would reach the library cut to them
    rows = _lib.load().moe_fp8_b200_plan_rows(*whole) if whole == given and max(whole) < 1 << 31 and min(whole) >= 0 else -1
    if rows < 0:
        raise ValueError(f"no plan for {num_tokens} tokens, top_k {top_k} (1 .. {_lib.PLAN_MAX_TOP_K}), {num_experts} experts "
                         f"(1 .. {_lib.PLAN_MAX_EXPERTS}), align {align} (1 .. 1024)")
    return int(rows)


class ExpertPlan:
    """Which packed row every (token, expert) pair has.  Rows are ordered by expert, within an expert by pair
    t * top_k + k; each expert starts a multiple of `align` rows after the one before it.

      pair_row       int32 [T, top_k]    row of each pair, -1 where its expert is not one of this plan's
      row_pair       int32 [capacity]    pair of each row, -1 in an expert's padding and behind the last expert
      expert_offset  int32 [E + 1]       first row of each expert, and the end of the last one
      expert_count   int32 [E]           pairs of each expert

    Made by sort_tokens, or from four tensors of one's own (to be filled, or filled elsewhere).  All of these are read-only."""
    # the C struct holds the same addresses and sizes
    __slots__ = ("_pair_row", "_row_pair", "_expert_offset", "_expert_count", "_align", "_num_tokens", "_top_k", "_num_experts",
                 "_capacity", "_device", "_index", "_c", "_arrays")
    (pair_row, row_pair, expert_offset, expert_count, align, num_tokens, top_k, num_experts, capacity, device,
     index) = (property(operator.attrgetter(name)) for name in __slots__[:11])

    def __init__(self, pair_row, row_pair, expert_offset, expert_count, *, align: int = 1):
        index = _on_gpu("pair_row", pair_row)
        if pair_row.dim() != 2:
            raise ValueError(f"pair_row must have shape (tokens, top_k), got {tuple(pair_row.shape)}")
        T, K = pair_row.shape
        E = expert_count.shape[0] if isinstance(expert_count, torch.Tensor) and expert_count.dim() == 1 else 0
        self._num_tokens, self._top_k, self._num_experts, self._align = T, K, E, align
        self._capacity = capacity = plan_rows(T, K, E, align)
        self._pair_row, self._row_pair, self._expert_offset, self._expert_count = pair_row, row_pair, expert_offset, expert_count
        self._device, self._index = pair_row.device, index
        self._arrays = (pair_row, row_pair, expert_offset, expert_count)
        i32 = torch.int32
        self._c = C.byref(_lib.Plan(T, K, E, align, _packed("pair_row", pair_row, i32, (T, K), index),
                                    _packed("row_pair", row_pair, i32, (capacity,), index),
                                    _packed("expert_offset", expert_offset, i32, (E + 1,), index),
                                    _packed("expert_count", expert_count, i32, (E,), index)))

    @classmethod
    def empty(cls, num_tokens: int, top_k: int, num_experts: int, align: int = 1, device="cuda") -> "ExpertPlan":
        """A plan to be filled."""
        def ints(*shape):
            return torch.empty(shape, dtype=torch.int32, device=device)
        capacity = plan_rows(num_tokens, top_k, num_experts, align)
        T, K, E = int(num_tokens), int(top_k), int(num_experts)
        return cls(ints(T, K), ints(capacity), ints(E + 1), ints(E), align=int(align))

    @property
    def _filled(self):
        """The versions of the arrays that a backward pass reads: any write to them changes these, through whichever object it went."""
        return self._pair_row._version, self._expert_offset._version, self._expert_count._version

    def _for_backward(self):
        """The plan that a backward pass keeps, and its state: this one, if the versions of its arrays say when they are written.  They
        do not for pieces of a larger buffer, whose version moves with the other pieces too, nor for tensors of the inference
        mode, which have none: then a plan with copies, which no one else knows."""
        read = (self._pair_row, self._expert_offset, self._expert_count)
        if all(t.untyped_storage().nbytes() == 4 * t.numel() and not t.is_inference() for t in read):
            return self, self._filled
        plan = ExpertPlan(self._pair_row.clone(), self._row_pair, self._expert_offset.clone(), self._expert_count.clone(),
                          align=self._align)
        return plan, plan._filled


def _check_plan(plan):
    if not isinstance(plan, ExpertPlan):
        raise TypeError("plan must be an ExpertPlan")
    return plan._index


def _ids(topk_idx, num_experts, first_expert, align, plan):
    """The plan to fill for these ids."""
    index = _on_gpu("topk_idx", topk_idx)
    if type(first_expert) is not int or not 0 <= first_expert <= _SMALL:
        # the library counts on from it modulo 2^64
        if not -1 << 63 <= operator.index(first_expert) <= (1 << 63) - max(1, int(num_experts)):
            raise ValueError(f"first_expert {first_expert}: experts from it on are not 64-bit ids")
    if topk_idx.dtype not in _ID_BITS:
        raise TypeError(f"topk_idx must be int32 or int64, got {topk_idx.dtype}")
    if topk_idx.dim() != 2:
        raise ValueError(f"topk_idx must have shape (tokens, top_k), got {tuple(topk_idx.shape)}")
    if not topk_idx.is_contiguous():
        raise ValueError("topk_idx must be contiguous")
    T, K = topk_idx.shape
    if plan is None:
        return ExpertPlan.empty(T, K, num_experts, align, topk_idx.device)
    if _check_plan(plan) != index:
        raise ValueError(f"plan must live on {topk_idx.device}, got {plan._device}")
    if (plan._num_tokens, plan._top_k, plan._num_experts, plan._align) != (T, K, num_experts, align):
        raise ValueError(f"plan is for {plan._num_tokens} tokens, top_k {plan._top_k}, {plan._num_experts} experts, align "
                         f"{plan._align}; the call has {T}, {K}, {num_experts}, {align}")
    return plan


def sort_tokens(topk_idx, num_experts: int, *, first_expert: int = 0, align: int = 1,
                plan: Optional[ExpertPlan] = None) -> ExpertPlan:
    """Sorts the (token, expert) pairs of topk_idx [T, top_k] (int32 or int64) by expert.  The plan's experts are
    [first_expert, first_expert + num_experts); pairs of other experts (an id of -1, another GPU's expert) have no row."""
    plan = _ids(topk_idx, num_experts, first_expert, align, plan)
    _call(_lib.load().moe_fp8_b200_sort_tokens, plan._index, topk_idx.data_ptr(), _ID_BITS[topk_idx.dtype], first_expert,
          plan._c)
    _written(plan._arrays)
    return plan


def _rows_for(x, plan, rows):
    """Arguments of the copy to packed rows: the matrix, and its C arguments."""
    kind = _row_type("x", x)
    H = x.shape[1]
    xp, xs = _matrix("x", x, plan._num_tokens, H, x.dtype, plan._index)
    fresh = rows is None
    if fresh:
        rows = torch.empty((plan._capacity, H), dtype=x.dtype, device=plan._device)
    else:
        _result("rows", rows)
    rp, rs = _matrix("rows", rows, plan._capacity, H, x.dtype, plan._index)
    return rows, (xp, xs, rp, rs, kind, H, plan._c, int(fresh))


def _wants_grad(a, b=None):
    return (a.requires_grad or (b is not None and b.requires_grad)) and torch.is_grad_enabled()


def dispatch(x, plan: ExpertPlan, rows=None):
    """rows[r] = x[token of row r], zeros in the experts' padding; rows behind the last expert stay as they were (in
    a new matrix: zeros).  x [T, hidden], rows [plan.capacity, hidden]: bfloat16, float16 or float32, any row stride.
    Differentiable in x (not together with `rows`)."""
    _check_plan(plan)
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if _forward_ad._current_level >= 0:
        _no_tangents(x=x)
    if _wants_grad(x):
        if rows is not None:
            raise ValueError("rows cannot be given where x requires a gradient")
        return _Dispatch.apply(x, plan)
    rows, args = _rows_for(x, plan, rows)
    _call(_lib.load().moe_fp8_b200_dispatch_rows, plan._index, *args)
    if not args[-1]:
        _written((rows,))
    return rows


def sort_and_dispatch(x, topk_idx, num_experts: int, *, first_expert: int = 0, align: int = 1,
                      plan: Optional[ExpertPlan] = None, rows=None) -> Tuple[torch.Tensor, ExpertPlan]:
    """sort_tokens and dispatch in one call: (rows, plan)."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if _forward_ad._current_level >= 0:
        _no_tangents(x=x)
    plan = _ids(topk_idx, num_experts, first_expert, align, plan)
    if _wants_grad(x):
        if rows is not None:
            raise ValueError("rows cannot be given where x requires a gradient")
        return dispatch(x, sort_tokens(topk_idx, num_experts, first_expert=first_expert, align=align, plan=plan)), plan
    rows, args = _rows_for(x, plan, rows)
    _call(_lib.load().moe_fp8_b200_sort_and_dispatch, plan._index, topk_idx.data_ptr(), _ID_BITS[topk_idx.dtype], first_expert,
          *args)
    _written(plan._arrays if args[-1] else (rows, *plan._arrays))
    return rows, plan


def _combine(y, weights, plan, out):
    kind = _row_type("y", y)
    H = y.shape[1]
    yp, ys = _matrix("y", y, plan._capacity, H, y.dtype, plan._index)
    wp = None if weights is None else _packed("weights", weights, torch.float32, (plan._num_tokens, plan._top_k), plan._index)
    fresh = out is None
    if fresh:
        out = torch.empty((plan._num_tokens, H), dtype=y.dtype, device=plan._device)
    else:
        _result("out", out)
    op, os = _matrix("out", out, plan._num_tokens, H, y.dtype, plan._index)
    _call(_lib.load().moe_fp8_b200_combine_rows, plan._index, yp, ys, wp, op, os, kind, H, plan._c)
    if not fresh:
        _written((out,))
    return out


def combine(y, weights, plan: ExpertPlan, out=None):
    """out[t] = sum over token t's rows of weights[t, k] * y[row], in fp32 and pair order, rounded once; zeros for a token
    without rows.  y [plan.capacity, hidden], weights fp32 [T, top_k].  Padding and unused rows of y are not read.
    Differentiable in y and weights (not together with `out`)."""
    _check_plan(plan)
    if not isinstance(y, torch.Tensor) or not isinstance(weights, torch.Tensor):
        raise TypeError("y and weights must be torch.Tensors")
    if _forward_ad._current_level >= 0:
        _no_tangents(y=y, weights=weights)
    if _wants_grad(y, weights):
        if out is not None:
            raise ValueError("out cannot be given where y or weights require a gradient")
        return _Combine.apply(y, weights, plan)
    return _combine(y, weights, plan, out)


def dispatch_backward(grad_rows, plan: ExpertPlan, out=None):
    """Gradient of dispatch's x from that of its rows: out[t] = the sum of token t's rows.  Not differentiable itself."""
    _check_plan(plan)
    if _forward_ad._current_level >= 0:
        _no_tangents(grad_rows=grad_rows)
    if isinstance(grad_rows, torch.Tensor) and _wants_grad(grad_rows):
        raise ValueError("dispatch_backward has no gradient: call it under torch.no_grad()")
    return _combine(grad_rows, None, plan, out)


def combine_backward(grad_out, y, weights, plan: ExpertPlan, grad_y=None, grad_weights=None, *, need_y: bool = True,
                     need_weights: bool = True):
    """Gradients of combine: (grad_y [plan.capacity, hidden], grad_weights fp32 [T, top_k]).  grad_y is zero in the
    experts' padding and untouched behind the last expert (in a new matrix: zero there too); grad_weights is 0 where a pair has no row.  A gradient that is
    not needed is None; y is read for grad_weights only, weights for grad_y only, and either may be None without it.  Not
    differentiable itself."""
    _check_plan(plan)
    if _forward_ad._current_level >= 0:
        _no_tangents(grad_out=grad_out, y=y, weights=weights)
    kind = _row_type("grad_out", grad_out)
    H, dtype, device, index = grad_out.shape[1], grad_out.dtype, plan._device, plan._index
    gp, gs = _matrix("grad_out", grad_out, plan._num_tokens, H, dtype, index)
    yp, ys, wp, dp, ds, dwp = None, 0, None, None, 0, None
    wanted = grad_out.requires_grad
    if need_weights or y is not None:
        yp, ys = _matrix("y", y, plan._capacity, H, dtype, index)
        wanted |= y.requires_grad
    if need_y or weights is not None:
        wp = _packed("weights", weights, torch.float32, (plan._num_tokens, plan._top_k), index)
        wanted |= weights.requires_grad
    if wanted and torch.is_grad_enabled():
        raise ValueError("combine_backward has no gradient: call it under torch.no_grad()")
    fresh = grad_y is None
    if need_y:
        if fresh:
            grad_y = torch.empty((plan._capacity, H), dtype=dtype, device=device)
        else:
            _result("grad_y", grad_y)
        dp, ds = _matrix("grad_y", grad_y, plan._capacity, H, dtype, index)
    fresh_weights = grad_weights is None
    if need_weights:
        if fresh_weights:
            grad_weights = torch.empty((plan._num_tokens, plan._top_k), dtype=torch.float32, device=device)
        else:
            _result("grad_weights", grad_weights)
        dwp = _packed("grad_weights", grad_weights, torch.float32, (plan._num_tokens, plan._top_k), index)
    _call(_lib.load().moe_fp8_b200_combine_rows_backward, index, gp, gs, yp, ys, wp, dp, ds, dwp, kind, H, plan._c,
          int(fresh))
    if need_y and not fresh:
        _written((grad_y,))
    if need_weights and not fresh_weights:
        _written((grad_weights,))
    return grad_y if need_y else None, grad_weights if need_weights else None


def matvec_w4(x, codes, scales, *, zeros=None, plan: Optional[ExpertPlan] = None, by_token: bool = False, gated: bool = False,
              out=None):
    """Products of a few rows with 4-bit weights: y[r, n] = sum_k (code[n, k] - zero[n, g]) * scale[n, g] * x[r, k] with
    g = k // group: exact products of codes and x, summed in fp32, rounded once.

      codes   uint8 [E, n, k / 2]          two codes 0 .. 15 per byte, the even column in the low half
      scales  x's dtype [E, n, k / group]  group 32, 64 or 128
      zeros   uint8 [E, n, k / group]      zero points 0 .. 15; None: 8 everywhere

    With a plan, its rows meet their expert's weights: x is [plan.capacity, k], or [T, k] with `by_token`; rows of `out`
    [plan.capacity, n] without a pair stay as they were (in a new matrix: undefined).  Without one, codes, scales and zeros
    are those of a single matrix (no E), and x and out have as many rows as x.
    gated: the weights hold n / 2 linear rows, then n / 2 gated ones, and out [.., n / 2] is silu(gated) * linear.
    x is bfloat16 or float16; n a multiple of 16, k of the group and at most 8192.  The weights are read once per eight
    rows of an expert: for decode batches.

    Equal calls give equal bits.  The order of a sum depends on how many rows the expert has, and on the values, so that a row's
    last bits may differ between batches.  A weight that never arrives (a wait of a second) leaves NaN in the results, and no
    error.  Not differentiable."""
    index = _on_gpu("x", x)
    kind = _row_type("x", x)
    if kind == _lib.FP32:
        raise TypeError("x must be bfloat16 or float16, got torch.float32")
    if _forward_ad._current_level >= 0:
        _no_tangents(x=x, scales=scales)
    if _wants_grad(x) or (isinstance(scales, torch.Tensor) and _wants_grad(scales)):
        raise ValueError("matvec_w4 has no gradient: call it under torch.no_grad()")
    if plan is not None and _check_plan(plan) != index:
        raise ValueError(f"plan must live on {x.device}, got {plan._device}")
    if by_token and plan is None:
        raise ValueError("by_token needs a plan")
    K = x.shape[1]
    E = 1 if plan is None else plan._num_experts
    if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor):
        raise TypeError("codes and scales must be torch.Tensors")
    lead = () if plan is None else (E,)
    if codes.dim() != len(lead) + 2 or scales.dim() != len(lead) + 2:
        raise ValueError(f"codes and scales must have {len(lead) + 2} dimensions{' (one matrix, no plan)' if plan is None else ''}")
    N, G = codes.shape[-2], scales.shape[-1]
    if G < 1 or K % G or K % 2:
        raise ValueError(f"scales of {G} groups do not divide {K} columns")
    rows = x.shape[0] if plan is None else plan._capacity
    if rows >= 1 << 31 or N >= 1 << 31:
        raise ValueError(f"{rows} rows by {N} are too many")
    cp = _packed("codes", codes, torch.uint8, (*lead, N, K // 2), index)
    sp = _packed("scales", scales, x.dtype, (*lead, N, G), index)
    zp = None if zeros is None else _packed("zeros", zeros, torch.uint8, (*lead, N, G), index)
    xp, xs = _matrix("x", x, plan._num_tokens if by_token else rows, K, x.dtype, index)
    columns = N // 2 if gated else N
    fresh = out is None
    if fresh:
        out = torch.empty((rows, columns), dtype=x.dtype, device=x.device)
    else:
        _result("out", out)
    op, os = _matrix("out", out, rows, columns, x.dtype, index)
    _call(_lib.load().moe_fp8_b200_matvec_w4, index, xp, xs, int(by_token), C.byref(_lib.W4(cp, sp, zp, E, N, K, K // G)),
          int(gated), op, os, kind, None if plan is None else plan._c, rows)
    if not fresh:
        _written((out,))
    return out


def _plain_rows(grad):
    # autograd may hand in a broadcast gradient (of a sum, say)
    return grad if grad.stride(1) == 1 else grad.contiguous()


def _same_plan(ctx):
    if ctx.plan._filled != ctx.filled:
        raise RuntimeError("the plan was filled anew since the forward pass: keep one plan per pass")
    return ctx.plan


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan, ctx.filled = plan._for_backward()
        return dispatch(x.detach(), plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_rows):
        return dispatch_backward(_plain_rows(grad_rows), _same_plan(ctx)), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, plan):
        ctx.plan, ctx.filled = plan._for_backward()
        # what neither gradient reads may be written, and freed, before the backward pass
        need_y, need_weights, _ = ctx.needs_input_grad
        ctx.save_for_backward(y if need_weights else None, weights if need_y else None)
        return _combine(y.detach(), weights.detach(), plan, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        y, weights = ctx.saved_tensors
        grad_y, grad_weights = combine_backward(_plain_rows(grad_out), y, weights, _same_plan(ctx),
                                                need_y=ctx.needs_input_grad[0], need_weights=ctx.needs_input_grad[1])
        return grad_y, grad_weights, None
