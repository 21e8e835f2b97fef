"""Operators around the experts of one block: tokens to expert order and back without the hops between
(:func:`expert_sort`, :func:`expert_unsort`), the experts' products on 4-bit weights (:func:`w4_pack`,
:func:`expert_linear_w4`) and what stands between two blocks (:func:`block_norm`).

They have no counterpart in the reference, which leaves them to the layer around it.  As everywhere in ``terrace.ops``
the kernels of the library are the only implementation: a tensor that is not on a ROCm device raises, and every call
enqueues on the current stream of its tensors' device.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import _hip

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_MAX_EXPERTS = 2048
_MAX_WIDTH = 16384


def _ops():
    from .. import ops           # deferred: the package imports this module
    return ops


def _ready(*tensors):
    """The library is loaded and the tensors share one ROCm device, which is returned."""
    _ops()._require()
    _hip.need_device(*tensors)
    given = [t for t in tensors if t is not None]
    dev = given[0].device
    for t in given[1:]:
        if t.device != dev:
            raise RuntimeError(f"terrace: tensors on {dev} and on {t.device} in one call")
    return dev


def _call(dev, name, *args):
    """One library call with ``dev`` current: a kernel is launched from the device its stream belongs to."""
    if dev.index == torch.cuda.current_device():
        _hip.call(name, *args)
    else:
        with torch.cuda.device(dev):
            _hip.call(name, *args)


def _movable_rows(t):
    """``t`` as the row movers take it: packed, or on a kilobyte pitch; else a packed copy."""
    pitch = t.stride(0) * t.element_size() if t.shape[0] > 1 else 0
    if _hip.is_rows(t) and not t.is_contiguous() and pitch % 1024 == 0 and t.data_ptr() % 16 == 0 and \
            (t.shape[1] * t.element_size()) % 16 == 0:
        return t
    return t.contiguous()


def _aligned(t):
    """``t`` packed and on a 16-byte boundary (a copy only when it is not)."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# --------------------------------------------------------------------------------------
# tokens to expert order and back
# --------------------------------------------------------------------------------------

class ExpertPlan(NamedTuple):
    """Where :func:`expert_sort` put each (token, expert) pair."""
    where: torch.Tensor                 # [T, k] int64: its row in expert order, -1 for a pair without an expert
    tokens_per_expert: torch.Tensor     # [n_experts] int64
    offsets: torch.Tensor               # [n_experts + 1] int64: first row of each expert; the last entry counts all pairs
    status: torch.Tensor                # the library's status words: FAULT_ID_RANGE when an id was >= n_experts


def _sort_raw(x, expert_idx, n_experts):
    dev = x.device
    T, k = expert_idx.shape
    x = _movable_rows(x)
    expert_idx = expert_idx.contiguous()
    rows = _hip.empty_rows(T * k, x)
    # the index planes share one allocation: [T*k] places, [n] counts, [n + 1] offsets, 2 words of status
    n = n_experts
    planes = torch.empty((T * k + 2 * n + 3,), dtype=torch.int64, device=dev)
    where, counts, offsets, words = planes.split((T * k, n, n + 1, 2))
    need = _hip.query("terrace_expert_sort_workspace", T, k, n)
    ws = _hip.workspace(need, dev) if need > 256 else None
    base = planes.data_ptr()
    _call(dev, "terrace_expert_sort", x.data_ptr(), expert_idx.data_ptr(), T, _hip.row_arg(x), k, n, rows.data_ptr(), base,
          base + 8 * T * k, base + 8 * (T * k + n), base + 8 * (T * k + 2 * n + 1), _hip.ptr(ws),
          0 if ws is None else ws.numel(), _hip.stream(dev))
    return rows, where.view(T, k), counts, offsets, words.view(torch.int32)


class _ExpertSortFn(torch.autograd.Function):
    """rows[where[t, j]] = x[t]; adjoint: a token sums the gradients of its k rows in column order."""

    @staticmethod
    def forward(ctx, x, expert_idx, n_experts):
        rows, where, counts, offsets, status = _sort_raw(x, expert_idx, n_experts)
        ctx.save_for_backward(where)
        ctx.mark_non_differentiable(where, counts, offsets, status)
        ctx.set_materialize_grads(False)
        ctx.dtype = x.dtype
        return rows, where, counts, offsets, status

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        (where,) = ctx.saved_tensors
        if g is None:
            return None, None, None
        return _ops().combine(g.contiguous(), where, None, out_dtype=ctx.dtype), None, None


def expert_sort(x, expert_idx, n_experts: int):
    """``x`` [T, H] to expert order: ``(rows [T*k, H], plan)`` with ``rows[plan.where[t, j]] = x[t]``.

    ``expert_idx`` [T, k] int64 names the experts of each token (``t_route``'s first result).  The pairs of one expert
    keep their order (token, then column).  An id below 0 is a pair without an expert here -- another rank's, or masked
    -- and one past ``n_experts`` is treated the same and reported in ``plan.status``; such a pair has ``where`` -1, and
    the rows behind the last live one are zeros.  A token may have no expert at all.  ``rows`` carries gradients to ``x``
    (any dtype may be sorted; gradients need a float one).  ``plan.tokens_per_expert`` is what :func:`expert_linear_w4`
    takes, ``plan.where`` what ``combine`` takes.  At most 2048 experts.  Up to 2048 pairs the call is one launch."""
    _ready(x, expert_idx)
    if x.dim() != 2 or expert_idx.dim() != 2 or x.shape[0] != expert_idx.shape[0]:
        raise RuntimeError(f"expert_sort: x {tuple(x.shape)} and expert_idx {tuple(expert_idx.shape)} must be [T, H] "
                           f"and [T, k]")
    if expert_idx.dtype != torch.int64:
        raise RuntimeError("expert_sort: expert_idx must be int64")
    if not 0 < n_experts <= _MAX_EXPERTS or expert_idx.shape[1] < 1:
        raise RuntimeError(f"expert_sort: 1 to {_MAX_EXPERTS} experts and at least one column, got {n_experts} and "
                           f"{expert_idx.shape[1]}")
    if torch.is_grad_enabled() and x.requires_grad:
        rows, *plan = _ExpertSortFn.apply(x, expert_idx, int(n_experts))
    else:
        rows, *plan = _sort_raw(x, expert_idx, int(n_experts))
    return rows, ExpertPlan(*plan)


class _ExpertUnsortFn(torch.autograd.Function):
    """y[t] = sum_j weights[t, j] * rows[where[t, j]]; adjoint: one pass over dy and the rows."""

    @staticmethod
    def forward(ctx, rows, weights, where, offsets, out_dtype):
        rows = rows.contiguous()
        ctx.save_for_backward(rows, weights, where, offsets)
        ctx.set_materialize_grads(False)
        return _ops().combine(rows, where, weights, out_dtype=out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weights, where, offsets = ctx.saved_tensors
        if dy is None:
            return (None,) * 5
        dy = dy.contiguous()
        T, k = where.shape
        want_rows, want_w = ctx.needs_input_grad[0], weights is not None and ctx.needs_input_grad[1]
        d_rows = torch.empty_like(rows) if want_rows else None
        w = None if weights is None else weights.contiguous()
        d_w = torch.empty_like(w) if want_w else None
        _call(rows.device, "terrace_expert_unsort_grad", rows.data_ptr(), _hip.float_code(rows.dtype), dy.data_ptr(),
              _hip.float_code(dy.dtype), where.data_ptr(), _hip.ptr(w), 0 if w is None else _hip.float_code(w.dtype), T, k,
              rows.shape[1], rows.shape[0], offsets.data_ptr() + 8 * (offsets.numel() - 1), _hip.ptr(d_rows),
              _hip.ptr(d_w), _hip.stream(rows.device))
        return d_rows, d_w, None, None, None


def expert_unsort(rows, weights, plan: ExpertPlan, out_dtype=None):
    """The way back: ``y[t] = sum_j weights[t, j] * rows[plan.where[t, j]]``, summed in fp32 in column order and rounded
    once to ``out_dtype`` (default: ``rows.dtype``).

    ``rows`` [T*k, H] float32 / bfloat16 / float16 in the order of ``plan`` (a plan of :func:`expert_sort`),
    ``weights`` [T, k] of any of these types, or None for plain sums.  A pair without an expert contributes nothing and
    a token without any is a zero row, whatever ``rows`` holds behind the live rows.  Carries gradients to ``rows``
    (zeros behind the live rows) and ``weights`` (0 where there is no expert)."""
    dev = _ready(rows, weights, plan.where, plan.offsets)
    where = plan.where
    if rows.dim() != 2 or rows.shape[0] != where.numel():
        raise RuntimeError(f"expert_unsort: rows {tuple(rows.shape)} does not have one row per pair of the plan "
                           f"({where.numel()})")
    if rows.dtype not in _FLOATS or (weights is not None and weights.dtype not in _FLOATS) or \
            (out_dtype or rows.dtype) not in _FLOATS:
        raise RuntimeError("expert_unsort: rows, weights and the result are float32, bfloat16 or float16")
    if weights is not None and weights.shape != where.shape:
        raise RuntimeError(f"expert_unsort: weights {tuple(weights.shape)} must match the plan's {tuple(where.shape)}")
    if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)):
        return _ExpertUnsortFn.apply(rows, weights, where, plan.offsets, out_dtype)
    if dev.index == torch.cuda.current_device():
        return _ops().combine(rows, where, weights, out_dtype=out_dtype)
    with torch.cuda.device(dev):
        return _ops().combine(rows, where, weights, out_dtype=out_dtype)


# --------------------------------------------------------------------------------------
# the experts' products on 4-bit weights
# --------------------------------------------------------------------------------------

class W4Weights:
    """4-bit weights laid out for :func:`expert_linear_w4` by :func:`w4_pack`: ``n_experts`` matrices [N, K] in groups of
    ``group`` along K, for rows of ``dtype``."""

    __slots__ = ("codes", "scales", "zeros", "n_experts", "N", "K", "group", "dtype", "device")

    def __init__(self, codes, scales, zeros, n_experts, N, K, group, dtype):
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.n_experts, self.N, self.K, self.group, self.dtype, self.device = n_experts, N, K, group, dtype, codes.device


def w4_pack(codes, scales, zeros=None) -> W4Weights:
    """Lay 4-bit weights out for :func:`expert_linear_w4`, once per weight; the inputs may be freed afterwards.

    ``codes`` uint8 [E, N, K/2] (or [N, K/2] for one matrix): two codes a byte, even k in the low nibble; ``scales``
    bfloat16 or float16 [E, N, K/group], ``zeros`` uint8 of the same shape holding 0..15, or None for 8 everywhere.
    ``weight = scale * (code - zero)``.  ``group`` is 32, 64 or 128."""
    _ready(codes, scales, zeros)
    if codes.dim() == 2:
        codes, scales = codes.unsqueeze(0), scales.unsqueeze(0)
        zeros = None if zeros is None else zeros.unsqueeze(0)
    if codes.dtype != torch.uint8 or codes.dim() != 3 or scales.dim() != 3 or scales.shape[:2] != codes.shape[:2]:
        raise RuntimeError(f"w4_pack: codes must be uint8 [E, N, K/2] and scales [E, N, K/group], got "
                           f"{codes.dtype} {tuple(codes.shape)} and {tuple(scales.shape)}")
    if scales.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"w4_pack: scales must be bfloat16 or float16, got {scales.dtype}")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise RuntimeError("w4_pack: zeros must be a uint8 plane of the scales' shape")
    E, N, half = codes.shape
    K = 2 * half
    group = K // scales.shape[2] if scales.shape[2] else 0
    if group not in (32, 64, 128) or group * scales.shape[2] != K:
        raise RuntimeError(f"w4_pack: {scales.shape[2]} groups over K={K}: groups of 32, 64 or 128 are taken")
    dev = codes.device
    sizes = [_hip.query("terrace_w4_packed_bytes", E, N, K, group, what) for what in range(3)]
    if not sizes[0]:
        raise RuntimeError(f"w4_pack: {E} matrices of {N} x {K} are not taken")
    codes, scales = codes.contiguous(), scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    out_codes = torch.empty((sizes[0],), dtype=torch.uint8, device=dev)
    out_scales = torch.empty((sizes[1] // 2,), dtype=scales.dtype, device=dev)
    out_zeros = None if zeros is None else torch.empty((sizes[2],), dtype=torch.uint8, device=dev)
    _call(dev, "terrace_w4_pack", codes.data_ptr(), scales.data_ptr(), _hip.ptr(zeros), _hip.float_code(scales.dtype), E, N, K,
          group, out_codes.data_ptr(), out_scales.data_ptr(), _hip.ptr(out_zeros), _hip.stream(dev))
    return W4Weights(out_codes, out_scales, out_zeros, E, N, K, group, scales.dtype)


def expert_linear_w4(rows, tokens_per_expert, weights: W4Weights, swiglu: bool = False):
    """``out[i] = W[e] rows[i]`` for the rows ``i`` of expert ``e``: [P, N], or with ``swiglu`` the [P, N/2] product
    ``silu(a[:, :N/2]) * a[:, N/2:]`` of its halves, taken before the one rounding.

    ``rows`` [P, K] of the weights' dtype in expert order and ``tokens_per_expert`` [E] int64 as :func:`expert_sort`,
    ``hopb_scatter`` and ``regroup`` (drop-less) give them; None with a single matrix: all rows are its rows.  Rows past
    the last expert's give zero rows.  Made for serving, where an expert holds a few rows: the weights are read once per
    16, 32 or 64 rows of an expert.  No gradients: a call that would need them raises."""
    w = weights
    dev = _ready(rows, tokens_per_expert, w.codes)
    if rows.dim() != 2 or rows.shape[1] != w.K or rows.dtype != w.dtype:
        raise RuntimeError(f"expert_linear_w4: rows must be {w.dtype} [P, {w.K}], got {rows.dtype} {tuple(rows.shape)}")
    if tokens_per_expert is None:
        if w.n_experts != 1:
            raise RuntimeError(f"expert_linear_w4: tokens_per_expert is needed with {w.n_experts} experts")
    elif tokens_per_expert.dtype != torch.int64 or tuple(tokens_per_expert.shape) != (w.n_experts,):
        raise RuntimeError(f"expert_linear_w4: tokens_per_expert must be int64 [{w.n_experts}], got "
                           f"{tokens_per_expert.dtype} {tuple(tokens_per_expert.shape)}")
    if swiglu and w.N % 2:
        raise RuntimeError(f"expert_linear_w4: swiglu needs an even number of columns, got {w.N}")
    if rows.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("expert_linear_w4: forward only (4-bit weights are for serving); call it under no_grad")
    rows = _aligned(rows)
    counts = None if tokens_per_expert is None else tokens_per_expert.contiguous()
    P = rows.shape[0]
    out = torch.empty((P, w.N // 2 if swiglu else w.N), dtype=w.dtype, device=dev)
    _call(dev, "terrace_w4_linear", rows.data_ptr(), _hip.float_code(w.dtype), P, _hip.ptr(counts), w.codes.data_ptr(),
          w.scales.data_ptr(), _hip.ptr(w.zeros), w.n_experts, w.N, w.K, w.group, int(swiglu), out.data_ptr(),
          _hip.stream(dev))
    return out


# --------------------------------------------------------------------------------------
# between two blocks
# --------------------------------------------------------------------------------------

def _norm_vectors(post_weight, gate, pre_weight, kind):
    """The (pointer, dtype) arguments of the three vectors, the gate's kind after its own."""
    def one(v):
        return (None, 0) if v is None else (v.data_ptr(), _hip.float_code(v.dtype))
    return (*one(post_weight), *one(gate), kind, *one(pre_weight))


def _norm_forward(y, residual, post_weight, gate, kind, pre_weight, scale, eps, want_stats):
    """(h or None, n or None, stats or None) of 2-D packed inputs."""
    dev = residual.device
    T, H = residual.shape
    y_dtype = residual.dtype if y is None else y.dtype
    h = None if y is None else torch.empty_like(residual)
    n = None if pre_weight is None else torch.empty((T, H), dtype=y_dtype, device=dev)
    stats = torch.empty((T, 2), dtype=torch.float32, device=dev) if want_stats else None
    _call(dev, "terrace_block_norm", _hip.ptr(y), _hip.float_code(y_dtype), residual.data_ptr(),
          _hip.float_code(residual.dtype), *_norm_vectors(post_weight, gate, pre_weight, kind), scale, eps, T, H,
          _hip.ptr(h), _hip.ptr(n), _hip.ptr(stats), _hip.stream(dev))
    return h, n, stats


class _BlockNormFn(torch.autograd.Function):
    """(h, n) of :func:`block_norm` on 2-D packed inputs; h or n is None where it is not made."""

    @staticmethod
    def forward(ctx, y, residual, post_weight, gate, pre_weight, kind, scale, eps):
        h, n, stats = _norm_forward(y, residual, post_weight, gate, kind, pre_weight, scale, eps, True)
        ctx.save_for_backward(y, residual, post_weight, gate, pre_weight, stats)
        ctx.set_materialize_grads(False)
        ctx.norm = (kind, scale, eps)
        return h, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dn):
        y, residual, post_weight, gate, pre_weight, stats = ctx.saved_tensors
        kind, scale, eps = ctx.norm
        dev = residual.device
        T, H = residual.shape
        dh, dn = _aligned(dh), _aligned(dn)
        wanted = [torch.empty_like(t) if t is not None and need else None
                  for t, need in zip((y, residual, post_weight, gate, pre_weight), ctx.needs_input_grad)]
        d_y, d_residual, d_post, d_gate, d_pre = wanted
        y_dtype = residual.dtype if y is None else y.dtype
        need = d_post is not None or d_pre is not None or (d_gate is not None and kind == _hip.GATE_CHANNEL)
        ws = _hip.workspace(_hip.query("terrace_block_norm_grad_workspace", T, H), dev) if need else None
        _call(dev, "terrace_block_norm_grad", _hip.ptr(y), _hip.float_code(y_dtype), residual.data_ptr(),
              _hip.float_code(residual.dtype), *_norm_vectors(post_weight, gate, pre_weight, kind), scale, eps, T, H,
              stats.data_ptr(), _hip.ptr(dh), _hip.ptr(dn), *(_hip.ptr(t) for t in wanted), _hip.ptr(ws),
              0 if ws is None else ws.numel(), _hip.stream(dev))
        return d_y, d_residual, d_post, d_gate, d_pre, None, None, None


def block_norm(y, residual, post_weight=None, gate=None, pre_weight=None, *, scale: float = 1.0, eps: float = 1e-6):
    """What stands between two blocks, in one pass: ``(h, n)`` with

        p = y / rms(y) * post_weight          (the norm after a block; ``post_weight`` None: p = y)
        h = residual + scale * gate * p       (``gate`` [H] per channel or [..., 1] per token; None: 1)
        n = h / rms(h) * pre_weight           (the norm before the next block; ``pre_weight`` None: n is None)

    and ``rms(v) = sqrt(mean(v^2) + eps)``.  ``y`` and ``residual`` are [..., H] of one shape, float32, bfloat16 or float16;
    the residual may be float32 beside a 16-bit ``y``.  ``h`` has the residual's dtype, ``n`` has ``y``'s; all arithmetic is
    fp32 and each output is rounded once (``n`` comes from the unrounded ``h``).  ``y`` None is the entry of the first
    block: ``h`` is ``residual`` itself and ``n`` its norm.  Carries gradients to all five tensors.  H is at most 16384."""
    dev = _ready(y, residual, post_weight, gate, pre_weight)
    shape = residual.shape
    if residual.dim() < 1 or (y is not None and y.shape != shape):
        raise RuntimeError(f"block_norm: y and residual must have one shape [..., H], got "
                           f"{None if y is None else tuple(y.shape)} and {tuple(shape)}")
    if y is None and (post_weight is not None or gate is not None):
        raise RuntimeError("block_norm: post_weight and gate need a y")
    H = shape[-1]
    if any(t is not None and t.dtype not in _FLOATS for t in (y, residual, post_weight, gate, pre_weight)) or \
            (y is not None and residual.dtype not in (y.dtype, torch.float32)):
        raise RuntimeError("block_norm: float32, bfloat16 or float16; the residual of y's dtype or float32")
    if not 0 < H <= _MAX_WIDTH:
        raise RuntimeError(f"block_norm: rows of {H} elements; 1 to {_MAX_WIDTH} are taken")
    for name, v in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if v is not None and tuple(v.shape) != (H,):
            raise RuntimeError(f"block_norm: {name} must be [{H}], got {tuple(v.shape)}")
    kind = _hip.GATE_NONE
    if gate is not None:
        if tuple(gate.shape) == (H,):
            kind = _hip.GATE_CHANNEL
        elif gate.shape == shape[:-1] + (1,):
            kind = _hip.GATE_TOKEN
        else:
            raise RuntimeError(f"block_norm: gate must be [{H}] or {list(shape[:-1]) + [1]}, got {tuple(gate.shape)}")
    scale, eps = float(scale), float(eps)
    if y is None and pre_weight is None:
        return residual, None
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                           for t in (y, residual, post_weight, gate, pre_weight))
    flat = residual.dim() != 2
    y2 = y.reshape(-1, H) if flat and y is not None else y
    r2 = residual.reshape(-1, H) if flat else residual
    g2 = gate.reshape(-1, 1) if flat and kind == _hip.GATE_TOKEN else gate
    args = [_aligned(t) for t in (y2, r2, post_weight, g2, pre_weight)]
    if grad:
        h, n = _BlockNormFn.apply(*args, kind, scale, eps)
    else:
        h, n, _ = _norm_forward(args[0], args[1], args[2], args[3], kind, args[4], scale, eps, False)
    h = residual if y is None else h
    if flat:
        h, n = h.reshape(shape), None if n is None else n.reshape(shape)
    return h, n
