"""Operators around the experts of one block: tokens to expert order and back without the hops between
(:func:`expert_sort`, :func:`expert_unsort`), the experts' products on 4-bit weights (:func:`w4_pack`,
:func:`expert_linear_w4`) and what stands between two blocks (:func:`block_norm`).

They have no counterpart in the reference, which leaves them to the layer around it.  As everywhere in ``terrace.ops``
the kernels of the library are the only implementation: a tensor that is not on a ROCm device raises, and every call
enqueues on the current stream of its tensors' device.  Gradients are those of reverse mode; a tensor with a forward-mode
tangent raises.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _hip
from .. import ops as _ops

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_CODE = {torch.float32: _hip.F32, torch.bfloat16: _hip.BF16, torch.float16: _hip.F16}
_MAX_EXPERTS = 2048
_MAX_WIDTH = 16384
_MAX_GRAD_TOKENS = (1 << 24) - 1025          # one workgroup a token and 1024 for the rows of none, below 2^32 threads
_CURRENT = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _ready(*tensors) -> int:
    """The library is loaded and the tensors (None: absent) share one ROCm device, whose index is returned; none carries
    a forward-mode tangent."""
    _ops._require()
    _hip.refuse_tangents(*tensors)
    index = -1
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            _hip.need_device(t)
        at = t.get_device()
        if index < 0:
            index = at
        elif at != index:
            raise RuntimeError(f"terrace: tensors on cuda:{index} and on cuda:{at} in one call")
    return index


def _enqueue(index: int, name: str, *args):
    """One library call on the current stream of device ``index``, with that device current: a kernel is launched from
    the device its stream belongs to."""
    if index == _CURRENT():
        _hip.call(name, *args, _hip.raw_stream(index))
    else:
        with torch.cuda.device(index):
            _hip.call(name, *args, _hip.raw_stream(index))


def _at(t):
    """Address of a tensor for an argument that may be absent."""
    return None if t is None else t.data_ptr()


def _movable_rows(t):
    """``t`` as the row movers take it: packed, or on a kilobyte pitch; else a packed copy."""
    if t.is_contiguous():
        return t
    pitch = t.stride(0) * t.element_size() if t.shape[0] > 1 else 0
    if _hip.is_rows(t) and pitch % 1024 == 0 and t.data_ptr() % 16 == 0 and (t.shape[1] * t.element_size()) % 16 == 0:
        return t
    return t.contiguous()


def _aligned(t):
    """``t`` packed and on a 16-byte boundary (a copy only when it is not)."""
    if t is None:
        return None
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# --------------------------------------------------------------------------------------
# tokens to expert order and back
# --------------------------------------------------------------------------------------

class ExpertPlan:
    """Where :func:`expert_sort` put each (token, expert) pair.  The planes share one allocation and become tensors of
    their own when first read:

    ``where``              [T, k] int64: the pair's row in expert order, -1 for a pair without an expert
    ``tokens_per_expert``  [n_experts] int64
    ``offsets``            [n_experts + 1] int64: first row of each expert; the last entry counts the pairs with one
    ``status``             the library's status words: FAULT_ID_RANGE when an id was >= n_experts"""

    __slots__ = ("planes", "T", "k", "n_experts", "_made")

    def __init__(self, planes, T, k, n_experts):
        if planes.dtype != torch.int64 or planes.numel() != self.words(T, k, n_experts) or not planes.is_contiguous():
            raise RuntimeError("ExpertPlan: the planes do not match the geometry")
        self.planes, self.T, self.k, self.n_experts, self._made = planes, T, k, n_experts, {}

    @staticmethod
    def words(T, k, n_experts):
        """int64 words of the planes: places, counts, offsets, status."""
        return T * k + 2 * n_experts + 3

    def _plane(self, name, lo, n):
        t = self._made.get(name)
        if t is None:
            t = self._made[name] = self.planes[lo:lo + n]
        return t

    @property
    def where(self):
        return self._plane("where", 0, self.T * self.k).view(self.T, self.k)

    @property
    def tokens_per_expert(self):
        return self._plane("tokens_per_expert", self.T * self.k, self.n_experts)

    @property
    def offsets(self):
        return self._plane("offsets", self.T * self.k + self.n_experts, self.n_experts + 1)

    @property
    def status(self):
        return self._plane("status", self.T * self.k + 2 * self.n_experts + 1, 2).view(torch.int32)


def _sort_raw(index, x, expert_idx, planes, T, k, n):
    x = _movable_rows(x)
    expert_idx = expert_idx.contiguous()
    if x.is_contiguous():
        rows, row_bytes = torch.empty((T * k, x.shape[1]), dtype=x.dtype, device=x.device), x.shape[1] * x.element_size()
    else:
        rows, row_bytes = _hip.empty_rows(T * k, x), _hip.row_arg(x)
    need = _hip.query("terrace_expert_sort_workspace", T, k, n)
    ws = _hip.workspace(need, x.device) if need > 256 else None      # 256: the one-launch form, which needs none
    base = planes.data_ptr()
    counts = base + 8 * T * k
    src, dst = (x.data_ptr(), rows.data_ptr()) if rows.numel() else (None, None)
    _enqueue(index, "terrace_expert_sort", src, expert_idx.data_ptr(), T, row_bytes, k, n, dst, base, counts,
             counts + 8 * n, counts + 8 * (2 * n + 1), _at(ws), need if ws is not None else 0)
    return rows


def _combine(index, rows, where_at, weights, T, k, out_dtype):
    """The combine over the [T, k] places at address ``where_at``: rows packed, weights packed or None."""
    out = torch.empty((T, rows.shape[1]), dtype=out_dtype, device=rows.device)
    _enqueue(index, "terrace_combine", rows.data_ptr(), rows.shape[0], _CODE[rows.dtype], where_at, _at(weights),
             0 if weights is None else _CODE[weights.dtype], T, k, rows.shape[1], out.data_ptr(), _CODE[out_dtype])
    return out


class _ExpertSortFn(torch.autograd.Function):
    """rows[where[t, j]] = x[t]; adjoint: a token sums the gradients of its k rows in column order."""

    @staticmethod
    def forward(ctx, x, expert_idx, planes, T, k, n):
        ctx.save_for_backward(planes)
        ctx.geom = (T, k, x.dtype)
        return _sort_raw(x.get_device(), x, expert_idx, planes, T, k, n)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        _hip.refuse_tangents(g)
        (planes,) = ctx.saved_tensors
        T, k, dtype = ctx.geom
        return _combine(g.get_device(), g.contiguous(), planes.data_ptr(), None, T, k, dtype), None, None, None, None, None


def expert_sort(x, expert_idx, n_experts: int):
    """``x`` [T, H] to expert order: ``(rows [T*k, H], plan)`` with ``rows[plan.where[t, j]] = x[t]``.

    ``expert_idx`` [T, k] int64 names the experts of each token (``t_route``'s first result).  The pairs of one expert
    keep their order (token, then column).  An id below 0 is a pair without an expert here -- another rank's, or masked
    -- and one past ``n_experts`` is treated the same and reported in ``plan.status``; such a pair has ``where`` -1, and
    the rows behind the last live one are zeros.  A token may have no expert at all.  ``rows`` carries gradients to ``x``
    (any dtype may be sorted; gradients need float32, bfloat16 or float16).  ``plan.tokens_per_expert`` is what
    :func:`expert_linear_w4` takes, ``plan.where`` what ``combine`` takes.  At most 2048 experts.  Up to 2048 pairs (4096
    over at most 1024 tokens) the call is one launch."""
    index = _ready(x, expert_idx)
    if x.dim() != 2 or expert_idx.dim() != 2 or x.shape[0] != expert_idx.shape[0]:
        raise RuntimeError(f"expert_sort: x {tuple(x.shape)} and expert_idx {tuple(expert_idx.shape)} must be [T, H] "
                           f"and [T, k]")
    if expert_idx.dtype != torch.int64:
        raise RuntimeError("expert_sort: expert_idx must be int64")
    T, k = expert_idx.shape
    n = int(n_experts)
    if not 0 < n <= _MAX_EXPERTS or k < 1:
        raise RuntimeError(f"expert_sort: 1 to {_MAX_EXPERTS} experts and at least one column, got {n} and {k}")
    planes = torch.empty((ExpertPlan.words(T, k, n),), dtype=torch.int64, device=x.device)
    if x.requires_grad and torch.is_grad_enabled():
        if x.dtype not in _FLOATS:
            raise RuntimeError(f"expert_sort: gradients need float32, bfloat16 or float16 rows, got {x.dtype}")
        rows = _ExpertSortFn.apply(x, expert_idx, planes, T, k, n)
    else:
        rows = _sort_raw(index, x, expert_idx, planes, T, k, n)
    return rows, ExpertPlan(planes, T, k, n)


class _ExpertUnsortFn(torch.autograd.Function):
    """y[t] = sum_j weights[t, j] * rows[where[t, j]]; adjoint: one pass over dy and the rows."""

    @staticmethod
    def forward(ctx, rows, weights, planes, T, k, n, out_dtype):
        ctx.save_for_backward(rows, weights, planes)
        ctx.geom = (T, k, n)
        return _combine(rows.get_device(), rows, planes.data_ptr(), weights, T, k, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _hip.refuse_tangents(dy)
        rows, weights, planes = ctx.saved_tensors
        T, k, n = ctx.geom
        dy = dy.contiguous()
        d_rows = torch.empty_like(rows) if ctx.needs_input_grad[0] else None
        d_w = torch.empty_like(weights) if weights is not None and ctx.needs_input_grad[1] else None
        where = planes.data_ptr()
        _enqueue(rows.get_device(), "terrace_expert_unsort_grad", rows.data_ptr(), _CODE[rows.dtype], dy.data_ptr(),
                 _CODE[dy.dtype], where, _at(weights), 0 if weights is None else _CODE[weights.dtype], T, k, rows.shape[1],
                 rows.shape[0], where + 8 * (T * k + 2 * n), _at(d_rows), _at(d_w))
        return d_rows, d_w, None, None, None, None, None


def expert_unsort(rows, weights, plan: ExpertPlan, out_dtype=None):
    """The way back: ``y[t] = sum_j weights[t, j] * rows[plan.where[t, j]]``, summed in fp32 in column order and rounded
    once to ``out_dtype`` (default: ``rows.dtype``).

    ``rows`` [T*k, H] float32 / bfloat16 / float16 in the order of ``plan`` (a plan of :func:`expert_sort`),
    ``weights`` [T, k] of any of these types, or None for plain sums.  A pair without an expert contributes nothing and
    a token without any is a zero row, whatever ``rows`` holds behind the live rows.  Carries gradients to ``rows``
    (zeros behind the live rows) and ``weights`` (0 where there is no expert), for up to 2^24 - 1025 tokens."""
    index = _ready(rows, weights, plan.planes)
    T, k = plan.T, plan.k
    out_dtype = out_dtype or rows.dtype
    if rows.dim() != 2 or rows.shape[0] != T * k:
        raise RuntimeError(f"expert_unsort: rows {tuple(rows.shape)} does not have one row per pair of the plan ({T * k})")
    if rows.dtype not in _CODE or out_dtype not in _CODE or (weights is not None and weights.dtype not in _CODE):
        raise RuntimeError("expert_unsort: rows, weights and the result are float32, bfloat16 or float16")
    if weights is not None and weights.shape != (T, k):
        raise RuntimeError(f"expert_unsort: weights {tuple(weights.shape)} must match the plan's {(T, k)}")
    rows = rows.contiguous()
    weights = None if weights is None else weights.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)):
        if T > _MAX_GRAD_TOKENS:
            raise RuntimeError(f"expert_unsort: gradients for up to {_MAX_GRAD_TOKENS} tokens, got {T}")
        return _ExpertUnsortFn.apply(rows, weights, plan.planes, T, k, plan.n_experts, out_dtype)
    return _combine(index, rows, plan.planes.data_ptr(), weights, T, k, out_dtype)


# --------------------------------------------------------------------------------------
# the experts' products on 4-bit weights
# --------------------------------------------------------------------------------------

class W4Weights:
    """4-bit weights laid out for :func:`expert_linear_w4` by :func:`w4_pack`: ``n_experts`` matrices [N, K] in groups of
    ``group`` along K, for rows of ``dtype``.

    To store them, keep the planes ``codes``, ``scales`` and ``zeros`` (None: 8 everywhere) with the five numbers and the
    dtype, and hand them to the constructor again; the layout is this build's own.  The planes are checked against the
    numbers by the first product after any attribute was set; resizing a plane's storage behind it is not seen."""

    __slots__ = ("codes", "scales", "zeros", "n_experts", "N", "K", "group", "dtype", "device", "_sound")

    def __init__(self, codes, scales, zeros, n_experts, N, K, group, dtype):
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.n_experts, self.N, self.K, self.group, self.dtype, self.device = n_experts, N, K, group, dtype, codes.device

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        object.__setattr__(self, "_sound", False)

    def check(self):
        """Raises RuntimeError unless the planes are what :func:`w4_pack` lays out for these sizes."""
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError(f"W4Weights: bfloat16 or float16, got {self.dtype}")
        planes = (("codes", self.codes, torch.uint8, 1, 16), ("scales", self.scales, self.dtype, 2, 8),
                  ("zeros", self.zeros, torch.uint8, 1, 8))
        for what, (name, t, dtype, width, boundary) in enumerate(planes):
            if t is None and name == "zeros":
                continue
            need = _hip.query("terrace_w4_packed_bytes", self.n_experts, self.N, self.K, self.group, what)
            if not need:
                raise RuntimeError(f"W4Weights: {self.n_experts} matrices of {self.N} x {self.K} in groups of {self.group} are "
                                   f"not taken")
            if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.numel() * width != need or not t.is_contiguous() or \
                    t.device != self.device or t.data_ptr() % boundary:
                raise RuntimeError(f"W4Weights: {name} must hold {need} bytes of {dtype}, packed, on {self.device} and a "
                                   f"{boundary}-byte boundary, as w4_pack lays them out")
        object.__setattr__(self, "_sound", True)


def w4_pack(codes, scales, zeros=None) -> W4Weights:
    """Lay 4-bit weights out for :func:`expert_linear_w4`, once per weight; the inputs may be freed afterwards.

    ``codes`` uint8 [E, N, K/2] (or [N, K/2] for one matrix): two codes a byte, even k in the low nibble; ``scales``
    bfloat16 or float16 [E, N, K/group], ``zeros`` uint8 of the same shape (the low four bits count), or None for 8
    everywhere.
    ``weight = scale * (code - zero)``.  ``group`` is 32, 64 or 128."""
    index = _ready(codes, scales, zeros)
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
    _enqueue(index, "terrace_w4_pack", codes.data_ptr(), scales.data_ptr(), _at(zeros), _CODE[scales.dtype], E, N, K, group,
             out_codes.data_ptr(), out_scales.data_ptr(), _at(out_zeros))
    return W4Weights(out_codes, out_scales, out_zeros, E, N, K, group, scales.dtype)


def expert_linear_w4(rows, tokens_per_expert, weights: W4Weights, swiglu: bool = False):
    """``out[i] = W[e] rows[i]`` for the rows ``i`` of expert ``e``: [P, N], or with ``swiglu`` the [P, N/2] product
    ``silu(a[:, :N/2]) * a[:, N/2:]`` of its halves, taken before the one rounding.

    ``rows`` [P, K] of the weights' dtype in expert order and ``tokens_per_expert`` [E] int64 as :func:`expert_sort`,
    ``hopb_scatter`` and ``regroup`` (drop-less) give them; None with a single matrix: all rows are its rows.  Rows past
    the last expert's give zero rows.  Infinities, NaN and very large values in a row give what the sum gives; a row
    with an infinity takes some hundred times as long.  Made for serving, where an expert holds a few rows: the weights are read once per
    16, 32 or 64 rows of an expert.  At most 2^30 rows; refused is also a launch of 2^32 threads, which takes some hundred
    thousand experts of a few rows each (``include/terrace_hip.h`` has the sum).  No gradients: a call that would need them
    raises."""
    w = weights
    index = _ready(rows, tokens_per_expert, w.codes)
    if not w._sound:
        w.check()
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
    out = torch.empty((P, w.N // 2 if swiglu else w.N), dtype=w.dtype, device=w.device)
    _enqueue(index, "terrace_w4_linear", rows.data_ptr(), _CODE[w.dtype], P, _at(counts), w.codes.data_ptr(),
             w.scales.data_ptr(), _at(w.zeros), w.n_experts, w.N, w.K, w.group, 1 if swiglu else 0, out.data_ptr())
    return out


# --------------------------------------------------------------------------------------
# between two blocks
# --------------------------------------------------------------------------------------

def _norm_inputs(y, residual, post_weight, gate, kind, pre_weight, scale, eps, T, H):
    """The arguments that the two entry points share."""
    y_code = _CODE[residual.dtype if y is None else y.dtype]
    return (_at(y), y_code, residual.data_ptr(), _CODE[residual.dtype],
            _at(post_weight), 0 if post_weight is None else _CODE[post_weight.dtype],
            _at(gate), 0 if gate is None else _CODE[gate.dtype], kind,
            _at(pre_weight), 0 if pre_weight is None else _CODE[pre_weight.dtype], scale, eps, T, H)


def _norm_forward(y, residual, post_weight, gate, kind, pre_weight, scale, eps, want_stats):
    """(h or None, n or None, stats or None) of 2-D packed inputs."""
    T, H = residual.shape
    h = None if y is None else torch.empty_like(residual)
    n = None if pre_weight is None else torch.empty_like(residual if y is None else y)
    stats = torch.empty((T, 2), dtype=torch.float32, device=residual.device) if want_stats else None
    _enqueue(residual.get_device(), "terrace_block_norm",
             *_norm_inputs(y, residual, post_weight, gate, kind, pre_weight, scale, eps, T, H), _at(h), _at(n), _at(stats))
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
        _hip.refuse_tangents(dh, dn)
        y, residual, post_weight, gate, pre_weight, stats = ctx.saved_tensors
        kind, scale, eps = ctx.norm
        T, H = residual.shape
        dh, dn = _aligned(dh), _aligned(dn)
        wanted = [torch.empty_like(t) if need and t is not None else None
                  for t, need in zip((y, residual, post_weight, gate, pre_weight), ctx.needs_input_grad)]
        ws, need = None, 0
        if wanted[2] is not None or wanted[4] is not None or (wanted[3] is not None and kind == _hip.GATE_CHANNEL):
            need = _hip.query("terrace_block_norm_grad_workspace", T, H)
            ws = _hip.workspace(need, residual.device)
        _enqueue(residual.get_device(), "terrace_block_norm_grad",
                 *_norm_inputs(y, residual, post_weight, gate, kind, pre_weight, scale, eps, T, H), stats.data_ptr(), _at(dh),
                 _at(dn), *(_at(t) for t in wanted), _at(ws), need)
        return (*wanted, None, None, None)


def block_norm(y, residual, post_weight=None, gate=None, pre_weight=None, *, scale: float = 1.0, eps: float = 1e-6):
    """What stands between two blocks, in one pass: ``(h, n)`` with

        p = y / rms(y) * post_weight          (the norm after a block; ``post_weight`` None: p = y)
        h = residual + scale * gate * p       (``gate`` [H] per channel or [..., 1] per token; None: 1)
        n = h / rms(h) * pre_weight           (the norm before the next block; ``pre_weight`` None: n is None)

    and ``rms(v) = sqrt(mean(v^2) + eps)``.  ``y`` and ``residual`` are [..., H] of one shape, float32, bfloat16 or float16;
    the residual may be float32 beside a 16-bit ``y``.  ``h`` has the residual's dtype, ``n`` has ``y``'s; all arithmetic is
    fp32 and each output is rounded once (``n`` comes from the unrounded ``h``).  ``y`` None is the entry of the first
    block: ``h`` is ``residual`` itself and ``n`` its norm.  Carries gradients to all five tensors.  H is at most 16384."""
    tensors = (y, residual, post_weight, gate, pre_weight)
    _ready(*tensors)
    shape = residual.shape
    if residual.dim() < 1 or (y is not None and y.shape != shape):
        raise RuntimeError(f"block_norm: y and residual must have one shape [..., H], got "
                           f"{None if y is None else tuple(y.shape)} and {tuple(shape)}")
    if y is None and (post_weight is not None or gate is not None):
        raise RuntimeError("block_norm: post_weight and gate need a y")
    H = shape[-1]
    grad = False
    for t in tensors:
        if t is not None:
            if t.dtype not in _CODE:
                raise RuntimeError(f"block_norm: float32, bfloat16 or float16, got {t.dtype}")
            grad = grad or t.requires_grad
    if y is not None and residual.dtype != y.dtype and residual.dtype != torch.float32:
        raise RuntimeError(f"block_norm: the residual has y's dtype or float32, got {residual.dtype} beside {y.dtype}")
    if not 0 < H <= _MAX_WIDTH:
        raise RuntimeError(f"block_norm: rows of {H} elements; 1 to {_MAX_WIDTH} are taken")
    if post_weight is not None and post_weight.shape != (H,):
        raise RuntimeError(f"block_norm: post_weight must be [{H}], got {tuple(post_weight.shape)}")
    if pre_weight is not None and pre_weight.shape != (H,):
        raise RuntimeError(f"block_norm: pre_weight must be [{H}], got {tuple(pre_weight.shape)}")
    kind = _hip.GATE_NONE
    if gate is not None:
        if gate.shape == (H,):
            kind = _hip.GATE_CHANNEL
        elif gate.shape == shape[:-1] + (1,):
            kind = _hip.GATE_TOKEN
        else:
            raise RuntimeError(f"block_norm: gate must be [{H}] or {list(shape[:-1]) + [1]}, got {tuple(gate.shape)}")
    if y is None and pre_weight is None:
        return residual, None
    scale, eps = float(scale), float(eps)
    flat = len(shape) != 2
    y2 = y.reshape(-1, H) if flat and y is not None else y
    r2 = residual.reshape(-1, H) if flat else residual
    g2 = gate.reshape(-1, 1) if flat and kind == _hip.GATE_TOKEN else gate
    y2, r2, w_post, g2, w_pre = _aligned(y2), _aligned(r2), _aligned(post_weight), _aligned(g2), _aligned(pre_weight)
    if grad and torch.is_grad_enabled():
        h, n = _BlockNormFn.apply(y2, r2, w_post, g2, w_pre, kind, scale, eps)
    else:
        h, n, _ = _norm_forward(y2, r2, w_post, g2, kind, w_pre, scale, eps, False)
    h = residual if y is None else h
    if flat:
        h, n = h.reshape(shape), None if n is None else n.reshape(shape)
    return h, n
