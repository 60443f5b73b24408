"""Dense feed-forward operators in 16 bits: what a mixture-of-experts model computes beside its routed experts (dense layers, an
always-on expert that the checkpoint keeps in bf16 or fp16), forward and backward.

``gated_linear``  both projections, the activation and the product in one kernel; weight order and activations are the routed
                  layer's (``w13``: gate rows, then up rows; SwiGLU with its limit, or SiTU)
``fused_linear``  a projection with bias, activation and residual in its epilogue

Tensors are bf16 or fp16, one type per call, on one GPU; sums are fp32 and rounded once. Rows may have any pitch, the values of a
row must be neighbours; x and weights whose rows do not start on 16 bytes are copied to rows that do, within the call. Calls run
on the current stream, allocate through torch only, and may be captured.

Called with gradients enabled and an input that requires one, the two operators record themselves for ``backward()``; that
form cannot be captured into a CUDA graph (capture the forward call with ``return_preact=True`` and ``*_backward`` instead, which
record nothing). The backward pass rounds the gradient of the pre-activations to the type once, as its products' operand: in
fp16 that is 0 below 3e-8 and infinite beyond 65504, so losses are scaled as for any fp16 training. Forward-mode differentiation is not offered: a tensor with a tangent is refused.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from .. import native_runtime as nr
from ._dispatch import OpNotEligible
from .moe_fused_mxfp4 import SITU, SWIGLU

_DTYPE = {torch.bfloat16: 0, torch.float16: 1}
_LINEAR_ACT = {None: 0, "none": 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}
# tokens, inputs, weight rows that the kernels take
_MOST = 2 ** 27

_entries = {}


def _entry(name):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(nr.load_library(), name)
    return fn


# the handle alone: a Stream object around it costs a microsecond of a decode step's dozen
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name, index, *args):
    """The C entry on the current stream of device `index`, which becomes the current device for the call."""
    if index == torch.cuda.current_device():
        rc = _entry(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = _entry(name)(*args, _raw_stream(index))
    if rc:
        nr.check(rc, name)


def _matrix(t, shape, dtype, index):
    """The row pitch of a matrix that is just what the kernels read (this shape and type, this device, rows of neighbours), else 0."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == index:
        row, step = t.stride()
        if step == 1:
            if shape[0] == 1:
                return shape[1] + 7 & -8
            if row >= shape[1]:
                return row
    return 0


def _vector(t, n, dtype, index):
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == (n,) and t.get_device() == index and t.is_contiguous()


def _check_tensor(name, t):
    if not isinstance(t, torch.Tensor):
        raise OpNotEligible(f"{name} must be a tensor")


def _check(name, t, dtype, index):
    _check_tensor(name, t)
    if t.dtype is not dtype:
        raise OpNotEligible(f"{name} must be {dtype}, like the other tensors of the call, got {t.dtype}")
    if t.get_device() != index:
        raise OpNotEligible(f"{name} must be on the device of x, got {t.device}")


def _pitch(name, t):
    """Elements from one row of a 2-D tensor to the next."""
    T, n = t.shape
    row, step = t.stride()
    if T > 0 and n > 1 and step != 1:      # (of no rows, an expanded gradient has any)
        raise OpNotEligible(f"the values of a row of {name} must be neighbours in memory")
    if T <= 1:
        return (n + 7) // 8 * 8
    if row < n:
        raise OpNotEligible(f"the rows of {name} must not overlap")
    return row


def _span(t):
    """First byte and the one behind the last of a tensor's memory."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _apart(name, out, others):
    a, b = _span(out)
    for other_name, t in others:
        if t is not None:
            c, d = _span(t)
            if a < d and c < b and not _side_by_side(out, a, t, c):
                raise OpNotEligible(f"{name} must not overlap {other_name}")


def require_apart(name, out, *others):
    """Refuses a tensor `out`, called `name`, that shares memory with any of the others: pairs of a name and a tensor or None."""
    _check_tensor(name, out)
    for other_name, t in others:
        if t is not None:
            _check_tensor(other_name, t)
    _apart(name, out, others)


def _side_by_side(t, a, u, c):
    """Whether two matrices are different columns of one wider one."""
    if t.dim() != 2 or u.dim() != 2 or t.stride() != u.stride() or t.stride(1) != 1:
        return False
    pitch, gap = t.stride(0), (c - a) // t.element_size()
    return pitch > 0 and t.shape[1] <= gap % pitch and gap % pitch + u.shape[1] <= pitch


def _rows2d(name, t, cols):
    """A result tensor of the caller, or a tensor that goes with the result, as [T, cols] without a copy."""
    if t.dim() < 1 or t.shape[-1] != cols:
        raise OpNotEligible(f"{name} must have {cols} columns")
    if t.dim() == 2:
        return t
    try:
        return t.view(-1, cols)
    except RuntimeError:
        raise OpNotEligible(f"{name} must be viewable as rows of {cols}")


def _inputs(x, w, gated, what):
    if not (isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor)):
        raise OpNotEligible(f"{what}: tensors expected")
    if x.dtype not in _DTYPE:
        raise OpNotEligible(f"x must be bfloat16 or float16, got {x.dtype}")
    _check("the weight", w, x.dtype, x.get_device())
    shape, wshape = x.shape, w.shape
    if len(shape) < 1 or len(wshape) != 2 or wshape[1] != shape[-1]:
        raise OpNotEligible(f"{what}: x [..., n_in] and a weight [rows, n_in] expected")
    if wshape[1] < 1 or wshape[0] < 1:
        raise OpNotEligible(f"{what}: feature counts must be positive")
    if gated and wshape[0] % 2:
        raise OpNotEligible("w13 must hold gate rows followed by up rows: an even row count")
    x2 = x if len(shape) == 2 else x.reshape(-1, shape[-1])
    if x2.shape[0] > _MOST or wshape[0] > _MOST or wshape[1] > _MOST:
        raise OpNotEligible(f"{what}: more than 2^27 tokens, inputs or weight rows")
    return x2


def _bias(bias, rows, x):
    if bias is None:
        return None
    _check("the bias", bias, x.dtype, x.get_device())
    if bias.shape != (rows,) or rows > 1 and bias.stride(0) != 1:
        raise OpNotEligible(f"the bias must be contiguous [{rows}]")
    return bias.data_ptr()


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_tangent(*tensors):
    """Refuses a tensor that carries a tangent of forward-mode differentiation (there is none outside a dual level)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:      # (asking a tensor costs 3 us)
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise OpNotEligible("forward-mode differentiation is not offered: a tensor of the call carries a tangent")


def _no_capture():
    if torch.cuda.is_current_stream_capturing():
        raise OpNotEligible("recording for backward() cannot be captured into a CUDA graph: capture the forward call with "
                            "return_preact=True on detached tensors and its *_backward")


def _resident(x):
    if not x.is_cuda:
        raise OpNotEligible("inputs must be CUDA-resident (there is no CPU path)")


def _given_out(out, shape, x, others):
    """A result tensor of the caller, as rows."""
    _check("out", out, x.dtype, x.get_device())
    if out.shape != shape:
        raise OpNotEligible(f"out must be {tuple(shape)}, got {tuple(out.shape)}")
    _apart("out", out, others)
    out2 = _rows2d("out", out, shape[-1])
    _pitch("out", out2)
    return out2


def _result(out, out2, shape, x):
    """The result tensor, as the caller sees it and as rows."""
    if out is None:
        out = x.new_empty(shape)
        return out, out if len(shape) == 2 else out.view(-1, shape[-1])
    increment_version(out)
    return out, out2


def _new_preact(x, T, rows):
    """Room for fp32 pre-activations [T, rows], each row on 32 bytes."""
    if rows & 7:
        return x.new_empty_strided((T, rows), (rows + 7 & -8, 1), dtype=torch.float32)
    return x.new_empty((T, rows), dtype=torch.float32)


_NO_ROOM = (None, None, 0)


def _forward_work(x, xp, ldx, wp, ldw, T, n_in, rows):
    """(tensor to keep, pointer, bytes) of the room for copies of x and w, where their alignment calls for them."""
    if not ((xp | wp) & 15 or (ldx | ldw) & 7):
        return _NO_ROOM
    nbytes = _entry("vk_cuda_dense_forward_workspace_bytes")(xp, ldx, wp, ldw, T, n_in, rows)
    work = x.new_empty((nbytes,), dtype=torch.uint8)
    return work, work.data_ptr(), nbytes


# ---------------------------------------------------------------------------
# gated projection
# ---------------------------------------------------------------------------

def _gated_kind(activation, swiglu_limit, beta):
    if activation not in (SWIGLU, SITU):
        raise OpNotEligible("activation must be SWIGLU or SITU")
    if not swiglu_limit >= 0:
        raise OpNotEligible("swiglu_limit must not be negative (0 for none)")
    if activation == SITU and not beta > 0:
        raise OpNotEligible("SiTU needs a positive beta")


def gated_linear(x: torch.Tensor, w13: torch.Tensor, b13: torch.Tensor | None = None, *, activation: int = SWIGLU,
                 swiglu_limit: float = 0.0, beta: float = 4.0, linear_beta: float = 25.0, out: torch.Tensor | None = None,
                 return_preact: bool = False):
    """``h [..., ispp] = act(x Wg^T + bg) * (x Wu^T + bu)`` for x ``[..., hidden]`` and w13 ``[2 * ispp, hidden]`` (gate rows, then
    up rows; b13 ``[2 * ispp]`` likewise). SwiGLU: gate * sigmoid(gate) * up, the gate clamped from above and up from both sides
    at `swiglu_limit` if that is positive; SiTU: beta tanh(gate / beta) sigmoid(gate) * linear_beta tanh(up / linear_beta) (up
    itself if linear_beta is not positive).

    ``return_preact``: also return what ``gated_linear_backward`` needs, the pre-activations in fp32, ``[T, 2 * ispp]`` (T: all
    leading dimensions of x together)."""
    _no_tangent(x, w13, b13, out)
    if out is None and type(x) is torch.Tensor and isinstance(w13, torch.Tensor):
        # the ordinary call, checked at once: what it does not cover is looked at below piece by piece
        shape, index, dtype, wshape = x.shape, x.get_device(), x.dtype, w13.shape
        if (len(shape) == 2 and index >= 0 and dtype in _DTYPE and len(wshape) == 2 and _MOST >= wshape[1] == shape[1] > 0
                and 0 < wshape[0] <= _MOST and not wshape[0] & 1 and 0 < shape[0] <= _MOST
                and (activation == SWIGLU or activation == SITU and beta > 0) and swiglu_limit >= 0
                and (ldx := _matrix(x, shape, dtype, index)) and (ldw := _matrix(w13, wshape, dtype, index))
                and (b13 is None or _vector(b13, wshape[0], dtype, index)) and not _wants_grad(x, w13, b13)):
            T, rows = shape[0], wshape[0]
            h = x.new_empty((T, rows // 2))
            preact = _new_preact(x, T, rows) if return_preact else None
            xp, wp = x.data_ptr(), w13.data_ptr()
            work, room, nbytes = _forward_work(x, xp, ldx, wp, ldw, T, shape[1], rows) if (xp | wp) & 15 or (ldx | ldw) & 7 else _NO_ROOM
            _call("vk_cuda_gated_linear", index, xp, ldx, wp, ldw, None if b13 is None else b13.data_ptr(),
                  h.data_ptr(), rows // 2, None if preact is None else preact.data_ptr(), rows + 7 & -8, _DTYPE[dtype], T, shape[1], rows // 2,
                  activation, swiglu_limit, beta, linear_beta, room, nbytes)
            return (h, preact) if return_preact else h
    x2 = _inputs(x, w13, True, "gated_linear")
    _gated_kind(activation, swiglu_limit, beta)
    rows, ispp = w13.shape[0], w13.shape[0] // 2
    b = _bias(b13, rows, x)
    T, hidden = x2.shape
    shape = (*x.shape[:-1], ispp)
    ldx, ldw = _pitch("x", x2), _pitch("w13", w13)
    out2 = None if out is None else _given_out(out, shape, x, (("x", x), ("w13", w13), ("b13", b13)))
    _resident(x)
    if _wants_grad(x, w13, b13, out):
        if out is not None or return_preact:
            raise OpNotEligible("gated_linear: out and return_preact are for calls that record no gradient")
        return _GatedLinear.apply(x, w13, b13, activation, swiglu_limit, beta, linear_beta)
    h, h2 = _result(out, out2, shape, x)
    preact = _new_preact(x, T, rows) if return_preact else None
    if T > 0:
        work, room, nbytes = _forward_work(x, x2.data_ptr(), ldx, w13.data_ptr(), ldw, T, hidden, rows)
        _call("vk_cuda_gated_linear", x.get_device(), x2.data_ptr(), ldx, w13.data_ptr(), ldw, b, h2.data_ptr(), _pitch("out", h2),
              None if preact is None else preact.data_ptr(), rows + 7 & -8, _DTYPE[x.dtype], T, hidden, ispp, activation, swiglu_limit, beta,
              linear_beta, room, nbytes)
    return (h, preact) if return_preact else h


def gated_linear_backward(dh: torch.Tensor, x: torch.Tensor, w13: torch.Tensor, preact: torch.Tensor, *, activation: int = SWIGLU,
                          swiglu_limit: float = 0.0, beta: float = 4.0, linear_beta: float = 25.0, bias_grad: bool = False,
                          x_grad: bool = True, w_grad: bool = True):
    """``(dx, dw13, db13)`` for the gradient dh of ``gated_linear``'s result; ``preact`` as that call returned it, the other
    arguments as it was given. What is not asked for is None."""
    _gated_kind(activation, swiglu_limit, beta)
    if preact is None:
        raise OpNotEligible("gated_linear_backward needs the forward call's pre-activations")
    return _backward("vk_cuda_gated_linear_backward", dh, x, w13, preact, True, bias_grad, x_grad, w_grad,
                     (activation, swiglu_limit, beta, linear_beta))


# ---------------------------------------------------------------------------
# projection with epilogue
# ---------------------------------------------------------------------------

def _linear_kind(activation):
    kind = _LINEAR_ACT.get(activation) if activation is None or isinstance(activation, str) else None
    if kind is None:
        raise OpNotEligible(f"activation must be None, 'silu', 'gelu' or 'gelu_tanh', got {activation!r}")
    return kind


def fused_linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
                 residual: torch.Tensor | None = None, out: torch.Tensor | None = None, return_preact: bool = False):
    """``y [..., n_out] = act(x w^T + bias) + residual`` for x ``[..., n_in]``, w ``[n_out, n_in]``; activation None, "silu",
    "gelu" (erf) or "gelu_tanh"; residual of y's shape (not broadcast). ``out`` may be the residual itself.

    ``return_preact``: also return what ``fused_linear_backward`` needs: the pre-activations in fp32, ``[T, n_out]``, or None
    where there is no activation."""
    act = _linear_kind(activation)
    _no_tangent(x, w, bias, residual, out)
    if out is None and type(x) is torch.Tensor and isinstance(w, torch.Tensor):
        # the ordinary call, checked at once: what it does not cover is looked at below piece by piece
        shape, index, dtype, wshape = x.shape, x.get_device(), x.dtype, w.shape
        T, n_out, ldr = shape[0] if shape else 0, wshape[0] if wshape else 0, 0
        if (len(shape) == 2 and index >= 0 and dtype in _DTYPE and len(wshape) == 2 and _MOST >= wshape[1] == shape[1] > 0
                and 0 < n_out <= _MOST and 0 < T <= _MOST
                and (ldx := _matrix(x, shape, dtype, index)) and (ldw := _matrix(w, wshape, dtype, index))
                and (bias is None or _vector(bias, n_out, dtype, index))
                and (residual is None or isinstance(residual, torch.Tensor) and (ldr := _matrix(residual, (T, n_out), dtype, index)))
                and not _wants_grad(x, w, bias, residual)):
            n_in = shape[1]
            y = x.new_empty((T, n_out))
            preact = _new_preact(x, T, n_out) if return_preact and act else None
            xp, wp = x.data_ptr(), w.data_ptr()
            work, room, nbytes = _forward_work(x, xp, ldx, wp, ldw, T, n_in, n_out) if (xp | wp) & 15 or (ldx | ldw) & 7 else _NO_ROOM
            _call("vk_cuda_fused_linear", index, xp, ldx, wp, ldw, None if bias is None else bias.data_ptr(),
                  None if residual is None else residual.data_ptr(), ldr, y.data_ptr(), n_out,
                  None if preact is None else preact.data_ptr(), n_out + 7 & -8, _DTYPE[dtype], T, n_in, n_out, act, room, nbytes)
            return (y, preact) if return_preact else y
    x2 = _inputs(x, w, False, "fused_linear")
    n_out = w.shape[0]
    b = _bias(bias, n_out, x)
    shape = (*x.shape[:-1], n_out)
    ldx, ldw = _pitch("x", x2), _pitch("w", w)
    r2, ldr = None, 0
    if residual is not None:
        _check("the residual", residual, x.dtype, x.get_device())
        if residual.shape != shape:
            raise OpNotEligible(f"the residual must be {shape}, got {tuple(residual.shape)}")
        r2 = _rows2d("the residual", residual, n_out)
        ldr = _pitch("the residual", r2)
    out2 = None
    if out is not None:
        _check_tensor("out", out)
        in_place = residual is not None and out.data_ptr() == residual.data_ptr() and out.stride() == residual.stride()
        out2 = _given_out(out, shape, x, (("x", x), ("w", w), ("the bias", bias), ("the residual", None if in_place else residual)))
    _resident(x)
    if _wants_grad(x, w, bias, residual, out):
        if out is not None or return_preact:
            raise OpNotEligible("fused_linear: out and return_preact are for calls that record no gradient")
        return _FusedLinear.apply(x, w, bias, residual, activation)
    T, n_in = x2.shape
    y, y2 = _result(out, out2, shape, x)
    preact = _new_preact(x, T, n_out) if return_preact and act else None
    if T > 0:
        work, room, nbytes = _forward_work(x, x2.data_ptr(), ldx, w.data_ptr(), ldw, T, n_in, n_out)
        _call("vk_cuda_fused_linear", x.get_device(), x2.data_ptr(), ldx, w.data_ptr(), ldw, b, None if r2 is None else r2.data_ptr(), ldr,
              y2.data_ptr(), _pitch("out", y2), None if preact is None else preact.data_ptr(), n_out + 7 & -8, _DTYPE[x.dtype], T, n_in, n_out,
              act, room, nbytes)
    return (y, preact) if return_preact else y


def fused_linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, preact: torch.Tensor | None = None, *,
                          activation: str | None = None, bias_grad: bool = False, x_grad: bool = True, w_grad: bool = True):
    """``(dx, dw, dbias)`` for the gradient dy of ``fused_linear``'s result; ``preact`` as that call returned it (None without an
    activation). What is not asked for is None. The residual's gradient is dy."""
    act = _linear_kind(activation)
    if act and preact is None:
        raise OpNotEligible("fused_linear_backward needs the forward call's pre-activations")
    return _backward("vk_cuda_fused_linear_backward", dy, x, w, preact if act else None, False, bias_grad, x_grad, w_grad, (act,))


def _backward(entry, dy, x, w, preact, gated, bias_grad, x_grad, w_grad, kind):
    _no_tangent(dy, x, w, preact)
    ordinary, ldp = False, 0
    if type(x) is torch.Tensor and isinstance(w, torch.Tensor) and isinstance(dy, torch.Tensor):
        # the ordinary call, checked at once: what it does not cover is looked at below piece by piece
        shape, index, dtype, wshape = x.shape, x.get_device(), x.dtype, w.shape
        ordinary = (len(shape) == 2 and index >= 0 and dtype in _DTYPE and len(wshape) == 2 and _MOST >= wshape[1] == shape[1] > 0
                    and 0 < wshape[0] <= _MOST and not (gated and wshape[0] & 1) and 0 < shape[0] <= _MOST
                    and (ldx := _matrix(x, shape, dtype, index)) and (ldw := _matrix(w, wshape, dtype, index))
                    and (ld_dy := _matrix(dy, (shape[0], wshape[0] >> gated), dtype, index))
                    and (preact is None or isinstance(preact, torch.Tensor) and (ldp := _matrix(preact, (shape[0], wshape[0]), torch.float32, index))))
    if ordinary:
        (T, n_in), rows = shape, wshape[0]
        n_out = rows >> gated
        dy2, x2 = dy, x
    else:
        x2 = _inputs(x, w, gated, entry[8:])
        rows, (T, n_in) = w.shape[0], x2.shape
        n_out = rows // 2 if gated else rows
        dtype = x.dtype
        _check("the result's gradient", dy, dtype, x.get_device())
        if dy.shape != (*x.shape[:-1], n_out):
            raise OpNotEligible(f"the result's gradient must be {(*x.shape[:-1], n_out)}, got {tuple(dy.shape)}")
        dy2 = dy if dy.dim() == 2 else dy.reshape(-1, n_out)
        if preact is not None:
            _check("preact", preact, torch.float32, x.get_device())
            if preact.shape != (T, rows):
                raise OpNotEligible(f"preact must be {(T, rows)}, got {tuple(preact.shape)}")
        ldx, ldw, ld_dy = _pitch("x", x2), _pitch("the weight", w), _pitch("the result's gradient", dy2)
        ldp = 0 if preact is None else _pitch("preact", preact)
        _resident(x)
        index = x.get_device()
    dx = x.new_empty(x.shape) if x_grad else None
    dw = x.new_empty((rows, n_in)) if w_grad else None
    db = x.new_empty((rows,)) if bias_grad else None
    if dx is None and dw is None and db is None:
        return None, None, None
    xp, wp = x2.data_ptr(), w.data_ptr()
    nbytes = _entry("vk_cuda_dense_backward_workspace_bytes")(xp, ldx, wp, ldw, T, n_in, n_out, gated)
    work = x.new_empty((nbytes,), dtype=torch.uint8)
    _call(entry, index, dy2.data_ptr(), ld_dy, xp, ldx, wp, ldw, None if preact is None else preact.data_ptr(), ldp,
          None if dx is None else dx.data_ptr(), n_in, None if dw is None else dw.data_ptr(), n_in, None if db is None else db.data_ptr(),
          _DTYPE[dtype], T, n_in, n_out, *kind, work.data_ptr(), nbytes)
    return dx, dw, db


# ---------------------------------------------------------------------------
# recording for backward()
# ---------------------------------------------------------------------------

def _neighbours(t):
    """A gradient as autograd hands it over (it may be an expanded number), with rows that the kernels take."""
    return t if t.stride(-1) == 1 and (t.dim() < 2 or t.stride(-2) >= t.shape[-1]) else t.contiguous()


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, b13, activation, swiglu_limit, beta, linear_beta):
        _no_capture()
        ctx.kw = dict(activation=activation, swiglu_limit=swiglu_limit, beta=beta, linear_beta=linear_beta)
        h, preact = gated_linear(x, w13, b13, return_preact=True, **ctx.kw)
        ctx.save_for_backward(x, w13, preact)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        _no_capture()
        x, w13, preact = ctx.saved_tensors
        nx, nw, nb = ctx.needs_input_grad[:3]
        dx, dw, db = gated_linear_backward(_neighbours(dh), x, w13, preact, x_grad=nx, w_grad=nw, bias_grad=nb, **ctx.kw)
        return dx, dw, db, None, None, None, None


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation):
        _no_capture()
        ctx.activation = activation
        y, preact = fused_linear(x, w, bias, activation=activation, residual=residual, return_preact=True)
        ctx.save_for_backward(x, w, preact)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _no_capture()
        x, w, preact = ctx.saved_tensors
        nx, nw, nb, n_residual, _ = ctx.needs_input_grad
        dx = dw = db = None
        if nx or nw or nb:
            dx, dw, db = fused_linear_backward(_neighbours(dy), x, w, preact, activation=ctx.activation, x_grad=nx, w_grad=nw,
                                               bias_grad=nb)
        return dx, dw, db, dy if n_residual else None, None
