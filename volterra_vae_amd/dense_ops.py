"""Layers and loss of a network equaliser: `linear`, `gated_linear` and `topk_distillation` over the HIP kernels.

Tensors in, kernels enqueued on the current HIP stream of the tensors' device; float32, bfloat16 or float16, one type for all
tensors of a call, on a GPU only.  Matrices need unit stride inside a row; rows may lie apart (up to 2^22 elements), and rows of inputs
may overlap (windows that slide over one received sequence are a matrix with the row stride `samples_per_symbol`).

Two ways to train: the functions named above are differentiable; `linear_forward` / `linear_backward`, `gated_forward` /
`gated_backward` and `topk_distillation_step` are the same passes with every gradient an explicit result, for training loops
that run without autograd, and for HIP graphs: these are what to capture (a backward pass of autograd that is captured while an
eager graph of the same leaves lives ends the process).  Forward-mode derivatives are refused.

`torch.ops.v2vae.linear`, `torch.ops.v2vae.gated_linear` and `torch.ops.v2vae.topk_distillation` are the differentiable forms as
registered ops.  Where a dispatch mode is at work (fake tensors, make_fx and what else traces a program), every pass enters the graph
as an op with a shape function (`torch.ops.v2vae.linear_forward`, `linear_backward`, `gated_forward`, `gated_backward`,
`distillation_forward`, `distillation_backward`, `distillation_step`).
"""
from __future__ import annotations

import functools
from typing import List, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import Dense, Distill, check, lib

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "tanh": 4}
MAX_TEACHER_ENTRIES = 1024
MAX_ROW_STRIDE = 1 << 22
_NAMES = list(ACTIVATIONS)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_tensor(t, name, dim, like=None, dtype=None):
    try:  # what passes, first: these checks run before every launch
        want = dtype if dtype is not None else (like.dtype if like is not None else t.dtype)
        index = t.get_device()
        if (t.dtype is want and (like is not None or want in _DTYPES) and index >= 0 and (like is None or index == like.get_device())
                and t.dim() == dim and (t.stride(-1) == 1 or t.shape[-1] <= 1) and not t.is_neg()):
            return
    except (AttributeError, IndexError):
        pass
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor (got {type(t).__name__})")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on the GPU: these kernels have no CPU implementation")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if dtype is None and like is None:
        if t.dtype not in _DTYPES:
            raise NotImplementedError(f"{name}: float32, bfloat16 or float16 only (got {t.dtype})")
    elif t.dtype != want:
        raise ValueError(f"{name} is {t.dtype}, expected {want}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimension{'s' if dim > 1 else ''} (got {t.dim()})")
    if t.is_neg():
        raise ValueError(f"{name} is a negation that is not carried out yet (pass {name}.resolve_neg())")
    raise ValueError(f"{name} must have unit stride in its last dimension")


# How many dispatch modes are at work.  They have to see an op, not the addresses of tensors that they may follow or that have no memory.
_modes = torch._C._len_torch_dispatch_stack


def _refuse_tangents(*tensors):
    """Inside a forward-mode level: the kernels carry no tangents, and a dual tensor's derivative would be lost without a word."""
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("forward-mode derivatives: these operators have a backward pass only")


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _activation(kind):
    try:
        return ACTIVATIONS[kind]
    except KeyError:
        raise ValueError(f"activation {kind!r} is none of {', '.join(ACTIVATIONS)}") from None


def _p(t):
    return None if t is None else t.data_ptr()


def _enqueue(fn, name, t, *args):
    """fn(*args, stream) with t's device current and its current stream."""
    index = t.get_device()
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, name)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(gated, backward, description):
    f = lib.v2vae_gated_workspace_bytes if gated else lib.v2vae_linear_workspace_bytes
    return f(Dense.from_buffer_copy(description), backward)


def _workspace(gated, backward, d, x):
    """Scratch memory of one call, from torch's allocator: of the current stream, or of the graph that is being captured."""
    size = _workspace_bytes(gated, backward, bytes(d))
    return torch.empty(max(size, 256), dtype=torch.uint8, device=x.device) if size or backward else None


def _check_layer(x, weight, name, bias, bias_name):
    try:  # what passes, first
        dtype, index = x.dtype, x.get_device()
        n, k = weight.shape
        if (weight.dtype is dtype and weight.get_device() == index and k == x.shape[1] and n > 0 and k > 0
                and (weight.stride(1) == 1 or k == 1) and not weight.is_neg()
                and (bias is None or (bias.dtype is dtype and bias.get_device() == index and bias.shape == (n,)
                                      and (bias.stride(0) == 1 or n == 1) and not bias.is_neg()))):
            return
    except (AttributeError, ValueError, IndexError):
        pass
    _check_tensor(weight, name, 2, like=x)
    if weight.shape[1] != x.shape[1]:
        raise ValueError(f"{name}: {weight.shape[1]} columns, x has {x.shape[1]}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{name}: empty")
    if bias is not None:
        _check_tensor(bias, bias_name, 1, like=x)
        if bias.shape[0] != weight.shape[0]:
            raise ValueError(f"{bias_name}: {bias.shape[0]} values, {name} has {weight.shape[0]} rows")


def _dense(x, w, act, w2=None, residual=None, dy=None):
    return Dense(_DTYPES[x.dtype], act, x.shape[0], x.shape[1], w.shape[0], _row_stride(x), _row_stride(w),
                 0 if w2 is None else _row_stride(w2), 0 if residual is None else _row_stride(residual),
                 0 if dy is None else _row_stride(dy))


def _check_grad(dy, name, x, n):
    _check_tensor(dy, name, 2, like=x)
    if tuple(dy.shape) != (x.shape[0], n):
        raise ValueError(f"{name}: expected {(x.shape[0], n)}, got {tuple(dy.shape)}")


def _incoming(dy):
    """A gradient in a layout that the kernels take: autograd chose the one that it comes in."""
    return (dy if (dy.shape[1] <= 1 or dy.stride(1) == 1) and dy.stride(0) <= MAX_ROW_STRIDE else dy.contiguous()).resolve_neg()


def _check_kept(kept, shape, x):
    _check_tensor(kept, "the kept pre-activations", len(shape), like=x, dtype=torch.float32)
    if tuple(kept.shape) != shape or not kept.is_contiguous():
        raise ValueError(f"the kept pre-activations: expected a contiguous {shape}, got {tuple(kept.shape)}")


# ------------------------------------------------------------------------------------------------ linear
def linear_forward(x, weight, bias=None, *, residual=None, activation="none",
                   keep=False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(y, z) for x [M, K], weight [N, K]: y = activation(x weight^T + bias) + residual, and, if `keep` and there is an
    activation, the float32 pre-activations z [M, N] that `linear_backward` wants (else None)."""
    act = _activation(activation)
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight, bias, residual)
    _check_tensor(x, "x", 2)
    _check_layer(x, weight, "weight", bias, "bias")
    m, n = x.shape[0], weight.shape[0]
    if residual is not None:
        _check_tensor(residual, "residual", 2, like=x)
        if tuple(residual.shape) != (m, n):
            raise ValueError(f"residual: expected {(m, n)}, got {tuple(residual.shape)}")
    if _modes():
        y, z = torch.ops.v2vae.linear_forward(x, weight, bias, residual, activation, bool(keep))
        return y, z if keep and act else None
    d = _dense(x, weight, act, residual=residual)
    y = x.new_empty((m, n))
    z = torch.empty((m, n), dtype=torch.float32, device=x.device) if keep and act else None
    ws = None if m <= 16 and x.dtype is not torch.float32 else _workspace(False, 0, d, x)  # few 16-bit rows need none
    _enqueue(lib.v2vae_linear_fwd, "v2vae_linear_fwd", x, d, x.data_ptr(), weight.data_ptr(), _p(bias), _p(residual), y.data_ptr(), _p(z),
             _p(ws))
    return y, z


def linear_backward(dy, x, weight, z=None, *, activation="none", need=(True, True, True)):
    """(dx, dweight, dbias) of `linear_forward` given dy [M, N] and the kept z; None where `need` says so.  The residual's
    gradient is dy."""
    act = _activation(activation)
    _check_tensor(x, "x", 2)
    _check_layer(x, weight, "weight", None, "")
    m, n = x.shape[0], weight.shape[0]
    _check_grad(dy, "dy", x, n)
    if act:
        if z is None:
            raise ValueError("z: the pre-activations of linear_forward(..., keep=True) are needed with an activation")
        _check_kept(z, (m, n), x)
    return _linear_backward(dy, x, weight, z, act, need)


def _linear_backward(dy, x, weight, z, act, need):
    if forward_ad._current_level >= 0:
        _refuse_tangents(dy, x, weight, z)
    if _modes():
        grads = torch.ops.v2vae.linear_backward(dy, x, weight, z if act else None, _NAMES[act], [bool(q) for q in need[:3]])
        return tuple(g if q else None for g, q in zip(grads, need))
    m, k, n = x.shape[0], x.shape[1], weight.shape[0]
    d = _dense(x, weight, act, dy=dy)
    new = lambda wanted, *shape: x.new_empty(shape) if wanted else None  # noqa: E731
    dx, dw, db = new(need[0], m, k), new(need[1], n, k), new(need[2], n)
    ws = _workspace(False, 1, d, x)
    _enqueue(lib.v2vae_linear_bwd, "v2vae_linear_bwd", x, d, _p(x), _p(weight), _p(z) if act else None, _p(dy), _p(dx), _p(dw), _p(db), _p(ws))
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, z = linear_forward(x, weight, bias, residual=residual, activation=activation,
                              keep=any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, z)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, dw, db = _linear_backward(_incoming(dy), x, weight, z, ACTIVATIONS[ctx.activation], need)
        return dx, dw, db, dy if need[3] else None, None


def _flat(t):
    return t if t is None or t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _grads_wanted(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
           activation: str = "none") -> torch.Tensor:
    """activation(x weight^T + bias) + residual for x [..., K], weight [N, K], bias [N], residual [..., N], in one kernel.

    activation: none, relu, silu, gelu (erf form) or tanh.  Differentiable in every tensor.  Sums are float32; the backward pass
    works from float32 pre-activations and rounds dy * activation' to the tensors' type once before the two products (float16: beyond
    65504 it becomes infinite there, however small the sums it enters)."""
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("x must be a tensor [..., K]")
    if residual is not None and tuple(residual.shape[:-1]) != tuple(x.shape[:-1]):
        raise ValueError(f"residual: expected {tuple(x.shape[:-1])} rows, got {tuple(residual.shape[:-1])}")
    flat = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if _grads_wanted(x, weight, bias, residual):
        y = _Linear.apply(flat, weight, bias, _flat(residual), activation)
    else:
        y = linear_forward(flat, weight, bias, residual=_flat(residual), activation=activation)[0]
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[-1])


# ------------------------------------------------------------------------------------------------ gated block
def gated_forward(x, weight_gate, weight_up, bias_gate=None, bias_up=None, *, activation="silu",
                  keep=False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(h, gu) for x [M, K], weights [N, K]: h = activation(x weight_gate^T + bias_gate) * (x weight_up^T + bias_up), and, if
    `keep`, the float32 pre-activations gu [2, M, N] (gate, up) that `gated_backward` wants (else None)."""
    act = _activation(activation)
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight_gate, weight_up, bias_gate, bias_up)
    _check_tensor(x, "x", 2)
    _check_layer(x, weight_gate, "weight_gate", bias_gate, "bias_gate")
    _check_layer(x, weight_up, "weight_up", bias_up, "bias_up")
    if weight_up.shape != weight_gate.shape:
        raise ValueError(f"weight_up: expected {tuple(weight_gate.shape)}, got {tuple(weight_up.shape)}")
    m, n = x.shape[0], weight_gate.shape[0]
    if _modes():
        h, gu = torch.ops.v2vae.gated_forward(x, weight_gate, weight_up, bias_gate, bias_up, activation, bool(keep))
        return h, gu if keep else None
    d = _dense(x, weight_gate, act, w2=weight_up)
    h = x.new_empty((m, n))
    gu = torch.empty((2, m, n), dtype=torch.float32, device=x.device) if keep else None
    ws = None if m <= 16 and x.dtype is not torch.float32 else _workspace(True, 0, d, x)
    _enqueue(lib.v2vae_gated_fwd, "v2vae_gated_fwd", x, d, x.data_ptr(), weight_gate.data_ptr(), weight_up.data_ptr(), _p(bias_gate),
             _p(bias_up), h.data_ptr(), _p(gu), _p(ws))
    return h, gu


def gated_backward(dh, x, weight_gate, weight_up, gu, *, activation="silu", need=(True, True, True, True, True)):
    """(dx, dweight_gate, dweight_up, dbias_gate, dbias_up) of `gated_forward` given dh [M, N] and the kept gu; None where
    `need` says so."""
    act = _activation(activation)
    _check_tensor(x, "x", 2)
    _check_layer(x, weight_gate, "weight_gate", None, "")
    _check_layer(x, weight_up, "weight_up", None, "")
    if weight_up.shape != weight_gate.shape:
        raise ValueError(f"weight_up: expected {tuple(weight_gate.shape)}, got {tuple(weight_up.shape)}")
    m, n = x.shape[0], weight_gate.shape[0]
    _check_grad(dh, "dh", x, n)
    _check_kept(gu, (2, m, n), x)
    return _gated_backward(dh, x, weight_gate, weight_up, gu, act, need)


def _gated_backward(dh, x, weight_gate, weight_up, gu, act, need):
    if forward_ad._current_level >= 0:
        _refuse_tangents(dh, x, weight_gate, weight_up, gu)
    if _modes():
        grads = torch.ops.v2vae.gated_backward(dh, x, weight_gate, weight_up, gu, _NAMES[act], [bool(q) for q in need[:5]])
        return tuple(g if q else None for g, q in zip(grads, need))
    m, k, n = x.shape[0], x.shape[1], weight_gate.shape[0]
    d = _dense(x, weight_gate, act, w2=weight_up, dy=dh)
    new = lambda wanted, *shape: x.new_empty(shape) if wanted else None  # noqa: E731
    out = [new(need[0], m, k), new(need[1], n, k), new(need[2], n, k), new(need[3], n), new(need[4], n)]
    ws = _workspace(True, 1, d, x)
    _enqueue(lib.v2vae_gated_bwd, "v2vae_gated_bwd", x, d, _p(x), _p(weight_gate), _p(weight_up), _p(gu), _p(dh), *[_p(t) for t in out], _p(ws))
    return tuple(out)


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight_gate, weight_up, bias_gate, bias_up, activation):
        h, gu = gated_forward(x, weight_gate, weight_up, bias_gate, bias_up, activation=activation, keep=True)
        ctx.save_for_backward(x, weight_gate, weight_up, gu)
        ctx.activation = activation
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, weight_gate, weight_up, gu = ctx.saved_tensors
        return (*_gated_backward(_incoming(dh), x, weight_gate, weight_up, gu, ACTIVATIONS[ctx.activation], ctx.needs_input_grad), None)


def gated_linear(x: torch.Tensor, weight_gate: torch.Tensor, weight_up: torch.Tensor, bias_gate: Optional[torch.Tensor] = None,
                 bias_up: Optional[torch.Tensor] = None, *, activation: str = "silu") -> torch.Tensor:
    """Gated feed-forward block: activation(x weight_gate^T + bias_gate) * (x weight_up^T + bias_up) for x [..., K], weights
    [N, K], both projections, the activation and the product in one kernel.  Differentiable in every tensor; the gradients of both
    pre-activations are rounded to the tensors' type as in `linear`."""
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("x must be a tensor [..., K]")
    flat = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if _grads_wanted(x, weight_gate, weight_up, bias_gate, bias_up):
        h = _Gated.apply(flat, weight_gate, weight_up, bias_gate, bias_up, activation)
    else:
        h = gated_forward(flat, weight_gate, weight_up, bias_gate, bias_up, activation=activation)[0]
    return h if x.dim() == 2 else h.view(*x.shape[:-1], h.shape[-1])


# ------------------------------------------------------------------------------------------------ distillation
def _check_distill(logits, teacher_logits, teacher_index, temperature):
    if forward_ad._current_level >= 0:
        _refuse_tangents(logits, teacher_logits)
    _check_tensor(logits, "logits", 2)
    if getattr(teacher_logits, "dtype", None) not in _DTYPES:
        raise NotImplementedError("teacher_logits: a float32, bfloat16 or float16 tensor")
    if getattr(teacher_index, "dtype", None) not in (torch.int32, torch.int64):
        raise ValueError("teacher_index: an int32 or int64 tensor")
    _check_tensor(teacher_logits, "teacher_logits", 2, like=logits, dtype=teacher_logits.dtype)
    _check_tensor(teacher_index, "teacher_index", 2, like=logits, dtype=teacher_index.dtype)
    m, v = logits.shape
    k = teacher_logits.shape[1]
    if v < 1:
        raise ValueError("logits: no classes")
    if not 1 <= k <= MAX_TEACHER_ENTRIES:
        raise ValueError(f"teacher_logits: 1 ... {MAX_TEACHER_ENTRIES} entries a row (got {k})")
    if teacher_logits.shape[0] != m or tuple(teacher_index.shape) != (m, k):
        raise ValueError(f"teacher_logits and teacher_index: expected {(m, k)}, got {tuple(teacher_logits.shape)} and "
                         f"{tuple(teacher_index.shape)}")
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"temperature: 1e-4 ... 1e4 (got {temperature})")


def _distill(logits, teacher_logits, teacher_index, temperature):
    return Distill(_DTYPES[logits.dtype], _DTYPES[teacher_logits.dtype], 32 if teacher_index.dtype == torch.int32 else 64,
                   teacher_logits.shape[1], logits.shape[0], logits.shape[1], _row_stride(logits), _row_stride(teacher_logits),
                   _row_stride(teacher_index), temperature, 0)


def _check_weight(weight, logits):
    if forward_ad._current_level >= 0:
        _refuse_tangents(weight)
    _check_tensor(weight, "row_weight", 1, like=logits, dtype=torch.float32)
    if weight.shape[0] != logits.shape[0]:
        raise ValueError(f"row_weight: expected {logits.shape[0]} values, got {weight.shape[0]}")


def topk_distillation_step(logits, teacher_logits, teacher_index, row_weight, *, temperature: float = 1.0):
    """(loss [M] float32, grad [M, V]): the losses of `topk_distillation` and d(sum of row_weight * loss) / d logits, one pass."""
    _check_distill(logits, teacher_logits, teacher_index, temperature)
    _check_weight(row_weight, logits)
    if _modes():
        return torch.ops.v2vae.distillation_step(logits, teacher_logits, teacher_index, row_weight, temperature)
    d = _distill(logits, teacher_logits, teacher_index, temperature)
    loss, grad = row_weight.new_empty(row_weight.shape), logits.new_empty(logits.shape)
    _enqueue(lib.v2vae_distill_step, "v2vae_distill_step", logits, d, _p(logits), _p(teacher_logits), _p(teacher_index), _p(row_weight),
             _p(loss), _p(grad))
    return loss, grad


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_index, temperature):
        _check_distill(logits, teacher_logits, teacher_index, temperature)
        ctx.d, loss, stats = _distill_forward(logits, teacher_logits, teacher_index, temperature, True)
        ctx.save_for_backward(logits, teacher_logits, teacher_index, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, weight):
        if forward_ad._current_level >= 0:
            _refuse_tangents(weight)
        logits, teacher_logits, teacher_index, stats = ctx.saved_tensors
        # hooks on saved tensors may give them back with other strides than the forward pass saw
        d = ctx.d
        if d is not None and (logits.stride(0) != d.ld_logits or teacher_logits.stride(0) != d.ld_teacher or teacher_index.stride(0) != d.ld_index):
            d = None
        weight = weight.contiguous().resolve_neg()
        return _distill_backward(weight, logits, teacher_logits, teacher_index, stats, ctx.temperature, d), None, None, None


def _distill_forward(logits, teacher_logits, teacher_index, temperature, keep):
    """(argument block, loss, statistics), the last two as asked for; no block in a trace."""
    if _modes():
        loss, stats = torch.ops.v2vae.distillation_forward(logits, teacher_logits, teacher_index, temperature, keep)
        return None, loss, stats if keep else None
    m = logits.shape[0]
    d = _distill(logits, teacher_logits, teacher_index, temperature)
    loss = torch.empty(m, dtype=torch.float32, device=logits.device)
    stats = loss.new_empty((m, 2)) if keep else None
    _enqueue(lib.v2vae_distill_fwd, "v2vae_distill_fwd", logits, d, _p(logits), _p(teacher_logits), _p(teacher_index), _p(loss), _p(stats))
    return d, loss, stats


def _distill_backward(weight, logits, teacher_logits, teacher_index, stats, temperature, d=None):
    if _modes():
        return torch.ops.v2vae.distillation_backward(weight, logits, teacher_logits, teacher_index, stats, temperature)
    if d is None:
        d = _distill(logits, teacher_logits, teacher_index, temperature)
    grad = logits.new_empty(logits.shape)
    _enqueue(lib.v2vae_distill_bwd, "v2vae_distill_bwd", logits, d, _p(logits), _p(teacher_logits), _p(teacher_index), _p(stats), _p(weight),
             _p(grad))
    return grad


def topk_distillation(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor, *,
                      temperature: float = 1.0) -> torch.Tensor:
    """Per-row distillation losses [M] (float32) of student logits [M, V] against a teacher's top logits [M, k] at the classes
    teacher_index [M, k] (int32 or int64):

        p = softmax(teacher / T),  q = softmax(logits / T),  loss = T^2 sum_j p_j (log p_j - log q[index_j])

    An entry with index < 0 or a teacher logit of -inf is absent; a row without present entries has loss and gradient 0; a class
    that a row names twice counts twice.  An index >= V makes the row NaN.  Differentiable in `logits`; the teacher is not.  Rows
    of the three matrices may lie any distance apart, but may not overlap.  Computed in float32, the loss is off by up to about
    T^2 2^-20 (2 + |log q|)."""
    if isinstance(teacher_logits, torch.Tensor) and teacher_logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("teacher_logits: the loss is not differentiable in the teacher (pass teacher_logits.detach())")
    if isinstance(logits, torch.Tensor) and _grads_wanted(logits):
        return _Distillation.apply(logits, teacher_logits, teacher_index, temperature)
    _check_distill(logits, teacher_logits, teacher_index, temperature)
    return _distill_forward(logits, teacher_logits, teacher_index, temperature, False)[1]


# ------------------------------------------------------------------------------------------------ registered ops
# The passes, for what traces a program.  An op returns tensors only: what a pass leaves out is empty there.
def _filled(like, *tensors):
    return tuple(like.new_empty(0) if t is None else t for t in tensors)


@torch.library.custom_op("v2vae::linear_forward", mutates_args=(), device_types="cuda")
def _op_linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], residual: Optional[torch.Tensor],
                       activation: str, keep: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    y, z = linear_forward(x, weight, bias, residual=residual, activation=activation, keep=keep)
    return _filled(x, y, z)


@_op_linear_forward.register_fake
def _(x, weight, bias, residual, activation, keep):
    shape = (x.shape[0], weight.shape[0])
    return _filled(x, x.new_empty(shape), x.new_empty(shape, dtype=torch.float32) if keep and activation != "none" else None)


@torch.library.custom_op("v2vae::linear_backward", mutates_args=(), device_types="cuda")
def _op_linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, z: Optional[torch.Tensor], activation: str,
                        need: List[bool]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _filled(x, *linear_backward(dy, x, weight, z, activation=activation, need=need))


@_op_linear_backward.register_fake
def _(dy, x, weight, z, activation, need):
    shapes = (x.shape, weight.shape, weight.shape[:1])
    return _filled(x, *(x.new_empty(s) if q else None for s, q in zip(shapes, need)))


@torch.library.custom_op("v2vae::gated_forward", mutates_args=(), device_types="cuda")
def _op_gated_forward(x: torch.Tensor, weight_gate: torch.Tensor, weight_up: torch.Tensor, bias_gate: Optional[torch.Tensor],
                      bias_up: Optional[torch.Tensor], activation: str, keep: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return _filled(x, *gated_forward(x, weight_gate, weight_up, bias_gate, bias_up, activation=activation, keep=keep))


@_op_gated_forward.register_fake
def _(x, weight_gate, weight_up, bias_gate, bias_up, activation, keep):
    m, n = x.shape[0], weight_gate.shape[0]
    return _filled(x, x.new_empty((m, n)), x.new_empty((2, m, n), dtype=torch.float32) if keep else None)


@torch.library.custom_op("v2vae::gated_backward", mutates_args=(), device_types="cuda")
def _op_gated_backward(dh: torch.Tensor, x: torch.Tensor, weight_gate: torch.Tensor, weight_up: torch.Tensor, gu: torch.Tensor, activation: str,
                       need: List[bool]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _filled(x, *gated_backward(dh, x, weight_gate, weight_up, gu, activation=activation, need=need))


@_op_gated_backward.register_fake
def _(dh, x, weight_gate, weight_up, gu, activation, need):
    shapes = (x.shape, weight_gate.shape, weight_up.shape, weight_gate.shape[:1], weight_up.shape[:1])
    return _filled(x, *(x.new_empty(s) if q else None for s, q in zip(shapes, need)))


@torch.library.custom_op("v2vae::distillation_forward", mutates_args=(), device_types="cuda")
def _op_distillation_forward(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor, temperature: float,
                             keep: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    _check_distill(logits, teacher_logits, teacher_index, temperature)
    _, loss, stats = _distill_forward(logits, teacher_logits, teacher_index, temperature, keep)
    return _filled(loss, loss, stats)


@_op_distillation_forward.register_fake
def _(logits, teacher_logits, teacher_index, temperature, keep):
    m = logits.shape[0]
    return logits.new_empty(m, dtype=torch.float32), logits.new_empty((m, 2) if keep else 0, dtype=torch.float32)


@torch.library.custom_op("v2vae::distillation_backward", mutates_args=(), device_types="cuda")
def _op_distillation_backward(weight: torch.Tensor, logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor,
                              stats: torch.Tensor, temperature: float) -> torch.Tensor:
    _check_distill(logits, teacher_logits, teacher_index, temperature)
    _check_weight(weight, logits)
    return _distill_backward(weight, logits, teacher_logits, teacher_index, stats.contiguous(), temperature)


@_op_distillation_backward.register_fake
def _(weight, logits, teacher_logits, teacher_index, stats, temperature):
    return logits.new_empty(logits.shape)


@torch.library.custom_op("v2vae::distillation_step", mutates_args=(), device_types="cuda")
def _op_distillation_step(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor, row_weight: torch.Tensor,
                          temperature: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return topk_distillation_step(logits, teacher_logits, teacher_index, row_weight, temperature=temperature)


@_op_distillation_step.register_fake
def _(logits, teacher_logits, teacher_index, row_weight, temperature):
    return row_weight.new_empty(row_weight.shape), logits.new_empty(logits.shape)


# The differentiable forms.
_LIBRARY = torch.library.Library("v2vae", "FRAGMENT")
_LIBRARY.define("linear(Tensor x, Tensor weight, Tensor? bias=None, *, Tensor? residual=None, str activation='none') -> Tensor")
_LIBRARY.define("gated_linear(Tensor x, Tensor weight_gate, Tensor weight_up, Tensor? bias_gate=None, Tensor? bias_up=None, *, "
                "str activation='silu') -> Tensor")
_LIBRARY.define("topk_distillation(Tensor logits, Tensor teacher_logits, Tensor teacher_index, *, float temperature=1.0) -> Tensor")
for _name, _fn in (("linear", linear), ("gated_linear", gated_linear), ("topk_distillation", topk_distillation)):
    _LIBRARY.impl(_name, _fn, "CompositeImplicitAutograd")
