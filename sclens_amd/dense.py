"""Dense operators on torch tensors of one MI355X: the product with bias, activation and residual, its gradient, and the orthogonal
factor of a matrix by products. They stand beside the per-call drop-ins of `sclens_amd.api` (`_wishart_matrix`, `corr_mat`, `_get_eigen`):
scores of cells outside a decomposition (`linear` with the centring as the bias), covariates taken out of a matrix (the residual), heads
and encoders trained on the signals (`linear`, `linear_backward`, an `orthogonalize`d update), bases of two runs or members turned onto
each other (`orthogonalize` of `corr_mat(V1, V2)`).

Element types are torch.bfloat16, torch.float16 and torch.float32; sums are held in 32 bits and rounded once. What 16-bit types hold in 16 bits
between two products: `linear_backward` the gradient of the activation's argument (fp16 under a scale), `orthogonalize` its iterates (fp16
under scales); the single-launch forms of small sizes keep 32 bits.

Calls are queued on the tensors' device on torch's current stream of that device; they neither block nor synchronise, and can be captured
into a graph after one eager call of the same thread (which creates the thread's context). They record no autograd graph and propagate
no tangents (tensors that ask for either are refused): gradients are the explicit call.

torch has to be imported before the library is first used (importing this module does it): both then run on one HIP runtime and torch's
streams are valid for the library.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import Context

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
#: steep quintic step: five of them bring the singular values above about 1e-2 of the norm into 0.7 .. 1.2
UPDATE_STEP = (3.4445, -4.7750, 2.0315)
#: p(1) = 1, p'(1) = p''(1) = 0: converges cubically to the orthogonal factor from there
POLAR_STEP = (1.875, -1.25, 0.375)

_local = threading.local()


def _context(index: int, ctx: Optional[Context]) -> Context:
    if ctx is None:
        try:
            ctx = _local.contexts[index]
        except (AttributeError, KeyError):
            if not hasattr(_local, "contexts"):
                _local.contexts, _local.sizes = {}, {}
            ctx = _local.contexts[index] = Context(index)  # one host thread per context
    else:
        if ctx.device != index:
            raise ValueError(f"the tensors are on device {index}, the context on device {ctx.device}")
        if not hasattr(_local, "sizes"):
            _local.contexts, _local.sizes = {}, {}
    if not _lib.shares_torch_runtime:
        raise RuntimeError("libsclens_hip.so was loaded before torch and runs on another HIP runtime: import torch (or sclens_amd.dense) "
                           "before the first use of sclens_amd")
    return ctx


def _no_graph(name: str, t: torch.Tensor) -> None:
    """neither of autograd's modes: a result of these calls would lack its graph or its tangent in silence"""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: these operators record no graph (torch.no_grad() and the explicit gradient)")
    # (inside a dual level only: unpacking costs as much as all other checks of a tensor)
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a forward-mode tangent: these operators propagate none")


def _first(name: str, t) -> int:
    """checks of the tensor that sets the element type and the device; its device's index"""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} has to be a torch tensor")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name}: element type {t.dtype} (bfloat16, float16 or float32 expected)")
    _no_graph(name, t)
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}, expected a GPU")
    return t.get_device()


def _other(name: str, t, like: torch.Tensor, index: int, shape) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} has to be a torch tensor")
    if t.dtype is not like.dtype or not t.is_cuda or t.get_device() != index:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, expected {like.dtype} on {like.device}")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    _no_graph(name, t)


def _ld(name: str, t: torch.Tensor) -> int:
    """leading dimension of t as a matrix of rows along its last axis"""
    shape, stride = t.shape, t.stride()
    cols = shape[-1]
    if len(shape) == 2:
        ld = stride[0] if shape[0] > 1 else cols
    elif t.numel() == 0 or len(shape) == 1 or t.is_contiguous():
        ld = cols
    else:
        try:
            v = t.view(-1, cols)
        except RuntimeError:
            raise ValueError(f"{name}: the leading axes of strides {stride} do not join into one; call .contiguous()") from None
        ld = v.stride(0) if v.size(0) > 1 else cols
    if (cols > 1 and stride[-1] != 1 or ld < cols) and t.numel():
        if cols > 1 and stride[-1] != 1:
            raise ValueError(f"{name}: rows have to be contiguous (strides {stride}); call .contiguous()")
        raise ValueError(f"{name}: rows overlap (strides {stride}); call .contiguous()")
    return ld if ld > 0 else 1


def _rows(shape) -> int:
    n = 1
    for s in shape[:-1]:
        n *= s
    return n


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r} (one of {', '.join(ACTIVATIONS)})")
    return ACTIVATIONS[name]


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# the raw handle of torch's current stream of a device (the function its own compiled code uses, where there is one)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _run(fn, key, ctx: Context, like: torch.Tensor, index: int, *args):
    """the call with its workspace: the size the last call of these sizes needed is tried first, then what the library asks for"""
    sizes = _local.sizes
    size = sizes.get(key, 0)
    n = C.c_int64(size)
    stream = _raw_stream(index)
    ws = like.new_empty(size, dtype=torch.uint8) if size else None
    rc = fn(ctx.h, stream, *args, ws.data_ptr() if size else None, n)
    if rc == 8:  # SCLENS_ERR_WORKSPACE: nothing was launched
        if len(sizes) > 4096:
            sizes.clear()
        sizes[key] = size = n.value
        ws = like.new_empty(size, dtype=torch.uint8)
        rc = fn(ctx.h, stream, *args, ws.data_ptr(), n)
    if rc != 0:
        ctx.check(rc)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
           activation: str = "none", save_preact: bool = False,
           ctx: Optional[Context] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """activation(x @ weight.T + bias) + residual in one pass: x [..., K], weight [N, K], bias [N], residual [..., N] -> [..., N].

    `save_preact` also returns the argument of the activation, which `linear_backward` reads. activation: "none", "relu", "silu",
    "gelu" (z Phi(z)) or "gelu_tanh". One row (or a few) streams the weights once: the form for serving."""
    act = _activation(activation)
    index = _first("x", x)
    if not isinstance(weight, torch.Tensor) or x.dim() < 1 or weight.dim() != 2 or weight.size(1) != x.size(-1):
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(getattr(weight, 'shape', ()))}: expected [..., K] and [N, K]")
    _other("weight", weight, x, index, weight.shape)
    shape = x.shape
    N, K = weight.shape
    out_shape = (*shape[:-1], N)
    if bias is not None:
        _other("bias", bias, x, index, (N,))
        if N > 1 and bias.stride(0) != 1:
            raise ValueError("bias has to be contiguous")
    ldr = N
    if residual is not None:
        _other("residual", residual, x, index, out_shape)
        ldr = _ld("residual", residual)
    M = shape[0] if len(shape) == 2 else _rows(shape)
    ldx, ldw = _ld("x", x), _ld("weight", weight)
    ctx = _context(index, ctx)
    y = x.new_empty(out_shape)
    z = x.new_empty(out_shape) if save_preact else None
    dt = DTYPES[x.dtype]
    _run(ctx.lib.sclens_hip_linear, (1, dt, M, N, K), ctx, x, index, dt, M, N, K, x.data_ptr(), ldx, weight.data_ptr(), ldw, _p(bias),
         _p(residual), ldr, act, y.data_ptr(), N or 1, _p(z), N or 1)
    return (y, z) if save_preact else y


def linear_backward(grad: torch.Tensor, x: Optional[torch.Tensor], weight: Optional[torch.Tensor], preact: Optional[torch.Tensor] = None,
                    activation: str = "none", need_x: bool = True, need_weight: bool = True, need_bias: bool = True,
                    ctx: Optional[Context] = None):
    """Gradients of `linear`: (dx, dweight, dbias), those not needed None. grad [..., N] is the gradient of the result (and already that
    of the residual), preact what `linear(save_preact=True)` returned (not needed for "none"; relu'(0) = 0). x may be None if
    need_weight is false, weight if need_x is false. All leading axes are summed over in dweight and dbias, in a fixed order."""
    act = _activation(activation)
    index = _first("grad", grad)
    shape = grad.shape
    if len(shape) < 1:
        raise ValueError("grad: expected [..., N]")
    N = shape[-1]
    lead = shape[:-1]
    M = _rows(shape)
    if need_weight and x is None or need_x and weight is None:
        raise ValueError("dweight needs x, dx needs weight")
    K = x.size(-1) if x is not None else (weight.size(-1) if weight is not None else 0)
    if x is not None:
        _other("x", x, grad, index, (*lead, K))
    if weight is not None:
        _other("weight", weight, grad, index, (N, K))
    ldz = N or 1
    if act:
        if preact is None:
            raise ValueError(f"the gradient of {activation!r} needs preact (linear(..., save_preact=True))")
        _other("preact", preact, grad, index, shape)
        ldz = _ld("preact", preact)
    lddy = _ld("grad", grad)
    ldx = _ld("x", x) if need_weight else K or 1
    ldw = _ld("weight", weight) if need_x else K or 1
    ctx = _context(index, ctx)
    dx = grad.new_empty((*lead, K)) if need_x else None
    dw = grad.new_empty((N, K)) if need_weight else None
    db = grad.new_empty((N,)) if need_bias else None
    dt = DTYPES[grad.dtype]
    _run(ctx.lib.sclens_hip_linear_backward, (2, dt, M, N, K, need_x, need_weight, need_bias), ctx, grad, index, dt, M, N, K, grad.data_ptr(),
         lddy, _p(x) if need_weight else None, ldx, _p(weight) if need_x else None, ldw, _p(preact) if act else None, ldz, act, _p(dx),
         K or 1, _p(dw), K or 1, _p(db))
    return dx, dw, db


def orthogonalize(x: torch.Tensor, steps: int = 5, coefficients: Union[Sequence[float], Sequence[Sequence[float]]] = UPDATE_STEP,
                  eps: float = 1e-7, ctx: Optional[Context] = None) -> torch.Tensor:
    """x [..., rows, cols] with its singular values driven towards 1, by products: x0 = x / (|x|_F + eps), then per step (a, b, c)
    x <- a x + (b A + c A A) x with A = x x' on the shorter side, so that every singular value s becomes a s + b s^3 + c s^5.

    `coefficients`: one triple, used `steps` times, or a sequence of triples, one per step. [UPDATE_STEP] * 5 is an optimiser's update;
    [UPDATE_STEP] * 5 + [POLAR_STEP] * 3 converges to the orthogonal factor (singular values well above 1e-2 of the norm). Every matrix
    of the leading axes is worked on by itself."""
    index = _first("x", x)
    if x.dim() < 2:
        raise ValueError(f"x {tuple(x.shape)}: expected [..., rows, cols]")
    coef = [float(v) for v in coefficients] if len(coefficients) == 3 and not hasattr(coefficients[0], "__len__") else None
    if coef is not None:
        if int(steps) < 1:
            raise ValueError("at least one step")
        coef = coef * int(steps)
    else:
        if len(coefficients) < 1 or any(len(t) != 3 for t in coefficients):
            raise ValueError("coefficients: one (a, b, c) or a sequence of them, one per step")
        coef = [float(v) for t in coefficients for v in t]
    rows, cols = x.shape[-2:]
    batch = 1
    for s in x.shape[:-2]:
        batch *= s
    v = x
    if x.dim() > 3:
        try:
            v = x.view(batch, rows, cols)
        except RuntimeError:
            raise ValueError(f"x: the leading axes of strides {x.stride()} do not join into one; call .contiguous()") from None
    stride = v.stride(0) if v.dim() == 3 and batch > 1 else rows * cols
    ld = v.stride(-2) if rows > 1 else cols
    if x.numel() and (cols > 1 and v.stride(-1) != 1 or ld < cols):
        raise ValueError(f"x: rows have to be contiguous and apart (strides {x.stride()}); call .contiguous()")
    ctx = _context(index, ctx)
    y = x.new_empty(x.shape)
    dt = DTYPES[x.dtype]
    arr = (C.c_double * len(coef))(*coef)
    _run(ctx.lib.sclens_hip_orthogonalize, (3, dt, batch, rows, cols, len(coef)), ctx, x, index, dt, batch, rows, cols, x.data_ptr(), stride,
         ld or 1, y.data_ptr(), rows * cols, cols or 1, len(coef) // 3, arr, float(eps))
    return y
