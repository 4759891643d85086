"""torch.library operator boundary.

Keeps the reference's operator names and schemas so existing call sites bind unchanged:

  rten::materialize_fwd / rten::materialize_bwd     src/rten_cpp/RandumbTensor.py:371-390
  rten::scale_bias_bwd                              src/rten_cpp/RandumbTensor.py:414-420
  rten::embed_fwd / rten::embed_bwd                 src/rten_cpp/RandumbTensor.py:1121-1134
  rten_cpp::sq5_gen_2d / rten_cpp::materialize_fwd  src/rten_cpp/csrc/rten.cpp:36-39, ops.py:8-13

and adds the operators of the matrix-coefficient layer ``W = S @ C`` that fill the slot the
reference left to ``fakeMM`` (RandumbTensor.py:771-791, 942-946):

  rten::rlinear_fwd(x, coef, seed, out_features, row0=0) -> y
  rten::rlinear_bwd(dy, x, coef, seed, row0, need_dx, need_dc) -> (dx, dc)
  rten::noise(rows, cols, seed, row0, dtype, device) -> S

and the loss over a large vocabulary, which keeps no logits (the reference ends in F.cross_entropy on all of them,
modded-nanogpt/train_gpt2.py:236-240):

  rten::noise_ce_fwd / rten::noise_ce_bwd     logits z S^T over regenerated noise rows
  rten::linear_ce_fwd / rten::linear_ce_bwd   logits x W^T over a stored matrix
  rten::matmul_nt_fwd / rten::matmul_nt_bwd   z = x C^T in front of a noise head
  noise_cross_entropy, rlinear_cross_entropy, linear_cross_entropy   the differentiable functions on top of them

Every operator is functional (fresh outputs, current stream), has a fake (meta) kernel so
FakeTensor / torch.compile tracing works, and -- like the reference (RandumbTensor.py:438-448) --
a CPU registration that raises ``NotImplementedError``: there is no CPU implementation.
"""
from __future__ import annotations

import functools
from typing import List, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.library import custom_op

from . import kernels as K


def _cpu_raises(name):
    def _impl(*args, **kwargs):
        raise NotImplementedError(f"Unsupported CPU implementation of {name} called.")
    return _impl


# ------------------------------------------------------------------------------------------------
# matrix-coefficient layer
# ------------------------------------------------------------------------------------------------
@custom_op("rten::rlinear_fwd", mutates_args=(), device_types="cuda")
def rlinear_fwd(x: torch.Tensor, coef: torch.Tensor, seed: int, out_features: int, row0: int = 0) -> torch.Tensor:
    assert x.dim() == 2, "rlinear_fwd expects x flattened to [T, K]"
    return K.linear_fwd(x.contiguous(), coef.contiguous(), seed, out_features, row0)


@rlinear_fwd.register_fake
def _(x, coef, seed, out_features, row0=0):
    return x.new_empty((x.shape[0], out_features))


rlinear_fwd.register_kernel("cpu")(_cpu_raises("rlinear_fwd"))


@custom_op("rten::rlinear_bwd", mutates_args=(), device_types="cuda")
def rlinear_bwd(dy: torch.Tensor, x: torch.Tensor, coef: torch.Tensor, seed: int, row0: int, need_dx: bool,
                need_dc: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    dx, dc = K.linear_bwd(dy.contiguous(), x.contiguous(), coef.contiguous(), seed, row0, need_dx, need_dc)
    # custom ops cannot return None: an empty tensor stands for "not requested"
    if dx is None:
        dx = x.new_empty((0,))
    if dc is None:
        dc = coef.new_empty((0,))
    return dx, dc


@rlinear_bwd.register_fake
def _(dy, x, coef, seed, row0, need_dx, need_dc):
    return (x.new_empty(x.shape) if need_dx else x.new_empty((0,)),
            coef.new_empty(coef.shape) if need_dc else coef.new_empty((0,)))


rlinear_bwd.register_kernel("cpu")(_cpu_raises("rlinear_bwd"))


def _rlinear_setup(ctx, inputs, output):
    x, coef, seed, out_features, row0 = inputs
    ctx.save_for_backward(x, coef)
    ctx.seed = seed
    ctx.row0 = row0


def _rlinear_backward(ctx, dy):
    x, coef = ctx.saved_tensors
    need_dx, need_dc = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
    dx, dc = rlinear_bwd(dy, x, coef, ctx.seed, ctx.row0, need_dx, need_dc)
    return (dx if need_dx else None), (dc if need_dc else None), None, None, None


rlinear_fwd.register_autograd(_rlinear_backward, setup_context=_rlinear_setup)


def rlinear(x: torch.Tensor, coef: torch.Tensor, seed: int, out_features: int, row0: int = 0,
            bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = x @ (S @ coef).T (+ bias) for x of shape [..., K]; differentiable in x and coef."""
    lead = x.shape[:-1]
    y = rlinear_fwd(x.reshape(-1, x.shape[-1]), coef, seed, out_features, row0)
    y = y.reshape(*lead, out_features)
    if bias is not None:
        y = y + bias
    return y


@custom_op("rten::noise", mutates_args=(), device_types="cuda")
def noise(rows: int, cols: int, seed: int, row0: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    return K.noise(rows, cols, seed, row0, 0, dtype, device)


@noise.register_fake
def _(rows, cols, seed, row0, dtype, device):
    return torch.empty((rows, cols), dtype=dtype, device=device)


# ------------------------------------------------------------------------------------------------
# cross entropy over a large vocabulary
# ------------------------------------------------------------------------------------------------
class _Once(torch.autograd.Function):
    """A gradient whose own gradient does not exist: it says so when it is asked for."""

    @staticmethod
    def forward(ctx, t):
        return t.view_as(t)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("cross entropy: second derivatives are not implemented")


def _first_order(backward):
    """Marks the gradients that ``backward`` returns under create_graph=True.  (torch's once_differentiable does that only where the
    incoming gradient takes part in autograd; that of a loss does not, and a penalty on the gradient would drop out silently.)"""
    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        again = torch.is_grad_enabled()
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not again:
            return out
        return tuple(_Once.apply(t.detach().requires_grad_()) if isinstance(t, torch.Tensor) else t for t in out)
    return wrapper


@custom_op("rten::noise_ce_fwd", mutates_args=(), device_types="cuda")
def noise_ce_fwd(z: torch.Tensor, target: torch.Tensor, seed: int, out_features: int, row0: int, ignore_index: Optional[int], reduction: str,
                 need_grad: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    loss, aux, unit = K.ce_fwd(z, None, target, ignore_index, reduction, seed, out_features, row0, need_grad)
    return loss, aux, unit if unit is not None else aux.new_empty((0,))


@noise_ce_fwd.register_fake
def _(z, target, seed, out_features, row0, ignore_index, reduction, need_grad):
    T = z.shape[0]
    return (z.new_empty((T,) if reduction == "none" else (), dtype=torch.float32), z.new_empty((2 * T + 1,), dtype=torch.float32),
            z.new_empty(z.shape if need_grad else (0,), dtype=torch.float32))


noise_ce_fwd.register_kernel("cpu")(_cpu_raises("noise_ce_fwd"))


@custom_op("rten::noise_ce_bwd", mutates_args=(), device_types="cuda")
def noise_ce_bwd(dloss: torch.Tensor, unit: torch.Tensor, aux: torch.Tensor, reduction: str, dtype: torch.dtype) -> torch.Tensor:
    return K.ce_scale(unit, dloss, aux, reduction, dtype)


@noise_ce_bwd.register_fake
def _(dloss, unit, aux, reduction, dtype):
    return torch.empty_like(unit, dtype=dtype)


noise_ce_bwd.register_kernel("cpu")(_cpu_raises("noise_ce_bwd"))


def _noise_ce_setup(ctx, inputs, output):
    _, aux, unit = output
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(aux, unit)
    ctx.save_for_backward(aux, unit)
    ctx.reduction, ctx.has_unit, ctx.dtype = inputs[6], inputs[7], inputs[0].dtype


@_first_order
def _noise_ce_backward(ctx, dloss, daux, dunit):
    aux, unit = ctx.saved_tensors
    if dloss is None or not ctx.needs_input_grad[0]:
        return (None,) * 8
    if not ctx.has_unit:
        raise RuntimeError("noise_ce_fwd was called with need_grad=False: it kept nothing for a backward pass")
    return (noise_ce_bwd(dloss, unit, aux, ctx.reduction, ctx.dtype),) + (None,) * 7


noise_ce_fwd.register_autograd(_noise_ce_backward, setup_context=_noise_ce_setup)


@custom_op("rten::linear_ce_fwd", mutates_args=(), device_types="cuda")
def linear_ce_fwd(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: Optional[int], reduction: str
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    loss, aux, _ = K.ce_fwd(x, weight, target, ignore_index, reduction)
    return loss, aux


@linear_ce_fwd.register_fake
def _(x, weight, target, ignore_index, reduction):
    T = x.shape[0]
    return x.new_empty((T,) if reduction == "none" else (), dtype=torch.float32), x.new_empty((2 * T + 1,), dtype=torch.float32)


linear_ce_fwd.register_kernel("cpu")(_cpu_raises("linear_ce_fwd"))


@custom_op("rten::linear_ce_bwd", mutates_args=(), device_types="cuda")
def linear_ce_bwd(dloss: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, aux: torch.Tensor, ignore_index: Optional[int],
                  reduction: str, need_dx: bool, need_dw: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    dx, dw = K.ce_bwd(dloss, x, weight, target, aux, ignore_index, reduction, need_dx, need_dw)
    return dx if dx is not None else x.new_empty((0,)), dw if dw is not None else weight.new_empty((0,))


@linear_ce_bwd.register_fake
def _(dloss, x, weight, target, aux, ignore_index, reduction, need_dx, need_dw):
    return x.new_empty(x.shape if need_dx else (0,)), weight.new_empty(weight.shape if need_dw else (0,))


linear_ce_bwd.register_kernel("cpu")(_cpu_raises("linear_ce_bwd"))


def _linear_ce_setup(ctx, inputs, output):
    x, weight, target, ctx.ignore_index, ctx.reduction = inputs
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, weight, target, output[1])


@_first_order
def _linear_ce_backward(ctx, dloss, daux):
    x, weight, target, aux = ctx.saved_tensors
    need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
    if dloss is None or not (need_dx or need_dw):
        return (None,) * 5
    dx, dw = linear_ce_bwd(dloss, x, weight, target, aux, ctx.ignore_index, ctx.reduction, need_dx, need_dw)
    return dx if need_dx else None, dw if need_dw else None, None, None, None


linear_ce_fwd.register_autograd(_linear_ce_backward, setup_context=_linear_ce_setup)


@custom_op("rten::matmul_nt_fwd", mutates_args=(), device_types="cuda")
def matmul_nt_fwd(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    return K.gemm_dense(a.contiguous(), b.contiguous(), True, True)


@matmul_nt_fwd.register_fake
def _(a, b):
    return a.new_empty((a.shape[0], b.shape[0]))


matmul_nt_fwd.register_kernel("cpu")(_cpu_raises("matmul_nt_fwd"))


@custom_op("rten::matmul_nt_bwd", mutates_args=(), device_types="cuda")
def matmul_nt_bwd(grad: torch.Tensor, a: torch.Tensor, b: torch.Tensor, need_da: bool, need_db: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    da, db = _matmul_nt_grads(grad, a, b, need_da, need_db)
    return da if need_da else a.new_empty((0,)), db if need_db else b.new_empty((0,))


@matmul_nt_bwd.register_fake
def _(grad, a, b, need_da, need_db):
    return a.new_empty(a.shape if need_da else (0,)), b.new_empty(b.shape if need_db else (0,))


matmul_nt_bwd.register_kernel("cpu")(_cpu_raises("matmul_nt_bwd"))


def _matmul_nt_grads(grad, a, b, need_da, need_db):
    grad = grad.contiguous()
    return (K.gemm_dense(grad, b.contiguous(), True, False) if need_da else None,       # grad @ b
            K.gemm_dense(grad, a.contiguous(), False, False) if need_db else None)      # grad^T @ a


@_first_order
def _matmul_nt_backward(ctx, grad):
    a, b = ctx.saved_tensors
    need_da, need_db = ctx.needs_input_grad
    da, db = matmul_nt_bwd(grad, a, b, need_da, need_db)
    return da if need_da else None, db if need_db else None


matmul_nt_fwd.register_autograd(_matmul_nt_backward, setup_context=lambda ctx, inputs, output: ctx.save_for_backward(*inputs))


def _eager(*ts: torch.Tensor) -> bool:
    """Plain CUDA tensors outside of any tracing and of torch.func's transforms: the kernels can be called without going through the
    dispatcher, which costs more than they do on small problems."""
    return not torch.compiler.is_compiling() and all([t.is_cuda and type(t) in (torch.Tensor, torch.nn.Parameter) for t in ts]) \
        and not torch._C._len_torch_dispatch_stack() and not torch._C._are_functorch_transforms_active()


def _no_tangents(*ts: torch.Tensor) -> None:
    """Forward-mode differentiation is not implemented: raises where a tangent would be dropped."""
    if forward_ad._current_level >= 0 and any([forward_ad.unpack_dual(t).tangent is not None for t in ts]):
        raise RuntimeError("cross entropy: forward-mode differentiation is not implemented")


class _NoiseCE(torch.autograd.Function):
    """noise_ce_fwd / noise_ce_bwd for eager calls that take part in autograd."""

    @staticmethod
    def forward(ctx, z, target, seed, out_features, row0, ignore_index, reduction):
        loss, aux, unit = K.ce_fwd(z, None, target, ignore_index, reduction, seed, out_features, row0, True)
        ctx.save_for_backward(aux, unit)
        ctx.reduction, ctx.dtype = reduction, z.dtype
        return loss

    @staticmethod
    @_first_order
    def backward(ctx, dloss):
        aux, unit = ctx.saved_tensors
        return K.ce_scale(unit, dloss, aux, ctx.reduction, ctx.dtype), None, None, None, None, None, None


class _LinearCE(torch.autograd.Function):
    """linear_ce_fwd / linear_ce_bwd for eager calls that take part in autograd."""

    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        loss, aux, _ = K.ce_fwd(x, weight, target, ignore_index, reduction)
        ctx.save_for_backward(x, weight, target, aux)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @_first_order
    def backward(ctx, dloss):
        x, weight, target, aux = ctx.saved_tensors
        dx, dw = K.ce_bwd(dloss, x, weight, target, aux, ctx.ignore_index, ctx.reduction, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx, dw, None, None, None


class _MatmulNT(torch.autograd.Function):
    """a[L, P] @ b[Q, P].T on the library's product kernels: matmul_nt_fwd / matmul_nt_bwd for eager calls that take part in autograd."""

    @staticmethod
    def forward(ctx, a, b):
        ctx.save_for_backward(a, b)
        return K.gemm_dense(a.contiguous(), b.contiguous(), True, True)

    @staticmethod
    @_first_order
    def backward(ctx, grad):
        return _matmul_nt_grads(grad, *ctx.saved_tensors, *ctx.needs_input_grad)


def noise_cross_entropy(z: torch.Tensor, seed: int, out_features: int, target: torch.Tensor, row0: int = 0, ignore_index: Optional[int] = -100,
                        reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits ``z @ S[row0:row0 + out_features].T`` (noise of ``seed`` in z's type) against ``target``,
    for z of shape [..., R] and int64 target of shape [...]; differentiable in z.

    The logits are never kept: the loss and, when z takes part in autograd, its gradient come out of one pass over the noise in
    pieces.  Rows whose target is ``ignore_index`` (None: no such value) count for nothing, whatever they contain; any other
    target outside [0, out_features) makes its row's loss and gradient NaN.  Returns float32: a scalar for reduction "mean" (over
    the rows that count; NaN when there are none) and "sum", the rows' losses in target's shape for "none"."""
    lead = z.shape[:-1]
    if tuple(target.shape) != tuple(lead):
        raise RuntimeError(f"noise_cross_entropy: target {tuple(target.shape)} does not match z {tuple(z.shape)}")
    _no_tangents(z)
    z2, t = z.reshape(-1, z.shape[-1]), target.reshape(-1)
    need = torch.is_grad_enabled() and z.requires_grad
    if not _eager(z2, t):
        loss = noise_ce_fwd(z2, t, seed, out_features, row0, ignore_index, reduction, need)[0]
    elif need:
        loss = _NoiseCE.apply(z2, t, seed, out_features, row0, ignore_index, reduction)
    else:
        loss = K.ce_fwd(z2, None, t, ignore_index, reduction, seed, out_features, row0)[0]
    return loss.reshape(lead) if reduction == "none" else loss


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: Optional[int] = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits ``x @ weight.T`` against ``target``, for x of shape [..., K], weight [V, K] of the same
    type and int64 target of shape [...]; differentiable in x and weight.  The logits are never kept: the backward recomputes
    them in pieces of the vocabulary.  ignore_index, other targets, reduction and result as ``noise_cross_entropy``."""
    lead = x.shape[:-1]
    if tuple(target.shape) != tuple(lead):
        raise RuntimeError(f"linear_cross_entropy: target {tuple(target.shape)} does not match x {tuple(x.shape)}")
    _no_tangents(x, weight)
    x2, t = x.reshape(-1, x.shape[-1]), target.reshape(-1)
    if not _eager(x2, weight, t):
        loss = linear_ce_fwd(x2, weight, t, ignore_index, reduction)[0]
    elif torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        loss = _LinearCE.apply(x2, weight, t, ignore_index, reduction)
    else:
        loss = K.ce_fwd(x2, weight, t, ignore_index, reduction)[0]
    return loss.reshape(lead) if reduction == "none" else loss


def rlinear_cross_entropy(x: torch.Tensor, coef: torch.Tensor, seed: int, out_features: int, target: torch.Tensor, row0: int = 0,
                          ignore_index: Optional[int] = -100, reduction: str = "mean") -> torch.Tensor:
    """``cross_entropy(rlinear(x, coef, seed, out_features, row0), target)`` without the logits: z = x C^T (rounded to x's type, as
    the layer's forward keeps it), then ``noise_cross_entropy``; differentiable in x and coef.  Rows of x whose target is ignored
    are taken as zeros, so whatever they hold reaches neither the loss nor a gradient."""
    lead = x.shape[:-1]
    if tuple(target.shape) != tuple(lead):
        raise RuntimeError(f"rlinear_cross_entropy: target {tuple(target.shape)} does not match x {tuple(x.shape)}")
    if coef.dim() != 2 or coef.shape[1] != x.shape[-1] or coef.dtype != x.dtype:
        raise RuntimeError(f"rlinear_cross_entropy: coef {tuple(coef.shape)} {coef.dtype} does not match x {tuple(x.shape)} {x.dtype}")
    _no_tangents(x, coef)
    x2 = x.reshape(-1, x.shape[-1])
    if ignore_index is not None:
        x2 = x2.masked_fill((target.reshape(-1) == ignore_index).unsqueeze(1), 0.0)
    z = _MatmulNT.apply(x2, coef) if _eager(x2, coef) else matmul_nt_fwd(x2, coef)
    loss = noise_cross_entropy(z, seed, out_features, target.reshape(-1), row0, ignore_index, reduction)
    return loss.reshape(lead) if reduction == "none" else loss


# ------------------------------------------------------------------------------------------------
# reference operators (1-D coefficient vector)
# ------------------------------------------------------------------------------------------------
@custom_op("rten::materialize_fwd", mutates_args=(), device_types="cuda")
def materialize_fwd(coefs: torch.Tensor, size: List[int], strides: List[int], seed: int,
                    scale_bias: Optional[torch.Tensor], fused_bias: bool) -> torch.Tensor:
    assert not (fused_bias and scale_bias is None), "scale_bias not initialized but fused_bias is True"
    sb = scale_bias.detach().reshape(1).float().contiguous() if fused_bias else None
    return K.materialize_fwd(coefs.float().contiguous(), size, strides, seed, sb)


@materialize_fwd.register_fake
def _(coefs, size, strides, seed, scale_bias, fused_bias):
    return coefs.new_empty(size, dtype=torch.float32)


materialize_fwd.register_kernel("cpu")(_cpu_raises("materialize_fwd"))


@custom_op("rten::materialize_bwd", mutates_args=(), device_types="cuda")
def materialize_bwd(dout: torch.Tensor, dcoefs_size: int, seed: int) -> torch.Tensor:
    assert dout.is_contiguous(), "dout is not contiguous, backwards pass might give incorrect results."
    return K.materialize_bwd(dout, dcoefs_size, seed)


@materialize_bwd.register_fake
def _(dout, dcoefs_size, seed):
    return dout.new_empty((dcoefs_size,), dtype=torch.float32)


materialize_bwd.register_kernel("cpu")(_cpu_raises("materialize_bwd"))


@custom_op("rten::scale_bias_bwd", mutates_args=(), device_types="cuda")
def scale_bias_bwd(dout: torch.Tensor, seed: int) -> torch.Tensor:
    assert dout.is_contiguous(), "dout is not contiguous, backwards pass might give incorrect results."
    return K.scale_bias_bwd(dout, seed)


@scale_bias_bwd.register_fake
def _(dout, seed):
    return dout.new_empty((1,), dtype=torch.float32)


scale_bias_bwd.register_kernel("cpu")(_cpu_raises("scale_bias_bwd"))


def _mat_setup(ctx, inputs, output):
    coefs, size, strides, seed, scale_bias, fused_bias = inputs
    ctx.dcoefs_size = coefs.numel()
    ctx.seed = seed
    ctx.coef_dtype = coefs.dtype
    ctx.fused_bias = fused_bias
    ctx.bias_dtype = scale_bias.dtype if scale_bias is not None else None
    ctx.bias_shape = scale_bias.shape if scale_bias is not None else None
    ctx.view_size, ctx.view_strides = list(size), list(strides)


def _natural_order(grad: torch.Tensor, size: List[int], strides: List[int]) -> torch.Tensor:
    """Gradient of a strided view, laid out in the order of the virtual tensor's own elements.

    Element ``n`` of the virtual tensor always uses noise row ``n``; a view (a transpose, say) only changes which ``n`` sits
    at which output position: ``sq = sum_d index_d * stride_d`` (src/rten_cpp/RandumbTensor.py:264).  The backward kernels
    walk the noise rows in order (:304-359), so the incoming gradient is scattered back to ``flat[sq]`` first; positions
    the view does not reach keep a zero gradient."""
    expect, acc = [], 1
    for d in reversed(size):
        expect.append(acc)
        acc *= d
    if list(strides) == list(reversed(expect)):
        return grad.contiguous()
    extent = 1 + sum((d - 1) * st for d, st in zip(size, strides)) if all(d > 0 for d in size) else 0
    flat = grad.new_zeros((extent,))
    flat.as_strided(size, strides).copy_(grad)
    return flat


def _mat_backward(ctx, grad):
    grad = _natural_order(grad, ctx.view_size, ctx.view_strides)
    dcoefs = materialize_bwd(grad, ctx.dcoefs_size, ctx.seed).to(ctx.coef_dtype)
    dscale_bias = None
    if ctx.fused_bias:
        dscale_bias = scale_bias_bwd(grad, ctx.seed).to(ctx.bias_dtype).reshape(ctx.bias_shape)
    return dcoefs, None, None, None, dscale_bias, None


materialize_fwd.register_autograd(_mat_backward, setup_context=_mat_setup)


# ------------------------------------------------------------------------------------------------
# embedding rows of a virtual (vocab, rowsize) matrix (reference: RandumbTensor.py:1121-1160)
# ------------------------------------------------------------------------------------------------
@custom_op("rten::embed_fwd", mutates_args=(), device_types="cuda")
def embed_fwd(idx: torch.Tensor, coefs: torch.Tensor, rowsize: int, seed: int) -> torch.Tensor:
    return K.embed_fwd(idx, coefs.float().contiguous(), rowsize, seed)


@embed_fwd.register_fake
def _(idx, coefs, rowsize, seed):
    return coefs.new_empty((*idx.shape, rowsize), dtype=torch.float32)


embed_fwd.register_kernel("cpu")(_cpu_raises("embed_fwd"))


@custom_op("rten::embed_bwd", mutates_args=(), device_types="cuda")
def embed_bwd(idx: torch.Tensor, dout: torch.Tensor, dcoefs_size: int, rowsize: int, seed: int) -> torch.Tensor:
    return K.embed_bwd(idx, dout.contiguous(), dcoefs_size, rowsize, seed)


@embed_bwd.register_fake
def _(idx, dout, dcoefs_size, rowsize, seed):
    return dout.new_empty((dcoefs_size,), dtype=torch.float32)


embed_bwd.register_kernel("cpu")(_cpu_raises("embed_bwd"))


def _embed_setup(ctx, inputs, output):
    idx, coefs, rowsize, seed = inputs
    ctx.save_for_backward(idx)
    ctx.dcoefs_size = coefs.numel()
    ctx.rowsize = rowsize
    ctx.seed = seed
    ctx.coef_dtype = coefs.dtype


def _embed_backward(ctx, grad):
    (idx,) = ctx.saved_tensors
    dcoefs = embed_bwd(idx, grad.contiguous(), ctx.dcoefs_size, ctx.rowsize, ctx.seed).to(ctx.coef_dtype)
    return None, dcoefs, None, None


embed_fwd.register_autograd(_embed_backward, setup_context=_embed_setup)


def rt_mm(mat1: torch.Tensor, coefs: torch.Tensor, size: List[int], strides: List[int], seed: int,
          scale_bias: Optional[torch.Tensor] = None, fused_bias: bool = False) -> torch.Tensor:
    """``mat1[L, P] @ RT[P, Q]`` for a RandumbTensor in the 1-D coefficient form, same call as the reference's
    experimental ``rt_mm`` / ``rt_mm_grouped`` (src/rten_cpp/RandumbTensor.py:634-645, 758-769).

    Every element of RT costs ``M`` hashes, so regenerating RT tiles inside a product would repeat that work once
    per row block of ``mat1``; RT is materialised once (``rten::materialize_fwd``, differentiable in ``coefs`` and
    ``scale_bias``) and multiplied by the library's own product kernels (differentiable in ``mat1``).
    """
    P, Q = size
    assert mat1.dim() == 2 and mat1.size(1) == P, f"mm shape mismatch, received mat1 shape {tuple(mat1.size())} and rt shape {size}"
    rt = materialize_fwd(coefs, list(size), list(strides), seed, scale_bias, fused_bias)
    return _DenseMM.apply(mat1, rt.to(mat1.dtype))


class _DenseMM(torch.autograd.Function):
    """a[L, P] @ b[P, Q] on the library's product kernels (tensor cores for bf16, CUDA cores for float32)."""

    @staticmethod
    def forward(ctx, a, b):
        ctx.save_for_backward(a, b)
        return K.gemm_dense(a.contiguous(), b.contiguous(), True, False)

    @staticmethod
    def backward(ctx, grad):
        a, b = ctx.saved_tensors
        grad = grad.contiguous()
        da = K.gemm_dense(grad, b.contiguous(), True, True) if ctx.needs_input_grad[0] else None      # grad @ b^T
        db = K.gemm_dense(a.contiguous(), grad, False, False) if ctx.needs_input_grad[1] else None   # a^T @ grad
        return da, db


# C++-namespace twins of the reference (rten.cpp:36-39); registered from Python onto the same C ABI.
@custom_op("rten_cpp::sq5_gen_2d", mutates_args=())
def sq5_gen_2d(M: int, N: int, seed: int) -> torch.Tensor:
    return K.noise(M, N, seed, 0, 0, torch.float32, torch.device("cuda", torch.cuda.current_device()))


@sq5_gen_2d.register_fake
def _(M, N, seed):
    return torch.empty((M, N), dtype=torch.float32, device="cuda")


@custom_op("rten_cpp::materialize_fwd", mutates_args=(), device_types="cuda")
def materialize_fwd_cpp(coef: torch.Tensor, seed: int, P: int, Q: int, stride_P: int, stride_Q: int) -> torch.Tensor:
    assert coef.dim() == 1 and coef.is_contiguous()
    return K.materialize_fwd(coef.float(), [P, Q], [stride_P, stride_Q], seed)


@materialize_fwd_cpp.register_fake
def _(coef, seed, P, Q, stride_P, stride_Q):
    return coef.new_empty((P, Q), dtype=torch.float32)
