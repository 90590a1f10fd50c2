"""PyTorch custom operators and modules over hipgemm_amd.dense: products of 16-bit
activations with 16-bit weights, with gradients.

Importing this module registers, in the ``hipgemm`` namespace:

  torch.ops.hipgemm.linear(x, weight, bias=None, activation="none", residual=None,
                           out_dtype=None) -> Tensor
  torch.ops.hipgemm.gated_linear(x, weight, bias=None, activation="silu",
                                 out_dtype=None) -> Tensor

with the arguments and rules of the functions of the same names (but an x, weight and
bias of any strides and alignment, which are copied where they have to be), and fake
(meta) implementations, so that they trace under torch.compile, torch.export and
FakeTensorMode.  They may be captured in CUDA graphs.  CPU tensors raise HipGemmError:
there is no CPU path.

linear and gated_linear here are differentiable, once and in reverse mode: where a gradient
is wanted the forward pass keeps z in float32 (linear only with an activation) and the
backward pass is hipgemm's linear_backward or gated_linear_backward.  Gradients come in
their tensors' types; sums and z are fp32, dz is rounded to x's type.  The operators
themselves record no gradient.  Tensors with a tangent of forward mode raise HipGemmError,
and the operators wherever forward mode is on.  A backward pass may be captured into
a graph, with leaves of its own: p.detach().requires_grad_() of each parameter, over the same
memory.  (Leaves that an eager graph still alive has too end the process inside torch at the
capture's end, whatever the operators: their accumulation belongs to that graph's stream.)

DenseLinear   torch.nn.Linear with an activation and a residual in its epilogue
GatedMLP      the feed-forward half of a layer: x + down(act(gate(x)) * up(x))
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from . import ACTIVATIONS, HipGemmError, dense
from .torch_ops import _plain_buffers, _plain_eager
from .torch_serving import _rows as _aligned_rows

__all__ = ["linear", "gated_linear", "DenseLinear", "GatedMLP"]


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x where its rows are as the products take them, else a copy: also of rows further apart
    than they address, as the last token's of each of several long sequences."""
    if x.dim() == 2 and x.shape[0] > 1 and x.stride(0) > dense._MAX_LD:
        return x.clone(memory_format=torch.contiguous_format)
    return _aligned_rows(x)


def _unit(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t where its last dimension has unit stride and its rows do not overlap, else a copy."""
    if t is None or t.numel() == 0:
        return t
    if t.dim() == 1:
        return t.contiguous()
    if t.stride(1) == 1 and (t.shape[0] == 1 or t.stride(0) >= t.shape[1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_shapes(x, weight, bias, activation, residual, gated):
    if activation not in ACTIVATIONS:
        raise HipGemmError(f"unknown activation {activation!r}")
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]:
        raise HipGemmError(f"K mismatch: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    n = weight.shape[0]
    if gated and n % 16:
        raise HipGemmError("weight must have 2 N rows, N a multiple of 8")
    if bias is not None and tuple(bias.shape) != (n,):
        raise HipGemmError(f"bias must have {n} elements")
    n = n // 2 if gated else n
    if residual is not None and tuple(residual.shape) != (x.shape[0], n):
        raise HipGemmError(f"residual must be {(x.shape[0], n)}, got {tuple(residual.shape)}")
    return n


def _fake_shapes(x, weight, bias, activation, residual, out_dtype, gated):
    """_check_shapes, and what the kernels refuse by types and devices: a trace refuses what
    the call itself would."""
    n = _check_shapes(x, weight, bias, activation, residual, gated)
    operands, inputs, outputs = dense._types()
    if x.dtype not in operands or weight.dtype != x.dtype:
        raise HipGemmError(f"x and weight must both be bfloat16 or float16, got {x.dtype} and "
                           f"{weight.dtype}")
    if x.shape[1] % 8:
        raise HipGemmError(f"K must be a multiple of 8, got {x.shape[1]}")
    for name, t in (("bias", bias), ("residual", residual)):
        if t is not None and t.dtype not in inputs:
            raise HipGemmError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if out_dtype is not None and out_dtype not in outputs:
        raise HipGemmError("out_dtype must be bfloat16, float16 or float32")
    if any(t is not None and t.device != x.device for t in (weight, bias, residual)):
        raise HipGemmError(f"all tensors must be on {x.device}")
    return n


def _refuse_tangents():
    raise HipGemmError("linear and gated_linear have no forward-mode derivative")


def _tangents(*tensors) -> bool:
    """A tensor carries a tangent, or hides behind a transform whether it does; call it where
    forward mode is on."""
    return any(t is not None and (torch._C._functorch.is_functorch_wrapped_tensor(t)
                                  or forward_ad.unpack_dual(t).tangent is not None)
               for t in tensors)


def _forward_mode() -> bool:
    return forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()


def _op_checks():
    """What an operator's body is given has lost its tangents, and torch would take them for
    zeros.  (Calls whose tensors have been looked at turn forward mode off.)"""
    if _forward_mode():
        _refuse_tangents()


@torch.library.custom_op("hipgemm::linear", mutates_args=())
def _linear_op(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               activation: str = "none", residual: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    _op_checks()
    return dense.linear(_rows(x), _rows(weight), bias=_unit(bias), activation=activation,
                        residual=_unit(residual), out_dtype=out_dtype)


@_linear_op.register_fake
def _linear_fake(x, weight, bias=None, activation="none", residual=None, out_dtype=None):
    n = _fake_shapes(x, weight, bias, activation, residual, out_dtype, False)
    return x.new_empty((x.shape[0], n), dtype=out_dtype or x.dtype)


@torch.library.custom_op("hipgemm::gated_linear", mutates_args=())
def _gated_op(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
              activation: str = "silu", out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    _op_checks()
    return dense.gated_linear(_rows(x), _rows(weight), bias=_unit(bias), activation=activation,
                              out_dtype=out_dtype)


@_gated_op.register_fake
def _gated_fake(x, weight, bias=None, activation="silu", out_dtype=None):
    n = _fake_shapes(x, weight, bias, activation, None, out_dtype, True)
    return x.new_empty((x.shape[0], n), dtype=out_dtype or x.dtype)


# The pair that autograd records: the forward pass with its z, and the backward pass.

@torch.library.custom_op("hipgemm::linear_with_pre", mutates_args=())
def _linear_pre(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                activation: str, residual: Optional[torch.Tensor],
                out_dtype: Optional[torch.dtype],
                gated: bool) -> tuple[torch.Tensor, torch.Tensor]:
    _op_checks()
    x, weight, bias = _rows(x), _rows(weight), _unit(bias)
    if gated:
        return dense.gated_linear(x, weight, bias=bias, activation=activation,
                                  out_dtype=out_dtype, save_pre=True)
    if not ACTIVATIONS[activation]:  # nothing to keep
        y = dense.linear(x, weight, bias=bias, residual=_unit(residual), out_dtype=out_dtype)
        return y, x.new_empty(0, dtype=torch.float32)
    return dense.linear(x, weight, bias=bias, activation=activation, residual=_unit(residual),
                        out_dtype=out_dtype, save_pre=True)


@_linear_pre.register_fake
def _linear_pre_fake(x, weight, bias, activation, residual, out_dtype, gated):
    n = _fake_shapes(x, weight, bias, activation, residual, out_dtype, gated)
    pre = (x.shape[0], weight.shape[0]) if gated or ACTIVATIONS[activation] else (0,)
    return (x.new_empty((x.shape[0], n), dtype=out_dtype or x.dtype),
            x.new_empty(pre, dtype=torch.float32))


@torch.library.custom_op("hipgemm::linear_backward", mutates_args=())
def _linear_grad(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, pre: torch.Tensor,
                 activation: str, gated: bool, need_x: bool, need_weight: bool,
                 need_bias: bool, bias_dtype: torch.dtype
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _op_checks()
    back = dense.gated_linear_backward if gated else dense.linear_backward
    dx, dw, db = back(_unit(dy), _rows(x), _rows(weight), pre if pre.dim() == 2 else None,
                      activation=activation, need_x=need_x, need_weight=need_weight,
                      need_bias=need_bias, bias_dtype=bias_dtype)
    none = x.new_empty(0)
    return (none if dx is None else dx, none.clone() if dw is None else dw,
            none.clone() if db is None else db)


@_linear_grad.register_fake
def _linear_grad_fake(dy, x, weight, pre, activation, gated, need_x, need_weight, need_bias,
                      bias_dtype):
    return (x.new_empty(tuple(x.shape) if need_x else (0,)),
            weight.new_empty(tuple(weight.shape) if need_weight else (0,)),
            weight.new_empty((weight.shape[0],) if need_bias else (0,),
                             dtype=bias_dtype if need_bias else None))


def _setup(ctx, inputs, output):
    x, weight, bias, ctx.activation, residual, _, ctx.gated = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.bias_dtype = x.dtype if bias is None else bias.dtype
    ctx.residual_dtype = None if residual is None else residual.dtype
    ctx.mark_non_differentiable(output[1])
    # z has no gradient: none is made (zeros of z's size, in float32, for every pass).
    ctx.set_materialize_grads(False)


def _backward(ctx, dy, _):
    x, weight, pre = ctx.saved_tensors
    if _forward_mode():
        if _tangents(dy, x, weight):
            _refuse_tangents()
        with forward_ad._set_fwd_grad_enabled(False):
            return _backward(ctx, dy, _)
    need = ctx.needs_input_grad
    dx = dw = db = dr = None
    if dy is None:
        return (None,) * 7
    if any(need[:3]):
        dx, dw, db = torch.ops.hipgemm.linear_backward(
            dy, x, weight, pre, ctx.activation, ctx.gated, need[0], need[1], need[2],
            ctx.bias_dtype)
    if need[4]:
        dr = dy.to(ctx.residual_dtype)
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, dr,
            None, None)


_linear_pre.register_autograd(_backward, setup_context=_setup)


def _wanted(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _call(x, weight, bias, activation, residual, out_dtype, gated):
    if _forward_mode():
        if _tangents(x, weight, bias, residual):
            _refuse_tangents()
        with forward_ad._set_fwd_grad_enabled(False):
            return _call(x, weight, bias, activation, residual, out_dtype, gated)
    activation = activation or "none"
    if x.dim() != 2:
        lead = x.shape[:-1]
        if residual is not None:
            if residual.shape[:-1] != lead:
                raise HipGemmError(f"residual must be {(*lead, weight.shape[0])}, got "
                                   f"{tuple(residual.shape)}")
            residual = residual.unsqueeze(0).flatten(0, -2)
        y = _call(x.unsqueeze(0).flatten(0, -2), weight, bias, activation, residual, out_dtype,
                  gated)
        return y.reshape(*lead, y.shape[-1])
    _check_shapes(x, weight, bias, activation, residual, gated)
    if _wanted(x, weight, bias, residual):
        return torch.ops.hipgemm.linear_with_pre(x, weight, bias, activation, residual, out_dtype,
                                                 gated)[0]
    # (the call itself where nothing watches the operations, as in Fp8Linear)
    if _plain_eager(x) and _plain_buffers(weight, bias, residual):
        x, weight, bias = _rows(x), _rows(weight), _unit(bias)
        if gated:
            return dense.gated_linear(x, weight, bias=bias, activation=activation,
                                      out_dtype=out_dtype)
        return dense.linear(x, weight, bias=bias, activation=activation,
                            residual=_unit(residual), out_dtype=out_dtype)
    if gated:
        return torch.ops.hipgemm.gated_linear(x, weight, bias, activation, out_dtype)
    return torch.ops.hipgemm.linear(x, weight, bias, activation, residual, out_dtype)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x @ weight.T + bias) + residual, differentiable in all four (hipgemm_amd.linear).
    x (..., K), residual (..., N)."""
    return _call(x, weight, bias, activation, residual, out_dtype, False)


def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 activation: Optional[str] = "silu",
                 out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(gate) * up, [gate | up] = x @ weight.T + bias, differentiable
    (hipgemm_amd.gated_linear).  x (..., K), weight (2N, K): gate rows, then up rows."""
    return _call(x, weight, bias, activation, None, out_dtype, True)


class DenseLinear(torch.nn.Module):
    """y = act(x W^T + b) [+ residual] with W (out x in) and x bfloat16 or float16, trainable.
    in_features must be a multiple of 8."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 activation: Optional[str] = None, device=None,
                 dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if in_features % 8:
            raise HipGemmError("in_features must be a multiple of 8")
        if activation not in ACTIVATIONS:
            raise HipGemmError(f"unknown activation {activation!r}")
        like = torch.nn.Linear(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.weight, self.bias = like.weight, like.bias
        self.activation = activation or "none"

    @property
    def in_features(self) -> int:
        return self.weight.shape[1]

    @property
    def out_features(self) -> int:
        return self.weight.shape[0]

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, activation: Optional[str] = None):
        """With a Linear's own parameters."""
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, activation,
                device="meta", dtype=linear.weight.dtype)
        m.weight, m.bias = linear.weight, linear.bias
        return m

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise HipGemmError(f"x must have {self.in_features} features, got {tuple(x.shape)}")
        return linear(x, self.weight, self.bias, self.activation, residual)


class GatedMLP(torch.nn.Module):
    """residual + down(act(gate(x)) * up(x)): two calls, gated_linear and linear with the
    residual in its epilogue.  w13 (2 hidden x dim): gate rows, then up rows, as in MoE; w2
    (dim x hidden); dim and hidden multiples of 8.  Trainable."""

    def __init__(self, dim: int, hidden: int, activation: Optional[str] = "silu", device=None,
                 dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if dim % 8 or hidden % 8:
            raise HipGemmError("dim and hidden must be multiples of 8")
        if activation not in ACTIVATIONS:
            raise HipGemmError(f"unknown activation {activation!r}")

        def weight(n, k):
            return torch.nn.Linear(k, n, bias=False, device=device, dtype=dtype).weight

        self.w13, self.w2 = weight(2 * hidden, dim), weight(dim, hidden)
        self.activation = activation or "none"

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.shape[-1] != self.w13.shape[1]:
            raise HipGemmError(f"x must have {self.w13.shape[1]} features, got {tuple(x.shape)}")
        h = gated_linear(x, self.w13, activation=self.activation)
        return linear(h, self.w2, residual=residual)
