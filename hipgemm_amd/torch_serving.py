"""PyTorch custom operators and modules over hipgemm_amd.serving: products with
4-bit weights and mixture-of-experts layers.

Importing this module registers, in the ``hipgemm`` namespace:

  torch.ops.hipgemm.w4_gemm(x, weight, scales, zeros=None, format="int4",
                            group_size=128, bias=None, activation="none",
                            out_dtype=None)
  torch.ops.hipgemm.moe_route(logits, k, scoring="softmax", renormalize=True,
                              scale=1.0) -> (weights, ids)
  torch.ops.hipgemm.moe_experts(x, ids, weights, w13, scales13, w2, scales2,
                                zeros13=None, zeros2=None, format="e4m3",
                                group_size=128, activation="silu",
                                out_dtype=None)

with the arguments and rules of the functions of the same names (but an x of any
strides and alignment, which is copied where it has to be), and fake (meta)
implementations, so that they trace under torch.compile, torch.export and
FakeTensorMode.  They may be captured in CUDA graphs.  CPU tensors raise
HipGemmError: there is no CPU path.  They record no gradient.

W4Linear   torch.nn.Linear with 4-bit weights
MoE        a mixture-of-experts layer: router, choice of experts, gated MLPs

quantize_w4 packs a weight for them.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ACTIVATIONS, HipGemmError
from . import serving
from .torch_ops import _plain_buffers, _plain_eager, quantize_rows

__all__ = ["w4_gemm", "moe_route", "moe_experts", "quantize_w4", "W4Linear", "MoE"]


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x where its rows are as the kernels take them (unit stride, on 16 bytes), else
    a copy: views of any strides are what a Linear is given."""
    if (x.dim() == 2 and x.stride(1) == 1 and x.data_ptr() % 16 == 0 and
            (x.shape[0] <= 1 or (x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1]))):
        return x
    return x.clone(memory_format=torch.contiguous_format)


@torch.library.custom_op("hipgemm::w4_gemm", mutates_args=())
def w4_gemm(x: torch.Tensor, weight: torch.Tensor, scales: torch.Tensor,
            zeros: Optional[torch.Tensor] = None, format: str = "int4",
            group_size: int = 128, bias: Optional[torch.Tensor] = None,
            activation: str = "none",
            out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return serving.w4_gemm(_rows(x), weight, scales, zeros, format=format,
                           group_size=group_size, bias=bias,
                           activation=activation, out_dtype=out_dtype)


@w4_gemm.register_fake
def _w4_gemm_fake(x, weight, scales, zeros=None, format="int4", group_size=128,
                  bias=None, activation="none", out_dtype=None):
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != 2 * weight.shape[1]:
        raise HipGemmError(f"K mismatch: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    if format not in serving.W4_FORMATS:
        raise HipGemmError(f"unknown format {format!r}")
    if activation not in ACTIVATIONS:
        raise HipGemmError(f"unknown activation {activation!r}")
    if group_size <= 0 or group_size % 32:
        raise HipGemmError("group_size must be a multiple of 32")
    if tuple(scales.shape) != (weight.shape[0], -(-x.shape[1] // group_size)):
        raise HipGemmError(f"scales must be (N, groups), got {tuple(scales.shape)}")
    return x.new_empty((x.shape[0], weight.shape[0]), dtype=out_dtype or x.dtype)


@torch.library.custom_op("hipgemm::moe_route", mutates_args=())
def moe_route(logits: torch.Tensor, k: int, scoring: str = "softmax",
              renormalize: bool = True,
              scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    return serving.moe_route(logits, k, scoring=scoring, renormalize=renormalize,
                             scale=scale)


@moe_route.register_fake
def _moe_route_fake(logits, k, scoring="softmax", renormalize=True, scale=1.0):
    if logits.dim() != 2 or scoring not in serving.MOE_SCORING:
        raise HipGemmError("logits must be 2-D, scoring softmax or sigmoid")
    shape = (logits.shape[0], k)
    return (logits.new_empty(shape, dtype=torch.float32),
            logits.new_empty(shape, dtype=torch.int32))


@torch.library.custom_op("hipgemm::moe_experts", mutates_args=())
def moe_experts(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
                w13: torch.Tensor, scales13: torch.Tensor, w2: torch.Tensor,
                scales2: torch.Tensor, zeros13: Optional[torch.Tensor] = None,
                zeros2: Optional[torch.Tensor] = None, format: str = "e4m3",
                group_size: int = 128, activation: str = "silu",
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return serving.moe_experts(_rows(x), ids, weights, w13, scales13, w2, scales2,
                               zeros13=zeros13, zeros2=zeros2, format=format,
                               group_size=group_size, activation=activation,
                               out_dtype=out_dtype)


@moe_experts.register_fake
def _moe_experts_fake(x, ids, weights, w13, scales13, w2, scales2, zeros13=None,
                      zeros2=None, format="e4m3", group_size=128,
                      activation="silu", out_dtype=None):
    if format not in serving.MOE_FORMATS:
        raise HipGemmError(f"unknown format {format!r}")
    if activation not in ACTIVATIONS:
        raise HipGemmError(f"unknown activation {activation!r}")
    per = 1 if format == "e4m3" else 2
    if (x.dim() != 2 or w13.dim() != 3 or w2.dim() != 3 or ids.shape != weights.shape
            or w13.shape[2] * per != x.shape[1] or w13.shape[1] != 2 * per * w2.shape[2]
            or w2.shape[:2] != (w13.shape[0], x.shape[1])):
        raise HipGemmError(f"shapes do not fit: x {tuple(x.shape)}, w13 "
                           f"{tuple(w13.shape)}, w2 {tuple(w2.shape)}")
    return x.new_empty(tuple(x.shape), dtype=out_dtype or x.dtype)


# Magnitudes of e2m1 by code, and the middles between them.
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_E2M1_MID = tuple((a + b) / 2 for a, b in zip(_E2M1, _E2M1[1:]))


def quantize_w4(weight: torch.Tensor, format: str = "int4", group_size: int = 128,
                scale_dtype: torch.dtype = torch.bfloat16):
    """(codes, scales) of a (..., K) weight, each group of group_size elements of
    a row by its largest magnitude: symmetric int4 (codes 1-15 around 8, scale
    amax / 7) or fp4 (nearest e2m1, scale amax / 6).  scale_dtype: float32,
    bfloat16, float16, or uint8 for E8M0 (rounded up to a power of two).  Codes
    are rounded against the scale as stored."""
    if format not in serving.W4_FORMATS:
        raise HipGemmError(f"format must be one of {sorted(serving.W4_FORMATS)}")
    K = weight.shape[-1]
    if group_size <= 0 or group_size % 32 or K % 32:
        raise HipGemmError("K and group_size must be multiples of 32")
    groups = -(-K // group_size)
    w = torch.nn.functional.pad(weight.detach().float(), (0, groups * group_size - K))
    w = w.unflatten(-1, (groups, group_size))
    s = w.abs().amax(-1) / (7.0 if format == "int4" else 6.0)
    s = torch.where(s > 0, s, torch.ones_like(s))
    if scale_dtype == torch.uint8:
        m, e = torch.frexp(s)  # s = m 2^e, 1/2 <= m < 1
        e = torch.where(m > 0.5, e, e - 1).clamp(-127, 127)
        scales, s = (e + 127).to(torch.uint8), torch.ldexp(torch.ones_like(s), e)
    else:
        scales = s.to(scale_dtype)
        s = scales.float()
    v = w / s[..., None]
    if format == "int4":
        q = (v.round().clamp(-8, 7) + 8).to(torch.uint8)
    else:
        q = torch.bucketize(v.abs(), torch.tensor(_E2M1_MID, device=v.device)).to(torch.uint8)
        q = q | (v < 0).to(torch.uint8) << 3
    q = q.flatten(-2)[..., :K]
    return (q[..., 0::2] | q[..., 1::2] << 4).contiguous(), scales.contiguous()


class W4Linear(torch.nn.Module):
    """y = act(x W^T + b) with W (out x in) held as 4-bit codes and scales per
    group of a row (and zero points for int4, if given), x bfloat16 or float16.
    in_features must be a multiple of 32."""

    def __init__(self, weight: torch.Tensor, scales: torch.Tensor,
                 zeros: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, format: str = "int4",
                 group_size: int = 128, activation: Optional[str] = None):
        super().__init__()
        if format not in serving.W4_FORMATS:
            raise HipGemmError(f"format must be one of {sorted(serving.W4_FORMATS)}")
        if activation not in ACTIVATIONS:
            raise HipGemmError(f"unknown activation {activation!r}")
        if weight.dim() != 2 or 2 * weight.shape[1] % 32:
            raise HipGemmError("weight must be 2-D, in_features a multiple of 32")
        if group_size <= 0 or group_size % 32 or tuple(scales.shape) != (
                weight.shape[0], -(-2 * weight.shape[1] // group_size)):
            raise HipGemmError("scales must be (out_features, groups of a row)")
        self.register_buffer("weight", weight.contiguous())
        self.register_buffer("scales", scales.contiguous())
        self.register_buffer("zeros", None if zeros is None else zeros.contiguous())
        self.register_buffer("bias", None if bias is None else
                             bias.to(torch.float32).contiguous())
        self.format, self.group_size = format, group_size
        self.activation = activation or "none"

    @property
    def in_features(self) -> int:
        return 2 * self.weight.shape[1]

    @property
    def out_features(self) -> int:
        return self.weight.shape[0]

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, format: str = "int4",
                    group_size: int = 128, scale_dtype: torch.dtype = torch.bfloat16,
                    activation: Optional[str] = None):
        """Quantise a Linear's weight (quantize_w4)."""
        w, s = quantize_w4(linear.weight, format, group_size, scale_dtype)
        return cls(w, s, None, linear.bias.detach() if linear.bias is not None else None,
                   format, group_size, activation)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise HipGemmError(f"x must have {self.in_features} features, got {tuple(x.shape)}")
        x2 = x.reshape(-1, self.in_features)
        kw = dict(format=self.format, group_size=self.group_size, bias=self.bias,
                  activation=self.activation)
        # (as in Fp8Linear: the call itself where nothing watches the operations)
        if _plain_eager(x2) and _plain_buffers(self.weight, self.scales, self.zeros,
                                               self.bias):
            y = serving.w4_gemm(_rows(x2), self.weight, self.scales, self.zeros, **kw)
        else:
            y = torch.ops.hipgemm.w4_gemm(x2, self.weight, self.scales, self.zeros, **kw)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], self.out_features)


class MoE(torch.nn.Module):
    """A mixture-of-experts layer for decoding: router logits x gate^T (in
    gate's type), each token's k experts (moe_route), their gated MLPs weighted
    and summed (moe_experts).  gate: (E, D);  w13 (E, 2F, D), w2 (E, D, F) with
    their scales in one of moe_experts' formats."""

    def __init__(self, gate: torch.Tensor, w13: torch.Tensor, scales13: torch.Tensor,
                 w2: torch.Tensor, scales2: torch.Tensor, k: int,
                 format: str = "e4m3", group_size: int = 128,
                 scoring: str = "softmax", renormalize: bool = True,
                 scale: float = 1.0, activation: Optional[str] = "silu"):
        super().__init__()
        if format not in serving.MOE_FORMATS or scoring not in serving.MOE_SCORING:
            raise HipGemmError(f"unknown format {format!r} or scoring {scoring!r}")
        if activation not in ACTIVATIONS:
            raise HipGemmError(f"unknown activation {activation!r}")
        if w13.dim() != 3 or w2.dim() != 3 or gate.dim() != 2 or not (
                gate.shape[0] == w13.shape[0] == w2.shape[0]) \
                or gate.shape[1] != w2.shape[1]:
            raise HipGemmError("gate must be (E, D), w13 (E, 2F, D), w2 (E, D, F)")
        if not 1 <= k <= gate.shape[0]:
            raise HipGemmError("k must be 1 .. E")
        for name, t in (("gate", gate), ("w13", w13), ("scales13", scales13),
                        ("w2", w2), ("scales2", scales2)):
            self.register_buffer(name, t.contiguous())
        self.k, self.format, self.group_size = k, format, group_size
        self.scoring, self.renormalize, self.scale = scoring, renormalize, scale
        self.activation = activation or "none"

    @classmethod
    def from_weights(cls, gate: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor,
                     k: int, format: str = "e4m3", group_size: int = 128,
                     scale_dtype: torch.dtype = torch.bfloat16, **kw):
        """Quantise the experts' weights: e4m3 by rows, 4-bit by groups."""
        def pack(w):
            if format == "e4m3":
                q, s = quantize_rows(w.detach().flatten(0, 1))
                return q.unflatten(0, w.shape[:2]), s.unflatten(0, w.shape[:2])
            return quantize_w4(w, format, group_size, scale_dtype)
        return cls(gate.detach(), *pack(w13), *pack(w2), k, format, group_size, **kw)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x2 = x.reshape(-1, x.shape[-1])
        experts = (self.w13, self.scales13, self.w2, self.scales2)
        plain = _plain_eager(x2) and _plain_buffers(self.gate, *experts)
        if plain:
            x2 = _rows(x2)
        logits = torch.nn.functional.linear(x2.to(self.gate.dtype), self.gate)
        route = dict(scoring=self.scoring, renormalize=self.renormalize, scale=self.scale)
        kw = dict(format=self.format, group_size=self.group_size,
                  activation=self.activation)
        if plain:
            weights, ids = serving.moe_route(logits, self.k, **route)
            y = serving.moe_experts(x2, ids, weights, *experts, **kw)
        else:
            weights, ids = torch.ops.hipgemm.moe_route(logits, self.k, **route)
            y = torch.ops.hipgemm.moe_experts(x2, ids, weights, *experts, **kw)
        return y if x.dim() == 2 else y.reshape(x.shape)
