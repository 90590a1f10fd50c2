"""Operators of LLM serving with quantised weights and 16-bit activations
(include/hipgemm.h: hipgemm_w4_gemm and its neighbours), on torch tensors.

w4_gemm      products with 4-bit weights and group scales
moe_route    a router's choice of experts for each token
moe_experts  the experts' gated MLPs of a few tokens, e4m3 or 4-bit weights

Like the rest of the package these run on the GPU only, on the current stream
or the one given, and raise HipGemmError for arguments that they do not take.
None of them records a gradient.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

from . import (ACTIVATIONS, OUT_BF16, OUT_F16, OUT_F32, HipGemmError, _check,
               _torch, hipErrorInvalidValue, lib)

__all__ = ["w4_gemm", "W4Desc", "w4_gemm_raw", "w4_select", "moe_select", "W4_FORMATS",
           "moe_route", "MOE_SCORING", "moe_experts", "MoeDesc", "MoeMatrix",
           "moe_experts_raw", "moe_workspace_size", "MOE_FORMATS"]

# include/hipgemm.h codes
W4_FORMATS = {"int4": 0, "fp4": 1}
MOE_FORMATS = {**W4_FORMATS, "e4m3": 2}
MOE_SCORING = {"softmax": 0, "sigmoid": 1}
_vp, _ci, _ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


class W4Desc(ctypes.Structure):
    """hipgemm_w4_desc (include/hipgemm.h)."""
    _fields_ = [("size", ctypes.c_size_t), ("x", _vp), ("weight", _vp),
                ("scales", _vp), ("zeros", _vp), ("y", _vp), ("bias", _vp),
                ("M", _ci), ("N", _ci), ("K", _ci), ("group_size", _ci),
                ("ldx", _ll), ("ldw", _ll), ("lds", _ll), ("ldy", _ll),
                ("x_type", _ci), ("format", _ci), ("scale_type", _ci),
                ("out_dtype", _ci), ("activation", _ci)]


class MoeMatrix(ctypes.Structure):
    """hipgemm_moe_matrix (include/hipgemm.h)."""
    _fields_ = [("weight", _vp), ("scales", _vp), ("zeros", _vp), ("ldw", _ll),
                ("expert_w", _ll), ("lds", _ll), ("expert_s", _ll)]


class MoeDesc(ctypes.Structure):
    """hipgemm_moe_desc (include/hipgemm.h)."""
    _fields_ = [("size", ctypes.c_size_t), ("x", _vp), ("ids", _vp),
                ("weights", _vp), ("w13", MoeMatrix), ("w2", MoeMatrix),
                ("y", _vp), ("workspace", _vp),
                ("workspace_bytes", ctypes.c_size_t), ("ldx", _ll), ("ldy", _ll),
                ("T", _ci), ("k", _ci), ("E", _ci), ("D", _ci), ("F", _ci),
                ("group_size", _ci), ("x_type", _ci), ("format", _ci),
                ("scale_type", _ci), ("out_dtype", _ci), ("activation", _ci)]


_MOE_BYTES = ctypes.sizeof(MoeDesc)
_W4_BYTES = ctypes.sizeof(W4Desc)


@functools.lru_cache(maxsize=1)
def _types():
    """Codes by dtype: activations, scales, outputs."""
    t = _torch()
    return ({t.bfloat16: 1, t.float16: 2},
            {t.float32: 0, t.bfloat16: 1, t.float16: 2, t.uint8: 3},
            {t.bfloat16: OUT_BF16, t.float16: OUT_F16, t.float32: OUT_F32})


def _bad(msg: str):
    raise HipGemmError(msg, hipErrorInvalidValue)


def _stream_handle(t, stream) -> int:
    if stream is not None:
        return stream.cuda_stream
    return _torch()._C._cuda_getCurrentRawStream(t.get_device())


def _on(stream):
    """Memory that is allocated here belongs to `stream` (None: the current one):
    what the current stream has freed and may still read is not written over."""
    return contextlib.nullcontext() if stream is None else _torch().cuda.stream(stream)


def w4_gemm_raw(desc: "W4Desc", stream: int = 0) -> int:
    """Call hipgemm_w4_gemm; returns hipError_t."""
    return int(lib().hipgemm_w4_gemm(ctypes.byref(desc), stream or None))


def w4_select(desc: "W4Desc") -> tuple:
    """(kernel, tile rows, tile columns) that hipgemm_w4_gemm takes for a descriptor;
    kernel: "vectors" (no tiles), "split" or "tiles"."""
    plan = (_ci * 3)()
    _check(lib().hipgemm_w4_select(ctypes.byref(desc), plan), "hipgemm_w4_select")
    return (("vectors", "split", "tiles")[plan[0]], *plan[1:])


def w4_gemm(x, weight, scales, zeros=None, *, format: str = "int4",
            group_size: int = 128, bias=None, activation=None, out_dtype=None,
            out=None, stream=None):
    """out[m, n] = round(act(sum_k x[m, k] w[n, k] + bias[n])) with 4-bit
    weights: w[n, k] = (q[n, k] - zeros[n, k // group_size]) *
    scales[n, k // group_size] ("int4", q 0-15, zeros 8 where None), or
    e2m1(q[n, k]) * scales[...] ("fp4").

    x (M, K): bfloat16 or float16, K a multiple of 32.  weight (N, K / 2): uint8,
    element 2i in the low nibble of byte i (or float4_e2m1fn_x2).  scales
    (N, ceil(K / group_size)): bfloat16, float16, float32, or uint8 for E8M0
    (2^(e - 127)); zeros: uint8 of that shape and strides.  group_size: a
    multiple of 32.  bias: float32 (N).  activation as for gemm().  out_dtype:
    bfloat16, float16 or float32, x's where None.  Rows have unit stride; those
    of x and weight start on 16 bytes.  Sums are fp32, weights are not rounded.
    """
    torch = _torch()
    x_types, s_types, o_types = _types()
    if x.dim() != 2 or weight.dim() != 2 or scales.dim() != 2:
        _bad("x, weight and scales must be 2-D")
    (M, K), N = x.shape, weight.shape[0]
    xt = x_types.get(x.dtype)
    if xt is None:
        _bad(f"x must be bfloat16 or float16, got {x.dtype}")
    fmt = W4_FORMATS.get(format)
    if fmt is None:
        _bad(f"format must be one of {sorted(W4_FORMATS)}")
    if weight.dtype != torch.uint8:
        if weight.dtype != torch.float4_e2m1fn_x2 or fmt != 1:
            _bad(f"weight must be uint8 (or float4_e2m1fn_x2 for fp4), got {weight.dtype}")
    if 2 * weight.shape[1] != K:
        _bad(f"K mismatch: x has {K}, weight {2 * weight.shape[1]}")
    if group_size <= 0 or group_size % 32 or K % 32:
        _bad("K and group_size must be multiples of 32")
    groups = -(-K // group_size)
    st = s_types.get(scales.dtype)
    if st is None or scales.shape != (N, groups):
        _bad(f"scales must be ({N}, {groups}) bfloat16, float16, float32 or uint8, "
             f"got {tuple(scales.shape)} {scales.dtype}")
    lds = scales.stride(0) if N > 1 else groups
    zp = 0
    if zeros is not None:
        if fmt != 0:
            _bad("zeros belong to int4")
        if zeros.dtype != torch.uint8 or zeros.shape != scales.shape or not zeros.is_cuda:
            _bad("zeros must be uint8 of the shape of scales, on the GPU")
        if zeros.stride() != scales.stride() and zeros.numel() > 1:
            with _on(stream):
                zeros = torch.empty_strided(scales.shape, scales.stride(), dtype=torch.uint8,
                                            device=zeros.device).copy_(zeros)
        zp = zeros.data_ptr()
    if not (x.is_cuda and weight.is_cuda and scales.is_cuda):
        _bad("x, weight and scales must be device tensors")
    if ((K > 1 and x.stride(1) != 1) or (K > 2 and weight.stride(1) != 1)
            or (groups > 1 and scales.stride(1) != 1)):
        _bad("x, weight and scales must have unit stride along K")
    if activation not in ACTIVATIONS:
        _bad(f"activation must be one of {sorted(k for k in ACTIVATIONS if k)}")
    out_dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    ot = o_types.get(out_dtype)
    if ot is None:
        _bad("out_dtype must be bfloat16, float16 or float32")
    if out is None:
        # (a bare new_empty is the quickest there is, by 0.3 us of 8)
        if stream is None:
            out = (x.new_empty((M, N)) if out_dtype is x.dtype else
                   x.new_empty((M, N), dtype=out_dtype))
        else:
            with _on(stream):
                out = x.new_empty((M, N), dtype=out_dtype)
    elif (out.dtype != out_dtype or tuple(out.shape) != (M, N) or not out.is_cuda
          or (N > 1 and out.stride(1) != 1)):
        _bad(f"out must be a ({M}, {N}) {out_dtype} device tensor with unit column stride")
    bp = 0
    if bias is not None:
        if not (bias.is_cuda and bias.dtype == torch.float32 and tuple(bias.shape) == (N,)
                and (N <= 1 or bias.stride(0) == 1)):
            _bad(f"bias must be a contiguous float32 device vector of {N} elements")
        bp = bias.data_ptr()
    d = W4Desc(_W4_BYTES, x.data_ptr(), weight.data_ptr(), scales.data_ptr(), zp,
               out.data_ptr(), bp, M, N, K, group_size,
               x.stride(0) if M > 1 else K, weight.stride(0) if N > 1 else K // 2,
               lds, out.stride(0) if M > 1 else N, xt, fmt, st, ot,
               ACTIVATIONS[activation])
    _check(lib().hipgemm_w4_gemm(ctypes.byref(d), _stream_handle(x, stream)), "hipgemm_w4_gemm")
    return out


def moe_route(logits, k: int, *, scoring: str = "softmax", renormalize: bool = True,
              scale: float = 1.0, stream=None):
    """The k experts of largest logit for each token, in order (equal logits: the
    lower index first), and their weights: (weights (T, k) float32, ids (T, k)
    int32).

    logits (T, E): float32, bfloat16 or float16, unit stride along E.  scoring:
    "softmax" over all experts, or "sigmoid" of each; renormalize divides a
    token's k weights by their sum; scale multiplies them.  A logit of -inf is
    never chosen: a token with fewer than k others gets id -1 and weight 0 in the
    remaining places.  Up to 1024 experts, k up to 64."""
    torch = _torch()
    if logits.dim() != 2 or not logits.is_cuda:
        _bad("logits must be a 2-D device tensor")
    kind = _types()[1].get(logits.dtype)
    if kind is None or kind > 2:
        _bad(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    T, E = logits.shape
    if E > 1 and logits.stride(1) != 1:
        _bad("logits must have unit stride along the experts")
    code = MOE_SCORING.get(scoring)
    if code is None:
        _bad(f"scoring must be one of {sorted(MOE_SCORING)}")
    shape = (T, k if k > 0 else 0)
    if stream is None:
        weights = (logits.new_empty(shape) if kind == 0 else
                   logits.new_empty(shape, dtype=torch.float32))
        ids = logits.new_empty(shape, dtype=torch.int32)
    else:
        with _on(stream):
            weights = logits.new_empty(shape, dtype=torch.float32)
            ids = logits.new_empty(shape, dtype=torch.int32)
    _check(lib().hipgemm_moe_route(
        logits.data_ptr(), kind, T, E, k, logits.stride(0) if T > 1 else E, code,
        int(renormalize), scale, weights.data_ptr(), ids.data_ptr(),
        _stream_handle(logits, stream)), "hipgemm_moe_route")
    return weights, ids


def moe_select(T: int, k: int, E: int, D: int, F: int, format: str = "e4m3",
               out_dtype=None) -> dict:
    """How moe_experts runs the first turn of such a call (out_dtype: bfloat16 where
    None): empty pair by pair; grouped, up_rows and down_rows (tokens of a tile), up_waves and down_waves (that
    share a row's K), parts (of F, of part_len each)."""
    plan = (_ci * 7)()
    out = OUT_BF16 if out_dtype is None else _types()[2].get(out_dtype, -1)
    _check(lib().hipgemm_moe_select(T, k, E, D, F, MOE_FORMATS.get(format, -1), out, plan),
           "hipgemm_moe_select")
    names = ("up_rows", "up_waves", "down_rows", "down_waves", "parts", "part_len")
    return dict(zip(names, plan[1:])) if plan[0] else {}


def moe_experts_raw(desc: "MoeDesc", stream: int = 0) -> int:
    """Call hipgemm_moe_experts; returns hipError_t."""
    return int(lib().hipgemm_moe_experts(ctypes.byref(desc), stream or None))


def moe_workspace_size(T: int, k: int, E: int, D: int, F: int) -> int:
    """Workspace bytes hipgemm_moe_experts needs."""
    return int(lib().hipgemm_moe_workspace_size(T, k, E, D, F))


_moe_ws_bytes = functools.lru_cache(maxsize=1024)(moe_workspace_size)


def _moe_matrix(name, w, s, z, shape, fmt, group):
    """The matrix' pointers and strides, and its scales' type; shape: (E, rows, K)."""
    torch = _torch()
    E, rows, K = shape
    if fmt == 2:
        dtypes, width, groups = (torch.float8_e4m3fn,), K, None
    else:
        dtypes = (torch.uint8, torch.float4_e2m1fn_x2) if fmt == 1 else (torch.uint8,)
        width, groups = K // 2, -(-K // group)
    if w.dtype not in dtypes or tuple(w.shape) != (E, rows, width) or not w.is_cuda \
            or w.stride(2) != 1:
        _bad(f"{name} must be a ({E}, {rows}, {width}) {dtypes[0]} device tensor with unit "
             f"stride along the last dimension, got {tuple(w.shape)} {w.dtype}")
    want = (E, rows) if groups is None else (E, rows, groups)
    st = _types()[1].get(s.dtype)
    if st is None or (fmt == 2 and st != 0) or tuple(s.shape) != want or not s.is_cuda:
        _bad(f"scales of {name} must be {want}" + (" float32" if fmt == 2 else
             " bfloat16, float16, float32 or uint8") + f", got {tuple(s.shape)} {s.dtype}")
    if groups is not None and groups > 1 and s.stride(2) != 1:
        _bad(f"scales of {name} must have unit stride along the groups")
    zp = 0
    if z is not None:
        if fmt != 0:
            _bad("zeros belong to int4")
        if z.dtype != torch.uint8 or tuple(z.shape) != want or not z.is_cuda \
                or z.stride() != s.stride():
            _bad(f"zeros of {name} must be uint8 of the shape and strides of its scales")
        zp = z.data_ptr()
    return MoeMatrix(w.data_ptr(), s.data_ptr(), zp, w.stride(1), w.stride(0),
                     s.stride(1), s.stride(0)), st


def moe_experts(x, ids, weights, w13, scales13, w2, scales2, *, zeros13=None,
                zeros2=None, format: str = "e4m3", group_size: int = 128,
                activation="silu", out_dtype=None, out=None, workspace=None, stream=None):
    """The experts of a mixture-of-experts layer on a few tokens:

        h[t, j] = act(x[t] @ W13[e, :F].T) * (x[t] @ W13[e, F:].T),  e = ids[t, j]
        out[t]  = round(sum_j weights[t, j] * (h[t, j] @ W2[e].T))

    x (T, D): bfloat16 or float16.  ids (T, k) int32 and weights (T, k) float32 as
    moe_route gives them; an id outside [0, E) is skipped.  w13 (E, 2F, D) (gate
    rows, then up rows) and w2 (E, D, F): float8_e4m3fn with float32 scales (E, 2F)
    and (E, D) ("e4m3"), or 4-bit codes (last dimension halved) with scales per
    group_size elements of a row, (E, rows, groups), as for w4_gemm ("int4",
    "fp4").  D, F and group_size are multiples of 32.  activation: of the gate
    (None, "relu", "gelu_tanh", "silu").  out_dtype: bfloat16, float16 or float32,
    x's where None; h is held to 16 significant bits, to 24 for float32 results.
    Made for up to 64 tokens; any number works, in turns of 512 / k that each read
    the chosen experts' weights (moe_select: how often).  workspace: a uint8 device
    tensor of moe_workspace_size bytes; allocated per call where None."""
    torch = _torch()
    x_types, _, o_types = _types()
    xt, fmt = x_types.get(x.dtype), MOE_FORMATS.get(format)
    if xt is None or x.dim() != 2 or not x.is_cuda:
        _bad(f"x must be a 2-D bfloat16 or float16 device tensor, got {x.dtype}")
    if fmt is None:
        _bad(f"format must be one of {sorted(MOE_FORMATS)}")
    if w13.dim() != 3 or ids.dim() != 2:
        _bad("w13 must be 3-D, ids 2-D")
    (T, D), (E, F2, _), k = x.shape, w13.shape, ids.shape[1]
    F = F2 // 2
    if F2 % 2 or D % 32 or F % 32:
        _bad("D and F must be multiples of 32")
    if fmt != 2 and (group_size <= 0 or group_size % 32):
        _bad("group_size must be a multiple of 32")
    if D > 1 and x.stride(1) != 1:
        _bad("x must have unit stride along D")
    for t, dtype, name in ((ids, torch.int32, "ids"), (weights, torch.float32, "weights")):
        if t.dtype != dtype or tuple(t.shape) != (T, k) or not t.is_cuda \
                or not t.is_contiguous():
            _bad(f"{name} must be a contiguous ({T}, {k}) {dtype} device tensor")
    if activation not in ACTIVATIONS:
        _bad(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)}")
    m13, s13 = _moe_matrix("w13", w13, scales13, zeros13, (E, F2, D), fmt, group_size)
    m2, s2 = _moe_matrix("w2", w2, scales2, zeros2, (E, D, F), fmt, group_size)
    if s13 != s2:
        _bad("scales13 and scales2 must have one dtype")
    out_dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    ot = o_types.get(out_dtype)
    if ot is None:
        _bad("out_dtype must be bfloat16, float16 or float32")
    if out is None:
        with _on(stream):
            out = torch.empty((T, D), dtype=out_dtype, device=x.device)
    elif (out.dtype != out_dtype or tuple(out.shape) != (T, D) or not out.is_cuda
          or out.stride(1) != 1):
        _bad(f"out must be a ({T}, {D}) {out_dtype} device tensor with unit column stride")
    need = _moe_ws_bytes(T, k, E, D, F)
    if workspace is None:
        with _on(stream):
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    elif workspace.dtype != torch.uint8 or not workspace.is_cuda \
            or not workspace.is_contiguous() or workspace.numel() < need:
        _bad(f"workspace must be a contiguous uint8 device tensor of {need} bytes")
    d = MoeDesc(_MOE_BYTES, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), m13, m2,
                out.data_ptr(), workspace.data_ptr(), workspace.numel(),
                x.stride(0) if T > 1 else D, out.stride(0) if T > 1 else D, T, k, E, D, F,
                group_size, xt, fmt, s13, ot, ACTIVATIONS[activation])
    _check(lib().hipgemm_moe_experts(ctypes.byref(d), _stream_handle(x, stream)),
           "hipgemm_moe_experts")
    return out
