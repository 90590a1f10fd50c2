"""Products of 16-bit activations with 16-bit weights and the epilogues of a
feed-forward block, with their backward passes (include/hipgemm.h: hipgemm_linear
and hipgemm_linear_backward), on torch tensors.

linear, linear_backward              y = act(x W^T + b) + r
gated_linear, gated_linear_backward  y = act(x Wg^T + bg) * (x Wu^T + bu)

Like the rest of the package these run on the GPU only, on the current stream or
the one given, and raise HipGemmError for arguments that they do not take.  They
record no gradient: hipgemm_amd.torch_dense has operators and modules that do.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import struct

from . import ACTIVATIONS, OUT_BF16, OUT_F16, OUT_F32, _check, _torch, lib
from .serving import _bad, _on

__all__ = ["linear", "linear_backward", "gated_linear", "gated_linear_backward",
           "LinearDesc", "LinearGradDesc", "linear_raw", "linear_backward_raw",
           "linear_workspace_size", "linear_backward_workspace_size", "linear_select",
           "linear_backward_select"]

_vp, _ci, _ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


class LinearDesc(ctypes.Structure):
    """hipgemm_linear_desc (include/hipgemm.h)."""
    _fields_ = [("size", ctypes.c_size_t), ("x", _vp), ("weight", _vp), ("bias", _vp),
                ("residual", _vp), ("y", _vp), ("pre", _vp), ("workspace", _vp),
                ("workspace_bytes", ctypes.c_size_t), ("ldx", _ll), ("ldw", _ll),
                ("ldr", _ll), ("ldy", _ll), ("ldp", _ll), ("M", _ci), ("N", _ci),
                ("K", _ci), ("gated", _ci), ("type", _ci), ("bias_type", _ci),
                ("residual_type", _ci), ("out_dtype", _ci), ("pre_dtype", _ci),
                ("activation", _ci)]


class LinearGradDesc(ctypes.Structure):
    """hipgemm_linear_grad_desc (include/hipgemm.h)."""
    _fields_ = [("size", ctypes.c_size_t), ("dy", _vp), ("x", _vp), ("weight", _vp),
                ("pre", _vp), ("dx", _vp), ("dw", _vp), ("db", _vp), ("workspace", _vp),
                ("workspace_bytes", ctypes.c_size_t), ("lddy", _ll), ("ldx", _ll),
                ("ldw", _ll), ("ldp", _ll), ("lddx", _ll), ("lddw", _ll), ("M", _ci),
                ("N", _ci), ("K", _ci), ("gated", _ci), ("type", _ci), ("dy_type", _ci),
                ("pre_type", _ci), ("dx_dtype", _ci), ("dw_dtype", _ci), ("db_dtype", _ci),
                ("activation", _ci)]


_DESC_BYTES = ctypes.sizeof(LinearDesc)
# The structures' bytes, in a fifth of the time that they take to fill.
_linear_desc = struct.Struct("@N7PN5q10i").pack
_grad_desc = struct.Struct("@N8PN6q11i0q").pack
_MAX_LD = 1 << 21  # of rows that the products read
_NOTHING = contextlib.nullcontext()
_GRAD_BYTES = ctypes.sizeof(LinearGradDesc)


@functools.lru_cache(maxsize=1)
def _types():
    """Codes by dtype: operands, inputs, outputs."""
    t = _torch()
    return ({t.bfloat16: 1, t.float16: 2}, {t.float32: 0, t.bfloat16: 1, t.float16: 2},
            {t.bfloat16: OUT_BF16, t.float16: OUT_F16, t.float32: OUT_F32})


def linear_raw(desc: "LinearDesc", stream: int = 0) -> int:
    """Call hipgemm_linear; returns hipError_t."""
    return int(lib().hipgemm_linear(ctypes.byref(desc), stream or None))


def linear_backward_raw(desc: "LinearGradDesc", stream: int = 0) -> int:
    """Call hipgemm_linear_backward; returns hipError_t."""
    return int(lib().hipgemm_linear_backward(ctypes.byref(desc), stream or None))


def linear_workspace_size(desc: "LinearDesc") -> int:
    """Workspace bytes hipgemm_linear needs for a descriptor."""
    return int(lib().hipgemm_linear_workspace_size(ctypes.byref(desc)))


def linear_backward_workspace_size(desc: "LinearGradDesc") -> int:
    """Workspace bytes hipgemm_linear_backward needs for a descriptor."""
    return int(lib().hipgemm_linear_backward_workspace_size(ctypes.byref(desc)))


def linear_select(desc: "LinearDesc") -> tuple:
    """(tile rows, tile columns, slices along K, first columns) that hipgemm_linear takes for
    a descriptor's sizes (include/hipgemm.h); tile rows 0: the kernel of a few rows."""
    plan = (_ci * 4)()
    _check(lib().hipgemm_linear_select(ctypes.byref(desc), plan), "hipgemm_linear_select")
    return tuple(plan)


def linear_backward_select(desc: "LinearGradDesc") -> tuple:
    """The same of hipgemm_linear_backward's two products: (of dx, of dw)."""
    plan = (_ci * 8)()
    _check(lib().hipgemm_linear_backward_select(ctypes.byref(desc), plan),
           "hipgemm_linear_backward_select")
    return tuple(plan[:4]), tuple(plan[4:])


def _launch(call, what, desc, index, stream):
    """call(desc, stream) with device `index` as the current one."""
    torch = _torch()
    c = torch._C
    if index != c._cuda_getDevice():
        with torch.cuda.device(index):
            return _launch(call, what, desc, index, stream)
    handle = c._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream
    code = call(desc, handle)
    if code:
        _check(code, what)


@functools.lru_cache(maxsize=4096)
def _forward_bytes(M, N, K, kind, device):
    """Workspace of a forward call (a pure function of its sizes; kind: 0 linear, 1 with a
    residual, 2 gated)."""
    d = LinearDesc(size=_DESC_BYTES, M=M, N=N, K=K, gated=int(kind == 2), type=1,
                   residual=int(kind == 1))
    return linear_workspace_size(d)


@functools.lru_cache(maxsize=4096)
def _backward_bytes(M, N, K, gated, code, act, dyt, aligned, whole, need_x, need_weight,
                    need_bias, device, dw_type=OUT_BF16):
    """Workspace of a backward call, of whose addresses and strides only those of dy matter:
    whether it starts on 16 bytes, and its rows (`whole`); and of whose results' types that of
    dw, since dx has the operands'."""
    d = LinearGradDesc(size=_GRAD_BYTES, M=M, N=N, K=K, gated=int(gated), type=code,
                       activation=act, dy_type=dyt, dy=16 if aligned else 2,
                       lddy=8 if whole else 1, dx=int(need_x), dw=int(need_weight),
                       db=int(need_bias), dw_dtype=dw_type)
    return linear_backward_workspace_size(d)


def _operand(t, name, dtype, index):
    """The row stride and the address of a matrix that the products read as it is."""
    if t.dtype is not dtype or t.get_device() != index:
        _bad(f"{name} must be a 2-D {dtype} tensor on device {index}, got {tuple(t.shape)} "
             f"{t.dtype} on {t.device}")
    rows, cols = t.shape
    ld, unit = t.stride()
    at = t.data_ptr()
    if unit != 1 and cols > 1:
        _bad(f"{name} must have unit stride along its rows")
    if rows <= 1:
        ld = cols
    if (at % 16 or ld % 8 or not cols <= ld <= _MAX_LD) and rows and cols:
        _bad(f"rows of {name} must start on 16 bytes, not overlap and be at most {_MAX_LD} "
             f"elements apart, got a stride of {ld}")
    return ld, at


def _matrix(t, name, shape, dtypes, index):
    """The code of a (M, N) matrix' type, its row stride and its address."""
    code = dtypes.get(t.dtype)
    if code is None or t.shape != shape or t.get_device() != index:
        _bad(f"{name} must be a {shape} bfloat16, float16 or float32 tensor on device {index}, "
             f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    ld, unit = t.stride()
    if unit != 1 and shape[1] > 1:
        _bad(f"{name} must have unit stride along its rows")
    if shape[0] <= 1:
        ld = shape[1]
    if ld < shape[1]:
        _bad(f"rows of {name} must not overlap")
    return code, ld, t.data_ptr()


def _sizes(x, weight, gated):
    """The code of the operands' type, M, rows of the weight, N, K and the device."""
    code = _types()[0].get(x.dtype)
    index = x.get_device()
    if code is None or index < 0 or x.dim() != 2:
        _bad(f"x must be a 2-D bfloat16 or float16 device tensor, got {x.dtype} on {x.device}")
    M, K = x.shape
    if weight.dim() != 2 or weight.shape[1] != K:
        _bad(f"K mismatch: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    N = rows = weight.shape[0]
    if K % 8:
        _bad(f"K must be a multiple of 8, got {K}")
    if gated:
        if N % 16:
            _bad(f"weight must have 2 N rows, N a multiple of 8, got {N}")
        N //= 2
    return code, M, rows, N, K, index


def _forward(x, weight, bias, activation, residual, out_dtype, out, save_pre, gated, stream):
    torch = _torch()
    _, inputs, outputs = _types()
    code, M, rows, N, K, index = _sizes(x, weight, gated)
    ldx, xp = _operand(x, "x", x.dtype, index)
    ldw, wp = _operand(weight, "weight", x.dtype, index)
    if activation not in ACTIVATIONS:
        _bad(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)}")
    bp = bt = rp = rt = ldr = 0
    if bias is not None:
        bt = inputs.get(bias.dtype)
        if (bt is None or bias.shape != (rows,) or bias.get_device() != index
                or (rows > 1 and bias.stride(0) != 1)):
            _bad(f"bias must be a contiguous bfloat16, float16 or float32 vector of {rows} "
                 f"elements on device {index}")
        bp = bias.data_ptr()
    if residual is not None:
        rt, ldr, rp = _matrix(residual, "residual", (M, N), inputs, index)
    out_dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    ot = outputs.get(out_dtype)
    if ot is None:
        _bad("out_dtype must be bfloat16, float16 or float32")
    pre_dtype = torch.float32 if save_pre is True else save_pre or torch.float32
    pt = outputs.get(pre_dtype)
    if pt is None:
        _bad("save_pre must be True, False, bfloat16, float16 or float32")
    kind = 2 if gated else 1 if residual is not None else 0
    memory = (x, M, N, K, rows, out, out_dtype, pre_dtype, save_pre, kind, index)
    if stream is not None:
        if stream.device != x.device:
            _bad(f"stream is on {stream.device}, x on {x.device}")
        with torch.cuda.stream(stream):
            out, ldy, yp, pre, workspace, need = _forward_memory(*memory)
    else:
        out, ldy, yp, pre, workspace, need = _forward_memory(*memory)
    d = _linear_desc(_DESC_BYTES, xp, wp, bp, rp, yp, 0 if pre is None else pre.data_ptr(),
                     workspace.data_ptr() if need else 0, need, ldx, ldw, ldr, ldy, rows, M, N,
                     K, int(gated), code, bt, rt, ot, pt, ACTIVATIONS[activation])
    _launch(lib().hipgemm_linear, "hipgemm_linear", d, index, stream)
    return (out, pre) if save_pre else out


def _forward_memory(x, M, N, K, rows, out, out_dtype, pre_dtype, save_pre, kind, index):
    """(out, its row stride and address, pre, workspace, its bytes): what of them has to be
    allocated is the current stream's."""
    if out is None:
        out, ldy = x.new_empty((M, N), dtype=out_dtype), N
        yp = out.data_ptr()
    else:
        if out.dtype != out_dtype:
            _bad(f"out must be {out_dtype}")
        _, ldy, yp = _matrix(out, "out", (M, N), _types()[2], index)
    pre = x.new_empty((M, rows), dtype=pre_dtype) if save_pre else None
    need = _forward_bytes(M, N, K, kind, index)
    workspace = x.new_empty(need, dtype=_torch().uint8) if need else None
    return out, ldy, yp, pre, workspace, need


def _backward(dy, x, weight, pre, activation, need_x, need_weight, need_bias, grad_dtype,
              bias_dtype, gated, stream):
    torch = _torch()
    _, inputs, outputs = _types()
    code, M, rows, N, K, index = _sizes(x, weight, gated)
    ldx, xp = _operand(x, "x", x.dtype, index)
    ldw, wp = _operand(weight, "weight", x.dtype, index)
    if activation not in ACTIVATIONS:
        _bad(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)}")
    dyt, lddy, dyp = _matrix(dy, "dy", (M, N), inputs, index)
    pp = pt = ldp = 0
    if gated or ACTIVATIONS[activation]:
        if pre is None:
            _bad("pre of the forward pass (save_pre) is needed")
        pt, ldp, pp = _matrix(pre, "pre", (M, rows), inputs, index)
    if stream is not None and stream.device != x.device:
        _bad(f"stream is on {stream.device}, x on {x.device}")
    grad_dtype = grad_dtype or x.dtype
    ot = outputs.get(grad_dtype)
    if ot is None:
        _bad("grad_dtype must be bfloat16, float16 or float32")
    bias_dtype = bias_dtype or grad_dtype
    bt = outputs.get(bias_dtype)
    if bt is None:
        _bad("bias_dtype must be bfloat16, float16 or float32")
    act = ACTIVATIONS[activation]
    need = _backward_bytes(M, N, K, gated, code, act, dyt, dyp % 16 == 0,
                           lddy % 8 == 0 and lddy <= _MAX_LD, need_x, need_weight, need_bias, index,
                           ot)
    with _on(stream) if stream is not None else _NOTHING:
        dx = x.new_empty((M, K)) if need_x else None
        dw = x.new_empty((rows, K), dtype=grad_dtype) if need_weight else None
        db = x.new_empty(rows, dtype=bias_dtype) if need_bias else None
        workspace = x.new_empty(need, dtype=torch.uint8) if need else None
    d = _grad_desc(_GRAD_BYTES, dyp, xp, wp, pp, 0 if dx is None else dx.data_ptr(),
                   0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(),
                   workspace.data_ptr() if need else 0, need, lddy, ldx, ldw, ldp, K, K, M, N, K,
                   int(gated), code, dyt, pt, outputs[x.dtype], ot, bt, act)
    _launch(lib().hipgemm_linear_backward, "hipgemm_linear_backward", d, index, stream)
    return dx, dw, db


def linear(x, weight, *, bias=None, activation=None, residual=None, out_dtype=None,
           out=None, save_pre=False, stream=None):
    """out[m, n] = round(act(z[m, n]) + residual[m, n]), z = x @ weight.T + bias.

    x (M, K) and weight (N, K): both bfloat16 or both float16, K a multiple of 8, rows of
    unit stride that start on 16 bytes, 2^21 elements apart at most.  bias (N) and residual (M, N): bfloat16, float16
    or float32.  activation as for gemm().  out_dtype: bfloat16, float16 or float32, x's
    where None.  out may be residual itself and overlaps nothing else.  Sums are fp32, and
    everything after them until the one rounding.  save_pre: returns (out, z), as
    linear_backward takes it: z in float32 where True, or of the type given (x's halves its
    memory and adds a rounding to the gradients)."""
    return _forward(x, weight, bias, activation, residual, out_dtype, out, save_pre, False,
                    stream)


def gated_linear(x, weight, *, bias=None, activation="silu", out_dtype=None, out=None,
                 save_pre=False, stream=None):
    """out[m, n] = round(act(z[m, n]) * z[m, N + n]), z = x @ weight.T + bias: the gate and
    up projections of a gated MLP, its activation and the product in one kernel.

    weight (2N, K): gate rows, then up rows (as moe_experts' w13), N a multiple of 8; bias
    (2N).  The rest as for linear; save_pre returns (out, z (M, 2N))."""
    return _forward(x, weight, bias, activation, None, out_dtype, out, save_pre, True, stream)


def linear_backward(dy, x, weight, pre=None, *, activation=None, need_x: bool = True,
                    need_weight: bool = True, need_bias: bool = False, grad_dtype=None,
                    bias_dtype=None, stream=None):
    """(dx, dweight, dbias) of linear, None where not needed: dz = dy * act'(z), dx = dz @
    weight, dweight = dz.T @ x, dbias = dz.sum(0).  (The residual's gradient is dy.)

    dy (M, N): bfloat16, float16 or float32.  pre: linear's z (save_pre); not needed without
    an activation.  dx has x's type, dweight grad_dtype (bfloat16, float16 or float32; x's
    type where None) and dbias bias_dtype (grad_dtype where None).  dz is rounded to x's type
    for the two products, half a step of every term; a float32 dweight is summed over dz in 24
    bits instead, at three times (bfloat16) or twice the operations.  Sums are fp32."""
    return _backward(dy, x, weight, pre, activation, need_x, need_weight, need_bias,
                     grad_dtype, bias_dtype, False, stream)


def gated_linear_backward(dy, x, weight, pre, *, activation="silu", need_x: bool = True,
                          need_weight: bool = True, need_bias: bool = False,
                          grad_dtype=None, bias_dtype=None, stream=None):
    """(dx, dweight, dbias) of gated_linear, None where not needed; as linear_backward, with
    [dg | du] = [dy * u * act'(g) | dy * act(g)] for dz, z = [g | u]."""
    return _backward(dy, x, weight, pre, activation, need_x, need_weight, need_bias,
                     grad_dtype, bias_dtype, True, stream)
