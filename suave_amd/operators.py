"""Operators around a classifier with many classes, on device tensors: its loss and gradients without the logits
(``linear_cross_entropy``), the orthogonalised update of hidden weight matrices (``orthogonalize``, ``muon_step``) and the
8-bit integer product that serves the head (``quantize_rows``, ``linear_quantized``).

Thin bindings of the C-ABI entry points of the same names (include/suave_hip.h): they check what the library cannot see
(devices, dtypes, strides), run on the current stream of the tensors' device, take scratch from torch's allocator (so calls
on different streams or in different captured graphs never share it) and never wait for the GPU.  No autograd: gradients are
outputs.
"""

from __future__ import annotations

import contextlib
import ctypes as C
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import lib as _lib
from .plan import LinearCeT, LinearQuantizedT, MuonMatrixT, OrthoMatrixT

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}  # SUAVE_DTYPE_F32, SUAVE_DTYPE_BF16


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# The checks below run on every call of operators that take ten microseconds: they build a message only when they fail.
def _device_of(name: str, t: torch.Tensor) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise _lib.SuaveHipError(f"{name} must be on a GPU device (there is no CPU fallback)")
    return t.device


def _matrix(name: str, t: torch.Tensor, dev: torch.device, dtypes, shape=None) -> int:
    """Checks a matrix whose rows are contiguous; returns its row stride in elements."""

    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{name} must be a matrix")
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must have one of the types {[str(d) for d in dtypes]}")
    rows, cols = t.shape
    if shape is not None and (rows, cols) != tuple(shape):
        raise ValueError(f"{name} must have the shape {tuple(shape)}")
    s0, s1 = t.stride()
    if s1 != 1 and cols > 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous")
    if rows <= 1:
        return cols or 1
    if s0 < cols:
        raise ValueError(f"{name}: rows must not overlap")
    return s0


def _vector(name: str, t: torch.Tensor, dev: torch.device, dtype: torch.dtype, n: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be a vector of {n} values")
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must have the type {dtype}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")


def _scalar(name: str, t: torch.Tensor, dev: torch.device, dtype: torch.dtype) -> None:
    if not isinstance(t, torch.Tensor) or t.numel() != 1 or t.device != dev or t.dtype is not dtype:
        raise ValueError(f"{name} must be one {dtype} value on {dev}")


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _on(dev: torch.device):
    """The device as the current one, where it is not."""

    return _NOTHING if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


_NOTHING = contextlib.nullcontext()


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    """Per-call scratch (torch's device allocations start at multiples of 512 bytes; the library checks for 256)."""

    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
                         class_weight: Optional[torch.Tensor] = None, weight_sum: Optional[torch.Tensor] = None,
                         loss_scale: float = 1.0, grad: bool = True, dx: Optional[torch.Tensor] = None,
                         dweight: Optional[torch.Tensor] = None, dbias: Optional[torch.Tensor] = None,
                         loss_sum: Optional[torch.Tensor] = None, loss_rows: float = 1.0) -> Dict[str, torch.Tensor]:
    """Class-weighted softmax cross entropy of ``x @ weight.T + bias`` against ``targets`` and its gradients
    (``suave_linear_ce``): what ``ClassificationHead.loss(linear(x), targets)`` and its backward give, without the
    ``[rows, classes]`` logits.

    ``x`` [rows, dim], ``weight`` [classes, dim]: float32 or bfloat16, rows contiguous, any row stride.  ``targets`` int32;
    a negative one leaves its row out, one beyond the classes makes the loss NaN.  ``weight_sum`` (one float32 value on the
    device) replaces the sum of the rows' class weights (data parallelism: that of the global batch).  Returns ``loss``
    (float32 scalar), ``row_loss`` [rows] (weighted, not divided), ``lse`` [rows] and, with ``grad``, ``dx``, ``dweight``
    (types of ``x`` / ``weight``) and ``dbias`` (float32), all multiplied by ``loss_scale``; buffers for them may be given.
    ``loss_sum`` (float64) += loss * ``loss_rows``."""

    dev = _device_of("x", x)
    ld_x = _matrix("x", x, dev, tuple(_DTYPES))
    n, d = int(x.shape[0]), int(x.shape[1])
    ld_w = _matrix("weight", weight, dev, (x.dtype,))
    c = int(weight.shape[0])
    if weight.shape[1] != d:
        raise ValueError(f"weight must have {d} columns, as x")
    _need(c >= 1 and d >= 1, "weight must have at least one row and one column")
    _vector("targets", targets, dev, torch.int32, n)
    if bias is not None:
        _vector("bias", bias, dev, torch.float32, c)
    if class_weight is not None:
        _vector("class_weight", class_weight, dev, torch.float32, c)
    if weight_sum is not None:
        _scalar("weight_sum", weight_sum, dev, torch.float32)
    if loss_sum is not None:
        _scalar("loss_sum", loss_sum, dev, torch.float64)
    with _on(dev):
        out = {"loss": torch.empty((), dtype=torch.float32, device=dev),
               "row_loss": torch.empty(n, dtype=torch.float32, device=dev), "lse": torch.empty(n, dtype=torch.float32, device=dev)}
        h = LinearCeT()
        if grad:
            out["dx"] = torch.empty((n, d), dtype=x.dtype, device=dev) if dx is None else dx
            out["dweight"] = torch.empty((c, d), dtype=x.dtype, device=dev) if dweight is None else dweight
            out["dbias"] = torch.empty(c, dtype=torch.float32, device=dev) if dbias is None else dbias
            h.ld_dx = d if dx is None else _matrix("dx", dx, dev, (x.dtype,), (n, d))
            h.ld_dweight = d if dweight is None else _matrix("dweight", dweight, dev, (x.dtype,), (c, d))
            if dbias is not None:
                _vector("dbias", dbias, dev, torch.float32, c)
            h.dx, h.dweight, h.dbias = (out[k].data_ptr() for k in ("dx", "dweight", "dbias"))
        else:
            _need(dx is None and dweight is None and dbias is None, "gradient buffers are given, but grad is False")
        h.dtype, h.n_classes, h.dim, h.n_rows = _DTYPES[x.dtype], c, d, n
        h.x, h.ld_x, h.weight, h.ld_weight = x.data_ptr(), ld_x, weight.data_ptr(), ld_w
        h.bias, h.targets, h.class_weight, h.weight_sum = _ptr(bias), targets.data_ptr(), _ptr(class_weight), _ptr(weight_sum)
        h.loss_scale, h.loss_rows = float(loss_scale), float(loss_rows)
        h.loss, h.loss_sum = out["loss"].data_ptr(), _ptr(loss_sum)
        h.row_loss, h.lse = out["row_loss"].data_ptr(), out["lse"].data_ptr()
        lib = _lib.load()
        nbytes = C.c_size_t(0)
        _lib.check(lib.suave_linear_ce_workspace_bytes(C.byref(h), C.byref(nbytes)), "suave_linear_ce_workspace_bytes")
        ws = _workspace(nbytes.value, dev)
        h.workspace, h.workspace_bytes = ws.data_ptr(), nbytes.value
        _lib.check(lib.suave_linear_ce(C.byref(h), _stream(dev)), "suave_linear_ce")
    return out


def orthogonalize(matrices: Sequence[torch.Tensor], *, steps: int = 5, eps: float = 1e-7,
                  out: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
    """Newton-Schulz orthogonalisation of a list of matrices at once (``suave_orthogonalize``): float32 or bfloat16 (one type
    for the list), rows contiguous, any row stride; ``out`` may be the matrices themselves.  ``steps`` times
    ``X <- (a I + b X X^T + c (X X^T)^2) X`` from ``X = U / (|U|_F + eps)``."""

    matrices = list(matrices)
    if not matrices:
        return []
    dev = _device_of("matrices[0]", matrices[0])
    dt = matrices[0].dtype
    _need(dt in _DTYPES, f"matrices must have one of the types {[str(d) for d in _DTYPES]}")
    lds = [_matrix(f"matrices[{i}]", t, dev, (dt,)) for i, t in enumerate(matrices)]
    _need(all(t.numel() > 0 for t in matrices), "a matrix needs at least one row and one column")
    with _on(dev):
        if out is None:
            out = [torch.empty(t.shape, dtype=dt, device=dev) for t in matrices]
        out = list(out)
        _need(len(out) == len(matrices), "out must have one matrix for each")
        arr = (OrthoMatrixT * len(matrices))()
        for i, (a, t, o) in enumerate(zip(arr, matrices, out)):
            a.ld_out = _matrix(f"out[{i}]", o, dev, (dt,), t.shape)
            a.in_, a.out, a.ld_in, a.rows, a.cols = t.data_ptr(), o.data_ptr(), lds[i], int(t.shape[0]), int(t.shape[1])
        lib = _lib.load()
        nbytes = C.c_size_t(0)
        _lib.check(lib.suave_orthogonalize_workspace_bytes(arr, len(matrices), _DTYPES[dt], C.byref(nbytes)),
                   "suave_orthogonalize_workspace_bytes")
        ws = _workspace(nbytes.value, dev)
        _lib.check(lib.suave_orthogonalize(arr, len(matrices), _DTYPES[dt], int(steps), float(eps), ws.data_ptr(), nbytes.value,
                                           _stream(dev)), "suave_orthogonalize")
    return out


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], *, lr,
              momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5, eps: float = 1e-7) -> None:
    """One Muon step in place on a list of float32 weight matrices (``suave_muon_step``): ``momentum`` averaging, the
    orthogonalised update of each matrix, ``param <- (1 - lr weight_decay) param - lr sqrt(max(1, rows / cols)) O``.  ``lr``: a
    number, or one for each matrix.  ``momenta`` start as zeros.  Rows contiguous, any row stride (views of a flat buffer)."""

    params, grads, momenta = list(params), list(grads), list(momenta)
    n = len(params)
    _need(len(grads) == n and len(momenta) == n, "params, grads and momenta must have the same length")
    lrs = [float(lr)] * n if not isinstance(lr, (list, tuple)) else [float(v) for v in lr]
    _need(len(lrs) == n, "lr must be a number or one for each matrix")
    if not n:
        return
    dev = _device_of("params[0]", params[0])
    f32 = (torch.float32,)
    arr = (MuonMatrixT * n)()
    for i, (a, p, g, m) in enumerate(zip(arr, params, grads, momenta)):
        a.ld_param = _matrix(f"params[{i}]", p, dev, f32)
        _need(p.numel() > 0, "a matrix needs at least one row and one column")
        a.ld_grad, a.ld_momentum = _matrix(f"grads[{i}]", g, dev, f32, p.shape), _matrix(f"momenta[{i}]", m, dev, f32, p.shape)
        a.param, a.grad, a.momentum = p.data_ptr(), g.data_ptr(), m.data_ptr()
        a.rows, a.cols, a.lr = int(p.shape[0]), int(p.shape[1]), lrs[i]
    with _on(dev):
        lib = _lib.load()
        nbytes = C.c_size_t(0)
        _lib.check(lib.suave_muon_workspace_bytes(arr, n, C.byref(nbytes)), "suave_muon_workspace_bytes")
        ws = _workspace(nbytes.value, dev)
        _lib.check(lib.suave_muon_step(arr, n, float(momentum), int(bool(nesterov)), float(weight_decay), int(steps), float(eps), ws.data_ptr(), nbytes.value,
                                       _stream(dev)), "suave_muon_step")


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` [rows, cols] (float32 / bfloat16) in 8 bits with one scale per row (``suave_quantize_rows``): ``(q, scale)``
    with ``q`` int8 [rows, cols], the nearest integers of ``x / scale`` within +-127 (rows start at multiples of 16 bytes), and ``scale``
    float32 [rows] = max |x| (1/127), as torch divides by 127.0 on the device.  The form ``linear_quantized`` takes a layer's weight in."""

    dev = _device_of("x", x)
    ld = _matrix("x", x, dev, tuple(_DTYPES))
    n, k = int(x.shape[0]), int(x.shape[1])
    _need(k >= 1, "x must have at least one column")
    with _on(dev):
        q = torch.empty((n, (k + 15) // 16 * 16), dtype=torch.int8, device=dev)
        scale = torch.empty(n, dtype=torch.float32, device=dev)
        _lib.check(_lib.load().suave_quantize_rows(x.data_ptr(), _DTYPES[x.dtype], n, k, ld, q.data_ptr(), int(q.shape[1]),
                                                   scale.data_ptr(), _stream(dev)), "suave_quantize_rows")
    return q[:, :k], scale


def linear_quantized(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ (weight * weight_scale[:, None]).T + bias`` with ``x`` quantised per row in the call and exact integer sums
    (``suave_linear_quantized``).  ``x`` [rows, in] float32 / bfloat16 and the result [rows, out] of the same type;
    ``weight`` int8 [out, in] and ``weight_scale`` float32 [out] as ``quantize_rows`` gives them: rows 16-byte aligned, a
    row stride that is a multiple of 16.  ``out`` may not overlap an input."""

    dev = _device_of("x", x)
    ld = _matrix("x", x, dev, tuple(_DTYPES))
    n, k = int(x.shape[0]), int(x.shape[1])
    ldw = _matrix("weight", weight, dev, (torch.int8,))
    c = int(weight.shape[0])
    if weight.shape[1] != k:
        raise ValueError(f"weight must have {k} columns, as x")
    _need(c >= 1 and k >= 1, "weight must have at least one row and one column")
    if c == 1:
        ldw = (k + 15) // 16 * 16
    _need(ldw % 16 == 0 and weight.data_ptr() % 16 == 0, "weight: rows must start at multiples of 16 bytes (quantize_rows)")
    held = weight.untyped_storage().nbytes() - weight.storage_offset() if k % 16 else c * ldw
    _need(held >= (c - 1) * ldw + (k + 15) // 16 * 16, "weight: the last row must be held up to a multiple of 16 (quantize_rows)")
    _vector("weight_scale", weight_scale, dev, torch.float32, c)
    if bias is not None:
        _vector("bias", bias, dev, torch.float32, c)
    with _on(dev):
        h = LinearQuantizedT()
        if out is None:
            out = torch.empty((n, c), dtype=x.dtype, device=dev)
            h.ld_out = c
        else:
            h.ld_out = _matrix("out", out, dev, (x.dtype,), (n, c))
        h.dtype, h.n_out, h.n_in, h.n_rows = _DTYPES[x.dtype], c, k, n
        h.x, h.ld_x, h.weight, h.ld_weight = x.data_ptr(), ld, weight.data_ptr(), ldw
        h.weight_scale, h.bias, h.out = weight_scale.data_ptr(), _ptr(bias), out.data_ptr()
        lib = _lib.load()
        nbytes = C.c_size_t(0)
        _lib.check(lib.suave_linear_quantized_workspace_bytes(C.byref(h), C.byref(nbytes)), "suave_linear_quantized_workspace_bytes")
        ws = _workspace(nbytes.value, dev)
        h.workspace, h.workspace_bytes = ws.data_ptr(), nbytes.value
        _lib.check(lib.suave_linear_quantized(C.byref(h), _stream(dev)), "suave_linear_quantized")
    return out
