"""Products with one operand held in few bits, beside `runner.gemm`.

Weights in 4 bits with group scales (serving):

    w = quantize_w4(weight, group=128)            # weight: out_features x in_features, f16 or bf16
    y = gemm_w4(x, w)                             # x @ W^T, from one row (a token) to thousands (a prompt)

Activations saved in 8 bits for the backward pass (training):

    saved = save8(x)                              # half the bytes of x; x can be freed
    dw = weight_grad8(saved, dy)                  # x^T @ dy, in fp32 (or rounded to dy's type), straight from the codes
    dw = weight_grad8(saved, dy, base=dw, out=dw) # added to the gradient of earlier micro batches

The formats and the exact rounding rules are described in include/subcuber_b200.h.  All compute happens in the CUDA
library, asynchronously on the current stream of the operands' device; every call can be captured into a graph.  A
workspace that is passed in serves one call at a time: calls that may overlap (other streams, two captured graphs that
are replayed at once) need one each.  The reference project has no counterpart.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .runner import KernelError

DTYPE_CODE = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 3}
HALF_TYPES = (torch.float16, torch.bfloat16)
GROUPS = (32, 64, 128)
ACT_BLOCK = 32   # channels of a token that share a step


def _matrix(name: str, t: torch.Tensor, dtypes) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor: this backend has no CPU path")
    if t.dim() != 2:
        raise ValueError(f"{name} must be a matrix")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, not {t.dtype}")
    # (the stride of an axis of one element is never used)
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have its rows in consecutive elements")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"the rows of {name} must not overlap")


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _same_device(*tensors) -> None:
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise ValueError(f"operands are on different devices: {sorted(map(str, devices))}")


def _output(name: str, t: Optional[torch.Tensor], shape, dtype, device) -> torch.Tensor:
    if t is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _matrix(name, t, (dtype,))
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {shape[0]} x {shape[1]}")
    return t


def _call(what: str, fn, device: torch.device, *args) -> None:
    # the library works on the current device: make the operands' device current where it is not
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc != 0:
        raise KernelError(what, rc)


class _Workspace:
    def check(self) -> None:
        """Wait for the call that used the workspace last and raise if a device-side wait gave up."""
        with torch.cuda.device(self.buf.device):
            rc = _lib.load().sb200_gemm_status(self.ptr, torch.cuda.current_stream(self.buf.device).cuda_stream)
        if rc != 0:
            raise KernelError("workspace", rc)

    def _allocate(self, nbytes: int, device) -> None:
        self.nbytes = nbytes
        self.buf = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
        self.ptr = self.buf.data_ptr() + (-self.buf.data_ptr()) % 256
        self.buf[:512].zero_()   # the status word


class WeightsW4:
    """Weights in 4 bits, in the library's order: `codes` uint8, `scales` in the activations' type, `zeros` uint8 or None
    (symmetric), all flat.  Made by `quantize_w4` or `pack_w4`."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor], n: int, k: int, group: int):
        lib = _lib.load()
        _check_w4(n, k, group)
        _same_device(codes, scales, zeros)
        nbytes, entries = int(lib.sb200_w4_codes_bytes(n, k)), int(lib.sb200_w4_table_entries(n, k, group))
        if scales.dtype not in HALF_TYPES:
            raise ValueError(f"scales must be one of {[str(d) for d in HALF_TYPES]}, not {scales.dtype}")
        for name, t, dtype, count in (("codes", codes, torch.uint8, nbytes), ("scales", scales, scales.dtype, entries),
                                      ("zeros", zeros, torch.uint8, entries)):
            if t is not None and (not t.is_cuda or t.dtype != dtype or t.numel() != count or not t.is_contiguous()):
                raise ValueError(f"{name} must be a packed CUDA tensor of {count} {dtype}")
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.n, self.k, self.group = n, k, group
        self.dtype, self.device = scales.dtype, scales.device
        self._zeros_ptr = zeros.data_ptr() if zeros is not None else None

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.zeros) if t is not None)


def _check_w4(n: int, k: int, group: int) -> None:
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}")
    if n <= 0 or k <= 0:
        raise ValueError("weights need at least one output and one input")


def _empty_w4(n: int, k: int, group: int, symmetric: bool, dtype, device) -> WeightsW4:
    lib = _lib.load()
    _check_w4(n, k, group)
    entries = int(lib.sb200_w4_table_entries(n, k, group))
    return WeightsW4(torch.empty(int(lib.sb200_w4_codes_bytes(n, k)), dtype=torch.uint8, device=device),
                     torch.empty(entries, dtype=dtype, device=device),
                     None if symmetric else torch.empty(entries, dtype=torch.uint8, device=device), n, k, group)


def quantize_w4(weight: torch.Tensor, group: int = 128, symmetric: bool = False) -> WeightsW4:
    """Quantise `weight` (out_features x in_features, f16 or bf16) to 4 bits, rounding to nearest within each group."""
    _matrix("weight", weight, HALF_TYPES)
    n, k = weight.shape
    w = _empty_w4(n, k, group, symmetric, weight.dtype, weight.device)
    _call("quantize_w4", _lib.load().sb200_w4_quantize, weight.device, DTYPE_CODE[weight.dtype], weight.data_ptr(), _ld(weight),
          n, k, group, w.codes.data_ptr(), w.scales.data_ptr(), w._zeros_ptr)
    return w


def pack_w4(q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, group: int = 128) -> WeightsW4:
    """Weights that another quantiser made: `q` [n, k] uint8 codes 0..15, `scales` [groups, n] f16 or bf16, `zeros`
    [groups, n] uint8 0..15 or None (then 8)."""
    _matrix("q", q, (torch.uint8,))
    _matrix("scales", scales, HALF_TYPES)
    n, k = q.shape
    _same_device(q, scales, zeros)
    _check_w4(n, k, group)
    if zeros is not None:
        _matrix("zeros", zeros, (torch.uint8,))
    for name, t in (("scales", scales), ("zeros", zeros)):
        if t is not None and tuple(t.shape) != (-(-k // group), n):
            raise ValueError(f"{name} must be a {-(-k // group)} x {n} table")
    w = _empty_w4(n, k, group, zeros is None, scales.dtype, q.device)
    _call("pack_w4", _lib.load().sb200_w4_pack, q.device, DTYPE_CODE[w.dtype], q.data_ptr(), _ld(q), scales.data_ptr(),
          _ld(scales), zeros.data_ptr() if zeros is not None else None, _ld(zeros) if zeros is not None else n, n, k, group,
          w.codes.data_ptr(), w.scales.data_ptr(), w._zeros_ptr)
    return w


def dequantize_w4(w: WeightsW4, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weights (out_features x in_features) that `w` stands for, rounded once to its type."""
    out = _output("out", out, (w.n, w.k), w.dtype, w.device)
    _same_device(w.codes, out)
    _call("dequantize_w4", _lib.load().sb200_w4_dequantize, w.device, DTYPE_CODE[w.dtype], w.codes.data_ptr(),
          w.scales.data_ptr(), w._zeros_ptr, w.n, w.k, w.group, out.data_ptr(), _ld(out))
    return out


def _tma_rows(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0 and _ld(t) % 8 == 0


class WorkspaceW4(_Workspace):
    """Device workspace for `gemm_w4` with up to `m` rows; for one call at a time.  `aligned`: the rows of x will start on 16
    bytes (the default expects packed rows); else there is room for a copy of x."""

    def __init__(self, m: int, w: WeightsW4, aligned: Optional[bool] = None):
        lib = _lib.load()
        with torch.cuda.device(w.device):  # a product is cut for the device that will run it
            self._allocate(int(lib.sb200_w4_gemm_workspace_bytes(DTYPE_CODE[w.dtype], m, w.n, w.k, w.group,
                                                                 int(w.k % 8 == 0 if aligned is None else aligned))), w.device)


def gemm_w4(x: torch.Tensor, w: WeightsW4, out: Optional[torch.Tensor] = None,
            workspace: Optional[WorkspaceW4] = None) -> torch.Tensor:
    """x @ W^T (m x out_features) for x (m x in_features) of the weights' type; sums in fp32."""
    _matrix("x", x, (w.dtype,))
    m = x.shape[0]
    if x.shape[1] != w.k:
        raise ValueError(f"x has {x.shape[1]} columns, the weights {w.k} inputs")
    out = _output("out", out, (m, w.n), w.dtype, x.device)
    _same_device(x, w.codes, out)
    if workspace is None:
        workspace = WorkspaceW4(m, w, _tma_rows(x))
    _call("gemm_w4", _lib.load().sb200_w4_gemm, w.device, DTYPE_CODE[w.dtype], x.data_ptr(), _ld(x), w.codes.data_ptr(),
          w.scales.data_ptr(), w._zeros_ptr, out.data_ptr(), _ld(out), m, w.n, w.k, w.group, workspace.ptr, workspace.nbytes)
    return out


class Checkpoint8:
    """Activations saved in 8 bits: `codes` [m, pitch] uint8 and `exponents` [m, exponent pitch] uint8 of m tokens x k
    channels; `dtype` is the activations'.  Made by `save8`."""

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, k: int, dtype: torch.dtype):
        if dtype not in HALF_TYPES:
            raise ValueError("saved activations are f16 or bf16")
        if k <= 0:
            raise ValueError("activations need at least one channel")
        _same_device(codes, exponents)
        for name, t, cols, unit in (("codes", codes, k, 16), ("exponents", exponents, -(-k // ACT_BLOCK), 4)):
            _matrix(name, t, (torch.uint8,))
            if t.shape[1] < cols or t.shape[1] % unit or _ld(t) % unit or t.data_ptr() % unit:
                raise ValueError(f"rows of {name} must hold {cols} bytes, padded and aligned to {unit}")
        if codes.shape[0] != exponents.shape[0]:
            raise ValueError("codes and exponents must have the same tokens")
        self.codes, self.exponents = codes, exponents
        self.m, self.k, self.dtype, self.device = codes.shape[0], k, dtype, codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()


def save8(x: torch.Tensor, out: Optional[Checkpoint8] = None) -> Checkpoint8:
    """Save activations x (tokens x channels, f16 or bf16) in 8 bits, into `out` where it is given."""
    _matrix("x", x, HALF_TYPES)
    m, k = x.shape
    if out is None:
        out = Checkpoint8(torch.empty((m, -(-k // 16) * 16), dtype=torch.uint8, device=x.device),
                          torch.empty((m, -(-k // (4 * ACT_BLOCK)) * 4), dtype=torch.uint8, device=x.device), k, x.dtype)
    elif (out.m, out.k, out.dtype) != (m, k, x.dtype):
        raise ValueError(f"out holds {out.m} x {out.k} {out.dtype}, x is {m} x {k} {x.dtype}")
    _same_device(x, out.codes)
    _call("save8", _lib.load().sb200_act8_save, x.device, DTYPE_CODE[x.dtype], x.data_ptr(), _ld(x), m, k, out.codes.data_ptr(),
          _ld(out.codes), out.exponents.data_ptr(), _ld(out.exponents))
    return out


def restore8(saved: Checkpoint8, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The activations (tokens x channels) that `saved` stands for, exact in its type."""
    out = _output("out", out, (saved.m, saved.k), saved.dtype, saved.device)
    _same_device(saved.codes, out)
    _call("restore8", _lib.load().sb200_act8_restore, saved.device, DTYPE_CODE[saved.dtype], saved.codes.data_ptr(),
          _ld(saved.codes), saved.exponents.data_ptr(), _ld(saved.exponents), saved.m, saved.k, out.data_ptr(), _ld(out))
    return out


class WorkspaceGrad8(_Workspace):
    """Device workspace for `weight_grad8` of `saved` against n output channels; for one call at a time.  `aligned`: the
    rows of dy will start on 16 bytes (the default expects packed rows); else there is room for a copy of dy."""

    def __init__(self, saved: Checkpoint8, n: int, out_dtype: torch.dtype = torch.float32, aligned: Optional[bool] = None):
        lib = _lib.load()
        with torch.cuda.device(saved.device):
            self._allocate(int(lib.sb200_act8_wgrad_workspace_bytes(DTYPE_CODE[saved.dtype], DTYPE_CODE[out_dtype], saved.m,
                                                                    n, saved.k, int(n % 8 == 0 if aligned is None else aligned))),
                           saved.device)


def weight_grad8(saved: Checkpoint8, dy: torch.Tensor, base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 out_dtype: torch.dtype = torch.float32, workspace: Optional[WorkspaceGrad8] = None) -> torch.Tensor:
    """base + X^T @ dy (in_features x out_features, the layout of `gemm`'s B) for the saved activations X and the output
    gradient dy (tokens x out_features) of the same type.  The result is fp32 or has dy's type; `base` and `out` have
    the result's type, and may be the same tensor."""
    _matrix("dy", dy, (saved.dtype,))
    n = dy.shape[1]
    if dy.shape[0] != saved.m:
        raise ValueError(f"dy has {dy.shape[0]} rows, {saved.m} tokens were saved")
    if n == 0:
        raise ValueError("dy needs at least one column")
    if out is not None:
        out_dtype = out.dtype
    if out_dtype not in (torch.float32, saved.dtype):
        raise ValueError(f"the gradient is float32 or {saved.dtype}")
    if base is not None:
        _matrix("base", base, (out_dtype,))
        if tuple(base.shape) != (saved.k, n):
            raise ValueError(f"base must be {saved.k} x {n}")
    out = _output("out", out, (saved.k, n), out_dtype, dy.device)
    _same_device(dy, saved.codes, out, base)
    if workspace is None:
        workspace = WorkspaceGrad8(saved, n, out_dtype, _tma_rows(dy))
    _call("weight_grad8", _lib.load().sb200_act8_wgrad, saved.device, DTYPE_CODE[saved.dtype], saved.codes.data_ptr(),
          _ld(saved.codes), saved.exponents.data_ptr(), _ld(saved.exponents), dy.data_ptr(), _ld(dy), DTYPE_CODE[out_dtype],
          base.data_ptr() if base is not None else None, _ld(base) if base is not None else n, out.data_ptr(), _ld(out),
          saved.m, n, saved.k, workspace.ptr, workspace.nbytes)
    return out
