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
are replayed at once) need one each.

Every wait inside a kernel is bounded.  A product whose wait gave up (2 s, or the bound in `opts`) leaves an incomplete result and
a status: `check=True` waits for the call and raises, or, with a workspace of one's own, its `check()` does at any time
before the next call that uses it.  Without either nothing is reported.

As with `runner.gemm` there is no autograd here: a result of tensors that require gradients does not.  The reference project has
no counterpart.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from .runner import KernelError

DTYPE_CODE = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 3}
HALF_TYPES = (torch.float16, torch.bfloat16)
GROUPS = (32, 64, 128)
ACT_BLOCK = 32   # channels of a token that share a step
MAX_EXTENT = 0x7fffff00  # of any axis: the library holds extents, rounded up to whole tiles, in 32 bits (ctypes would cut more bits off)


# handle of the current stream of a device (the public call builds a Stream object, which takes 2 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _matrix(name: str, t: torch.Tensor, dtypes) -> None:
    # (the stride of an axis of one element is never used)
    if t.is_cuda and t.dtype in dtypes and t.dim() == 2:
        rows, cols = t.shape
        ld, step = t.stride()
        if (step == 1 or cols <= 1) and (ld >= cols or rows <= 1) and rows <= MAX_EXTENT and cols <= MAX_EXTENT:
            return
        _extent(f"{name}'s rows", rows)
        _extent(f"{name}'s columns", cols)
        raise ValueError(f"{name} must have its rows in consecutive elements, rows that do not overlap")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor: this backend has no CPU path")
    if t.dim() != 2:
        raise ValueError(f"{name} must be a matrix")
    raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, not {t.dtype}")


def _extent(name: str, count: int) -> None:
    if not 0 <= count <= MAX_EXTENT:
        raise ValueError(f"{name}: {count}, must be 0 to {MAX_EXTENT}")


def _ld(t: torch.Tensor) -> int:
    # (a single row has no second one that could start off the 16-byte grid)
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else max(-(-cols // 8) * 8, 8)


def _same_device(first, *others) -> None:
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"operands are on different devices: {device} and {t.device}")


def _output(name: str, t: torch.Tensor, shape, dtype, device) -> None:
    _matrix(name, t, (dtype,))
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape[0]} x {shape[1]}")
    if t.device != device:
        raise ValueError(f"operands are on different devices: {device} and {t.device}")


_functions: dict = {}


def _call(what: str, device: torch.device, *args, behind=()) -> None:
    """Call the library's `what` on the current stream of `device`, with `device` current (`behind`: what follows the stream)."""
    fn = _functions.get(what)
    if fn is None:
        fn = _functions[what] = getattr(_lib.load(), what)
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index), *behind)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index), *behind)
    if rc != 0:
        raise KernelError(what, rc)


def _status(ptr: int, device) -> None:
    with torch.cuda.device(device):
        rc = _lib.load().sb200_gemm_status(ptr, _raw_stream(device.index))
    if rc != 0:
        raise KernelError("product with an operand in few bits", rc)


class _Workspace:
    def __init__(self, nbytes: int, device: torch.device):
        self.nbytes = nbytes
        self.device = device
        self.buf = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
        self.ptr = self.buf.data_ptr() + (-self.buf.data_ptr()) % 256
        self.buf[:512].zero_()   # the status word: products of a few rows leave it alone

    def _for(self, device: torch.device):
        if self.device != device:
            raise ValueError(f"the workspace is on {self.device}, the operands on {device}")
        return self.ptr, self.nbytes

    def check(self) -> None:
        """Wait for the calls so far and raise if a device-side wait of the last product in this workspace gave up (`gemm_w4` of up to 8
        rows has no waits and leaves the status of the product before it)."""
        _status(self.ptr, self.device)


def _check_w4(n: int, k: int, group: int) -> None:
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}")
    if n <= 0 or k <= 0:
        raise ValueError("weights need at least one output and one input")
    _extent("outputs", n)
    _extent("inputs", k)


class WeightsW4:
    """Weights in 4 bits (out_features n x in_features k), in the library's order: `codes` uint8, `scales` in the activations'
    type, `zeros` uint8 or None (symmetric), all flat.  Made by `quantize_w4` or `pack_w4`."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor], n: int, k: int, group: int):
        lib = _lib.load()
        _check_w4(n, k, group)
        nbytes, entries = int(lib.sb200_w4_codes_bytes(n, k)), int(lib.sb200_w4_table_entries(n, k, group))
        if scales.dtype not in HALF_TYPES:
            raise ValueError(f"scales must be one of {[str(d) for d in HALF_TYPES]}, not {scales.dtype}")
        for name, t, dtype, count in (("codes", codes, torch.uint8, nbytes), ("scales", scales, scales.dtype, entries),
                                      ("zeros", zeros, torch.uint8, entries)):
            if t is not None and (not t.is_cuda or t.dtype != dtype or t.numel() != count or not t.is_contiguous()):
                raise ValueError(f"{name} must be a packed CUDA tensor of {count} {dtype}")
        _same_device(codes, scales, zeros)
        self._tensors = (codes, scales, zeros)
        self._set(n, k, group, scales.dtype, scales.device, codes.data_ptr(), scales.data_ptr(),
                  zeros.data_ptr() if zeros is not None else None)
        # the status word of products that need no other workspace and are not checked
        self._own = torch.empty(512, dtype=torch.uint8, device=self.device)
        self._status_ptr = self._own.data_ptr() + (-self._own.data_ptr()) % 256

    def _set(self, n, k, group, dtype, device, codes_ptr, scales_ptr, zeros_ptr) -> None:
        self.n, self.k, self.group, self.dtype, self.device = n, k, group, dtype, device
        self._ptrs = (codes_ptr, scales_ptr, zeros_ptr)
        self._code = DTYPE_CODE[dtype]

    @classmethod
    def _empty(cls, n: int, k: int, group: int, symmetric: bool, dtype, device) -> "WeightsW4":
        """One allocation for everything; the tensors are made when they are asked for."""
        _check_w4(n, k, group)
        rows, blocks = -(-n // 16) * 16, -(-k // 128)
        nbytes, entries = rows * blocks * 64, rows * blocks * (128 // group)
        w = cls.__new__(cls)
        buf = torch.empty(512 + nbytes + entries * (2 if symmetric else 3), dtype=torch.uint8, device=device)
        base = buf.data_ptr()
        w._own, w._tensors, w._sizes = buf, None, (nbytes, entries, symmetric)
        w._status_ptr = base + (-base) % 256
        codes = base + 512
        w._set(n, k, group, dtype, device, codes, codes + nbytes, None if symmetric else codes + nbytes + 2 * entries)
        return w

    def _tensor(self, i: int):
        if self._tensors is None:
            nbytes, entries, symmetric = self._sizes
            b = self._own[512:]
            self._tensors = (b[:nbytes], b[nbytes:nbytes + 2 * entries].view(self.dtype),
                             None if symmetric else b[nbytes + 2 * entries:])
        return self._tensors[i]

    codes = property(lambda self: self._tensor(0))
    scales = property(lambda self: self._tensor(1))
    zeros = property(lambda self: self._tensor(2))

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.zeros) if t is not None)


def quantize_w4(weight: torch.Tensor, group: int = 128, symmetric: bool = False) -> WeightsW4:
    """Quantise `weight` (out_features x in_features, f16 or bf16) to 4 bits, rounding to nearest within each group."""
    _matrix("weight", weight, HALF_TYPES)
    n, k = weight.shape
    w = WeightsW4._empty(n, k, group, symmetric, weight.dtype, weight.device)
    _call("sb200_w4_quantize", w.device, w._code, weight.data_ptr(), _ld(weight), n, k, group, *w._ptrs)
    return w


def pack_w4(q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, group: int = 128) -> WeightsW4:
    """Weights that another quantiser made: `q` [n, k] uint8 codes 0..15, `scales` [groups, n] f16 or bf16, `zeros`
    [groups, n] uint8 0..15 or None (then 8)."""
    _matrix("q", q, (torch.uint8,))
    _matrix("scales", scales, HALF_TYPES)
    n, k = q.shape
    _check_w4(n, k, group)
    if zeros is not None:
        _matrix("zeros", zeros, (torch.uint8,))
    for name, t in (("scales", scales), ("zeros", zeros)):
        if t is not None and tuple(t.shape) != (-(-k // group), n):
            raise ValueError(f"{name} must be a {-(-k // group)} x {n} table")
    _same_device(q, scales, zeros)
    w = WeightsW4._empty(n, k, group, zeros is None, scales.dtype, q.device)
    _call("sb200_w4_pack", w.device, w._code, q.data_ptr(), _ld(q), scales.data_ptr(), _ld(scales),
          zeros.data_ptr() if zeros is not None else None, _ld(zeros) if zeros is not None else n, n, k, group, *w._ptrs)
    return w


def dequantize_w4(w: WeightsW4, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weights (out_features x in_features) that `w` stands for, rounded once to its type."""
    if out is None:
        out = torch.empty((w.n, w.k), dtype=w.dtype, device=w.device)
    else:
        _output("out", out, (w.n, w.k), w.dtype, w.device)
    _call("sb200_w4_dequantize", w.device, w._code, *w._ptrs, w.n, w.k, w.group, out.data_ptr(), _ld(out))
    return out


class WorkspaceW4(_Workspace):
    """Device workspace for `gemm_w4` with up to `m` rows; for one call at a time.  `aligned`: the rows of x will start on 16
    bytes (the default expects packed rows); else there is room for a copy of x.  From 65 rows on up to 64 MB, from 1280 rows on the
    weights in 16 bits besides."""

    def __init__(self, m: int, w: WeightsW4, aligned: Optional[bool] = None):
        _extent("rows", m)
        aligned = w.k % 8 == 0 if aligned is None else aligned
        with torch.cuda.device(w.device):  # a product is cut for the device that will run it
            super().__init__(int(_lib.load().sb200_w4_gemm_workspace_bytes(w._code, m, w.n, w.k, w.group, int(aligned))), w.device)


def gemm_w4(x: torch.Tensor, w: WeightsW4, out: Optional[torch.Tensor] = None, workspace: Optional[WorkspaceW4] = None,
            check: bool = False, opts=None) -> torch.Tensor:
    """x @ W^T (m x out_features) for x (m x in_features) of the weights' type; sums in fp32.  Up to 8 rows the codes and scales are
    exact, with more the weights are those of `dequantize_w4`, rounded to their type.  `out` must not overlap x.
    `check` synchronises and raises if a device-side wait gave up; `opts` (`runner.options`): the bound of those waits."""
    _matrix("x", x, (w.dtype,))
    m, k = x.shape
    if k != w.k:
        raise ValueError(f"x has {k} columns, the weights {w.k} inputs")
    if x.device != w.device:
        raise ValueError(f"operands are on different devices: {x.device} and {w.device}")
    if out is None:
        out = x.new_empty((m, w.n))   # (the type and device of the weights)
    else:
        _output("out", out, (m, w.n), w.dtype, w.device)
    ldx, x_ptr = _ld(x), x.data_ptr()
    if workspace is not None:
        ptr, nbytes = workspace._for(w.device)
    elif m <= 64 and x_ptr % 16 == 0 and ldx % 8 == 0 and not check:
        ptr, nbytes = w._status_ptr, 256     # few rows need a status word only; calls at once may share one that is not read
    else:
        workspace = WorkspaceW4(m, w, x_ptr % 16 == 0 and ldx % 8 == 0)
        ptr, nbytes = workspace.ptr, workspace.nbytes
    args = (w._code, x_ptr, ldx, *w._ptrs, out.data_ptr(), _ld(out), m, w.n, k, w.group, ptr, nbytes)
    if opts is None:
        _call("sb200_w4_gemm", w.device, *args)
    else:
        _call("sb200_w4_gemm_opt", w.device, *args, behind=(C.byref(opts),))
    if check:
        torch.cuda.current_stream(w.device).synchronize()
        if m > 8:                            # (below, the kernel has no waits and leaves the word alone)
            _status(ptr, w.device)
    return out


class Checkpoint8:
    """Activations saved in 8 bits: `codes` [m, pitch] uint8 and `exponents` [m, exponent pitch] uint8 of m tokens x k
    channels; `dtype` is the activations'.  Made by `save8`."""

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, k: int, dtype: torch.dtype):
        if dtype not in HALF_TYPES:
            raise ValueError("saved activations are f16 or bf16")
        if k <= 0:
            raise ValueError("activations need at least one channel")
        for name, t, cols, unit in (("codes", codes, k, 16), ("exponents", exponents, -(-k // ACT_BLOCK), 4)):
            _matrix(name, t, (torch.uint8,))
            if t.shape[1] < cols or t.shape[1] % unit or _ld(t) % unit or t.data_ptr() % unit:
                raise ValueError(f"rows of {name} must hold {cols} bytes, padded and aligned to {unit}")
        if codes.shape[0] != exponents.shape[0]:
            raise ValueError("codes and exponents must have the same tokens")
        _same_device(codes, exponents)
        self._tensors = (codes, exponents)
        self._set(codes.shape[0], k, dtype, codes.device, codes.data_ptr(), _ld(codes), exponents.data_ptr(), _ld(exponents))

    def _set(self, m, k, dtype, device, codes_ptr, pitch, exp_ptr, exp_pitch) -> None:
        self.m, self.k, self.dtype, self.device = m, k, dtype, device
        self._layout = (codes_ptr, pitch, exp_ptr, exp_pitch)
        self._code = DTYPE_CODE[dtype]

    @classmethod
    def _empty(cls, m: int, k: int, dtype, device) -> "Checkpoint8":
        """One allocation for both; the tensors are made when they are asked for."""
        if k <= 0:
            raise ValueError("activations need at least one channel")
        pitch, exp_pitch = -(-k // 16) * 16, -(-k // (4 * ACT_BLOCK)) * 4
        c = cls.__new__(cls)
        c._own, c._tensors = torch.empty(m * (pitch + exp_pitch), dtype=torch.uint8, device=device), None
        base = c._own.data_ptr()
        c._set(m, k, dtype, device, base, pitch, base + m * pitch, exp_pitch)
        return c

    def _tensor(self, i: int) -> torch.Tensor:
        if self._tensors is None:
            cut = self.m * self._layout[1]
            self._tensors = (self._own[:cut].view(self.m, self._layout[1]), self._own[cut:].view(self.m, self._layout[3]))
        return self._tensors[i]

    codes = property(lambda self: self._tensor(0))
    exponents = property(lambda self: self._tensor(1))

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()


def save8(x: torch.Tensor, out: Optional[Checkpoint8] = None) -> Checkpoint8:
    """Save activations x (tokens x channels, f16 or bf16) in 8 bits, into `out` where it is given."""
    _matrix("x", x, HALF_TYPES)
    m, k = x.shape
    if out is None:
        out = Checkpoint8._empty(m, k, x.dtype, x.device)
    elif (out.m, out.k, out.dtype) != (m, k, x.dtype):
        raise ValueError(f"out holds {out.m} x {out.k} {out.dtype}, x is {m} x {k} {x.dtype}")
    elif out.device != x.device:
        raise ValueError(f"operands are on different devices: {x.device} and {out.device}")
    _call("sb200_act8_save", out.device, out._code, x.data_ptr(), _ld(x), m, k, *out._layout)
    return out


def restore8(saved: Checkpoint8, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The activations (tokens x channels) that `saved` stands for, exact in its type."""
    if out is None:
        out = torch.empty((saved.m, saved.k), dtype=saved.dtype, device=saved.device)
    else:
        _output("out", out, (saved.m, saved.k), saved.dtype, saved.device)
    _call("sb200_act8_restore", saved.device, saved._code, *saved._layout, saved.m, saved.k, out.data_ptr(), _ld(out))
    return out


class WorkspaceGrad8(_Workspace):
    """Device workspace for `weight_grad8` of `saved` against n output channels; for one call at a time.  `aligned`: the
    rows of dy will start on 16 bytes (the default expects packed rows); else there is room for a copy of dy."""

    def __init__(self, saved: Checkpoint8, n: int, out_dtype: torch.dtype = torch.float32, aligned: Optional[bool] = None):
        if out_dtype != torch.float32 and out_dtype != saved.dtype:
            raise ValueError(f"the gradient is float32 or {saved.dtype}")
        _extent("output channels", n)
        aligned = n % 8 == 0 if aligned is None else aligned
        with torch.cuda.device(saved.device):
            super().__init__(int(_lib.load().sb200_act8_wgrad_workspace_bytes(saved._code, DTYPE_CODE[out_dtype], saved.m, n,
                                                                              saved.k, int(aligned))), saved.device)


def weight_grad8(saved: Checkpoint8, dy: torch.Tensor, base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 out_dtype: torch.dtype = torch.float32, workspace: Optional[WorkspaceGrad8] = None,
                 check: bool = False, opts=None) -> torch.Tensor:
    """base + X^T @ dy (in_features x out_features, the layout of `gemm`'s B) for the saved activations X and the output
    gradient dy (tokens x out_features) of the same type.  The result is fp32 or has dy's type; `base` and `out` have
    the result's type, and may be the same tensor; `out` overlaps no other operand.  `check` and `opts` as in `gemm_w4`."""
    _matrix("dy", dy, (saved.dtype,))
    m, n = dy.shape
    if m != saved.m:
        raise ValueError(f"dy has {m} rows, {saved.m} tokens were saved")
    if n == 0:
        raise ValueError("dy needs at least one column")
    if out is not None:
        out_dtype = out.dtype
    if out_dtype != torch.float32 and out_dtype != saved.dtype:
        raise ValueError(f"the gradient is float32 or {saved.dtype}")
    if base is not None:
        _output("base", base, (saved.k, n), out_dtype, saved.device)
    if dy.device != saved.device:
        raise ValueError(f"operands are on different devices: {dy.device} and {saved.device}")
    if out is None:
        out = torch.empty((saved.k, n), dtype=out_dtype, device=saved.device)
    else:
        _output("out", out, (saved.k, n), out_dtype, saved.device)
    lddy, dy_ptr = _ld(dy), dy.data_ptr()
    if workspace is None:
        workspace = WorkspaceGrad8(saved, n, out_dtype, dy_ptr % 16 == 0 and lddy % 8 == 0)
    ws_ptr, ws_bytes = workspace._for(saved.device)
    args = (saved._code, *saved._layout, dy_ptr, lddy, DTYPE_CODE[out_dtype], base.data_ptr() if base is not None else None,
            _ld(base) if base is not None else n, out.data_ptr(), _ld(out), m, n, saved.k, ws_ptr, ws_bytes)
    if opts is None:
        _call("sb200_act8_wgrad", saved.device, *args)
    else:
        _call("sb200_act8_wgrad_opt", saved.device, *args, behind=(C.byref(opts),))
    if check:
        workspace.check()
    return out
