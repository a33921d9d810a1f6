"""Operators of a readout: a network trained on SOAP rows and asked for answers.

Rows of ``Soap.compute_device`` go through a residual stream that is normalised
and stored in 8 bits (``rms_norm``), 8-bit matrix products whose scales belong
to blocks of 128 (``quantize``, ``matmul``), their gradients
(``rms_norm_backward``, and ``matmul`` on blocks along columns) and an AdamW
step over all tensors at once (``AdamW``).  The kernels are those of
libmdsoap.so; torch tensors hold the memory.  Every call runs on the current
stream of its tensors' device and returns without waiting (an optimizer's first
step, and the one after its tensors changed, makes a table and waits for it).
Nothing here takes part in autograd: results carry no graph, gradients are calls
of their own.  Rows are float32, bfloat16 or float16; convert float64 rows first.

One layer y = rms_norm(x + r) W^T and its gradients::

    weight = quantize(w, layout="tiles")                  # .rows is W, .columns its transpose
    n = rms_norm(x, g, residual=r, output="float8")       # n.output (blocks), n.sum, n.rstd
    y = matmul(n.output, weight.rows)
    d = quantize(dy, layout="both")
    x8 = quantize(n.sum, layout="columns", row_factor=n.rstd, col_factor=g)   # normalised rows, transposed
    dw = matmul(d.columns, x8.columns, dtype="float32")
    dn = matmul(d.rows, weight.columns)
    dx, dg = rms_norm_backward(dn, n.sum, n.rstd, g, dsum=dsum)
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Sequence

import torch

from . import _lib
from ._lib import AdamWParams, lib, raise_for

try:
    from . import _readout_call as _call
except ImportError as error:  # no second way: a missing build is an error, as with the library
    raise ImportError("readout calls not built; run `python -m mdescriptor_b200.build`") from error

_call.bind(*(ctypes.cast(f, ctypes.c_void_p).value
             for f in (lib.mdsoap_rms_norm, lib.mdsoap_rms_norm_backward, lib.mdsoap_quantize, lib.mdsoap_matmul,
                       lib.mdsoap_adamw_step)))
_call.use(torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.get_device, torch.Tensor.data_ptr)

BLOCK = 128

_DTYPES = {torch.float32: _lib.FLOAT32, torch.bfloat16: _lib.BFLOAT16, torch.float16: _lib.FLOAT16}
_NAMES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_CODES = torch.float8_e4m3fn


class Blocks(NamedTuple):
    """An 8-bit matrix: e4m3 ``values`` [rows, width] (row pitch a multiple of
    16) and float32 ``scales`` [rows, ceil(width / 128)], or
    [ceil(rows / 128), ceil(width / 128)] where they belong to tiles."""

    values: torch.Tensor
    scales: torch.Tensor

    def float(self) -> torch.Tensor:
        """The float32 values that the codes stand for."""
        rows, width = self.values.shape
        scales = self.scales.repeat_interleave(BLOCK, dim=1)[:, :width]
        if scales.shape[0] != rows:
            scales = scales.repeat_interleave(BLOCK, dim=0)[:rows]
        return self.values.float() * scales


class Quantized(NamedTuple):
    """Result of ``quantize``: ``rows`` is the matrix, ``columns`` its
    transpose, each in blocks along its own rows (None where not asked for)."""

    rows: Blocks | None
    columns: Blocks | None


class Norm(NamedTuple):
    """Result of ``rms_norm``: ``output`` (``Blocks`` or a tensor), the sum
    x + residual (x itself without a residual) and the row factors ``rstd``."""

    output: "Blocks | torch.Tensor"
    sum: torch.Tensor
    rstd: torch.Tensor


# Tells autograd that tensors were written in place, so that a graph that had
# kept their former values raises an error instead of using these.
_written = torch.autograd.graph.increment_version

# The handle of a device's current stream, without the Stream object around it.
_stream = torch._C._cuda_getCurrentRawStream


def _matrix(x: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, width, row pitch) of a 2-D CUDA tensor with unit column stride."""
    shape = x.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must have two dimensions, got {tuple(shape)}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    rows, width = shape
    stride, unit = x.stride()
    if unit != 1 and width > 1:
        raise ValueError(f"{name} must have unit column stride, got strides {x.stride()}")
    if stride < width:
        if rows > 1:
            raise ValueError(f"{name} has rows that overlap (strides {x.stride()})")
        stride = width
    return rows, width, stride


def _dtype(x: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    return code


def _vector(x: torch.Tensor | None, count: int, device: int, name: str) -> int | None:
    if x is None:
        return None
    if x.dtype != torch.float32 or x.shape != (count,) or not x.is_contiguous() or x.get_device() != device:
        raise ValueError(f"{name} must be a contiguous float32 vector of {count} on CUDA device {device}")
    return x.data_ptr()


def _same(x: torch.Tensor, like: torch.Tensor, name: str) -> int:
    """Row pitch of a matrix with the shape, type and device of ``like``."""
    if x.shape != like.shape or x.dtype != like.dtype or x.get_device() != like.get_device():
        raise ValueError(f"{name} must have shape {tuple(like.shape)}, type {like.dtype} and device {like.device}")
    return _matrix(x, name)[2]


def _empty_blocks(rows: int, width: int, scale_rows: int, device: torch.device) -> tuple[Blocks, int, int]:
    """New blocks, with their row pitch and scale pitch."""
    blocks = (width + BLOCK - 1) // BLOCK
    pitch, scale_pitch = (width + 15) // 16 * 16, (blocks + 3) // 4 * 4
    return Blocks(torch.empty_strided((rows, width), (pitch, 1), dtype=_CODES, device=device),
                  torch.empty_strided((scale_rows, blocks), (scale_pitch, 1), dtype=torch.float32, device=device)
                  ), pitch, scale_pitch


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
             output: str | None = None) -> Norm:
    """y = s (mean(s^2) + eps)^-1/2 weight of each row, s = x + residual.

    ``output`` "float8": y in 8 bits (``Blocks``); None: y in x's type.  ``sum``
    is s in x's type (x itself without a residual); with ``rstd`` it is what
    ``rms_norm_backward`` takes."""
    if output not in (None, "float8"):
        raise ValueError("output must be None or 'float8'")
    rows, width, stride = _matrix(x, "x")
    dtype = _dtype(x, "x")
    device, index = x.device, x.get_device()
    weight_ptr = _vector(weight, width, index, "weight")
    if residual is None:
        total, residual_ptr, residual_stride, sum_ptr = x, None, 0, None
    else:
        residual_stride = _same(residual, x, "residual")
        total = torch.empty_strided((rows, width), (width, 1), dtype=x.dtype, device=device)
        residual_ptr, sum_ptr = residual.data_ptr(), total.data_ptr()
    rstd = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=device)
    if output is None:
        out: Blocks | torch.Tensor = torch.empty_strided((rows, width), (width, 1), dtype=x.dtype, device=device)
        out_ptr, out_stride, scales_ptr, scale_stride = out.data_ptr(), width, None, 0
    else:
        out, out_stride, scale_stride = _empty_blocks(rows, width, rows, device)
        out_ptr, scales_ptr = out.values.data_ptr(), out.scales.data_ptr()
    if rows:
        status = _call.rms_norm(
            x.data_ptr(), rows, width, stride, residual_ptr, residual_stride, dtype, weight_ptr, eps, sum_ptr, width,
            rstd.data_ptr(), out_ptr, out_stride, scales_ptr, scale_stride, index, _stream(index))
        if status:
            raise_for(status)
    return Norm(out, total, rstd)


@lru_cache(maxsize=1024)
def _norm_backward_bytes(rows: int, width: int, dtype: int, device: int) -> int:
    value = ctypes.c_int64()
    raise_for(lib.mdsoap_rms_norm_backward_bytes(rows, width, dtype, device, ctypes.byref(value)))
    return value.value


def rms_norm_backward(dy: torch.Tensor, sum: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor,
                      dsum: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dweight) of ``rms_norm`` from its ``sum`` and ``rstd``.

    ``dsum`` is the gradient that reaches the sum past the norm (the residual
    stream's); dx is the gradient of x and of residual alike.  An 8-bit output
    passes its gradient through unchanged.  dweight is float32 and the same bits
    on every run."""
    rows, width, stride = _matrix(sum, "sum")
    dtype = _dtype(sum, "sum")
    dy_stride = _same(dy, sum, "dy")
    dsum_stride = 0 if dsum is None else _same(dsum, sum, "dsum")
    device = sum.get_device()
    rstd_ptr = _vector(rstd, rows, device, "rstd")
    weight_ptr = _vector(weight, width, device, "weight")
    bytes_ = _norm_backward_bytes(rows, width, dtype, device)
    dx = torch.empty((rows, width), dtype=sum.dtype, device=sum.device)
    dweight = torch.empty(width, dtype=torch.float32, device=sum.device)
    workspace = torch.empty(bytes_, dtype=torch.uint8, device=sum.device)
    raise_for(_call.rms_norm_backward(
        dy.data_ptr(), rows, width, dy_stride, sum.data_ptr(), stride, rstd_ptr, weight_ptr,
        None if dsum is None else dsum.data_ptr(), dsum_stride, dtype, dx.data_ptr(), width, dweight.data_ptr(),
        workspace.data_ptr(), bytes_, device, _stream(device)))
    return dx, dweight


def quantize(x: torch.Tensor, layout: str = "rows", row_factor: torch.Tensor | None = None,
             col_factor: torch.Tensor | None = None) -> Quantized:
    """8-bit blocks of x * row_factor[:, None] * col_factor.

    ``layout`` "rows": blocks along rows; "columns": of the transpose; "both":
    both from one read of x; "tiles" (weights): one scale for each tile of
    128 x 128, the matrix and its transpose."""
    if layout not in ("rows", "columns", "both", "tiles"):
        raise ValueError("layout must be 'rows', 'columns', 'both' or 'tiles'")
    rows, width, stride = _matrix(x, "x")
    dtype = _dtype(x, "x")
    device, index = x.device, x.get_device()
    row_ptr = _vector(row_factor, rows, index, "row_factor")
    col_ptr = _vector(col_factor, width, index, "col_factor")
    tiles = layout == "tiles"
    if tiles and (row_ptr or col_ptr):
        raise ValueError("tiles take no factors")
    by_rows = by_columns = codes = scales = codes_t = scales_t = None
    pitch = scale_pitch = pitch_t = scale_pitch_t = 0
    if layout != "columns":
        by_rows, pitch, scale_pitch = _empty_blocks(rows, width, (rows + BLOCK - 1) // BLOCK if tiles else rows, device)
        codes, scales = by_rows.values.data_ptr(), by_rows.scales.data_ptr()
    if layout != "rows":
        by_columns, pitch_t, scale_pitch_t = _empty_blocks(width, rows, (width + BLOCK - 1) // BLOCK if tiles else width,
                                                           device)
        codes_t, scales_t = by_columns.values.data_ptr(), by_columns.scales.data_ptr()
    if rows and width:
        status = _call.quantize(x.data_ptr(), rows, width, stride, dtype, row_ptr, col_ptr, tiles, codes, pitch, scales,
                                scale_pitch, codes_t, pitch_t, scales_t, scale_pitch_t, index, _stream(index))
        if status:
            raise_for(status)
    return Quantized(by_rows, by_columns)


def _blocks(b: Blocks, name: str, tiles: bool) -> tuple[int, int, int, int, int, int, bool]:
    """(rows, width, address, pitch, scales' address, their pitch, scales of tiles) of checked blocks."""
    values, scales = b
    rows, width, stride = _matrix(values, f"{name}.values")
    scale_rows, blocks, scale_stride = _matrix(scales, f"{name}.scales")
    if values.dtype != _CODES:
        raise ValueError(f"{name}.values must be float8_e4m3fn, got {values.dtype}")
    if scales.dtype != torch.float32 or scales.get_device() != values.get_device():
        raise ValueError(f"{name}.scales must be float32 on {values.device}")
    by_rows = scale_rows == rows
    if blocks != (width + 127) // 128 or not (by_rows or (tiles and scale_rows == (rows + 127) // 128)):
        raise ValueError(f"{name}.scales has shape {tuple(scales.shape)}, which fits no blocks of {tuple(values.shape)}")
    address = values.data_ptr()
    if (stride % 16 or address % 16) and rows and width:
        raise ValueError(f"{name}.values must start on 16 bytes and have a row pitch that is a multiple of 16")
    return rows, width, address, stride, scales.data_ptr(), scale_stride, not by_rows


@lru_cache(maxsize=4096)
def _matmul_bytes(m: int, n: int, k: int, tiles: bool, device: int) -> int:
    value = ctypes.c_int64()
    raise_for(lib.mdsoap_matmul_bytes(m, n, k, int(tiles), device, ctypes.byref(value)))
    return value.value


def matmul(a: Blocks, b: Blocks, dtype: str = "bfloat16", out: torch.Tensor | None = None,
           accumulate: bool = False) -> torch.Tensor:
    """a b^T [m, n] of two 8-bit matrices with blocks along their common width.

    ``b`` may carry scales of tiles (weights) or of its rows (the weight's
    gradient).  ``dtype`` "bfloat16" or "float32"; ``out`` takes the result, and
    with ``accumulate`` (float32) has it added.  Results whose copies or matrix
    instructions did not complete within a second are NaN, and ``check`` raises."""
    m, k, a_ptr, a_stride, a_scale_ptr, a_scale_stride, _ = _blocks(a, "a", False)
    n, k_b, b_ptr, b_stride, b_scale_ptr, b_scale_stride, tiles = _blocks(b, "b", True)
    if k != k_b:
        raise ValueError(f"a and b must have the same width, got {k} and {k_b}")
    device, index = a.values.device, a.values.get_device()
    if b.values.get_device() != index:
        raise ValueError("a and b must be on the same device")
    given = out is not None
    if not given:
        kind = _NAMES.get(dtype)
        if kind is None or kind is torch.float16:
            raise ValueError("dtype must be 'bfloat16' or 'float32'")
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty_strided((m, n), (n, 1), dtype=kind, device=device)
        out_stride = n
    else:
        kind = out.dtype
        if out.shape != (m, n) or out.get_device() != index or kind not in (torch.bfloat16, torch.float32):
            raise ValueError(f"out must be a bfloat16 or float32 matrix of shape {(m, n)} on {device}")
        out_stride = _matrix(out, "out")[2]
        if accumulate and kind != torch.float32:
            raise ValueError("accumulate needs a float32 out")
    bytes_ = _matmul_bytes(m, n, k, tiles, index)
    workspace = torch.empty(bytes_, dtype=torch.uint8, device=device) if bytes_ else None
    status = _call.matmul(
        a_ptr, m, a_stride, a_scale_ptr, a_scale_stride, b_ptr, n, b_stride, b_scale_ptr, b_scale_stride, tiles, k, _DTYPES[kind], accumulate, out.data_ptr(), out_stride,
        None if workspace is None else workspace.data_ptr(), bytes_, index, _stream(index))
    if status:
        raise_for(status)
    if given:
        _written(out)
    return out


def check(device: int = 0) -> None:
    """Wait for the current stream and raise if a product on ``device`` gave up waiting."""
    raise_for(lib.mdsoap_matmul_check(int(device), _stream(device)))


class AdamW:
    """AdamW over all of a readout's tensors in one launch.

    ``params``: contiguous CUDA tensors of one type (float32, bfloat16 or
    float16), updated in place, also where one has got other memory since the
    last step (``p.data = ...``).  ``state_bits`` 32 holds both moments in
    float32; 8 holds them as e4m3 codes with a scale for each 128 elements,
    rounded by dithering with random numbers of (seed, step, element).
    ``weight_decay``: one number, or one a tensor.  ``state``: moments to
    continue from (``exp_avg``, ``exp_avg_sq``, with 8 bits ``exp_avg_scale``
    and ``exp_avg_sq_scale``: lists like ``params``; ``step``: the steps
    taken), used in place; ``self.state`` has the same form.  A tensor of it
    that is replaced by another one is taken up by the next step."""

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float | Sequence[float] = 0.01, state_bits: int = 32, seed: int = 0,
                 state: dict | None = None) -> None:
        self._optimizer = None
        self.params = list(params)
        self.lr, self.betas, self.eps = float(lr), (float(betas[0]), float(betas[1])), float(eps)
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self.state_bits = state_bits
        self._seed = int(seed) & 0xFFFFFFFF
        count = len(self.params)
        if not count:
            raise ValueError("AdamW needs at least one tensor")
        decays = [float(weight_decay)] * count if isinstance(weight_decay, (int, float)) else [float(w) for w in weight_decay]
        if len(decays) != count:
            raise ValueError("weight_decay must be one number or one a tensor")
        self._decays = decays
        self._keys = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")[:4 if state_bits == 8 else 2]
        _, self.device, self._counts = self._check_params()
        if state is None:
            state = {"step": 0}
            for key in self._keys:
                scale = key.endswith("_scale")
                kind = torch.uint8 if state_bits == 8 and not scale else torch.float32
                state[key] = [torch.zeros((n + BLOCK - 1) // BLOCK if scale else n, dtype=kind, device=self.device)
                              for n in self._counts]
                if kind == torch.uint8:
                    state[key] = [t.view(_CODES) for t in state[key]]
        self.state = {"step": int(state["step"]), **{key: list(state[key]) for key in self._keys}}
        self._bind()

    def _check_params(self) -> tuple[int, torch.device, list[int]]:
        first = self.params[0]
        for p in self.params:
            if not p.is_cuda or not p.is_contiguous() or p.dtype != first.dtype or p.device != first.device:
                raise ValueError("params must be contiguous CUDA tensors of one type on one device")
        return _dtype(first, "params"), first.device, [p.numel() for p in self.params]

    def _bind(self) -> None:
        """Hands the tensors' addresses to the library.

        What it writes to stays alive with it (``_held``): a tensor that is
        replaced, or given other memory, cannot take the memory away from under
        a step, and its successor has another address, by which ``step`` sees it."""
        if len(self.params) != len(self._decays):
            raise ValueError(f"params must hold {len(self._decays)} tensors")
        dtype, device, numels = self._check_params()
        count = len(self.params)
        blocks = [(n + BLOCK - 1) // BLOCK for n in numels]
        arrays = {"params": self.params}
        for key in self._keys:
            sizes, want = (blocks if key.endswith("_scale") else numels,
                           _CODES if self.state_bits == 8 and not key.endswith("_scale") else torch.float32)
            tensors = self.state[key]
            if not isinstance(tensors, list):
                tensors = self.state[key] = list(tensors)
            if len(tensors) != count or any(t.numel() != n or t.dtype != want or t.device != device or
                                            not t.is_contiguous() for t, n in zip(tensors, sizes)):
                raise ValueError(f"state {key!r} must hold {count} contiguous {want} tensors that fit the params")
            arrays[key] = tensors
        pointers = {key: (ctypes.c_void_p * count)(*[t.data_ptr() for t in v]) for key, v in arrays.items()}
        counts = (ctypes.c_int64 * count)(*numels)
        decay = (ctypes.c_float * count)(*self._decays)
        address = {key: ctypes.cast(v, ctypes.c_void_p) for key, v in pointers.items()}
        handle = ctypes.c_void_p()
        raise_for(lib.mdsoap_adamw_create(ctypes.byref(AdamWParams(
            count, address["params"], address["exp_avg"], address["exp_avg_sq"], address.get("exp_avg_scale"),
            address.get("exp_avg_sq_scale"), ctypes.cast(counts, ctypes.c_void_p), ctypes.cast(decay, ctypes.c_void_p),
            dtype, self.state_bits, self._seed, device.index)), ctypes.byref(handle)))
        self.close()
        self._optimizer = handle
        self.device, self._index, self._counts = device, device.index, numels
        self._held = [t.detach() for v in arrays.values() for t in v]
        self._param_addresses = _call.addresses(self.params)
        self._moments = {key: list(arrays[key]) for key in self._keys}

    def _moved(self) -> bool:
        """Whether a tensor is not the one, or not where, the library writes to."""
        if _call.addresses(self.params) != self._param_addresses:
            return True
        state = self.state
        for key, held in self._moments.items():
            if not _call.identical(state[key], held):
                return True
        return False

    def step(self, grads: Sequence[torch.Tensor], lr: float | None = None, grad_scale: float = 1.0) -> None:
        """Update every tensor with its gradient (one type for all, times ``grad_scale``)."""
        if self._optimizer is None:
            raise ValueError("the optimizer is closed")
        if self._moved():
            self._bind()
        found = _call.gather(list(grads), self._counts, self._index)
        if found == 1:
            raise ValueError("grads must be one tensor for each of params, of its size")
        if found == 2:
            raise ValueError(f"grads must be contiguous tensors of one type on {self.device}")
        pointers, kind = found
        code = _DTYPES.get(kind)
        if code is None:
            raise ValueError(f"grads must be float32, bfloat16 or float16, got {kind}")
        step = self.state["step"] + 1
        status = _call.adamw_step(
            self._optimizer.value, pointers, code, step, self.lr if lr is None else lr,
            self.betas[0], self.betas[1], self.eps, grad_scale, _stream(self._index))
        if status:
            raise_for(status)
        _written(self.params)
        self.state["step"] = step

    def close(self) -> None:
        """Frees the optimizer's table on the device; no step can follow."""
        if self._optimizer:
            lib.mdsoap_adamw_destroy(self._optimizer)
            self._optimizer = None

    def __del__(self) -> None:
        try:
            self.close()
        except Exception:
            pass
