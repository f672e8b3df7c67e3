"""Tensor-level wrappers of the C ABI: they take CUDA tensors, pass raw pointers and the current stream.

Counterpart of the reference's launch wrappers in ``src/mlkit/kernels/packed_linear.py:181-313``,
``src/mlkit/kernels/hadamard.py:108-136`` and ``src/mlkit/kernels/launching.py:33-52``: work is queued
on the current CUDA stream of the tensor's device, nothing is synchronised and, apart from the
output tensor the caller passes in, nothing is allocated.
"""

import functools
import threading

import torch
from torch import Tensor

from mlkit_b200 import _native

DTYPE_TAGS = {torch.float16: _native.F16, torch.bfloat16: _native.BF16, torch.float32: _native.F32}
KERNEL_CHOICES = {"auto": _native.GEMV_AUTO, "scalar": _native.GEMV_SCALAR, "tiled": _native.GEMV_TILED,
                  "tmem": _native.GEMV_TMEM, "bulk": _native.GEMV_BULK, "stream": _native.GEMV_STREAM}

_workspaces: dict[tuple[int, int], Tensor] = {}


def matvec_workspace(device: torch.device, rows: int, outputs: int, width: int, bits: int) -> Tensor | None:
    """Zero-initialised scratch the tensor-memory matvec meets through (it splits K over CTAs), or
    ``None`` when the shape cannot use it.  One buffer per (device, stream) grows to the largest request;
    the kernel leaves it zeroed where it must be, so it is cleared only when (re)allocated.  Launches on
    one stream run in order and may share it."""
    need = _native.library().mkb_gemv_workspace_bytes(rows, outputs, width, bits)
    if need <= 0:
        return None
    key = (device.index if device.index is not None else torch.cuda.current_device(),
           torch.cuda.current_stream(device).cuda_stream)
    held = _workspaces.get(key)
    if held is None or held.numel() < need:
        held = _workspaces[key] = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=device)
    return held


def workspace_status() -> int:
    """Non-zero when a bounded wait expired inside any matvec that used one of the pooled workspaces
    (its results are not valid); synchronises with the devices."""
    import ctypes

    worst = 0
    for held in _workspaces.values():
        value = ctypes.c_int(0)
        with torch.cuda.device(held.device):
            check = _native.library().mkb_gemv_workspace_status(held.data_ptr(), held.numel(), ctypes.byref(value))
        _native.check(check, "workspace_status")
        worst = max(worst, value.value)
    return worst


def _tag(dtype: torch.dtype, what: str) -> int:
    try:
        return DTYPE_TAGS[dtype]
    except KeyError:
        raise ValueError(f"{what} dtype {dtype} is not supported (fp16, bf16, fp32)") from None


def _pointer(tensor: Tensor | None) -> int | None:
    return None if tensor is None else tensor.data_ptr()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(*tensors: Tensor | None) -> torch.device:
    device = None
    for tensor in tensors:
        if tensor is None:
            continue
        if not tensor.is_cuda:
            raise ValueError("mlkit_b200 kernels require CUDA tensors")
        if device is not None and tensor.device != device:
            raise ValueError("all tensors of one call must live on one device")
        device = tensor.device
    assert device is not None
    return device


def integer_grid_of(values: Tensor) -> tuple[bool, float]:
    """Whether ``values[c] == values[0] + c`` exactly with an integer ``values[0]``; and ``values[0]``."""
    table = values.detach().float().cpu()
    if table.numel() == 0:
        return False, 0.0
    low = float(table[0])
    exact = low == int(low) and abs(low) <= 512 and bool(
        torch.equal(table, low + torch.arange(table.numel(), dtype=torch.float32, device="cpu")))
    return exact, low


ROTATED_MAXIMUM_BYTES = 65536     # of fp32 activations the fused rotation holds in shared memory
ROTATED_PROFITABLE_BYTES = 16384  # up to here the fused launch measured faster than transform + matvec


def rotated_matvec_supported(rows: int, width: int, dtype: torch.dtype, *, profitable: bool = False) -> bool:
    """Whether ``packed_matvec_rotated`` may cover the input (the C entry point checks the layer as well).
    Every CTA of the matvec redoes the rotation, so its cost grows with the rows: measured on B200 at
    K = 4096 the fused launch wins at one row (6.4 against 7.0 us), ties at two and loses at four;
    ``profitable`` asks for the range where it wins."""
    limit = ROTATED_PROFITABLE_BYTES if profitable else ROTATED_MAXIMUM_BYTES
    return (dtype == torch.float16 and 1 <= rows <= 8 and width >= 512 and width & (width - 1) == 0
            and rows * width * 4 <= limit)


def packed_matvec_rotated(x: Tensor, signs: Tensor | None, packed: Tensor, scales: Tensor, values: Tensor,
                          bias: Tensor | None, out: Tensor, *, group: int, bits: int, integer_grid: bool,
                          grid_minimum: float, normalize: bool = True) -> Tensor:
    """``out = matvec(S(x * signs))`` in one launch (``mkb_gemv_hadamard``): equal to ``structured_transform``
    followed by ``packed_matvec`` bit for bit.  Raises ``ValueError`` where the fused launch does not apply."""
    device = _require_cuda(x, signs, packed, scales, values, bias, out)
    rows, width = x.shape
    if signs is not None and signs.dtype != torch.int8:
        raise ValueError("signs must be int8")
    if bias is not None and bias.dtype != x.dtype:
        bias = bias.to(x.dtype)
    with torch.cuda.device(device):
        status = _native.library().mkb_gemv_hadamard(
            x.data_ptr(), _pointer(signs), packed.data_ptr(), scales.data_ptr(), values.data_ptr(), _pointer(bias),
            out.data_ptr(), rows, out.shape[1], width, group, bits, values.numel(), _tag(x.dtype, "activation"),
            _tag(scales.dtype, "scale"), width * bits // 8, scales.stride(0) if scales.dim() == 2 else -(-width // group),
            int(integer_grid), float(grid_minimum), int(normalize), torch.cuda.current_stream().cuda_stream)
    _native.check(status, "packed_matvec_rotated")
    return out


_gemm_workspaces: dict[tuple[int, int], Tensor] = {}
GEMM_MAXIMUM_ROWS = 128


def gemm_workspace(device: torch.device, rows: int, outputs: int, width: int) -> Tensor:
    """Scratch of ``mkb_gemm``, one per (device, stream), grown to the largest request: a zeroed head whose last word is
    the status, then the partial sums."""
    need = _native.library().mkb_gemm_workspace_bytes(rows, outputs, width)
    if need <= 0:
        raise ValueError(f"no fused GEMM for {rows} rows, {outputs} outputs, width {width}")
    key = (device.index if device.index is not None else torch.cuda.current_device(),
           torch.cuda.current_stream(device).cuda_stream)
    held = _gemm_workspaces.get(key)
    if held is None or held.numel() < need:
        held = _gemm_workspaces[key] = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=device)
    return held


def gemm_status() -> int:
    """Non-zero when a bounded wait expired inside a fused GEMM that used a pooled workspace."""
    import ctypes

    worst = 0
    for held in _gemm_workspaces.values():
        value = ctypes.c_int(0)
        with torch.cuda.device(held.device):
            _native.check(_native.library().mkb_gemm_status(held.data_ptr(), ctypes.byref(value)), "gemm_status")
        worst = max(worst, value.value)
    return worst


def gemm_supported(rows: int, *, width: int, group: int, bits: int, dtype: torch.dtype, scales: Tensor,
                   zeros: Tensor | None, integer_grid: bool, grid_minimum: float, levels: int,
                   outputs: int | None = None) -> bool:
    """Whether ``packed_gemm`` covers the layer (the C entry point checks the same and more).  With ``outputs`` given,
    also whether it is a faster route than reconstruct + library GEMM whatever the layer: up to 32 rows, and up to 128
    for weights of 2^25 codes or more.  (``tile_gemm_rows`` draws the finer line that ``PackedLinear`` follows.)"""
    if not (1 <= rows <= GEMM_MAXIMUM_ROWS and bits == 4 and group == 128 and width % 128 == 0 and zeros is None
            and dtype == torch.float16 and scales.dtype == torch.float16 and bool(integer_grid)
            and float(grid_minimum) == -8.0 and levels == 16):
        return False
    return outputs is None or rows <= 32 or outputs * width >= 1 << 25


def packed_gemm(x: Tensor, packed: Tensor, scales: Tensor, values: Tensor, bias: Tensor | None, out: Tensor, *,
                group: int, bits: int, integer_grid: bool, grid_minimum: float) -> Tensor:
    """``out[M, N] = x[M, K] @ dequant(packed)^T (+ bias)`` for up to 128 fp16 rows of symmetric INT4 (``mkb_gemm``): the
    kernel of ``packed_tile_gemm`` with its partials in one workspace, for callers of the C ABI that own one."""
    device = _require_cuda(x, packed, scales, values, bias, out)
    rows, width = x.shape
    outputs = out.shape[1]
    if not x.is_contiguous() or not out.is_contiguous():
        raise ValueError("packed_gemm needs contiguous activations and outputs")
    if bias is not None and bias.dtype != x.dtype:
        bias = bias.to(x.dtype)
    with torch.cuda.device(device):
        workspace = gemm_workspace(device, rows, outputs, width)
        status = _native.library().mkb_gemm(
            x.data_ptr(), packed.data_ptr(), scales.data_ptr(), values.data_ptr(), None, _pointer(bias), out.data_ptr(),
            rows, outputs, width, group, bits, values.numel(), _tag(x.dtype, "activation"), _tag(scales.dtype, "scale"),
            width * bits // 8, scales.stride(0) if scales.dim() == 2 else -(-width // group), int(integer_grid),
            float(grid_minimum), workspace.data_ptr(), workspace.numel(), torch.cuda.current_stream().cuda_stream)
    _native.check(status, "packed_gemm")
    return out


def _status_pointer(device: torch.device, index: int, stream: int) -> int:
    """The status word the tile GEMMs of a (device, stream) share: the last one of a workspace head."""
    held = _gemm_workspaces.get((index, stream))
    if held is None:
        held = _gemm_workspaces[(index, stream)] = torch.zeros(1 << 20, dtype=torch.uint8, device=device)
    return held.data_ptr() + 65532


# Most rows for which the tile GEMM was not slower than reconstruct + library GEMM, measured on B200 over 32 shapes from
# 128 x 896 to 28672 x 4096, every codec, fp16 and bf16 (device time, weights cold in L2).  Both multiply at the tensor
# cores' rate; the tile GEMM saves writing the weight and reading it back, and pays its decode once per tile of up to 256
# rows, so the line moves up with the weight's size and down with the cost of the decode.  In us, tile / dense: 4 bits with
# offsets, 4096 x 4096, 768 rows 36.9 / 39.1, 1024 rows 45.3 / 43.9; 4 bits, 4864 x 896, 160 rows 10.8 / 11.2, 512 rows
# 15.1 / 11.8; 8 bits, 4096 x 4096, 128 rows 19.7 / 26.1, 1024 rows 85.6 / 42.3.
# By the width of the layer: (codes of the weight, most rows of: 4-bit integer grids; those with offsets; other codecs of up
# to 5 bits; 6 bits; 7 and 8 bits), the last line whose codes the weight reaches.  0: one tile of rows, the most of its
# decode.
_MI = 1 << 20
_TILE_ROWS = (
    (1024, ((0, (48, 48, 48, 48, 48)), (_MI, (96, 96, 96, 96, 64)), (4 * _MI, (160, 160, 160, 160, 64)))),
    (2048, ((0, (48, 48, 48, 48, 48)), (_MI, (128, 128, 96, 128, 128)), (2 * _MI, (160, 160, 160, 160, 128)),
            (3 * _MI, (192, 192, 192, 192, 0)), (8 * _MI, (448, 320, 224, 224, 0)), (16 * _MI, (1024, 1024, 448, 384, 0)))),
    (1 << 30, ((0, (48, 48, 48, 48, 48)), (_MI, (128, 128, 128, 128, 128)), (3 * _MI // 2, (160, 160, 160, 160, 128)),
               (2 * _MI, (256, 256, 192, 224, 192)), (3 * _MI, (384, 320, 192, 320, 192)), (4 * _MI, (384, 384, 192, 384, 192)),
               (6 * _MI, (448, 448, 224, 320, 0)), (8 * _MI, (448, 448, 256, 320, 0)), (9 * _MI, (896, 768, 448, 448, 0)),
               (24 * _MI, (1024, 1024, 640, 448, 0)), (56 * _MI, (1024, 1024, 768, 512, 256)))),
)


@functools.lru_cache(maxsize=4096)
def tile_gemm_rows(outputs: int, width: int, group: int, bits: int, integer_grid: bool, offsets: bool = False) -> int:
    """Most activation rows (fp16 or bf16) of a layer that ``packed_tile_gemm`` is the faster route for; 0 where it does
    not cover the layer (the C entry point checks the same and more)."""
    if not (2 <= bits <= 8 and group in (32, 64, 128) and width % 128 == 0 and width * bits // 8 % 16 == 0):
        return 0
    decoder = (1 if offsets else 0) if bits == 4 and integer_grid else 2 if bits <= 5 else 3 if bits == 6 else 4
    lines = next(lines for below, lines in _TILE_ROWS if width < below)
    rows = next(rows for codes, rows in reversed(lines) if outputs * width >= codes)[decoder]
    return rows or (176 if bits == 7 else 160) - (16 if offsets else 0)     # the tiles shared memory leaves room for


@functools.lru_cache(maxsize=64)
def _partial_bytes(rows: int, index: int) -> int:
    return _native.library().mkb_gemm_tile_partial_bytes(rows)


def packed_tile_gemm(x: Tensor, packed: Tensor, scales: Tensor, values: Tensor, zeros: Tensor | None, bias: Tensor | None,
                     out: Tensor, *, group: int, bits: int, integer_grid: bool, grid_minimum: float) -> Tensor:
    """``out[M, N] = x[M, K] @ dequant(packed)^T (+ bias)`` for any number of rows (``mkb_gemm_tile``); the weight is
    rounded to the type of ``x`` and never written to memory."""
    _require_cuda(x, packed, scales, values, zeros, bias, out)
    rows, width = x.shape
    if not x.is_contiguous() or not out.is_contiguous() or out.dtype != x.dtype or out.shape[0] != rows:
        raise ValueError("packed_tile_gemm needs contiguous activations and outputs of one type and number of rows")
    if zeros is not None and zeros.dtype != scales.dtype:
        raise ValueError("offsets must share the dtype of the scales")
    launch_tile_gemm(x, packed, scales, values, zeros, bias, out, rows, out.shape[1], width, group, bits, integer_grid,
                     grid_minimum)
    return out


def launch_tile_gemm(x: Tensor, packed: Tensor, scales: Tensor, values: Tensor, zeros: Tensor | None, bias: Tensor | None,
                     out: Tensor, rows: int, outputs: int, width: int, group: int, bits: int, integer_grid: bool,
                     grid_minimum: float) -> None:
    """``packed_tile_gemm`` of tensors a caller answers for: one device, contiguous, offsets of the scales' type."""
    index = x.get_device()
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return launch_tile_gemm(x, packed, scales, values, zeros, bias, out, rows, outputs, width, group, bits,
                                    integer_grid, grid_minimum)
    if bias is not None and bias.dtype != x.dtype:
        bias = bias.to(x.dtype)
    stream = torch.cuda.current_stream().cuda_stream
    size = _partial_bytes(rows, index)
    partials = x.new_empty(size, dtype=torch.uint8)
    status = _native.library().mkb_gemm_tile(
        x.data_ptr(), packed.data_ptr(), scales.data_ptr(), values.data_ptr(), _pointer(zeros), _pointer(bias), out.data_ptr(),
        rows, outputs, width, group, bits, values.numel(), _tag(x.dtype, "activation"), _tag(scales.dtype, "scale"),
        width * bits // 8, scales.stride(0) if scales.dim() == 2 else -(-width // group), int(integer_grid),
        float(grid_minimum), partials.data_ptr(), size, _status_pointer(x.device, index, stream), stream)
    if status:
        _native.check(status, "packed_tile_gemm")


def packed_matvec(x: Tensor, packed: Tensor, scales: Tensor, values: Tensor, zeros: Tensor | None,
                  bias: Tensor | None, out: Tensor, *, group: int, bits: int, integer_grid: bool = False,
                  grid_minimum: float = 0.0, kernel: str = "auto", packed_row_stride: int | None = None,
                  scale_row_stride: int | None = None, workspace: Tensor | None = None,
                  gated: bool = False) -> Tensor:
    """``out[m, n] = sum_k x[m, k] * (values[code[n, k]] * scales[n, k // group] (+ zeros)) (+ bias[n])``.

    ``x`` is ``[M, K]`` contiguous with ``M <= 8``; ``out`` is ``[M, N]`` in the dtype of ``x``.
    """
    device = _require_cuda(x, packed, scales, values, zeros, bias, out)
    rows, width = x.shape
    if gated:   # x is [rows, 2 * width] = gate | up; the kernel forms silu(gate) * up on load
        if width % 2:
            raise ValueError("a gated input has an even number of columns")
        width //= 2
    outputs = out.shape[-1]
    if not (x.is_contiguous() and out.is_contiguous()):
        raise ValueError("packed_matvec needs contiguous activations and output")
    if out.dtype != x.dtype or out.shape[0] != rows:
        raise ValueError("output must match the activations in dtype and rows")
    if zeros is not None and zeros.dtype != scales.dtype:
        raise ValueError("offsets must share the dtype of the scales")
    if bias is not None and bias.dtype != x.dtype:
        bias = bias.to(x.dtype)
    if packed_row_stride is None:
        packed_row_stride = width * bits // 8
    if scale_row_stride is None:
        scale_row_stride = scales.stride(0) if scales.dim() == 2 else -(-width // group)
    with torch.cuda.device(device):
        if workspace is None and kernel in ("auto", "tmem", "bulk") and x.dtype == torch.float16 and integer_grid:
            workspace = matvec_workspace(device, rows, outputs, width, bits)
        status = _native.library().mkb_gemv_ws(
            x.data_ptr(), packed.data_ptr(), scales.data_ptr(), values.data_ptr(), _pointer(zeros),
            _pointer(bias), out.data_ptr(), rows, outputs, width, group, bits, values.numel(),
            _tag(x.dtype, "activation"), _tag(scales.dtype, "scale"), packed_row_stride,
            scale_row_stride, int(integer_grid), float(grid_minimum),
            KERNEL_CHOICES[kernel] | (_native.GEMV_GATED if gated else 0), _pointer(workspace), 0 if workspace is None else workspace.numel(), _stream(device))
    _native.check(status, "packed_matvec")
    return out


class MatvecPlan:
    """The constant arguments of one layer's matvec, bound once.

    The per-call work is what the reference's direct launcher leaves
    (``src/mlkit/inference/packed_linear.py:181-245``): pass the activation and output pointers,
    the row count and the current stream.  The plan holds raw device pointers, so it must be rebuilt
    whenever the layer's buffers move (``PackedLinear._apply`` drops it).
    """

    __slots__ = ("function", "head", "tail", "outputs", "width", "bits", "dtype", "device", "device_index", "keep",
                 "integer_grid", "workspaces")

    def __init__(self, packed: Tensor, scales: Tensor, values: Tensor, zeros: Tensor | None, bias: Tensor | None,
                 *, outputs: int, width: int, group: int, bits: int, dtype: torch.dtype, integer_grid: bool,
                 grid_minimum: float, gated: bool = False) -> None:
        device = _require_cuda(packed, scales, values, zeros, bias)
        if zeros is not None and zeros.dtype != scales.dtype:
            raise ValueError("offsets must share the dtype of the scales")
        if bias is not None and bias.dtype != dtype:
            bias = bias.to(dtype)
        self.function = _native.library().mkb_gemv_ws
        self.head = (packed.data_ptr(), scales.data_ptr(), values.data_ptr(), _pointer(zeros), _pointer(bias))
        self.tail = (outputs, width, group, bits, values.numel(), _tag(dtype, "activation"),
                     _tag(scales.dtype, "scale"), width * bits // 8,
                     scales.stride(0) if scales.dim() == 2 else -(-width // group), int(integer_grid),
                     float(grid_minimum), _native.GEMV_AUTO | (_native.GEMV_GATED if gated else 0))
        self.outputs, self.width, self.bits, self.dtype, self.device = outputs, width, bits, dtype, device
        self.integer_grid = bool(integer_grid) and dtype == torch.float16 and zeros is None
        self.workspaces: dict[tuple[int, int], tuple[int | None, int, Tensor | None]] = {}
        self.device_index = device.index
        self.keep = (packed, scales, values, zeros, bias)  # the pointers above stay valid while these live

    def __call__(self, x: Tensor, out: Tensor) -> Tensor:
        """``x`` [M, width] and ``out`` [M, outputs]: contiguous, on the plan's device, dtype of the plan."""
        if torch.cuda.current_device() != self.device_index:
            with torch.cuda.device(self.device):
                return self(x, out)
        stream = torch.cuda.current_stream().cuda_stream
        rows = x.shape[0]
        held = self.workspaces.get((rows, stream))
        if held is None:  # (pointer, bytes, tensor kept alive) of the scratch for this row count and stream
            tensor = matvec_workspace(self.device, rows, self.outputs, self.width, self.bits) if self.integer_grid else None
            held = self.workspaces[(rows, stream)] = (_pointer(tensor), 0 if tensor is None else tensor.numel(), tensor)
        status = self.function(x.data_ptr(), *self.head, out.data_ptr(), rows, *self.tail, held[0], held[1], stream)
        if status:
            _native.check(status, "packed_matvec")
        return out


def dequantize(packed: Tensor, scales: Tensor | None, values: Tensor | None, zeros: Tensor | None, *,
               shape: tuple[int, int], group: int, bits: int, dtype: torch.dtype | None = torch.float16,
               codes: bool = False) -> tuple[Tensor | None, Tensor | None]:
    """Bit-exact reconstruction of a packed weight; returns ``(weight or None, codes or None)``."""
    device = _require_cuda(packed, scales, values, zeros)
    rows, width = shape
    weight = None if dtype is None else torch.empty(shape, device=device, dtype=dtype)
    unpacked = torch.empty(shape, device=device, dtype=torch.uint8) if codes else None
    if weight is None and unpacked is None:
        raise ValueError("dequantize needs at least one output")
    if weight is not None and (scales is None or values is None):
        raise ValueError("a dense weight needs scales and values")
    if rows * width == 0:
        return weight, unpacked
    if scales is not None and not scales.is_contiguous():
        raise ValueError("scales must be contiguous")
    stride = 0 if scales is None else (scales.stride(0) if scales.dim() == 2 else -(-width // group))
    with torch.cuda.device(device):
        status = _native.library().mkb_dequant(
            packed.data_ptr(), _pointer(scales), _pointer(values), _pointer(zeros), _pointer(weight),
            _pointer(unpacked), rows, width, group, bits, 0 if values is None else values.numel(),
            _native.F32 if scales is None else _tag(scales.dtype, "scale"),
            _native.F16 if dtype is None else _tag(dtype, "output"), stride, _stream(device))
    _native.check(status, "dequantize")
    return weight, unpacked


def rtn_encode(weight: Tensor, levels: Tensor, *, group: int, bits: int, integer_grid: bool, low: float, high: float,
               reciprocal: float, codes: bool = False) -> tuple[Tensor, Tensor, Tensor | None]:
    """Round-to-nearest encode and pack on the device: returns ``(packed uint8, scales fp16 [N, groups],
    codes uint8 [N, K] or None)``.  Raises ``ValueError`` for layouts whose groups or rows do not end
    on a byte (the caller then takes the tensor route)."""
    device = _require_cuda(weight, levels)
    rows, width = weight.shape
    source = weight if weight.is_contiguous() else weight.contiguous()
    group = min(group, width)
    packed = torch.empty(rows * width * bits // 8, dtype=torch.uint8, device=device)
    scales = torch.empty((rows, -(-width // group)), dtype=torch.float16, device=device)
    unpacked = torch.empty((rows, width), dtype=torch.uint8, device=device) if codes else None
    with torch.cuda.device(device):
        status = _native.library().mkb_rtn_encode(
            source.data_ptr(), levels.data_ptr(), packed.data_ptr(), scales.data_ptr(), _pointer(unpacked), rows, width,
            group, bits, levels.numel(), int(integer_grid), float(low), float(high), float(reciprocal),
            _tag(source.dtype, "weight"), _stream(device))
    _native.check(status, "rtn_encode")
    return packed, scales, unpacked


def checked_encode_supported(weight: Tensor, group: int) -> bool:
    """Whether ``rtn_encode_checked`` covers the layout (the C entry point checks the same): groups of 8 to 256 codes,
    a power of two, in rows of whole runs of eight."""
    rows, width = weight.shape
    group = min(group, width)
    return (weight.dtype in DTYPE_TAGS and weight.is_contiguous() and weight.data_ptr() % 16 == 0 and width % 8 == 0
            and 8 <= group <= 256 and group & (group - 1) == 0 and 0 < rows * (width + group) < 1 << 34)


def rtn_encode_checked(weight: Tensor, levels: Tensor | None, *, group: int, bits: int, integer_grid: bool, low: float, high: float,
                       reciprocal: float, asym: bool) -> tuple[Tensor, Tensor, Tensor | None, Tensor, Tensor]:
    """``rtn_encode`` of a weight in its own type, with offsets when ``asym``: returns ``(packed uint8, scales fp32,
    offsets fp32 or None, codes uint8, nonfinite int32 [1])``.  ``nonfinite`` is 1 when a weight is not finite.
    Integer grids need no ``levels``."""
    device = _require_cuda(weight, levels)
    rows, width = weight.shape
    group = min(group, width)
    packed = torch.empty(rows * width * bits // 8, dtype=torch.uint8, device=device)
    scales = torch.empty((rows, -(-width // group)), dtype=torch.float32, device=device)
    offsets = torch.empty_like(scales) if asym else None
    codes = torch.empty((rows, width), dtype=torch.uint8, device=device)
    nonfinite = torch.empty(1, dtype=torch.int32, device=device)
    with torch.cuda.device(device):
        status = _native.library().mkb_rtn_encode_checked(
            weight.data_ptr(), _pointer(levels), packed.data_ptr(), scales.data_ptr(), _pointer(offsets), codes.data_ptr(),
            nonfinite.data_ptr(), rows, width, group, bits, 1 if levels is None else levels.numel(), int(integer_grid), float(low), float(high),
            float(reciprocal), _tag(weight.dtype, "weight"), _stream(device))
    _native.check(status, "rtn_encode_checked")
    return packed, scales, offsets, codes, nonfinite


def dequantize_rows(packed: Tensor, scales: Tensor, values: Tensor, zeros: Tensor | None, rows: Tensor, *,
                    shape: tuple[int, int], group: int, bits: int, dtype: torch.dtype) -> Tensor:
    """Reconstruct the listed rows only: ``out[i] = weight[rows[i]]``."""
    device = _require_cuda(packed, scales, values, zeros, rows)
    total, width = shape
    rows = rows.reshape(-1).to(torch.int64).contiguous()
    out = torch.empty((rows.numel(), width), device=device, dtype=dtype)
    if rows.numel() == 0:
        return out
    with torch.cuda.device(device):
        status = _native.library().mkb_dequant_rows(
            packed.data_ptr(), scales.data_ptr(), values.data_ptr(), _pointer(zeros), rows.data_ptr(),
            out.data_ptr(), rows.numel(), total, width, group, bits, values.numel(),
            _tag(scales.dtype, "scale"), _tag(dtype, "output"), scales.stride(0), _stream(device))
    _native.check(status, "dequantize_rows")
    return out


def mix_supported(x: Tensor, signs: Tensor | None, out: Tensor, rows: int, factor: int, power: int) -> bool:
    """Whether ``mkb_hadamard_mix`` covers a transform whose basis is a Hadamard matrix (the C entry point checks the
    same), and is the faster kernel for it: a row per CTA needs rows to fill the GPU with.  14336 = 28 x 512 takes 6.1 us
    with the factor kernel and 7.2 with this one at 16 rows, 9.5 and 7.4 at 32; 18432 = 36 x 512, one CTA per SM, 9.9
    and 11.1 at 32, 13.0 and 11.3 at 64."""
    return (rows >= (32 if factor <= 32 else 64) and x.dtype in (torch.float16, torch.bfloat16)
            and 2 <= factor <= (32 if power == 1024 else 48)      # shared memory holds a row and its fp32 values
            and power in (128, 256, 512, 1024) and x.data_ptr() % 16 == 0 and out.data_ptr() % 8 == 0
            and (signs is None or signs.data_ptr() % 4 == 0))


def structured_transform(x: Tensor, *, factor: int, power: int, basis: Tensor | None = None,
                         signs: Tensor | None = None, inverse: bool = False, normalize: bool = True,
                         out: Tensor | None = None, hadamard_basis: bool = False) -> Tensor:
    """``(basis kron H_power)(x * signs)`` over the last axis, one fused launch; dtype preserved.  ``hadamard_basis``
    says that the entries of ``basis`` are all of one magnitude."""
    device = _require_cuda(x, basis, signs, out)
    width = x.shape[-1]
    if factor * power != width:
        raise ValueError("factor * power must equal the transform width")
    source = x if x.is_contiguous() else x.contiguous()
    if out is None:
        out = torch.empty_like(source)
    if signs is not None and (signs.dtype != torch.int8 or signs.numel() != width):
        raise ValueError("signs must be an int8 vector of the transform width")
    if basis is not None and (basis.dtype != torch.float32 or not basis.is_contiguous()):
        raise ValueError("basis must be a contiguous fp32 matrix")
    rows = source.numel() // width if width else 0
    library = _native.library()
    entry = library.mkb_hadamard
    if hadamard_basis and basis is not None and mix_supported(source, signs, out, rows, factor, power):
        entry = library.mkb_hadamard_mix
    with torch.cuda.device(device):
        status = entry(
            source.data_ptr(), _pointer(signs), _pointer(basis), out.data_ptr(), rows, width, factor,
            power, _tag(x.dtype, "activation"), int(inverse), int(normalize), _stream(device))
    _native.check(status, "structured_transform")
    return out


# ---- operators between the matvecs of a decode step (fp16, contiguous, caller-provided outputs) ----

def add_rmsnorm(residual: Tensor, delta: Tensor | None, weight: Tensor, normed: Tensor, eps: float) -> None:
    """``residual += delta`` (in place, when given) and ``normed = rms_norm(residual) * weight``."""
    rows, hidden = residual.shape
    status = _native.library().mkb_add_rmsnorm(residual.data_ptr(), _pointer(delta), weight.data_ptr(),
                                               normed.data_ptr(), rows, hidden, eps, _stream(residual.device))
    _native.check(status, "add_rmsnorm")


def rope_append(qkv: Tensor, positions: Tensor, k_cache: Tensor, v_cache: Tensor, *, q_heads: int, kv_heads: int,
                head_dim: int, theta: float) -> None:
    """Rotary embedding of the q and k heads of ``qkv`` in place, then k and v into the caches."""
    status = _native.library().mkb_rope_append(qkv.data_ptr(), positions.data_ptr(), k_cache.data_ptr(),
                                               v_cache.data_ptr(), qkv.shape[0], q_heads, kv_heads, head_dim,
                                               k_cache.shape[2], theta, _stream(qkv.device))
    _native.check(status, "rope_append")


def attention_decode(qkv: Tensor, positions: Tensor, k_cache: Tensor, v_cache: Tensor, out: Tensor, *,
                     q_heads: int, kv_heads: int, head_dim: int) -> None:
    """Single-token grouped-query attention over the cached positions ``0..positions[m]``."""
    status = _native.library().mkb_attention_decode(qkv.data_ptr(), positions.data_ptr(), k_cache.data_ptr(),
                                                    v_cache.data_ptr(), out.data_ptr(), qkv.shape[0], q_heads,
                                                    kv_heads, head_dim, k_cache.shape[2], head_dim ** -0.5,
                                                    _stream(qkv.device))
    _native.check(status, "attention_decode")


def rope_attention_decode(qkv: Tensor, positions: Tensor, k_cache: Tensor, v_cache: Tensor, out: Tensor, *,
                          q_heads: int, kv_heads: int, head_dim: int, theta: float, scale: float | None = None) -> None:
    """``rope_append`` and ``attention_decode`` in one launch (at most 8 query heads per key-value head);
    ``qkv`` is left unrotated."""
    if scale is None:
        scale = head_dim ** -0.5
    status = _native.library().mkb_rope_attention_decode(
        qkv.data_ptr(), positions.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), qkv.shape[0],
        q_heads, kv_heads, head_dim, k_cache.shape[2], theta, scale, _stream(qkv.device))
    _native.check(status, "rope_attention_decode")


def silu_mul(gate_up: Tensor, out: Tensor) -> None:
    """``out = silu(gate_up[:, :I]) * gate_up[:, I:]``."""
    status = _native.library().mkb_silu_mul(gate_up.data_ptr(), out.data_ptr(), gate_up.shape[0], out.shape[1],
                                            _stream(gate_up.device))
    _native.check(status, "silu_mul")


def argmax_keys(logits: Tensor, best: Tensor, offset: int = 0) -> Tensor:
    """``best[m]`` (int64 storage of an unsigned word) = sortable key of the row maximum of ``logits``
    ([M, width] fp16) in the high half, ``0xffffffff - (argmax + offset)`` in the low half."""
    status = _native.library().mkb_argmax(logits.data_ptr(), best.data_ptr(), logits.shape[0], logits.shape[1],
                                          logits.stride(0), offset, _stream(logits.device))
    _native.check(status, "argmax")
    return best


def tokens_of_keys(keys: Tensor) -> Tensor:
    """The token ids inside ``argmax_keys`` words."""
    return 0xFFFFFFFF - (keys & 0xFFFFFFFF)


# ---- operators over a paged cache, and on the logits ----

_raw_stream = torch._C._cuda_getCurrentRawStream      # torch.cuda.current_stream builds an object: 3 us of a call
_current_device, _capturing = torch._C._cuda_getDevice, torch._C._cuda_isCurrentStreamCapturing


# What a call of these operators checks depends on the layouts of its tensors alone (shapes, strides, dtypes, devices) and on
# plain numbers: calls whose layouts were checked before go straight to the C entry with the numbers made out then, which
# checks pointers and alignment itself.  The checks took 5 of the 13 us of an attention call's host side.
_Plan = tuple
_plans: dict[tuple, _Plan] = {}


def _planned(key: tuple, plan: _Plan) -> _Plan:
    if len(_plans) >= 4096:
        _plans.clear()
    _plans[key] = plan
    return plan


STATE_BYTES, STATES = 8192, 128     # of the attention over pages: zeroed words of one call at a time; states of a block


class _AttentionScratch:
    """Where the parts of a sequence meet, on one device: a state and a workspace for each.  Calls on one stream run in order and
    share theirs; the workspace grows to the largest request.  Captured calls may be replayed at any time, so each owns its
    state for good, also when its graph is gone (8 KB of a block that was cleared before), and has its workspace in the memory of its
    graph.  After every eager call there are STATES for the captures to come; only a call that is captured when none is left has its
    graph clear one.  The lock keeps host threads apart: a state is handed out once, and callers hold it until a call's launches are
    all in the stream.  (A call with weights makes two, and the second reads what the first left in the workspace, which threads
    on one stream share.)"""

    def __init__(self) -> None:
        self.lock = threading.RLock()
        self.streams: dict[int, tuple[int, Tensor]] = {}
        self.blocks: list[Tensor] = []
        self.left: list[int] = []

    def refill(self, index: int) -> None:
        block = torch.zeros(STATES * STATE_BYTES, dtype=torch.uint8, device=index)
        torch.cuda.current_stream(index).synchronize()        # other streams will use the states
        self.blocks.append(block)
        self.left = [block.data_ptr() + i * STATE_BYTES for i in range(STATES)] + self.left

    def of(self, index: int, stream: int, need: int) -> tuple[int, Tensor]:
        with self.lock:
            if _capturing():
                workspace = torch.empty(need + STATE_BYTES, dtype=torch.uint8, device=index)
                if self.left:
                    return self.left.pop(), workspace
                workspace[need:].zero_()
                return workspace.data_ptr() + need, workspace
            while len(self.left) < STATES + (stream not in self.streams):     # so that STATES are left
                self.refill(index)
            held = self.streams.get(stream)
            if held is None or held[1].numel() < need:
                held = self.streams[stream] = (self.left.pop() if held is None else held[0],
                                               torch.empty(need, dtype=torch.uint8, device=index))
            return held


_attention_scratch: dict[int, _AttentionScratch] = {}


def _scratch(index: int) -> _AttentionScratch:
    return _attention_scratch.get(index) or _attention_scratch.setdefault(index, _AttentionScratch())


def _check_pages(what: str, index: int, k_pages: Tensor, v_pages: Tensor, weights: Tensor | None, *tables: Tensor) -> None:
    """Pools, tables and accumulator of one layout on device ``index``."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape or v_pages.stride() != k_pages.stride() or v_pages.dtype != k_pages.dtype:
        raise ValueError(f"{what}: pages of keys and values must share one [pages, kv_heads, page, head_dim] layout and dtype")
    if k_pages.stride(3) != 1:
        raise ValueError(f"{what}: the head dimension of the pages must be contiguous")
    for table in tables:
        if table.dtype is not torch.int32 or table.dim() != 2 or table.stride(1) != 1:
            raise ValueError(f"{what}: page tables are int32 [rows, columns] with contiguous rows")
        if table.get_device() != index:
            raise ValueError("all tensors of one call must live on one device")
    if weights is not None and (weights.dtype is not torch.float32 or weights.shape != shape[:3] or not weights.is_contiguous()):
        raise ValueError(f"{what}: weights are a contiguous fp32 [pages, kv_heads, page] tensor")
    if k_pages.get_device() != index or v_pages.get_device() != index or (weights is not None and weights.get_device() != index):
        raise ValueError("all tensors of one call must live on one device")


def _check_rows(what: str, index: int, rows: int, *vectors: Tensor) -> None:
    for vector in vectors:
        if vector.dtype is not torch.int32 or vector.dim() != 1 or vector.shape[0] != rows or not vector.is_contiguous():
            raise ValueError(f"{what}: lengths and positions are contiguous int32 vectors of {rows} rows")
        if vector.get_device() != index:
            raise ValueError("all tensors of one call must live on one device")


def paged_attention_decode(q: Tensor, lengths: Tensor, k_pages: Tensor, v_pages: Tensor, tables: Tensor, out: Tensor, *,
                           scale: float | None = None, weights: Tensor | None = None) -> None:
    """Attention of one query token per sequence (``q`` [rows, q_heads, head_dim]) to the ``lengths`` slots of its paged cache
    (pools ``[pages, kv_heads, page, head_dim]``, page numbers ``tables`` int32 [rows, columns]) into ``out``.  An empty sequence
    and a row that is not in use (a negative length) give zeros.  ``weights`` (fp32 [pages, kv_heads, page]) adds up every
    slot's softmax weight over the query heads of its group; no page is then in the tables twice, as it may be without."""
    key = (q.shape, q.stride(), q.dtype, q.get_device(), lengths.shape, lengths.stride(), lengths.dtype, lengths.get_device(),
           k_pages.shape, k_pages.stride(), k_pages.dtype, k_pages.get_device(), v_pages.shape, v_pages.stride(), v_pages.dtype,
           v_pages.get_device(), tables.shape, tables.stride(), tables.dtype, tables.get_device(), out.shape, out.stride(), out.dtype,
           out.get_device(), scale, None if weights is None else
           (weights.shape, weights.stride(), weights.dtype, weights.get_device()))
    index, function, need, numbers = _plans.get(key) or _planned(key, _plan_attention(q, lengths, k_pages, v_pages, tables, out,
                                                                                     scale, weights))
    if _current_device() != index:
        with torch.cuda.device(index):
            return paged_attention_decode(q, lengths, k_pages, v_pages, tables, out, scale=scale, weights=weights)
    stream = _raw_stream(index)
    scratch = _scratch(index)
    with scratch.lock:
        state, workspace = scratch.of(index, stream, need)
        status = function(q.data_ptr(), lengths.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), tables.data_ptr(), out.data_ptr(),
                          None if weights is None else weights.data_ptr(), *numbers, state, workspace.data_ptr(), need, stream)
    if status:
        _native.check(status, "paged_attention_decode")


def _plan_attention(q: Tensor, lengths: Tensor, k_pages: Tensor, v_pages: Tensor, tables: Tensor, out: Tensor, scale: float | None,
                    weights: Tensor | None) -> _Plan:
    what, index, dtype = "paged_attention_decode", q.get_device(), q.dtype
    if index < 0:
        raise ValueError("mlkit_b200 kernels require CUDA tensors")
    if q.dim() != 3 or k_pages.dtype is not dtype:
        raise ValueError(f"{what}: queries are [rows, q_heads, head_dim] in the dtype of the pages")
    rows, q_heads, head_dim = q.shape
    row, head, step = q.stride()
    _check_pages(what, index, k_pages, v_pages, weights, tables)
    if step != 1 or k_pages.shape[3] != head_dim:
        raise ValueError(f"{what}: queries have contiguous heads of {k_pages.shape[3]}")
    _check_out(what, index, out, dtype, rows, q_heads, head_dim, tables)
    _check_rows(what, index, rows, lengths)
    return _attention_plan(index, "mkb_paged_attention_decode", q_heads, k_pages, tables, (row, head), (), scale, weights)


def _check_out(what: str, index: int, out: Tensor, dtype: torch.dtype, rows: int, q_heads: int, head_dim: int, tables: Tensor) -> None:
    if (out.dtype is not dtype or out.numel() != rows * q_heads * head_dim or not out.is_contiguous() or out.get_device() != index
            or out.dim() < 2 or out.shape[0] != rows):
        raise ValueError(f"{what}: the output is a contiguous [rows, q_heads, head_dim] in the dtype and on the device of the queries")
    if tables.shape[0] != rows:
        raise ValueError(f"{what}: a row of tables for each row of queries")


def _attention_plan(index: int, entry: str, q_heads: int, k_pages: Tensor, tables: Tensor, q_strides: tuple[int, ...],
                    theta: tuple[float, ...], scale: float | None, weights: Tensor | None) -> _Plan:
    """``(device, C entry, bytes of workspace, the entry's numbers)``."""
    pages, kv_heads, page, head_dim = k_pages.shape
    rows, columns = tables.shape
    library = _native.library()
    with torch.cuda.device(index):
        need = library.mkb_paged_attention_workspace_bytes(rows, q_heads, kv_heads, head_dim, page, columns, weights is not None)
    return (index, getattr(library, entry), need,
            (rows, q_heads, kv_heads, head_dim, page, columns, pages, *k_pages.stride()[:3], tables.stride(0), *q_strides, *theta,
             head_dim ** -0.5 if scale is None else scale, _tag(k_pages.dtype, "cache")))


def paged_rope_attention_decode(qkv: Tensor, positions: Tensor, lengths: Tensor, k_pages: Tensor, v_pages: Tensor, tables: Tensor,
                                out: Tensor, *, q_heads: int, kv_heads: int, head_dim: int, theta: float,
                                scale: float | None = None, weights: Tensor | None = None) -> None:
    """One decode step of attention over a paged cache: the new key of each row of ``qkv`` is rotated by ``positions`` and
    stored with its value in slot ``lengths`` of the sequence, and the rotated queries attend to slots ``0..lengths``.  ``qkv`` is
    left unrotated, ``lengths`` as they are; a row with a negative length is not in use (zeros, nothing stored).  Positions
    and lengths differ where slots were evicted.  ``weights`` as in ``paged_attention_decode``; a new slot begins at zero."""
    key = (qkv.shape, qkv.stride(), qkv.dtype, qkv.get_device(), positions.shape, positions.stride(), positions.dtype,
           positions.get_device(), lengths.shape, lengths.stride(), lengths.dtype, lengths.get_device(), k_pages.shape,
           k_pages.stride(), k_pages.dtype, k_pages.get_device(), v_pages.shape, v_pages.stride(), v_pages.dtype,
           v_pages.get_device(), tables.shape, tables.stride(), tables.dtype, tables.get_device(), out.shape, out.stride(), out.dtype,
           out.get_device(), q_heads, kv_heads, head_dim, theta, scale, None if weights is None else
           (weights.shape, weights.stride(), weights.dtype, weights.get_device()))
    index, function, need, numbers = _plans.get(key) or _planned(
        key, _plan_rope_attention(qkv, positions, lengths, k_pages, v_pages, tables, out, q_heads, kv_heads, head_dim, theta, scale,
                                  weights))
    if _current_device() != index:
        with torch.cuda.device(index):
            return paged_rope_attention_decode(qkv, positions, lengths, k_pages, v_pages, tables, out, q_heads=q_heads,
                                               kv_heads=kv_heads, head_dim=head_dim, theta=theta, scale=scale, weights=weights)
    stream = _raw_stream(index)
    scratch = _scratch(index)
    with scratch.lock:
        state, workspace = scratch.of(index, stream, need)
        status = function(qkv.data_ptr(), positions.data_ptr(), lengths.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                          tables.data_ptr(), out.data_ptr(), None if weights is None else weights.data_ptr(), *numbers, state,
                          workspace.data_ptr(), need, stream)
    if status:
        _native.check(status, "paged_rope_attention_decode")


def _plan_rope_attention(qkv: Tensor, positions: Tensor, lengths: Tensor, k_pages: Tensor, v_pages: Tensor, tables: Tensor,
                         out: Tensor, q_heads: int, kv_heads: int, head_dim: int, theta: float, scale: float | None,
                         weights: Tensor | None) -> _Plan:
    what, index, dtype = "paged_rope_attention_decode", qkv.get_device(), qkv.dtype
    if index < 0:
        raise ValueError("mlkit_b200 kernels require CUDA tensors")
    if qkv.dim() != 2 or k_pages.dtype is not dtype:
        raise ValueError(f"{what}: q | k | v is [rows, (q_heads + 2 * kv_heads) * head_dim] in the dtype of the pages")
    rows, width = qkv.shape
    row, step = qkv.stride()
    _check_pages(what, index, k_pages, v_pages, weights, tables)
    _, heads, _, depth = k_pages.shape
    if step != 1 or heads != kv_heads or depth != head_dim or width != (q_heads + 2 * kv_heads) * head_dim:
        raise ValueError(f"{what}: rows of {width} values and pages of {heads} heads of {depth} are not {q_heads} query and "
                         f"{kv_heads} key-value heads of {head_dim}")
    _check_out(what, index, out, dtype, rows, q_heads, head_dim, tables)
    _check_rows(what, index, rows, positions, lengths)
    return _attention_plan(index, "mkb_paged_rope_attention_decode", q_heads, k_pages, tables, (row,), (theta,), scale, weights)


def evict_pages(k_pages: Tensor, v_pages: Tensor, weights: Tensor, tables: Tensor, lengths: Tensor, new_tables: Tensor, *,
                budget: int, sinks: int = 0, recent: int = 0) -> Tensor:
    """Keep ``min(length, budget)`` slots of every sequence and head: the first ``sinks``, the last ``recent`` and the
    heaviest of the others by ``weights`` (a tie to the lower slot).  They are copied, in slot order, to the pages that
    ``new_tables`` names; these must be named once and be none of ``tables``.  Returns the kept slots, int32 [rows, kv_heads,
    budget], -1 behind the last.  The caller swaps the tables, sets the lengths and frees the old pages."""
    key = (k_pages.shape, k_pages.stride(), k_pages.dtype, k_pages.get_device(), v_pages.shape, v_pages.stride(), v_pages.dtype,
           v_pages.get_device(), weights.shape, weights.stride(), weights.dtype, weights.get_device(), tables.shape, tables.stride(),
           tables.dtype, tables.get_device(), lengths.shape, lengths.stride(), lengths.dtype, lengths.get_device(), new_tables.shape,
           new_tables.stride(), new_tables.dtype, new_tables.get_device(), budget, sinks, recent)
    index, function, shape, numbers = _plans.get(key) or _planned(key, _plan_evict(k_pages, v_pages, weights, tables, lengths,
                                                                                  new_tables, budget, sinks, recent))
    if _current_device() != index:
        with torch.cuda.device(index):
            return evict_pages(k_pages, v_pages, weights, tables, lengths, new_tables, budget=budget, sinks=sinks, recent=recent)
    kept = tables.new_empty(shape)
    status = function(k_pages.data_ptr(), v_pages.data_ptr(), weights.data_ptr(), tables.data_ptr(), lengths.data_ptr(),
                      new_tables.data_ptr(), kept.data_ptr(), *numbers, _raw_stream(index))
    if status:
        _native.check(status, "evict_pages")
    return kept


def _plan_evict(k_pages: Tensor, v_pages: Tensor, weights: Tensor, tables: Tensor, lengths: Tensor, new_tables: Tensor, budget: int,
                sinks: int, recent: int) -> _Plan:
    what, index = "evict_pages", k_pages.get_device()
    if index < 0:
        raise ValueError("mlkit_b200 kernels require CUDA tensors")
    _check_pages(what, index, k_pages, v_pages, weights, tables, new_tables)
    if k_pages.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{what}: pages are fp16 or bf16")
    pages, kv_heads, page, head_dim = k_pages.shape
    rows, columns = tables.shape
    if new_tables.shape[0] != rows:
        raise ValueError(f"{what}: a row of new tables for each row of tables")
    _check_rows(what, index, rows, lengths)
    return (index, _native.library().mkb_paged_evict, (rows, kv_heads, max(budget, 0)),
            (rows, kv_heads, head_dim, page, columns, new_tables.shape[1], pages, *k_pages.stride()[:3], tables.stride(0),
             new_tables.stride(0), budget, sinks, recent))


def adjust_logits(logits: Tensor, *, tokens: Tensor | None = None, lengths: Tensor | None = None, prompts: Tensor | None = None,
                  repetition: Tensor | None = None, frequency: Tensor | None = None, presence: Tensor | None = None,
                  bias_tokens: Tensor | None = None, bias: Tensor | None = None, mask: Tensor | None = None, offset: int = 0,
                  best: Tensor | None = None, picked: Tensor | None = None, out: Tensor | None = None) -> Tensor:
    """Penalties for the tokens of a history, sparse biases and a grammar's bit mask on ``logits`` [rows, width] of the tokens
    ``offset..offset + width``; in place unless ``out`` is given.  For token v, in fp32 and in this order:

    * v in ``tokens[m, :lengths[m]]``: divided by ``repetition[m]`` when positive, multiplied otherwise;
    * c times in ``tokens[m, prompts[m]:lengths[m]]``: less ``frequency[m] * c``, and less ``presence[m]`` when c > 0;
    * plus the ``bias`` of every entry of ``bias_tokens`` [rows, entries] that is v;
    * -inf where bit v % 32 of ``mask[m, v // 32]`` is 0.

    Ids outside ``offset..offset + width`` (-1 fills a row up) have no effect.  ``best`` (int64 [rows]) receives the words of
    ``argmax_keys`` for the result, ``picked`` (int64 [rows]) its greedy tokens."""
    if out is None:
        out = logits
    given = (logits, out, tokens, lengths, prompts, repetition, frequency, presence, bias_tokens, bias, mask, best, picked)
    key = (offset, *[None if t is None else (t.shape, t.stride(), t.dtype, t.get_device()) for t in given])
    index, function, numbers = _plans.get(key) or _planned(key, _plan_logits(*given, offset))
    if _current_device() != index:
        with torch.cuda.device(index):
            return adjust_logits(logits, tokens=tokens, lengths=lengths, prompts=prompts, repetition=repetition, frequency=frequency,
                                 presence=presence, bias_tokens=bias_tokens, bias=bias, mask=mask, offset=offset, best=best,
                                 picked=picked, out=out)
    status = function(*[None if t is None else t.data_ptr() for t in given], *numbers, _raw_stream(index))
    if status:
        _native.check(status, "adjust_logits")
    return out


def _plan_logits(logits: Tensor, out: Tensor, tokens: Tensor | None, lengths: Tensor | None, prompts: Tensor | None,
                 repetition: Tensor | None, frequency: Tensor | None, presence: Tensor | None, bias_tokens: Tensor | None,
                 bias: Tensor | None, mask: Tensor | None, best: Tensor | None, picked: Tensor | None, offset: int) -> _Plan:
    what, index = "adjust_logits", logits.get_device()
    if index < 0:
        raise ValueError("mlkit_b200 kernels require CUDA tensors")
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError(f"{what}: logits are [rows, width] with contiguous rows")
    rows, width = logits.shape
    if out.shape != logits.shape or out.dtype is not logits.dtype or out.stride(1) != 1 or out.get_device() != index:
        raise ValueError(f"{what}: the output matches the logits in shape, dtype and device, with contiguous rows")

    def vector(name: str, given: Tensor | None, kind: torch.dtype) -> None:
        if given is not None and (given.dtype is not kind or given.dim() != 1 or given.shape[0] != rows or not given.is_contiguous()
                                  or given.get_device() != index):
            raise ValueError(f"{what}: {name} must be a contiguous {kind} vector of {rows} rows on the device of the logits")

    def table(name: str, given: Tensor | None, *kinds: torch.dtype) -> tuple[int, int]:
        if given is None:
            return 0, 0
        if given.dim() != 2 or given.shape[0] != rows or given.dtype not in kinds or given.get_device() != index:
            raise ValueError(f"{what}: {name} must be {kinds[0]} [rows, entries] on the device of the logits")
        stride, step = given.stride()
        if step != 1 and given.shape[1] > 1:
            raise ValueError(f"{what}: {name} must have contiguous rows")
        return given.shape[1], stride

    for name, given, kind in (("lengths", lengths, torch.int32), ("prompts", prompts, torch.int32),
                              ("repetition", repetition, torch.float32), ("frequency", frequency, torch.float32),
                              ("presence", presence, torch.float32), ("best", best, torch.int64), ("picked", picked, torch.int64)):
        vector(name, given, kind)
    history = table("tokens", tokens, torch.int64, torch.int32)
    if (tokens is None) != (lengths is None):
        raise ValueError(f"{what}: a history needs its lengths")
    if tokens is None and not (prompts is None and repetition is None and frequency is None and presence is None):
        raise ValueError(f"{what}: penalties need a history of tokens")
    biases = table("bias_tokens", bias_tokens, torch.int32)
    if (bias is None) != (bias_tokens is None) or table("bias", bias, torch.float32) != biases:
        raise ValueError(f"{what}: biases need a token for every value, in the same layout")
    return (index, _native.library().mkb_adjust_logits,
            (rows, width, logits.stride(0), out.stride(0), *history, *biases, *table("mask", mask, torch.int32), offset,
             tokens is not None and tokens.dtype is torch.int64, _tag(logits.dtype, "logit")))


def decode_status() -> int:
    """Non-zero when a decode operator since the last call saw a cache position outside ``[0, capacity)``
    (it clamped the position and skipped the append; that step's results are not valid).  Synchronises."""
    import ctypes

    value = ctypes.c_int(0)
    _native.check(_native.library().mkb_decode_status(ctypes.byref(value)), "decode_status")
    return value.value
