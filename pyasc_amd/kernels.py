"""Typed host API over libasc_hip.so: torch device tensors in, kernels launched.

Every function checks on the host that the buffers hold everything the kernel
will touch (shape, dtype, device, layout) before it reaches the C ABI, so an
inconsistent call raises ValueError/TypeError here instead of faulting on the
GPU.  Launches are asynchronous on ``stream`` (default: torch's current stream).
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Any, Optional

import torch

from . import _native

_DTYPE_CODES = {
    torch.float32: _native.DT_FLOAT32,
    torch.float16: _native.DT_FLOAT16,
    torch.bfloat16: _native.DT_BFLOAT16,
    torch.int32: _native.DT_INT32,
    torch.int8: _native.DT_INT8,
    torch.int16: _native.DT_INT16,
}


def _stream(stream: Any) -> int:
    if stream is None:
        return _native.current_stream_handle()
    if isinstance(stream, int):
        return stream
    return int(stream.cuda_stream)


def _device_tensor(t: Any, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"'{name}' must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"'{name}' must be on the HIP device, got {t.device}")
    return t


def _stream_of(handle: int, device: torch.device) -> Any:
    """Stream ``handle`` as torch's.  0 is the default stream, which an ExternalStream cannot name."""
    return torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)


def workspace_on(handle: int, numel: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A workspace for the launches of one call on stream ``handle``, freed when the call returns.
    It comes from that stream's pool of torch's allocator: a block of another stream's pool may
    still be in use by work queued there, and would be handed out again before the launches have
    run, while a block of the launch stream's pool is ordered with them on both sides."""
    if handle == _native.current_stream_handle(device.index):
        return torch.empty(numel, dtype=dtype, device=device)
    with torch.cuda.stream(_stream_of(handle, device)):
        return torch.empty(numel, dtype=dtype, device=device)


def _held_by_a_graph(t: torch.Tensor) -> bool:
    """Whether ``t``, allocated during a capture, lies in a graph's own memory pool: torch keeps
    that for the graph's replays.  In a capture begun by other means the block is an ordinary
    one, which goes to the next allocation once it is freed."""
    if torch.cuda.get_allocator_backend() != "native":
        return False
    at = t.data_ptr()
    return any(s["address"] <= at < s["address"] + s["total_size"] and s.get("segment_pool_id", (0, 0)) != (0, 0)
               for s in torch.cuda.memory_snapshot())


def _contiguous(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_contiguous():
        raise ValueError(f"'{name}' must be contiguous")
    return t


def _code(t: torch.Tensor, name: str, allowed) -> int:
    if t.dtype not in allowed:
        raise TypeError(f"'{name}' has unsupported dtype {t.dtype}; expected one of {sorted(map(str, allowed))}")
    return _DTYPE_CODES[t.dtype]


# ---------------------------------------------------------------------------------------------- vadd

def vadd_covered(size: int, tile_size: int, tile_per_block: int, grid: int) -> int:
    """Elements written by asc2 vadd_kernel: [0, min(size, grid*tpb*tile))
    (python/test/asc2/kernels/test_vadd.py:22-28 with the store clipped at ``size``)."""
    return max(0, min(size, grid * tile_per_block * tile_size))


_VADD_DTYPES = (torch.float32, torch.float16, torch.bfloat16, torch.int32)


def vadd_check(x: torch.Tensor, y: torch.Tensor, out: torch.Tensor, size: int, tile_size: int, tile_per_block: int,
               grid: int) -> int:
    """Host checks of a vadd launch; returns the covered element count."""
    for t, n in ((x, "x"), (y, "y"), (out, "out")):
        _contiguous(_device_tensor(t, n), n)
    _code(x, "x", _VADD_DTYPES)
    if y.dtype != x.dtype or out.dtype != x.dtype:
        raise TypeError(f"vadd operands must share one dtype, got {x.dtype}, {y.dtype}, {out.dtype}")
    if tile_size <= 0 or tile_per_block < 0 or grid <= 0 or size < 0:
        raise ValueError(f"invalid vadd launch: size={size}, tile_size={tile_size}, "
                         f"tile_per_block={tile_per_block}, grid={grid}")
    covered = vadd_covered(size, tile_size, tile_per_block, grid)
    for t, n in ((x, "x"), (y, "y"), (out, "out")):
        if t.numel() < covered:
            raise ValueError(f"'{n}' holds {t.numel()} elements but the launch touches {covered}")
    return covered


def vadd(x: torch.Tensor, y: torch.Tensor, out: torch.Tensor, size: int, tile_size: int, tile_per_block: int,
         grid: int, stream: Any = None) -> None:
    vadd_check(x, y, out, size, tile_size, tile_per_block, grid)
    code = _DTYPE_CODES[x.dtype]
    _native.call("asc_vadd", code, x.data_ptr(), y.data_ptr(), out.data_ptr(), size, tile_size, tile_per_block,
                 grid, _stream(stream))


# -------------------------------------------------------------------------- leaky_relu / vmuladd / gelu

def _check_stream_operands(tensors, covered: int) -> int:
    """Common checks of the tiled elementwise kernels: contiguous device tensors of one
    float dtype, each holding at least the covered elements.  Returns the dtype code."""
    for t, n in tensors:
        _contiguous(_device_tensor(t, n), n)
    first = tensors[0][0]
    code = _code(first, tensors[0][1], (torch.float32, torch.float16, torch.bfloat16))
    for t, n in tensors:
        if t.dtype != first.dtype:
            raise TypeError(f"operands must share one dtype, got {first.dtype} and {t.dtype} ('{n}')")
        if t.numel() < covered:
            raise ValueError(f"'{n}' holds {t.numel()} elements but the launch touches {covered}")
    return code


def _check_tiling(size: int, tile_size: int, tile_per_block: int, grid: int, what: str) -> None:
    if tile_size <= 0 or tile_per_block < 0 or grid <= 0 or size < 0:
        raise ValueError(f"invalid {what} launch: size={size}, tile_size={tile_size}, "
                         f"tile_per_block={tile_per_block}, grid={grid}")


def leaky_relu_check(x: torch.Tensor, out: torch.Tensor, size: int, tile_size: int, tile_per_block: int,
                     grid: int) -> int:
    """Host checks of a leaky_relu launch; returns the covered element count."""
    _check_tiling(size, tile_size, tile_per_block, grid, "leaky_relu")
    covered = vadd_covered(size, tile_size, tile_per_block, grid)
    _check_stream_operands(((x, "x"), (out, "out")), covered)
    return covered


def leaky_relu(x: torch.Tensor, alpha: float, out: torch.Tensor, size: int, tile_size: int, tile_per_block: int,
               grid: int, stream: Any = None) -> None:
    """asc2 leaky_relu_kernel (python/test/asc2/kernels/test_leaky_relu.py:16-26):
    out = where(x >= 0, x, x * alpha) over the vadd-style covered range; ``alpha`` is
    used at its float value (a 0-dim bf16 tensor's exact value)."""
    leaky_relu_check(x, out, size, tile_size, tile_per_block, grid)
    _native.call("asc_leaky_relu", _DTYPE_CODES[x.dtype], x.data_ptr(), float(alpha), out.data_ptr(), size,
                 tile_size, tile_per_block, grid, _stream(stream))


def vmuladd_check(x: torch.Tensor, y: torch.Tensor, z: torch.Tensor, out: torch.Tensor, size: int, tile_size: int,
                  tile_per_block: int, grid: int) -> int:
    """Host checks of a vmuladd launch; returns the covered element count."""
    _check_tiling(size, tile_size, tile_per_block, grid, "vmuladd")
    covered = vadd_covered(size, tile_size, tile_per_block, grid)
    _check_stream_operands(((x, "x"), (y, "y"), (z, "z"), (out, "out")), covered)
    return covered


def vmuladd(x: torch.Tensor, y: torch.Tensor, z: torch.Tensor, out: torch.Tensor, size: int, tile_size: int,
            tile_per_block: int, grid: int, stream: Any = None) -> None:
    """asc2 vmuladd_kernel (python/test/asc2/kernels/test_vmuladd.py:16-31): out = x * y + z,
    multiply and add rounded separately."""
    vmuladd_check(x, y, z, out, size, tile_size, tile_per_block, grid)
    _native.call("asc_vmuladd", _DTYPE_CODES[x.dtype], x.data_ptr(), y.data_ptr(), z.data_ptr(), out.data_ptr(),
                 size, tile_size, tile_per_block, grid, _stream(stream))


def gelu_rows_check(x: torch.Tensor, out: torch.Tensor, num_rows: int, num_cols: int, tile_size: int,
                    grid: int) -> None:
    """Host checks of a gelu launch."""
    if tile_size <= 0 or grid <= 0 or num_rows < 0 or num_cols < 0:
        raise ValueError(f"invalid gelu launch: rows={num_rows}, cols={num_cols}, tile={tile_size}, grid={grid}")
    for t, n in ((x, "x"), (out, "out")):
        _contiguous(_device_tensor(t, n), n)
        if t.dtype != torch.float32:
            raise TypeError(f"gelu supports float32 only, '{n}' is {t.dtype}")
        if t.numel() < num_rows * num_cols:
            raise ValueError(f"'{n}' holds {t.numel()} elements but the launch touches {num_rows}x{num_cols}")


def gelu_rows(x: torch.Tensor, out: torch.Tensor, num_rows: int, num_cols: int, tile_size: int, approximate: bool,
              grid: int, stream: Any = None) -> None:
    """asc2 gelu_kernel (python/test/asc2/kernels/test_gelu.py:19-33) on fp32 rows.  A tile
    wider than the row computes the row's own columns (the padding is zeros and gelu is
    element-wise) and writes nothing past them."""
    gelu_rows_check(x, out, num_rows, num_cols, tile_size, grid)
    _native.call("asc_gelu_rows_f32", x.data_ptr(), out.data_ptr(), num_rows, num_cols, tile_size,
                 int(bool(approximate)), grid, _stream(stream))


# ------------------------------------------------------------------------------------------- softmax

def _check_softmax(x: torch.Tensor, out: torch.Tensor, rows: int, num_cols: int) -> str:
    """Checks the buffers; returns the entry-point suffix of their dtype ("f32" / "f16")."""
    for t, n in ((x, "x"), (out, "out")):
        _contiguous(_device_tensor(t, n), n)
        if t.dtype not in (torch.float32, torch.float16):
            raise TypeError(f"softmax supports float32 and float16, '{n}' is {t.dtype}")
        if t.numel() < rows * num_cols:
            raise ValueError(f"'{n}' holds {t.numel()} elements but the launch touches {rows}x{num_cols}")
    if out.dtype != x.dtype:
        raise TypeError(f"'out' must be {x.dtype}, got {out.dtype}")
    return "f32" if x.dtype == torch.float32 else "f16"


def _softmax_launch(x: torch.Tensor, out: torch.Tensor, num_rows: int, num_cols: int, size: int, grid: int,
                    fused: bool) -> str:
    """Checks a softmax launch (size is tile_size, or block_size when fused); returns the
    dtype suffix ("f32" / "f16")."""
    if size <= 0 or grid <= 0 or num_rows < 0 or num_cols < 0:
        raise ValueError(f"invalid softmax launch: rows={num_rows}, cols={num_cols}, "
                         f"{'block' if fused else 'tile'}={size}, grid={grid}")
    rows = softmax_blocks_covered(num_rows, size, grid) if fused else num_rows
    return _check_softmax(x, out, rows, num_cols)


def softmax_rows(x: torch.Tensor, out: torch.Tensor, num_rows: int, num_cols: int, tile_size: int, grid: int,
                 stream: Any = None) -> None:
    """asc2 softmax_kernel(x, out, num_rows, num_cols, tile_size) of
    python/test/asc2/kernels/test_softmax.py:16-27.  With tile_size > num_cols each row's
    statistics include the tile's tile_size - num_cols zero padding (the reference's padded
    load and whole-tile reductions) and each row writes its own num_cols outputs."""
    suffix = _softmax_launch(x, out, num_rows, num_cols, tile_size, grid, False)
    _native.call(f"asc_softmax_rows_{suffix}", x.data_ptr(), out.data_ptr(), num_rows, num_cols, tile_size, grid,
                 _stream(stream))


def softmax_blocks_covered(num_rows: int, block_size: int, grid: int) -> int:
    """Rows written by the fused asc2 softmax_kernel: [0, min(num_rows, grid*block_size))."""
    return max(0, min(num_rows, grid * block_size))


def softmax_blocks(x: torch.Tensor, out: torch.Tensor, num_rows: int, num_cols: int, block_size: int, grid: int,
                   stream: Any = None) -> None:
    """asc2 softmax_kernel(x, out, num_rows, num_cols, block_size) of
    python/test/asc2/kernels/test_softmax_fused.py:16-24."""
    suffix = _softmax_launch(x, out, num_rows, num_cols, block_size, grid, True)
    _native.call(f"asc_softmax_blocks_{suffix}", x.data_ptr(), out.data_ptr(), num_rows, num_cols, block_size,
                 grid, _stream(stream))


def softmax_plan(x: torch.Tensor, out: torch.Tensor, num_rows: int, num_cols: int, size: int, grid: int,
                 fused: bool) -> "_native.SoftmaxPlan":
    """A launch of softmax_rows (fused False, size = tile_size) or softmax_blocks (fused True,
    size = block_size) chosen by dtype and row length, as a kernel of the asc2_softmax code
    object with its grid, block and arguments (asc_softmax_plan); plan.grid == 0 when there is
    nothing to launch.  Same checks and errors as those two calls."""
    return _softmax_plan("asc_softmax_plan", x, out, num_rows, num_cols, size, grid, fused)


def softmax_dispatch(x: torch.Tensor, out: torch.Tensor, num_rows: int, num_cols: int, size: int, grid: int,
                     fused: bool) -> "_native.SoftmaxPlan":
    """The launch those two calls make (asc_softmax_dispatch), in softmax_plan's form."""
    return _softmax_plan("asc_softmax_dispatch", x, out, num_rows, num_cols, size, grid, fused)


def _softmax_plan(entry: str, x, out, num_rows, num_cols, size, grid, fused) -> "_native.SoftmaxPlan":
    suffix = _softmax_launch(x, out, num_rows, num_cols, size, grid, fused)
    plan = _native.SoftmaxPlan()
    _native.call(entry, _native.DT_FLOAT32 if suffix == "f32" else _native.DT_FLOAT16, int(fused), x.data_ptr(),
                 out.data_ptr(), num_rows, num_cols, size, grid, ctypes.byref(plan))
    return plan


# ---------------------------------------------------------------------------------- reductions, rms_norm

REDUCE_OPS = {"sum": 0, "max": 1, "min": 2, "prod": 3}


def reduce_f32(x: torch.Tensor, out: torch.Tensor, op: str, dim: Optional[int], stream: Any = None) -> None:
    """asc2.reduce_{sum,max,min,prod} of a 1-D or 2-D float32 tensor along ``dim`` (0 or 1 of
    a 2-D tensor) or over all elements (``dim=None``: the scalar is written to every element
    of ``out``, as asc2.full does in test_reduce_ops.py's kernel_all)."""
    if op not in REDUCE_OPS:
        raise ValueError(f"unknown reduction {op!r}; expected one of {sorted(REDUCE_OPS)}")
    for t, n in ((x, "x"), (out, "out")):
        _contiguous(_device_tensor(t, n), n)
        if t.dtype != torch.float32:
            raise TypeError(f"reductions support float32, '{n}' is {t.dtype}")
    if x.dim() == 1:
        rows, cols = 1, x.shape[0]
    elif x.dim() == 2:
        rows, cols = x.shape
    else:
        raise ValueError("x must be 1-D or 2-D")
    if dim is None:
        _reduce(x, out, op, rows, cols, -1, out.numel(), stream)
        return
    if x.dim() != 2 or dim not in (0, 1):
        raise ValueError(f"dim must be 0 or 1 of a 2-D tensor, got dim={dim} for shape {tuple(x.shape)}")
    need = rows if dim == 1 else cols
    if out.numel() != need:
        raise ValueError(f"out must hold {need} elements, holds {out.numel()}")
    _reduce(x, out, op, rows, cols, dim, need, stream)


# below this many elements no reduction uses a workspace (kSplitMinElems of csrc/reduce.hip)
_REDUCE_SPLIT_MIN = 1 << 18


def _reduce(x: torch.Tensor, out: torch.Tensor, op: str, rows: int, cols: int, dim: int, count: int, stream) -> None:
    """One reduction; one with few results over many elements gets a workspace (at most 64 KiB)
    for its partial results, from the launch stream's pool of torch's allocator as workspace_on's.
    Under a capture that torch does not know of, whose replays would find that workspace given
    to others, it runs without one."""
    handle = _stream(stream)
    args = (REDUCE_OPS[op], x.data_ptr(), out.data_ptr(), rows, cols, dim, count)
    nbytes = 0
    if dim != 1 and rows * cols >= _REDUCE_SPLIT_MIN:
        nbytes = _native.load_library().asc_reduce_f32_workspace(rows, cols, dim)
    if nbytes == 0:
        _native.call("asc_reduce_f32", *args, handle)
        return
    if handle == _native.current_stream_handle(x.device.index):
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        usable = not torch.cuda.is_current_stream_capturing() or _held_by_a_graph(workspace)
    else:
        with torch.cuda.stream(_stream_of(handle, x.device)):
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
            usable = not torch.cuda.is_current_stream_capturing() or _held_by_a_graph(workspace)
    if usable:
        _native.call("asc_reduce_f32_ws", *args, workspace.data_ptr(), nbytes, handle)
    else:
        _native.call("asc_reduce_f32", *args, handle)


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, out: torch.Tensor, num_rows: int, num_cols: int,
             epsilon: float, tile_size: Optional[int] = None, stream: Any = None) -> None:
    """asc2.rms_norm over the first ``tile_size`` (default: all) columns of each row:
    y = x / sqrt(mean(x^2) + epsilon) * gamma, fp32 or fp16 rows, fp32 gamma."""
    tile = num_cols if tile_size is None else int(tile_size)
    if num_rows < 0 or num_cols < 0 or not 0 < tile <= num_cols:
        raise ValueError(f"invalid rms_norm launch: rows={num_rows}, cols={num_cols}, tile={tile}")
    for t, n in ((x, "x"), (out, "out")):
        _contiguous(_device_tensor(t, n), n)
        if t.numel() < num_rows * num_cols:
            raise ValueError(f"'{n}' holds {t.numel()} elements but the launch touches {num_rows}x{num_cols}")
    code = _code(x, "x", (torch.float32, torch.float16))
    if out.dtype != x.dtype:
        raise TypeError(f"out must be {x.dtype}, got {out.dtype}")
    _contiguous(_device_tensor(gamma, "gamma"), "gamma")
    if gamma.dtype != torch.float32 or gamma.numel() < tile:
        raise ValueError(f"gamma must be float32 with at least {tile} elements")
    _native.call("asc_rms_norm", code, x.data_ptr(), gamma.data_ptr(), out.data_ptr(), num_rows, num_cols, tile,
                 float(epsilon), _stream(stream))


# -------------------------------------------------------------------------------------------- matmul

def _row_major_2d(t: torch.Tensor, name: str) -> int:
    """Leading dimension of a 2-D row-major (unit inner stride) tensor.  Rows must not
    overlap: a row stride below the row length (an expanded or as_strided view) would
    make the kernel read or write past the tensor's storage, and is refused."""
    if t.dim() != 2:
        raise ValueError(f"'{name}' must be 2-D, got shape {tuple(t.shape)}")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"'{name}' must have unit stride along its last dimension")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"'{name}' has row stride {t.stride(0)} below its row length {t.shape[1]}: "
                         "overlapping or expanded rows are not supported")
    return max(t.stride(0), t.shape[1], 1)


ACT_NONE, ACT_RELU, ACT_LEAKY_RELU = 0, 1, 2


def _matmul_args(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, relu: bool, bias: Optional[torch.Tensor],
                 leaky_alpha: Optional[float]) -> tuple:
    """Checks a matmul and returns the C arguments of asc_matmul_bias_act (and of
    asc_matmul_plan) without the stream: in/out dtype codes, pointers, M, N, K, the leading
    dimensions, the activation code and alpha."""
    for t, n in ((a, "a"), (b, "b"), (c, "c")):
        _device_tensor(t, n)
    in_code = _code(a, "a", (torch.float32, torch.float16, torch.bfloat16))
    if b.dtype != a.dtype:
        raise TypeError(f"a and b must share a dtype, got {a.dtype} and {b.dtype}")
    out_code = _code(c, "c", (torch.float32, torch.float16, torch.bfloat16))
    lda, ldb, ldc = _row_major_2d(a, "a"), _row_major_2d(b, "b"), _row_major_2d(c, "c")
    M, K = a.shape
    K2, N = b.shape
    if K2 != K:
        raise ValueError(f"inner dimensions differ: a is {tuple(a.shape)}, b is {tuple(b.shape)}")
    if tuple(c.shape) != (M, N):
        raise ValueError(f"c must be {(M, N)}, got {tuple(c.shape)}")
    if relu and leaky_alpha is not None:
        raise ValueError("relu and leaky_alpha are exclusive")
    bias_ptr = 0
    if bias is not None:
        _contiguous(_device_tensor(bias, "bias"), "bias")
        if bias.dtype != torch.float32 or bias.numel() != N:
            raise ValueError(f"bias must be float32 with {N} elements, got {bias.dtype} with {bias.numel()}")
        bias_ptr = bias.data_ptr()
    act = ACT_LEAKY_RELU if leaky_alpha is not None else (ACT_RELU if relu else ACT_NONE)
    return (in_code, out_code, a.data_ptr(), b.data_ptr(), c.data_ptr(), bias_ptr, M, N, K, lda, ldb, ldc, act,
            float(leaky_alpha or 0.0))


def matmul(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, relu: bool = False, stream: Any = None,
           bias: Optional[torch.Tensor] = None, leaky_alpha: Optional[float] = None) -> None:
    """c = cast(act(a @ b + bias)) with fp32 accumulation; the cast is chosen by c's dtype
    (float32: no cast; float16/bfloat16: RNE).  ``bias``: float32 with N elements (added
    per column), ``relu``: max(v, 0), ``leaky_alpha``: v >= 0 ? v : v * alpha (excludes relu)."""
    args = _matmul_args(a, b, c, relu, bias, leaky_alpha)
    if bias is None and leaky_alpha is None:
        in_code, out_code, ap, bp, cp, _, M, N, K, lda, ldb, ldc, _, _ = args
        _native.call("asc_matmul", in_code, out_code, ap, bp, cp, M, N, K, lda, ldb, ldc, int(bool(relu)),
                     _stream(stream))
        return
    _native.call("asc_matmul_bias_act", *args, _stream(stream))


def matmul_chained(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, workspace: Optional[torch.Tensor] = None,
                   stream: Any = None) -> None:
    """The asc2 chained matmul (python/test/asc2/kernels/test_matmul_l0c_to_l1.py:17-30):
    t = (a @ b) cast to a's dtype, c = cast(t @ b) to c's dtype, fp32 accumulation, N == K.
    ``workspace`` (a contiguous device tensor of at least M * N * 2 bytes) holds t; without
    one it is taken from the launch stream's pool of torch's allocator."""
    for t, n in ((a, "a"), (b, "b"), (c, "c")):
        _contiguous(_device_tensor(t, n), n)
    in_code = _code(a, "a", (torch.float16, torch.bfloat16))
    if b.dtype != a.dtype:
        raise TypeError(f"a and b must share a dtype, got {a.dtype} and {b.dtype}")
    out_code = _code(c, "c", (torch.float32, torch.float16, torch.bfloat16))
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError(f"a and b must be 2-D, got {tuple(a.shape)} and {tuple(b.shape)}")
    M, K = a.shape
    K2, N = b.shape
    if K2 != K or N != K:
        raise ValueError(f"the chained matmul needs b square and a's columns equal to its rows: a {tuple(a.shape)}, "
                         f"b {tuple(b.shape)}")
    if tuple(c.shape) != (M, N):
        raise ValueError(f"c must be {(M, N)}, got {tuple(c.shape)}")
    handle = _stream(stream)
    if workspace is None:
        workspace = workspace_on(handle, M * N, a.dtype, a.device)
    else:
        _contiguous(_device_tensor(workspace, "workspace"), "workspace")
    nbytes = workspace.numel() * workspace.element_size()
    _native.call("asc_matmul_chained", in_code, out_code, a.data_ptr(), b.data_ptr(), c.data_ptr(), M, N, K,
                 workspace.data_ptr(), nbytes, handle)


def matmul_plan(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, relu: bool = False,
                bias: Optional[torch.Tensor] = None, leaky_alpha: Optional[float] = None) -> "_native.LaunchPlan":
    """A launch of matmul(...)'s product by the kernel of its type on 256x256 tiles (fp32: 16x16
    blocks or 64x64 tiles), as a kernel of the asc2_matmul code object with its grid, block and
    argument blob (asc_matmul_plan); plan.grid == 0 when there is nothing to launch.  Same
    checks and errors as matmul."""
    plan = _native.LaunchPlan()
    _native.call("asc_matmul_plan", *_matmul_args(a, b, c, relu, bias, leaky_alpha), ctypes.byref(plan))
    return plan


def matmul_dispatch(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, relu: bool = False,
                    bias: Optional[torch.Tensor] = None, leaky_alpha: Optional[float] = None) -> "_native.LaunchPlan":
    """The launch matmul(...) makes (asc_matmul_dispatch), in matmul_plan's form."""
    plan = _native.LaunchPlan()
    _native.call("asc_matmul_dispatch", *_matmul_args(a, b, c, relu, bias, leaky_alpha), ctypes.byref(plan))
    return plan


def _matmul_i8_args(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, scale: Optional[torch.Tensor],
                    trunc19: bool) -> tuple:
    """Checks an int8 matmul and returns the C arguments of asc_matmul_i8_plan: pointers
    a, b, scale (0 for int32 output), c, then M, N, K, the dequant flag and trunc19."""
    for t, n in ((a, "a"), (b, "b"), (c, "c")):
        _contiguous(_device_tensor(t, n), n)
    _code(a, "a", (torch.int8,))
    _code(b, "b", (torch.int8,))
    if a.dim() != 2 or b.dim() != 2 or c.dim() != 2:
        raise ValueError("a, b and c must be 2-D")
    M, K = a.shape
    K2, N = b.shape
    if K2 != K or tuple(c.shape) != (M, N):
        raise ValueError(f"shape mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}, c {tuple(c.shape)}")
    if c.dtype == torch.int32:
        return (a.data_ptr(), b.data_ptr(), 0, c.data_ptr(), M, N, K, 0, 0)
    if c.dtype != torch.float16:
        raise TypeError(f"c must be int32 (accumulators) or float16 (dequantised), got {c.dtype}")
    if scale is None:
        raise ValueError("a float16 output needs the per-channel scale vector")
    _contiguous(_device_tensor(scale, "scale"), "scale")
    if scale.dtype != torch.float32 or scale.numel() != N:
        raise ValueError(f"scale must be float32 with {N} elements, got {scale.dtype} with {scale.numel()}")
    return (a.data_ptr(), b.data_ptr(), scale.data_ptr(), c.data_ptr(), M, N, K, 1, int(bool(trunc19)))


def matmul_i8(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, scale: Optional[torch.Tensor] = None,
              trunc19: bool = False, stream: Any = None) -> None:
    """int8 GEMM with exact int32 accumulation.  c int32: raw accumulators.  c float16:
    c = fp16(fp32(acc) * scale[n]) (scale required, fp32 of length N)."""
    ap, bp, sp, cp, M, N, K, dequant, t19 = _matmul_i8_args(a, b, c, scale, trunc19)
    if not dequant:
        _native.call("asc_matmul_i8_i32", ap, bp, cp, M, N, K, _stream(stream))
        return
    _native.call("asc_matmul_i8_dequant_f16", ap, bp, sp, cp, M, N, K, t19, _stream(stream))


def matmul_i8_plan(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, scale: Optional[torch.Tensor] = None,
                   trunc19: bool = False) -> "_native.LaunchPlan":
    """A launch of matmul_i8(...)'s product on 256x256 tiles, as a kernel of the asc2_matmul_i8
    code object with its grid, block and argument blob (asc_matmul_i8_plan).  Same checks as
    matmul_i8."""
    plan = _native.LaunchPlan()
    _native.call("asc_matmul_i8_plan", *_matmul_i8_args(a, b, c, scale, trunc19), ctypes.byref(plan))
    return plan


def matmul_i8_dispatch(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, scale: Optional[torch.Tensor] = None,
                       trunc19: bool = False) -> "_native.LaunchPlan":
    """The launch matmul_i8(...) makes (asc_matmul_i8_dispatch), in matmul_i8_plan's form."""
    plan = _native.LaunchPlan()
    _native.call("asc_matmul_i8_dispatch", *_matmul_i8_args(a, b, c, scale, trunc19), ctypes.byref(plan))
    return plan


# --------------------------------------------------------------------------------------- attention

FA_HEAD_DIMS = (64, 128)


def _attention_args(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, sm_scale: float,
                    causal: bool, lse: Optional[torch.Tensor]) -> tuple:
    """Checks an attention call and returns the C arguments of
    asc_flash_attention_fwd_bf16 without the stream."""
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (o, "o")):
        _contiguous(_device_tensor(t, n), n)
        if t.dtype != torch.bfloat16:
            raise TypeError(f"'{n}' must be bfloat16, got {t.dtype}")
        if t.dim() != 4 or tuple(t.shape) != tuple(q.shape):
            raise ValueError(f"'{n}' must be [batch, heads, seq_len, head_dim] like q {tuple(q.shape)}")
    batch, heads, seq_len, head_dim = q.shape
    if not sm_scale > 0:
        raise ValueError(f"sm_scale must be positive, got {sm_scale}")
    if head_dim not in FA_HEAD_DIMS:
        raise ValueError(f"head_dim {head_dim} not supported (supported: {FA_HEAD_DIMS})")
    lse_ptr = 0
    if lse is not None:
        _contiguous(_device_tensor(lse, "lse"), "lse")
        if lse.dtype != torch.float32 or lse.numel() != batch * heads * seq_len:
            raise ValueError("lse must be float32 [batch, heads, seq_len]")
        lse_ptr = lse.data_ptr()
    return (q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse_ptr, batch, heads, seq_len, head_dim,
            float(sm_scale), int(bool(causal)))


def flash_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, sm_scale: float,
                        causal: bool, lse: Optional[torch.Tensor] = None, stream: Any = None) -> None:
    """o = softmax(q k^T * sm_scale + causal mask) v for bf16 [batch, heads, seq, head_dim]."""
    _native.call("asc_flash_attention_fwd_bf16", *_attention_args(q, k, v, o, sm_scale, causal, lse),
                 _stream(stream))


def flash_attention_plan(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, sm_scale: float,
                         causal: bool, lse: Optional[torch.Tensor] = None) -> "_native.LaunchPlan":
    """A launch of flash_attention_fwd(...) without a split of the keys, as a kernel of the
    asc2_flash_attention code object with its grid, block and argument blob
    (asc_flash_attention_plan)."""
    plan = _native.LaunchPlan()
    _native.call("asc_flash_attention_plan", *_attention_args(q, k, v, o, sm_scale, causal, lse),
                 ctypes.byref(plan))
    return plan


def flash_attention_dispatch(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, sm_scale: float,
                             causal: bool, lse: Optional[torch.Tensor] = None) -> "_native.LaunchPlan":
    """The launch flash_attention_fwd(...) makes (asc_flash_attention_dispatch), in
    flash_attention_plan's form."""
    plan = _native.LaunchPlan()
    _native.call("asc_flash_attention_dispatch", *_attention_args(q, k, v, o, sm_scale, causal, lse),
                 ctypes.byref(plan))
    return plan


# ------------------------------------------------------------------- rotary positions, q/k norms

ROTARY_SCALINGS = (None, "linear", "ntk", "yarn")
MAX_ROTARY_HEAD_DIM = 512
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


_NO_ROWS = (0, 0, 0, 0)


def _current_device() -> int:
    c = _native._torch_c
    return torch.cuda.current_device() if c is None else c._cuda_getDevice()


def _here(t: torch.Tensor, name: str, device: int) -> torch.Tensor:
    """A tensor of the current device, the one that launches go to."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        _device_tensor(t, name)
        raise ValueError(f"'{name}' is on {t.device}, but the current device is cuda:{device}")
    return t


def _apart(t: torch.Tensor, name: str) -> None:
    """Refuses a tensor to write to whose elements may share a place."""
    shape, strides = t.shape, t.stride()
    if len(shape) == 4 and strides[3] == 1:  # [batch, rows, heads, head_dim] seen as [batch, heads, rows, head_dim]
        s0, s1, s2, _ = strides
        if s1 >= shape[3] and s2 >= s1 * shape[1] and s0 >= s2 * shape[2]:
            return
    span = 0  # of the dimensions so far, from the innermost
    for stride, size in sorted([x for x in zip(strides, shape) if x[1] > 1]):
        if stride <= span:
            raise ValueError(f"'{name}' is written but its elements overlap (strides {t.stride()})")
        span += stride * (size - 1)


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, device: int, shape: Optional[tuple] = None,
          written: bool = False, aligned: bool = False) -> tuple:
    """A [batch, heads, seq, head_dim] operand whose last dimension is contiguous as asc_rows_t's
    fields; ``aligned``: with rows that can be read and written 16 bytes at a time (16-bit elements)."""
    try:
        if t.get_device() != device:
            _here(t, name, device)
        size = t.shape
        if (size != shape if shape is not None else len(size) != 4):
            raise ValueError(f"'{name}' must be {list(shape) if shape else '[batch, heads, seq, head_dim]'}, "
                             f"got {tuple(size)}")
        s0, s1, s2, s3 = t.stride()
        at = t.data_ptr()
    except AttributeError:
        _device_tensor(t, name)  # says what it is instead of a tensor
        raise
    if t.dtype is not dtype:
        raise TypeError(f"'{name}' must be {dtype}, got {t.dtype}")
    if s3 != 1 and size[3] > 1:
        raise ValueError(f"the last dimension of '{name}' must be contiguous")
    if written and not t.is_contiguous():
        _apart(t, name)
    if aligned and (at | (s0 | s1 | s2) << 1) & 15:
        # a dimension of one element is not stepped over, whatever its stride
        s0, s1, s2 = (s if n > 1 else 0 for s, n in zip((s0, s1, s2), size))
        if (at | (s0 | s1 | s2) << 1) & 15:
            raise ValueError(f"'{name}' must be 16-byte aligned, with strides that are multiples of 8 elements "
                             f"(address {at:#x}, strides {t.stride()})")
    return at, s0, s1, s2


def _vector(t: torch.Tensor, name: str, dtype: torch.dtype, device: int, shape: tuple) -> int:
    """The address of a contiguous tensor of this type and shape."""
    _here(t, name, device)
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"'{name}' must be a contiguous {dtype} {list(shape)}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _launch(entry: str, *args: Any) -> None:
    """Calls an entry; what is left for it to refuse of a call's arguments is an error of their values."""
    code = getattr(_native._lib or _native.load_library(), entry)(*args)
    if code == _native.ERR_INVALID_ARG:
        raise ValueError(_native.last_error())
    if code != 0:
        _native.check(code, entry)


def _with_workspace(entry: str, args: bytes, device: torch.device, stream: Any) -> None:
    """Calls an entry with the workspace that it asks for, from the launch stream's pool as
    workspace_on's.  Under a capture that torch does not know of the workspace would go to others
    before the replays: refused."""
    handle = _stream(stream)
    nbytes = getattr(_native.load_library(), entry + "_workspace")(args)
    if nbytes == 0:
        _launch(entry, args, 0, 0, handle)
        return
    if handle == _native.current_stream_handle(device.index):
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        usable = not torch.cuda.is_current_stream_capturing() or _held_by_a_graph(workspace)
    else:
        with torch.cuda.stream(_stream_of(handle, device)):
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
            usable = not torch.cuda.is_current_stream_capturing() or _held_by_a_graph(workspace)
    if not usable:
        raise RuntimeError(f"{entry} needs a workspace: capture it with torch.cuda.graph")
    _launch(entry, args, workspace.data_ptr(), nbytes, handle)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, device: Any = None) -> tuple:
    """The angle per position of each of the rotary_dim / 2 pairs (float64, on ``device``, default
    the current one), base^(-2 i / rotary_dim), and the factor on the rotated values
    (``magnitude`` of rotary and qk_norm_rotary).  ``scaling`` extends a context of
    ``original_length`` tokens ``factor`` times:

    - "linear": every frequency divided by the factor;
    - "ntk": a larger base, base * factor^(rotary_dim / (rotary_dim - 2)), which leaves the first
      pair as it is and divides the last one's frequency by the factor;
    - "yarn": pairs that turn at least 32 times in the original length keep their frequency, those
      that turn less than once are divided by the factor, in between linearly in the number of
      turns; the magnitude is 0.1 ln(factor) + 1 (Peng et al., arXiv:2309.00071, sections 3.2-3.4).
      Parity with a trained model's own frequencies is unpinned: programs that ramp over the
      pairs' numbers between two rounded ends get others, and ``freqs`` can be theirs."""
    rotary_dim = int(rotary_dim)
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}; expected one of {ROTARY_SCALINGS}")
    if not base > 0 or not factor > 0:
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freqs = base ** (torch.arange(rotary_dim // 2, dtype=torch.float64) * (-2.0 / rotary_dim))
    magnitude = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        if original_length is None or original_length <= 0:
            raise ValueError("yarn scaling needs the original_length")
        turns = freqs * (original_length / (2 * math.pi))
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        freqs = freqs * keep + freqs / factor * (1.0 - keep)
        if factor > 1:
            magnitude = 0.1 * math.log(factor) + 1.0
    return freqs.to("cuda" if device is None else device), magnitude


_ROTARY = struct.Struct("@6i2f4q" + "P3q" * 6 + "P2q5P")  # asc_rotary_t


def _rotary_args(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor,
                 q_out: torch.Tensor, k_out: Optional[torch.Tensor], interleaved: bool, magnitude: float,
                 device: int, backward: bool = False, epsilon: float = 0.0, weights: Optional[tuple] = None,
                 grads: Optional[tuple] = None) -> bytes:
    """Checks the arguments of a rotary call and returns them as an asc_rotary_t.  ``weights``: those
    of q and k; ``grads``: the gradients of the results, and of the weights."""
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"'q' must be a torch.Tensor, got {type(q).__name__}")
    dtype = q.dtype
    if dtype not in _FLOATS:
        raise TypeError(f"'q' has unsupported dtype {dtype}; expected one of {sorted(map(str, _FLOATS))}")
    q_rows = _rows(q, "q", dtype, device)
    shape = q.shape
    batch, heads, seq, head_dim = shape
    if head_dim % 2 or not 0 < head_dim <= MAX_ROTARY_HEAD_DIM:
        raise ValueError(f"head_dim {head_dim} not supported (even, at most {MAX_ROTARY_HEAD_DIM})")
    qo_rows = _rows(q_out, "q_out", dtype, device, shape, True)
    k_rows = ko_rows = dq_rows = dk_rows = _NO_ROWS
    k_heads, w_q, w_k, dw_q, dw_k = 0, 0, 0, 0, 0
    if (k is None) != (k_out is None):
        raise ValueError("k and its result must be given together")
    if k is not None:
        k_rows = _rows(k, "k", dtype, device)
        k_shape = k.shape
        k_heads = k_shape[1]
        if k_shape != (batch, k_heads, seq, head_dim):
            raise ValueError(f"'k' must be {[batch, k_heads, seq, head_dim]}, got {tuple(k_shape)}")
        ko_rows = _rows(k_out, "k_out", dtype, device, k_shape, True)
    if weights is not None:
        if not epsilon >= 0:
            raise ValueError(f"epsilon must not be negative, got {epsilon}")
        w_q = _head_weight(weights[0], "q_weight", head_dim, device)
        if k is not None:
            w_k = _head_weight(weights[1], "k_weight", head_dim, device)
    if grads is not None:
        dq_rows = _rows(grads[0], "dq_out", dtype, device, shape)
        dw_q = _head_weight(grads[2], "dq_weight", head_dim, device)
        if k is not None:
            if grads[1] is None:
                raise ValueError("dk_out must be given with k")
            dk_rows = _rows(grads[1], "dk_out", dtype, device, k_shape)
            dw_k = _head_weight(grads[3], "dk_weight", head_dim, device)
    at_q, at_k = qo_rows[0], ko_rows[0]
    if (((at_q == q_rows[0] and qo_rows != q_rows) or (at_q == dq_rows[0] and qo_rows != dq_rows)) and q.numel() or
            ((at_k == k_rows[0] and ko_rows != k_rows) or (at_k == dk_rows[0] and ko_rows != dk_rows)) and k.numel()):
        raise ValueError("a result in place of its input must have the input's strides")
    if at_q and at_k and (at_q in (at_k, k_rows[0], dk_rows[0]) or at_k in (q_rows[0], dq_rows[0])):
        raise ValueError("a result of q must not lie in place of k's tensors, nor k's of q's")
    _here(positions, "positions", device)
    positions_dtype, positions_shape = positions.dtype, positions.shape
    if positions_dtype is not torch.int64 and positions_dtype is not torch.int32:
        raise TypeError(f"positions must be int32 or int64, got {positions_dtype}")
    if positions_shape == (batch, seq):
        batch_step, step = positions.stride()
    elif positions_shape == (seq,):
        batch_step, step = 0, positions.stride(0)
    else:
        raise ValueError(f"positions must be [seq] or [batch, seq] = {(batch, seq)}, got {tuple(positions_shape)}")
    _here(freqs, "freqs", device)
    pairs = freqs.numel()
    if freqs.dtype is not torch.float64 or freqs.dim() != 1 or 2 * pairs > head_dim or not freqs.is_contiguous():
        raise ValueError(f"'freqs' must be a contiguous float64 vector of at most {head_dim // 2} elements")
    return _ROTARY.pack(_DTYPE_CODES[dtype], head_dim, 2 * pairs, bool(interleaved), bool(backward),
                        positions_dtype is torch.int64, magnitude, epsilon, batch, heads, k_heads, seq, *q_rows,
                        *k_rows, *qo_rows, *ko_rows, *dq_rows, *dk_rows, positions.data_ptr(), batch_step, step,
                        freqs.data_ptr(), w_q, w_k, dw_q, dw_k)


def _head_weight(w: torch.Tensor, name: str, head_dim: int, device: int) -> int:
    return _vector(w, name, torch.float32, device, (head_dim,))


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor,
           q_out: torch.Tensor, k_out: Optional[torch.Tensor], interleaved: bool = False, magnitude: float = 1.0,
           backward: bool = False, stream: Any = None) -> None:
    """Rotary positions of queries and keys ([batch, heads, seq, head_dim] of any strides, k with
    its own number of heads or None) in one launch: pair i of the first 2 * len(freqs) columns,
    (i, i + len(freqs)) or, ``interleaved``, (2 i, 2 i + 1), turns by positions * freqs[i] and is
    multiplied by ``magnitude``; the other columns are copied.  ``backward`` gives the gradient:
    the turn the other way.  A result may lie in place of its input."""
    device = _current_device()
    _launch("asc_rotary", _rotary_args(q, k, positions, freqs, q_out, k_out, interleaved, magnitude, device, backward),
            _stream(stream))


def qk_norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor], q_weight: torch.Tensor,
                   k_weight: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor,
                   q_out: torch.Tensor, k_out: Optional[torch.Tensor], epsilon: float, interleaved: bool = False,
                   magnitude: float = 1.0, stream: Any = None) -> None:
    """rotary after an RMS norm of each head: x / sqrt(mean(x^2) + epsilon) * weight, the weights
    float32 [head_dim]."""
    device = _current_device()
    _launch("asc_qk_norm_rotary", _rotary_args(q, k, positions, freqs, q_out, k_out, interleaved, magnitude, device, False,
                                               epsilon, (q_weight, k_weight)), _stream(stream))


def qk_norm_rotary_bwd(dq_out: torch.Tensor, dk_out: Optional[torch.Tensor], q: torch.Tensor,
                       k: Optional[torch.Tensor], q_weight: torch.Tensor, k_weight: Optional[torch.Tensor],
                       positions: torch.Tensor, freqs: torch.Tensor, dq: torch.Tensor, dk: Optional[torch.Tensor],
                       dq_weight: torch.Tensor, dk_weight: Optional[torch.Tensor], epsilon: float,
                       interleaved: bool = False, magnitude: float = 1.0, stream: Any = None) -> None:
    """The gradient of qk_norm_rotary: from the results' gradients and its inputs, the gradients
    of q and k (dq may lie in place of dq_out or q) and of the weights (float32 [head_dim], summed
    over all rows in a fixed order, in float32 over a workgroup's rows and float64 over workgroups).
    A weight that q and k share has two gradients, to be added: one place for both is refused."""
    device = _current_device()
    args = _rotary_args(q, k, positions, freqs, dq, dk, interleaved, magnitude, device, False, epsilon,
                        (q_weight, k_weight), (dq_out, dk_out, dq_weight, dk_weight))
    _with_workspace("asc_qk_norm_rotary_bwd", args, q.device, stream)


# ------------------------------------------------- attention over other keys than the queries' own

_HALVES = (torch.float16, torch.bfloat16)


_ATTENTION = struct.Struct("@iifi6q" + "P3q" * 6 + "4PqP2q" + "P3q" * 4)  # asc_attention_t
_NO_GRADS = _NO_ROWS * 4
_NO_TREE = (0, 0, 0, 0, 0, 0)  # draft_lengths, block_table and its stride, tree_mask and its strides


def _kv_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, sm_scale: float, device: int,
             names: tuple, pages: bool = False, written: bool = True) -> tuple:
    """Checks queries, keys, values and o, a result where it is ``written``, and returns their rows;
    ``pages``: the first dimension of k is not the batch's."""
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"'q' must be a torch.Tensor, got {type(q).__name__}")
    dtype = q.dtype
    if dtype not in _HALVES:
        raise TypeError(f"'q' has unsupported dtype {dtype}; expected one of {sorted(map(str, _HALVES))}")
    q_rows = _rows(q, "q", dtype, device, None, False, True)
    shape = q.shape
    if shape[3] not in FA_HEAD_DIMS:
        raise ValueError(f"head_dim {shape[3]} not supported (supported: {FA_HEAD_DIMS})")
    o_rows = _rows(o, "o", dtype, device, shape, written, True)
    k_rows = _rows(k, names[0], dtype, device, None, False, True)
    k_shape = k.shape
    if k_shape[3] != shape[3] or (k_shape[0] != shape[0] and not pages):
        raise ValueError(f"'{names[0]}' {tuple(k_shape)} does not fit q {tuple(shape)}")
    v_rows = _rows(v, names[1], dtype, device, k_shape, False, True)
    if written and o_rows[0] in (q_rows[0], k_rows[0], v_rows[0]) and o_rows[0]:
        raise ValueError("'o' must not lie in place of an input")
    if k_shape[1] == 0 or shape[1] % k_shape[1]:
        raise ValueError(f"{shape[1]} query heads cannot share {k_shape[1]} key / value heads")
    if not 0 < sm_scale < math.inf:
        raise ValueError(f"sm_scale must be positive and finite, got {sm_scale}")
    return q_rows, o_rows, k_rows, v_rows


def cross_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, sm_scale: float,
                        kv_lengths: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                        stream: Any = None) -> None:
    """o = softmax(q k^T * sm_scale) v for float16 or bfloat16 queries [batch, heads, q_len, head_dim]
    over keys and values [batch, kv_heads, kv_len, head_dim] (an encoder's states: any length, heads
    a multiple of kv_heads, head_dim 64 or 128), all of any strides that are multiples of 8 elements
    with a contiguous last dimension.  ``kv_lengths`` (int32 [batch]): the keys of each sequence;
    what lies behind them is not read.  A sequence without keys gets zeros.  ``lse`` (float32
    [batch, heads, q_len]) receives the log-sum-exp, -inf without keys.  A length outside
    [0, kv_len] is not followed: its sequence's results are NaN."""
    device = _current_device()
    q_rows, o_rows, k_rows, v_rows = _kv_rows(q, k, v, o, sm_scale, device, ("k", "v"))
    batch, heads, q_len, head_dim = q.shape
    lse_at = 0 if lse is None else _vector(lse, "lse", torch.float32, device, (batch, heads, q_len))
    lengths = 0 if kv_lengths is None else _vector(kv_lengths, "kv_lengths", torch.int32, device, (batch,))
    args = _ATTENTION.pack(_DTYPE_CODES[q.dtype], head_dim, sm_scale, 0, batch, heads, k.shape[1], q_len, k.shape[2],
                           0, *q_rows, *o_rows, *k_rows, *v_rows, *_NO_ROWS, *_NO_ROWS, lse_at, lengths, *_NO_TREE,
                           *_NO_GRADS)
    _with_workspace("asc_cross_attention_fwd", args, q.device, stream)


def cross_attention_bwd(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                        lse: torch.Tensor, dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, sm_scale: float,
                        kv_lengths: Optional[torch.Tensor] = None, stream: Any = None) -> None:
    """The gradients of cross_attention_fwd: from the gradient ``do`` of o, its inputs and its o and
    lse, the gradients of q, k and v.  dk and dv are summed over the query heads that share a key /
    value head, in a fixed order, and are zeros behind a sequence's keys.  The probabilities and the
    scores' gradients are rounded to the inputs' type for their products: to its precision, whatever
    their size (in float16 they are held at powers of two that move with the largest of a row or key),
    but the gradients themselves end at the type's smallest value.  Above 192 keys the row sums of
    do * o are of the rounded o: rows that give few of many keys most of their probability have dq
    and dk off by up to three times a rounding."""
    device = _current_device()
    q_rows, o_rows, k_rows, v_rows = _kv_rows(q, k, v, o, sm_scale, device, ("k", "v"), written=False)
    dtype, shape = q.dtype, q.shape
    batch, heads, q_len, head_dim = shape
    lse_at = _vector(lse, "lse", torch.float32, device, (batch, heads, q_len))
    lengths = 0 if kv_lengths is None else _vector(kv_lengths, "kv_lengths", torch.int32, device, (batch,))
    do_rows = _rows(do, "do", dtype, device, shape, False, True)
    taken = [do_rows[0], q_rows[0], k_rows[0], v_rows[0], o_rows[0]]
    grads = ()
    for name, t, like in (("dq", dq, shape), ("dk", dk, k.shape), ("dv", dv, k.shape)):
        rows = _rows(t, name, dtype, device, like, True, True)
        if rows[0] in taken and t.numel():
            raise ValueError(f"'{name}' must not lie in place of an input or of another result")
        taken.append(rows[0])
        grads += rows
    args = _ATTENTION.pack(_DTYPE_CODES[dtype], head_dim, sm_scale, 0, batch, heads, k.shape[1], q_len, k.shape[2], 0,
                           *q_rows, *o_rows, *k_rows, *v_rows, *_NO_ROWS, *_NO_ROWS, lse_at, lengths, *_NO_TREE,
                           *do_rows, *grads)
    _with_workspace("asc_cross_attention_bwd", args, q.device, stream)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cache_lengths: torch.Tensor,
                   k_draft: torch.Tensor, v_draft: torch.Tensor, tree_mask: Optional[torch.Tensor],
                   o: torch.Tensor, sm_scale: float, block_table: Optional[torch.Tensor] = None,
                   draft_lengths: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                   stream: Any = None) -> None:
    """Attention of a tree of drafted tokens (a single one: plain decoding) over a cache and
    themselves: o = softmax(s) v with s = q k^T * sm_scale over the cached keys and the drafted ones
    that the mask names, for float16 or bfloat16 q [batch, heads, n, head_dim].

    - k_cache, v_cache: [batch, kv_heads, length, head_dim], or with ``block_table`` (int32
      [batch, pages of a sequence]) [pages, kv_heads, page size, head_dim]: key j of sequence b
      lies in page block_table[b, j // page_size], row j % page_size.  cache_lengths (int32
      [batch]): the cached keys, all of which every token attends.
    - k_draft, v_draft: [batch, kv_heads, n, head_dim], not in the cache yet.  tree_mask (bool
      [n, n] or [batch, n, n]): whether token i attends token j (its ancestors and itself); None: a
      chain, j <= i.  draft_lengths (int32 [batch]): tokens of each sequence, default n; the rows of
      o and lse behind them are left as they were, all of them where the number is negative.

    Strides and the last dimension as in cross_attention_fwd.  A token that attends nothing gets zeros
    and an lse of -inf.  A length outside the cache, a page outside it that a length reaches, or a
    number of drafted tokens above n is not followed: the sequence's results are NaN."""
    device = _current_device()
    q_rows, o_rows, k_rows, v_rows = _kv_rows(q, k_cache, v_cache, o, sm_scale, device, ("k_cache", "v_cache"),
                                              pages=block_table is not None)
    dtype = q.dtype
    batch, heads, n, head_dim = q.shape
    pages, kv_heads, kv_len, _ = k_cache.shape
    lse_at = 0 if lse is None else _vector(lse, "lse", torch.float32, device, (batch, heads, n))
    lengths = _vector(cache_lengths, "cache_lengths", torch.int32, device, (batch,))
    drafted = 0 if draft_lengths is None else _vector(draft_lengths, "draft_lengths", torch.int32, device, (batch,))
    shape = (batch, kv_heads, n, head_dim)
    kd_rows = _rows(k_draft, "k_draft", dtype, device, shape, False, True)
    vd_rows = _rows(v_draft, "v_draft", dtype, device, shape, False, True)
    if o_rows[0] in (kd_rows[0], vd_rows[0]) and o_rows[0]:
        raise ValueError("'o' must not lie in place of an input")
    page_size, table, table_stride = 0, 0, 0
    if block_table is not None:
        _here(block_table, "block_table", device)
        size = block_table.shape
        if block_table.dtype is not torch.int32 or len(size) != 2 or size[0] != batch:
            raise ValueError(f"'block_table' must be int32 [batch, pages], got {block_table.dtype} {tuple(size)}")
        table_stride, step = block_table.stride()
        if step != 1 and size[1] > 1:
            raise ValueError("the last dimension of 'block_table' must be contiguous")
        page_size, kv_len = kv_len, size[1] * kv_len
        if pages == 0 and kv_len:
            raise ValueError("a cache without pages needs a block_table without columns")
        table = block_table.data_ptr()
    mask, mask_batch, mask_row = 0, 0, 0
    if tree_mask is not None:
        _here(tree_mask, "tree_mask", device)
        size = tree_mask.shape
        if tree_mask.dtype is not torch.bool or (size != (batch, n, n) and size != (n, n)):
            raise ValueError(f"'tree_mask' must be bool [{n}, {n}] or [{batch}, {n}, {n}], got {tree_mask.dtype} "
                             f"{tuple(size)}")
        *outer, mask_row, step = tree_mask.stride()
        if step != 1 and n > 1:
            raise ValueError("the last dimension of 'tree_mask' must be contiguous")
        mask, mask_batch = tree_mask.data_ptr(), outer[0] if outer else 0
    args = _ATTENTION.pack(_DTYPE_CODES[dtype], head_dim, sm_scale, page_size, batch, heads, kv_heads, n, kv_len, pages,
                           *q_rows, *o_rows, *k_rows, *v_rows, *kd_rows, *vd_rows, lse_at, lengths, drafted, table,
                           table_stride, mask, mask_batch, mask_row, *_NO_GRADS)
    _with_workspace("asc_tree_attention", args, q.device, stream)


# -------------------------------------------------------------------------- a cache held in 8 bits

_CACHE_CODES = {torch.int8: _native.DT_INT8, torch.float8_e4m3fn: _native.DT_FLOAT8_E4M3}
_CACHE8 = struct.Struct("@6if6q" + "P3q" * 8 + "4Pq")  # asc_cache8_t


def _strided(t: torch.Tensor, name: str, device: int, dims: int, written: bool) -> tuple:
    """Address, strides and shape of a tensor of this device with so many dimensions."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        _here(t, name, device)
    shape = t.shape
    if len(shape) != dims:
        raise ValueError(f"'{name}' must have {dims} dimensions, got {tuple(shape)}")
    if written and not t.is_contiguous():
        _apart(t, name)
    return t.data_ptr(), t.stride(), shape


def _scales(t: torch.Tensor, name: str, device: int, pages: int, heads: int, rows: int, written: bool) -> tuple:
    """The scales of a cache, [pages, heads, blocks], as asc_rows_t's fields, and the rows of a block."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        _here(t, name, device)
    if t.dtype is not torch.float32:
        raise TypeError(f"'{name}' must be torch.float32, got {t.dtype}")
    size = t.shape
    blocks = size[2] if len(size) == 3 else -1
    if blocks <= 0 or rows % (16 * blocks) or size[0] != pages or size[1] != heads:
        if blocks != 0 or rows or size[0] != pages or size[1] != heads:
            raise ValueError(f"'{name}' must be [{pages}, {heads}, blocks] for blocks of a multiple of 16 rows that "
                             f"divide the {rows} of a page, got {tuple(size)}")
    if written and not t.is_contiguous():
        _apart(t, name)
    return t.data_ptr(), *t.stride(), (rows // blocks if rows else 16)


def _table(t: torch.Tensor, name: str, device: int, batch: int) -> tuple:
    """Address, row stride and width of an int32 table of pages."""
    at, (row, step), size = _strided(t, name, device, 2, False)
    if t.dtype is not torch.int32 or size[0] != batch:
        raise ValueError(f"'{name}' must be int32 [{batch}, pages], got {t.dtype} {tuple(size)}")
    if step != 1 and size[1] > 1:
        raise ValueError(f"the last dimension of '{name}' must be contiguous")
    return at, row, size[1]


def _cache8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
            block_table: Optional[torch.Tensor], batch: int, device: int, written: bool = False) -> tuple:
    """Checks a cache of 8 bits: its codes' and scales' rows, (cache dtype, head_dim, page_size, scale_block,
    kv_heads, kv_len, pages), and the table's address and stride."""
    if not isinstance(k_cache, torch.Tensor):
        raise TypeError(f"'k_cache' must be a torch.Tensor, got {type(k_cache).__name__}")
    dtype = k_cache.dtype
    code = _CACHE_CODES.get(dtype)
    if code is None:
        raise TypeError(f"'k_cache' has unsupported dtype {dtype}; expected one of {sorted(map(str, _CACHE_CODES))}")
    shape = k_cache.shape
    if len(shape) != 4:
        raise ValueError(f"'k_cache' must be [pages, kv_heads, rows, head_dim], got {tuple(shape)}")
    pages, heads, rows, head_dim = shape
    if head_dim not in FA_HEAD_DIMS:
        raise ValueError(f"head_dim {head_dim} not supported (supported: {FA_HEAD_DIMS})")
    fields = ()
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor) or t.get_device() != device:
            _here(t, name, device)
        if t.dtype is not dtype:
            raise TypeError(f"'{name}' must be {dtype}, got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"'{name}' must be {list(shape)}, got {tuple(t.shape)}")
        if written and not t.is_contiguous():
            _apart(t, name)
        at, (s0, s1, s2, s3) = t.data_ptr(), t.stride()
        if s3 != 1:
            raise ValueError(f"the last dimension of '{name}' must be contiguous")
        if (at | s0 | s1 | s2) & 15:
            s0, s1, s2 = (s if n > 1 else 0 for s, n in zip((s0, s1, s2), shape))
            if (at | s0 | s1 | s2) & 15:
                raise ValueError(f"'{name}' must be 16-byte aligned, with strides that are multiples of 16 "
                                 f"(address {at:#x}, strides {t.stride()})")
        fields += (at, s0, s1, s2)
    *ks_rows, block = _scales(k_scales, "k_scales", device, pages, heads, rows, written)
    *vs_rows, v_block = _scales(v_scales, "v_scales", device, pages, heads, rows, written)
    if block != v_block:
        raise ValueError(f"'k_scales' and 'v_scales' have blocks of {block} and {v_block} rows")
    fields += (*ks_rows, *vs_rows)
    if block_table is None:
        if pages != batch:
            raise ValueError(f"a cache without a block_table must have {batch} sequences, got {pages}")
        return fields, (code, head_dim, 0, block, heads, rows, pages), (0, 0)
    table, stride, width = _table(block_table, "block_table", device, batch)
    if rows == 0:
        raise ValueError("pages without rows")
    return fields, (code, head_dim, rows, block, heads, width * rows, pages), (table, stride)


def quantized_cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           k_scales: torch.Tensor, v_scales: torch.Tensor, cache_lengths: torch.Tensor,
                           block_table: Optional[torch.Tensor] = None, new_lengths: Optional[torch.Tensor] = None,
                           stream: Any = None) -> None:
    """Writes new keys and values into a cache held in 8 bits, behind the tokens that it holds.

    - k, v: float16 or bfloat16 [batch, kv_heads, n, head_dim] (64 or 128), rows 16-byte aligned, strides
      multiples of 8.  new_lengths (int32 [batch]): new tokens of each sequence, default n.
    - k_cache, v_cache: int8 or float8_e4m3fn codes, [batch, kv_heads, rows, head_dim], or with ``block_table``
      (int32 [batch, pages of a sequence]) [pages, kv_heads, page size, head_dim]: key j of sequence b lies in
      page block_table[b, j // page_size], row j % page_size.  cache_lengths (int32 [batch]): keys
      before the call; token i becomes key cache_lengths[b] + i.
    - k_scales, v_scales: float32 [pages, kv_heads, blocks], one for each block of page_size / blocks rows
      (a multiple of 16, below 2^33 / head_dim) and head; a code stands for itself times its block's scale.

    A block gets the least power of two (at least 2^-126) that holds its new rows' finite values, or keeps its
    scale where that is enough; where earlier rows' scale has to grow, their codes are rounded
    to the new one.  Rounded to nearest, ties to even; infinities become the largest code, NaN the NaN of e4m3 or 0
    of int8.  A sequence whose lengths do not fit the cache, and a block whose page lies outside it, are left
    as they were.  Pages that two sequences share must not be appended to."""
    device = _current_device()
    if not isinstance(k, torch.Tensor):
        raise TypeError(f"'k' must be a torch.Tensor, got {type(k).__name__}")
    dtype = k.dtype
    if dtype not in _HALVES:
        raise TypeError(f"'k' has unsupported dtype {dtype}; expected one of {sorted(map(str, _HALVES))}")
    rows = _rows(k, "k", dtype, device, None, False, True)
    shape = k.shape
    batch, heads, n, head_dim = shape
    rows += _rows(v, "v", dtype, device, shape, False, True)
    cache, sizes, table = _cache8(k_cache, v_cache, k_scales, v_scales, block_table, batch, device, True)
    if heads != sizes[4] or head_dim != sizes[1]:
        raise ValueError(f"'k' {tuple(shape)} does not fit the cache {tuple(k_cache.shape)}")
    lengths = _vector(cache_lengths, "cache_lengths", torch.int32, device, (batch,))
    news = 0 if new_lengths is None else _vector(new_lengths, "new_lengths", torch.int32, device, (batch,))
    args = _CACHE8.pack(_DTYPE_CODES[dtype], *sizes[:4], 0, 0.0, batch, 0, heads, n, *sizes[5:], *cache, *_NO_ROWS,
                        *_NO_ROWS, *rows, 0, lengths, news, *table)
    _launch("asc_quantized_cache_append", args, _stream(stream))


def quantized_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                         starts: torch.Tensor, k_out: Optional[torch.Tensor], v_out: Optional[torch.Tensor],
                         block_table: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                         stream: Any = None) -> None:
    """The values of keys starts[b] + i (int32 [batch]) of a cache held in 8 bits, as quantized_cache_append's,
    into k_out[b, :, i] and v_out[b, :, i] for i < counts[b] (int32 [batch], default n): float32, float16 or bfloat16
    [batch, kv_heads, n, head_dim], either may be None.  Rows behind counts[b] are left as they were.  A
    sequence whose keys do not fit the cache, and a key whose page lies outside it, give NaN."""
    device = _current_device()
    out = k_out if k_out is not None else v_out
    if not isinstance(out, torch.Tensor):
        raise TypeError("k_out or v_out must be a torch.Tensor")
    dtype, shape = out.dtype, out.shape
    if dtype not in _FLOATS or len(shape) != 4:
        raise TypeError(f"results must be floats [batch, kv_heads, n, head_dim], got {dtype} {tuple(shape)}")
    batch, heads, n, head_dim = shape
    rows = ()
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        at, *strides = _NO_ROWS if t is None else _rows(t, name, dtype, device, shape, True)
        if (at | (strides[0] | strides[1] | strides[2]) * out.element_size()) & 15:
            strides = [s if size > 1 else 0 for s, size in zip(strides, shape)]
            if (at | (strides[0] | strides[1] | strides[2]) * out.element_size()) & 15:
                raise ValueError(f"'{name}' must be 16-byte aligned, with strides that are multiples of 16 bytes")
        rows += (at, *strides)
    cache, sizes, table = _cache8(k_cache, v_cache, k_scales, v_scales, block_table, batch, device)
    if heads != sizes[4] or head_dim != sizes[1]:
        raise ValueError(f"results {tuple(shape)} do not fit the cache {tuple(k_cache.shape)}")
    lengths = _vector(starts, "starts", torch.int32, device, (batch,))
    news = 0 if counts is None else _vector(counts, "counts", torch.int32, device, (batch,))
    args = _CACHE8.pack(_DTYPE_CODES[dtype], *sizes[:4], 0, 0.0, batch, 0, heads, n, *sizes[5:], *cache, *_NO_ROWS,
                        *_NO_ROWS, *rows, 0, lengths, news, *table)
    _launch("asc_quantized_cache_read", args, _stream(stream))


def quantized_cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor,
                              v_scales: torch.Tensor, cache_lengths: torch.Tensor, o: torch.Tensor, sm_scale: float,
                              block_table: Optional[torch.Tensor] = None, new_lengths: Optional[torch.Tensor] = None,
                              causal: bool = True, lse: Optional[torch.Tensor] = None, stream: Any = None) -> None:
    """Attention of each sequence's newest tokens over a cache held in 8 bits that holds them already (as
    quantized_cache_append leaves it): o = softmax(q k^T * sm_scale) v for float16 or bfloat16 q and o [batch, heads,
    n, head_dim], heads a multiple of kv_heads.

    - cache_lengths (int32 [batch]): the keys of each sequence, the new ones among them.  new_lengths (int32 [batch]):
      its queries, default n, those of its last keys: with ``causal`` query i attends the first cache_lengths -
      new_lengths + i + 1 keys, else all.  Rows of o and lse behind new_lengths are left as they were, all of them
      where it is negative.
    - caches, scales and block_table as quantized_cache_append's; scales positive and finite.

    A query without keys gets zeros and an lse (float32 [batch, heads, n]) of -inf.  A length outside the cache and more
    queries than n are not followed: NaN; a page outside it gives NaN for the queries that attend its keys, and may
    for others of the sequence.  A key's probability times its V scale is rounded by up to 2^-11 of it, or 2^-33 of
    the largest that its query attends; float32 otherwise."""
    device = _current_device()
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"'q' must be a torch.Tensor, got {type(q).__name__}")
    dtype = q.dtype
    if dtype not in _HALVES:
        raise TypeError(f"'q' has unsupported dtype {dtype}; expected one of {sorted(map(str, _HALVES))}")
    q_rows = _rows(q, "q", dtype, device, None, False, True)
    shape = q.shape
    batch, heads, n, head_dim = shape
    o_rows = _rows(o, "o", dtype, device, shape, True, True)
    cache, sizes, table = _cache8(k_cache, v_cache, k_scales, v_scales, block_table, batch, device)
    kv_heads = sizes[4]
    if head_dim != sizes[1]:
        raise ValueError(f"'q' {tuple(shape)} does not fit the cache {tuple(k_cache.shape)}")
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} key / value heads")
    if not 0 < sm_scale < math.inf:
        raise ValueError(f"sm_scale must be positive and finite, got {sm_scale}")
    lse_at = 0 if lse is None else _vector(lse, "lse", torch.float32, device, shape[:3])
    lengths = _vector(cache_lengths, "cache_lengths", torch.int32, device, (batch,))
    news = 0 if new_lengths is None else _vector(new_lengths, "new_lengths", torch.int32, device, (batch,))
    args = _CACHE8.pack(_DTYPE_CODES[dtype], *sizes[:4], bool(causal), sm_scale, batch, heads, kv_heads, n, *sizes[5:], *cache,
                        *q_rows, *o_rows, *_NO_ROWS, *_NO_ROWS, lse_at, lengths, news, *table)
    _with_workspace("asc_quantized_cache_attention", args, q.device, stream)


# ------------------------------------------------------------------------------ pages of a cache

_PAGES_HEAD = struct.Struct("@8q3Pq4Pq3P")  # asc_pages_t before its tensors
_PAGE_TENSOR = struct.Struct("@2P7q")
_NO_PAGES = bytes(_PAGE_TENSOR.size * _native.MAX_PAGE_TENSORS)


def _page_tensors(caches: Any, results: Any, device: int) -> tuple:
    """The tensors of a cache as asc_page_tensor_t's, their number, and the pages of caches and results."""
    if isinstance(caches, torch.Tensor):
        caches = (caches,)
    if isinstance(results, torch.Tensor):
        results = (results,)
    if len(caches) != len(results) or len(caches) > _native.MAX_PAGE_TENSORS:
        raise ValueError(f"{len(caches)} caches and {len(results)} results (as many, at most {_native.MAX_PAGE_TENSORS})")
    packed, pages, to_pages = b"", None, None
    for x, y in zip(caches, results):
        _here(x, "caches", device)
        shape = x.shape
        if len(shape) < 2:
            raise ValueError(f"a cache must be [pages, heads, rows, ...], got {tuple(shape)}")
        strides = x.stride()
        to_shape, to_strides = shape, strides
        if y is not x:
            _here(y, "results", device)
            to_shape, to_strides = y.shape, y.stride()
            if y.dtype is not x.dtype or to_shape[1:] != shape[1:]:
                raise ValueError(f"a result {y.dtype} {tuple(to_shape)} does not fit its cache {x.dtype} {tuple(shape)}")
            if any(a != b for a, b, n in zip(strides[1:], to_strides[1:], shape[1:]) if n > 1):
                raise ValueError("a cache and its result must have the same strides within a page")
        if not y.is_contiguous():
            _apart(y, "results")
        if pages is None:
            pages, to_pages = shape[0], to_shape[0]
        elif shape[0] != pages or to_shape[0] != to_pages:
            raise ValueError(f"caches of {pages} and {shape[0]} pages, results of {to_pages} and {to_shape[0]}")
        size = x.element_size()
        row = size  # what lies behind a row's first element
        for n, s in zip(reversed(shape[3:]), reversed(strides[3:])):
            if s * size != row and n > 1:
                raise ValueError(f"the dimensions of a cache behind its rows must be contiguous (strides {strides})")
            row *= n
        if row == 0 or 0 in shape[1:]:
            raise ValueError(f"a cache without elements: {tuple(shape)}")
        rows, step = (shape[2], strides[2]) if len(shape) > 2 else (1, 0)
        packed += _PAGE_TENSOR.pack(x.data_ptr(), y.data_ptr(), strides[0] * size, to_strides[0] * size, shape[1], rows, row,
                                    strides[1] * size, step * size)
    return packed + _NO_PAGES[len(packed):], len(caches), pages or 0, to_pages or 0


def cache_copy_pages(caches: Any, results: Any, from_pages: torch.Tensor, to_pages: torch.Tensor,
                     stream: Any = None) -> None:
    """Page to_pages[i] of each result becomes page from_pages[i] of its cache (both int32 [pairs]): up to eight
    tensors whose first dimension is the pages (keys, values, their scales), of any type, in one launch.
    A result may be its cache.  Pairs with a page outside the tensors are left out.  A page that is written
    must be in no other pair: it would hold parts of both."""
    device = _current_device()
    tensors, number, pages, into = _page_tensors(caches, results, device)
    _here(from_pages, "from_pages", device)
    if from_pages.dim() != 1:
        raise ValueError(f"'from_pages' must be a vector, got {tuple(from_pages.shape)}")
    pairs = from_pages.numel()
    source = _vector(from_pages, "from_pages", torch.int32, device, (pairs,))
    target = _vector(to_pages, "to_pages", torch.int32, device, (pairs,))
    args = _PAGES_HEAD.pack(number, 1, pages, into, pairs, 0, 0, 0, source, target, *(0,) * 10) + tensors
    _launch("asc_cache_copy_pages", args, _stream(stream))


def _books(block_table: torch.Tensor, lengths: torch.Tensor, refcounts: torch.Tensor, refcounts_out: torch.Tensor,
           page_size: int, pages: Optional[int], device: int) -> tuple:
    """The bookkeeping that fork and compact share: batch, width, pages, and the addresses."""
    _here(block_table, "block_table", device)
    batch = block_table.shape[0] if block_table.dim() == 2 else -1
    table, stride, width = _table(block_table, "block_table", device, batch)
    _here(refcounts, "refcounts", device)
    pages = refcounts.numel() if pages is None else pages
    counts = _vector(refcounts, "refcounts", torch.int32, device, (pages,))
    counts_out = _vector(refcounts_out, "refcounts_out", torch.int32, device, (pages,))
    if page_size < 1:
        raise ValueError(f"page_size must be positive, got {page_size}")
    return batch, width, pages, table, stride, _vector(lengths, "lengths", torch.int32, device, (batch,)), counts, counts_out


def _table_out(t: torch.Tensor, device: int, rows: int, width: int) -> tuple:
    at, stride, columns = _table(t, "table_out", device, rows)
    if columns != width:
        raise ValueError(f"'table_out' must be [{rows}, {width}], got {tuple(t.shape)}")
    if not t.is_contiguous():
        _apart(t, "table_out")
    return at, stride


def cache_fork(caches: Any, block_table: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor,
               refcounts: torch.Tensor, page_size: int, table_out: torch.Tensor, lengths_out: torch.Tensor,
               refcounts_out: torch.Tensor, stream: Any = None) -> None:
    """The sequences of a paged cache become others: sequence i goes on from sequence parents[i] (int32 [new
    batch]; outside the batch: it holds nothing, so its pages are free if nobody else has them).

    - caches: up to eight tensors [pages, heads, rows, ...] of any type (keys, values, their scales);
      page_size is a multiple of each one's rows.
    - block_table (int32 [batch, width]), lengths (int32 [batch]): the sequences before; table_out (int32
      [new batch, width], -1 behind a sequence's pages) and lengths_out (int32 [new batch]): after.
    - refcounts (int32 [pages]): how many sequences hold a page, 0: free; refcounts_out, which may be
      refcounts: after.

    Full pages are shared.  The last page, where it is partly filled, stays with the first child; each other child
    gets a free page with its rows: the lowest free ones, in the children's order, -1 where there is none
    left.  A length outside the table is handed on, with a row of -1.  At most 4096 sequences."""
    device = _current_device()
    tensors, number, pages, _ = _page_tensors(caches, caches, device)
    batch, width, pages, table, stride, length, counts, counts_out = _books(
        block_table, lengths, refcounts, refcounts_out, page_size, pages if number else None, device)
    _here(parents, "parents", device)
    new = parents.numel()
    parent = _vector(parents, "parents", torch.int32, device, (new,))
    out, out_stride = _table_out(table_out, device, new, width)
    args = _PAGES_HEAD.pack(number, page_size, pages, pages, 0, batch, new, width, 0, 0, table, stride, length, parent,
                            counts, out, out_stride, _vector(lengths_out, "lengths_out", torch.int32, device, (new,)),
                            counts_out, 0) + tensors
    _with_workspace("asc_cache_fork", args, block_table.device, stream)


def cache_compact(caches: Any, block_table: torch.Tensor, lengths: torch.Tensor, refcounts: torch.Tensor,
                  page_size: int, table_out: torch.Tensor, refcounts_out: torch.Tensor, page_map: torch.Tensor,
                  stream: Any = None) -> None:
    """Brings the pages in use (refcounts > 0), U of them, to the front of a paged cache: the i-th of those at U and
    above moves into the i-th free one below.  Tensors (whose pages move whole, whatever their rows), tables and counts as
    cache_fork's; table_out may be block_table, refcounts_out refcounts.  page_map (int32 [pages]) receives each page's new place, -1 for free
    ones: holders outside the table have it to go by."""
    device = _current_device()
    tensors, number, pages, _ = _page_tensors(caches, caches, device)
    batch, width, pages, table, stride, length, counts, counts_out = _books(
        block_table, lengths, refcounts, refcounts_out, page_size, pages if number else None, device)
    out, out_stride = _table_out(table_out, device, batch, width)
    args = _PAGES_HEAD.pack(number, page_size, pages, pages, 0, batch, 0, width, 0, 0, table, stride, length, 0, counts,
                            out, out_stride, 0, counts_out,
                            _vector(page_map, "page_map", torch.int32, device, (pages,))) + tensors
    _with_workspace("asc_cache_compact", args, block_table.device, stream)


# ------------------------------------------------------------------ logits before a token is chosen

_LOGITS = struct.Struct("@2i3qPqPqPq6PqPq")  # asc_logits_t


def _matrix(t: torch.Tensor, name: str, dtype: torch.dtype, device: int, shape: tuple, written: bool = False) -> tuple:
    """Address and row stride of a matrix whose rows are contiguous."""
    at, (row, step), size = _strided(t, name, device, 2, written)
    if t.dtype is not dtype:
        raise TypeError(f"'{name}' must be {dtype}, got {t.dtype}")
    if size != shape:
        raise ValueError(f"'{name}' must be {list(shape)}, got {tuple(size)}")
    if step != 1 and size[1] > 1:
        raise ValueError(f"the last dimension of '{name}' must be contiguous")
    return at, row


def process_logits(logits: torch.Tensor, out: torch.Tensor, history: torch.Tensor, history_lengths: torch.Tensor,
                   prompt_lengths: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, stream: Any = None) -> None:
    """Logits [rows, vocabulary] (float32, float16 or bfloat16) before a token is chosen, into ``out`` (which may be
    logits), computed in float32 in this order:

    - a token of the row's history: x / repetition if x > 0, else x * repetition;
    - one that comes c times in it behind the prompt: x - frequency * c, and if c > 0 - presence;
    - x + bias (float32 [vocabulary] or [rows, vocabulary]);
    - -inf where its bit is 0 in mask (int32 [rows, ceil(vocabulary / 32)]: token t is bit t % 32 of word t // 32),
      whatever x is; a row whose mask leaves nothing is -inf throughout.

    history (int32 or int64 [rows, width]): the row's first history_lengths (int32 [rows]) tokens, of which the
    first prompt_lengths (int32 [rows], default none) are the prompt; tokens outside the vocabulary
    are passed over.  repetition, frequency, presence: float32 [rows].  A history length outside [0, width] gives
    NaN."""
    device = _current_device()
    if not isinstance(logits, torch.Tensor):
        raise TypeError(f"'logits' must be a torch.Tensor, got {type(logits).__name__}")
    dtype, shape = logits.dtype, logits.shape
    if dtype not in _FLOATS:
        raise TypeError(f"'logits' has unsupported dtype {dtype}; expected one of {sorted(map(str, _FLOATS))}")
    if len(shape) != 2:
        raise ValueError(f"'logits' must be [rows, vocabulary], got {tuple(shape)}")
    rows, vocab = shape
    x = _matrix(logits, "logits", dtype, device, shape)
    y = x if out is logits and logits.is_contiguous() else _matrix(out, "out", dtype, device, shape, True)
    _here(history, "history", device)
    wide = history.dtype is torch.int64
    if (not wide and history.dtype is not torch.int32) or history.dim() != 2:
        raise TypeError(f"'history' must be int32 or int64 [{rows}, width], got {history.dtype} {tuple(history.shape)}")
    width = history.shape[1]
    h = _matrix(history, "history", history.dtype, device, (rows, width))
    per_row = (rows,)
    lengths = _vector(history_lengths, "history_lengths", torch.int32, device, per_row)
    prompts = 0 if prompt_lengths is None else _vector(prompt_lengths, "prompt_lengths", torch.int32, device, per_row)
    r = 0 if repetition is None else _vector(repetition, "repetition", torch.float32, device, per_row)
    f = 0 if frequency is None else _vector(frequency, "frequency", torch.float32, device, per_row)
    p = 0 if presence is None else _vector(presence, "presence", torch.float32, device, per_row)
    b = m = (0, 0)
    if bias is not None:
        if isinstance(bias, torch.Tensor) and bias.dim() == 1:
            b = (_vector(bias, "bias", torch.float32, device, (vocab,)), 0)
        else:
            b = _matrix(bias, "bias", torch.float32, device, shape)
    if mask is not None:
        m = _matrix(mask, "mask", torch.int32, device, (rows, -(-vocab // 32)))
    _launch("asc_process_logits", _LOGITS.pack(_DTYPE_CODES[dtype], wide, rows, vocab, width, *x, *y, *h, lengths, prompts, r, f,
                                               p, *b, *m), _stream(stream))


# ------------------------------------------------------------------ element-wise tile operations

UNARY_OPS = ("abs", "ceil", "cos", "cosh", "erf", "exp", "exp2", "floor", "log", "log2", "negative", "relu",
             "rsqrt", "sin", "sinh", "sqrt", "tan", "tanh")
BINARY_OPS = ("add", "sub", "mul", "div", "maximum", "minimum", "left_shift", "right_shift")
COMPARE_OPS = ("equal", "not_equal", "greater", "greater_equal", "less", "less_equal")
_TILE_DTYPES = (torch.float32, torch.float16, torch.bfloat16, torch.int32, torch.int16)


def _flat(t: torch.Tensor, name: str, n: int) -> torch.Tensor:
    _contiguous(_device_tensor(t, name), name)
    if t.numel() < n:
        raise ValueError(f"'{name}' holds {t.numel()} elements, {n} needed")
    return t


def _scalar_parts(value: Any, dtype: torch.dtype):
    """(scalar_f, scalar_i) transport of a scalar operand for an element type."""
    if isinstance(value, torch.Tensor):
        if value.dim() != 0:
            raise ValueError("a scalar operand must be a 0-dim tensor or a python number")
        value = value.item()
    if dtype.is_floating_point:
        return float(value), 0
    if isinstance(value, float) and not value.is_integer():
        raise TypeError(f"an integer tile takes an integer scalar, got {value}")
    return 0.0, int(value)


def unary_f32(x: torch.Tensor, out: torch.Tensor, op: str, n: Optional[int] = None, stream=None) -> None:
    """out[:n] = op(x[:n]), fp32 (asc2 unary ops, python/asc/language/tile/unary_ops.py)."""
    if op not in UNARY_OPS:
        raise ValueError(f"unknown unary op {op!r}; expected one of {UNARY_OPS}")
    n = x.numel() if n is None else int(n)
    for t, name in ((x, "x"), (out, "out")):
        _flat(t, name, n)
        if t.dtype != torch.float32:
            raise TypeError(f"'{name}' must be float32, got {t.dtype}")
    _native.call("asc_unary_f32", UNARY_OPS.index(op), x.data_ptr(), out.data_ptr(), n, _stream(stream))


_FLOAT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def unary(x: torch.Tensor, out: torch.Tensor, op: str, n: Optional[int] = None, stream=None) -> None:
    """out[:n] = op(x[:n]) on float32 / float16 / bfloat16 (16-bit: fp32 op, one RNE rounding)."""
    if op not in UNARY_OPS:
        raise ValueError(f"unknown unary op {op!r}; expected one of {UNARY_OPS}")
    n = x.numel() if n is None else int(n)
    code = _code(x, "x", _FLOAT_DTYPES)
    if out.dtype != x.dtype:
        raise TypeError(f"'out' must be {x.dtype}, got {out.dtype}")
    _flat(x, "x", n)
    _flat(out, "out", n)
    _native.call("asc_unary", UNARY_OPS.index(op), code, x.data_ptr(), out.data_ptr(), n, _stream(stream))


def axpy(src: torch.Tensor, dst: torch.Tensor, scalar: float, n: Optional[int] = None, stream=None) -> None:
    """dst[:n] = src[:n] * scalar + dst[:n] (asc.axpy): float32 / float16 / bfloat16, the
    scalar rounded to the element type, fp32 math, one rounding of the result."""
    n = src.numel() if n is None else int(n)
    code = _code(src, "src", _FLOAT_DTYPES)
    if dst.dtype != src.dtype:
        raise TypeError(f"'dst' must be {src.dtype}, got {dst.dtype}")
    _flat(src, "src", n)
    _flat(dst, "dst", n)
    _native.call("asc_axpy", code, src.data_ptr(), dst.data_ptr(), float(_scalar_parts(scalar, src.dtype)[0]), n,
                 _stream(stream))


def transpose_batched(x: torch.Tensor, z: torch.Tensor, batch: int, rows: int, cols: int, stream=None) -> None:
    """z[b, c, r] = x[b, r, c] for row-major [batch, rows, cols] of 2- or 4-byte elements."""
    n = int(batch) * int(rows) * int(cols)
    _flat(x, "x", n)
    _flat(z, "z", n)
    if z.dtype != x.dtype:
        raise TypeError(f"'z' must be {x.dtype}, got {z.dtype}")
    _native.call("asc_transpose_batched", x.element_size(), x.data_ptr(), z.data_ptr(), int(batch), int(rows),
                 int(cols), _stream(stream))


def quant_i8(src: torch.Tensor, dst: torch.Tensor, scale: float, offset: float, n: Optional[int] = None,
             stream=None) -> None:
    """dst[:n] = saturate_int8(rint(src * scale + offset)) (asc.adv.quant): scale and offset
    in src's dtype, each operation rounded to it, ties to even, NaN -> 0."""
    n = src.numel() if n is None else int(n)
    code = _code(src, "src", _FLOAT_DTYPES)
    if dst.dtype != torch.int8:
        raise TypeError(f"'dst' must be int8, got {dst.dtype}")
    _flat(src, "src", n)
    _flat(dst, "dst", n)
    _native.call("asc_quant_i8", code, src.data_ptr(), dst.data_ptr(), float(scale), float(offset), n,
                 _stream(stream))


def binary(x: Any, y: Any, out: torch.Tensor, op: str, n: Optional[int] = None, stream=None) -> None:
    """out[:n] = op(x, y) with either operand a tensor or a scalar (asc2 binary ops,
    python/asc/language/tile/binary_ops.py); the result dtype is the tensor operand's."""
    if op not in BINARY_OPS:
        raise ValueError(f"unknown binary op {op!r}; expected one of {BINARY_OPS}")
    x_t, y_t = isinstance(x, torch.Tensor) and x.dim() > 0, isinstance(y, torch.Tensor) and y.dim() > 0
    if not (x_t or y_t):
        raise TypeError("at least one operand must be a tensor")
    ref = x if x_t else y
    n = ref.numel() if n is None else int(n)
    code = _code(ref, "x" if x_t else "y", _TILE_DTYPES)
    if out.dtype != ref.dtype:
        raise TypeError(f"'out' must be {ref.dtype}, got {out.dtype}")
    _flat(out, "out", n)
    mode, scalar = 0, None
    if x_t and y_t:
        if y.dtype != x.dtype:
            raise TypeError(f"operand dtypes differ: {x.dtype} and {y.dtype}")
        _flat(x, "x", n)
        _flat(y, "y", n)
    elif x_t:
        mode, scalar = 1, y
        _flat(x, "x", n)
    else:
        mode, scalar = 2, x
        _flat(y, "y", n)
    if op in ("left_shift", "right_shift"):
        if mode != 1 or ref.dtype.is_floating_point:
            raise TypeError(f"{op} takes an integer tensor and a scalar shift amount")
        bits = torch.iinfo(ref.dtype).bits
        shift = int(scalar.item()) if isinstance(scalar, torch.Tensor) else int(scalar)
        if not 0 <= shift < bits:
            raise ValueError(f"{op} amount {shift} is outside [0, {bits}) for {ref.dtype}")
    s_f, s_i = _scalar_parts(scalar, ref.dtype) if scalar is not None else (0.0, 0)
    # an unused operand slot gets the output buffer (valid for n elements), never NULL
    _native.call("asc_binary", BINARY_OPS.index(op), code, x.data_ptr() if x_t else out.data_ptr(),
                 y.data_ptr() if y_t else out.data_ptr(), out.data_ptr(), n, mode, s_f, s_i, _stream(stream))


def where_compare(x: torch.Tensor, y: Any, out: torch.Tensor, cmp: str, true_value=None, false_value=None,
                  n: Optional[int] = None, stream=None) -> None:
    """out = where(cmp(x, y), x, y) for a tensor y, or where(cmp(x, s), true_value,
    false_value) for a scalar s (asc2.where over a comparison, test_where.py)."""
    if cmp not in COMPARE_OPS:
        raise ValueError(f"unknown comparison {cmp!r}; expected one of {COMPARE_OPS}")
    n = x.numel() if n is None else int(n)
    code = _code(x, "x", _TILE_DTYPES)
    _flat(x, "x", n)
    _flat(out, "out", n)
    if out.dtype != x.dtype:
        raise TypeError(f"'out' must be {x.dtype}, got {out.dtype}")
    if isinstance(y, torch.Tensor) and y.dim() > 0:
        if y.dtype != x.dtype:
            raise TypeError(f"operand dtypes differ: {x.dtype} and {y.dtype}")
        _flat(y, "y", n)
        _native.call("asc_where_cmp", COMPARE_OPS.index(cmp), code, x.data_ptr(), y.data_ptr(), out.data_ptr(), n,
                     0, 0.0, 0, 0.0, 0.0, _stream(stream))
        return
    if true_value is None or false_value is None:
        raise ValueError("a scalar comparison needs true_value and false_value")
    s_f, s_i = _scalar_parts(y, x.dtype)
    _native.call("asc_where_cmp", COMPARE_OPS.index(cmp), code, x.data_ptr(), x.data_ptr(), out.data_ptr(), n, 1, s_f,
                 s_i, float(true_value), float(false_value), _stream(stream))


# ------------------------------------------------------------------- tile load / store, shape ops

def tile_offsets(tensor_shape, tile_shape, tile_id=None, offsets=None):
    """Offsets of a tile: exactly one of ``tile_id`` (-> tile_id * tile_shape) or
    ``offsets`` (python/asc/language/tile/memory_ops.py:24-31, 65-80)."""
    if (tile_id is None) == (offsets is None):
        raise ValueError("Exactly one of 'tile_id' or 'offsets' must be provided")
    if tile_shape is not None and len(tile_shape) != len(tensor_shape):
        raise RuntimeError("rank of 'tensor_shape' must match rank of 'shape'")
    if tile_id is not None:
        return [int(i) * int(s) for i, s in zip(tile_id, tile_shape)]
    if len(offsets) != len(tensor_shape):
        raise ValueError(f"{len(offsets)} offsets for a rank-{len(tensor_shape)} tensor")
    return [int(o) for o in offsets]


def tile_binary(x: torch.Tensor, y: torch.Tensor, z: torch.Tensor, op: str, tensor_shape, tile_shape, offsets,
                stream=None) -> None:
    """z[tile] = op(x[tile], y[tile]) for the tile at ``offsets`` of shape ``tile_shape``
    (None: one element) in 1-D / 2-D row-major tensors of ``tensor_shape``; the store
    clips at the tensor bounds (asc2.load, op, asc2.store)."""
    if op not in BINARY_OPS[:6]:
        raise ValueError(f"op {op!r} is not an element-wise binary op")
    shape = [int(v) for v in tensor_shape]
    if len(shape) not in (1, 2):
        raise NotImplementedError("tiles of 1-D and 2-D tensors")
    tile = [1] * len(shape) if tile_shape is None else [int(v) for v in tile_shape]
    if len(tile) != len(shape) or len(offsets) != len(shape):
        raise RuntimeError("rank of 'tensor_shape' must match rank of the tile and of 'offsets'")
    rows, cols = (1, shape[0]) if len(shape) == 1 else shape
    r0, c0 = (0, int(offsets[0])) if len(shape) == 1 else (int(offsets[0]), int(offsets[1]))
    h, w = (1, tile[0]) if len(shape) == 1 else tile
    if r0 < 0 or c0 < 0:
        raise ValueError(f"negative tile offsets {list(offsets)}")
    code = _code(x, "x", _TILE_DTYPES)
    for t, name in ((x, "x"), (y, "y"), (z, "z")):
        _flat(t, name, rows * cols)
        if t.dtype != x.dtype:
            raise TypeError(f"'{name}' must be {x.dtype}, got {t.dtype}")
    _native.call("asc_rect_binary", BINARY_OPS.index(op), code, x.data_ptr(), y.data_ptr(), z.data_ptr(), rows, cols,
                 r0, c0, h, w, _stream(stream))


def broadcast_rows(x: torch.Tensor, z: torch.Tensor, rows: int, cols: int, stream=None) -> None:
    """z[r, c] = x[c] for r < rows (asc2.broadcast_to from [1, cols]; rows = 1 copies)."""
    _flat(x, "x", cols)
    _flat(z, "z", rows * cols)
    if z.dtype != x.dtype:
        raise TypeError(f"'z' must be {x.dtype}, got {z.dtype}")
    _native.call("asc_broadcast_rows", x.element_size(), x.data_ptr(), z.data_ptr(), rows, cols, _stream(stream))


ATOMIC_OPS = ("add", "maximum", "minimum")


def atomic_tiles(x: torch.Tensor, z: torch.Tensor, op: str, n_tiles: int, tile_len: int, addend=0,
                 stream=None) -> None:
    """z[j] = op(z[j], x[b * tile_len + j] + addend) for b < n_tiles, each combine atomic
    (asc2.atomic_add / atomic_max / atomic_min, python/asc/language/tile/atomic_ops.py:19-33;
    the kernel of python/test/asc2/operations/test_atomic_ops.py:33-40).  The order in which
    the tiles' float sums land is unspecified."""
    if op not in ATOMIC_OPS:
        raise ValueError(f"unknown atomic op {op!r}; expected one of {ATOMIC_OPS}")
    n_tiles, tile_len = int(n_tiles), int(tile_len)
    if n_tiles < 0 or tile_len < 0:
        raise ValueError("n_tiles and tile_len must be non-negative")
    code = _code(x, "x", _TILE_DTYPES)
    _flat(x, "x", n_tiles * tile_len)
    _flat(z, "z", tile_len)
    if z.dtype != x.dtype:
        raise TypeError(f"'z' must be {x.dtype}, got {z.dtype}")
    c_f, c_i = _scalar_parts(addend, x.dtype)
    _native.call("asc_atomic_tiles", BINARY_OPS.index(op), code, x.data_ptr(), z.data_ptr(), n_tiles, tile_len, c_f,
                 c_i, _stream(stream))


def fill(z: torch.Tensor, value, n: Optional[int] = None, stream=None) -> None:
    """z[:n] = value in z's element type (asc2.full broadcast to the tensor and stored)."""
    n = z.numel() if n is None else int(n)
    code = _code(z, "z", _TILE_DTYPES)
    _flat(z, "z", n)
    c_f, c_i = _scalar_parts(value, z.dtype)
    _native.call("asc_fill", code, z.data_ptr(), n, c_f, c_i, _stream(stream))
