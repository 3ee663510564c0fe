"""Values in 8 bits with a float32 scale for each block of 128, and the ops that take them.

A block's scale is a / 448 with a = max(amax, 2^-100), and its codes are the e4m3 nearest to 448 x / a (csrc/kernels/blocks_quantize.cu).
Activations have a scale for each 128 values of a row, weights one for each 128 x 128; a matrix that a checkpoint brings in that form is
taken as it is."""

from __future__ import annotations

import torch

from . import _code, _count, _stream
from .library import KernelError, check, lib

BLOCK = 128                     # a block's edge
CODES = torch.float8_e4m3fn

_device = torch._C._cuda_getDevice


def _code_rows(values: torch.Tensor, what: str) -> int:
    """Bytes between the rows of a tensor of codes [.., N, K]."""
    if not isinstance(values, torch.Tensor) or values.dtype != CODES or not values.is_cuda:
        raise KernelError(f"{what}: expected codes in {CODES} on the device; there is no CPU path")
    K = values.shape[-1]
    ld = values.stride(-2) if values.shape[-2] > 1 else -(-K // 16) * 16
    if K < 1 or values.stride(-1) != 1 or ld < K or ld % 16 or values.data_ptr() % 16:
        raise KernelError(f"{what}: rows of codes have unit stride and start at multiples of 16 bytes, got {tuple(values.shape)} with strides {values.stride()}")
    return ld


def _scales(scales: torch.Tensor, values: torch.Tensor, shape: tuple, what: str) -> None:
    if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or tuple(scales.shape) != shape or not scales.is_contiguous() or scales.device != values.device:
        raise KernelError(f"{what}: expected contiguous float32 scales {shape} beside the codes")


class BlockRows:
    """Rows in blocks: `values` e4m3 [T, K] and `scales` float32 [ceil(K / 128), T], a block's scales of all rows side by side."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dim() != 2:
            raise KernelError(f"BlockRows: expected rows [T, K], got {tuple(values.shape)}")
        self.stride = _code_rows(values, "BlockRows")
        _scales(scales, values, (-(-values.shape[1] // BLOCK), values.shape[0]), "BlockRows")
        self.values, self.scales = values, scales

    shape = property(lambda self: self.values.shape)
    device = property(lambda self: self.values.device)


class BlockMatrix:
    """A matrix [N, K], or a stack of them [E, N, K], in blocks: `values` e4m3 and `scales` float32 [.., ceil(N / 128), ceil(K / 128)]."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dim() not in (2, 3):
            raise KernelError(f"BlockMatrix: expected a matrix or a stack of them, got {tuple(values.shape)}")
        self.stride = _code_rows(values, "BlockMatrix")
        N, K = values.shape[-2:]
        if values.dim() == 3 and values.shape[0] > 1 and values.stride(0) != N * self.stride:
            raise KernelError(f"BlockMatrix: the matrices of a stack lie one behind the other, got strides {values.stride()}")
        _scales(scales, values, tuple(values.shape[:-2]) + (-(-N // BLOCK), -(-K // BLOCK)), "BlockMatrix")
        self.values, self.scales = values, scales

    shape = property(lambda self: self.values.shape)
    device = property(lambda self: self.values.device)


def _room(shape: tuple, device) -> torch.Tensor:
    """A new tensor of codes whose rows start at multiples of 16 bytes."""
    K = shape[-1]
    room = torch.empty(shape[:-1] + (-(-K // 16) * 16,), dtype=CODES, device=device)
    return room if room.shape[-1] == K else room[..., :K]


def _plain(x: torch.Tensor, dims: tuple, what: str) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise KernelError(f"{what}: expected a CUDA tensor; there is no CPU path")
    _code(x.dtype)
    if x.dim() not in dims or x.shape[-1] < 1 or (x.stride(-1) != 1 and x.shape[-1] > 1):
        raise KernelError(f"{what}: expected rows with unit stride, got {tuple(x.shape)} with strides {x.stride()}")


def quantize_rows(x: torch.Tensor) -> BlockRows:
    """Rows x [T, K] (bfloat16 or float32; may be a column slice of wider rows) in blocks of 128 of a row."""
    _plain(x, (2,), "quantize_rows")
    if x.get_device() != _device():
        with torch.cuda.device(x.device):
            return quantize_rows(x)
    T, K = x.shape
    values = _room((T, K), x.device)
    scales = torch.empty((-(-K // BLOCK), T), dtype=torch.float32, device=x.device)
    rows = BlockRows(values, scales)
    check(lib().rlis_quantize_rows(x.data_ptr(), x.stride(0), values.data_ptr(), rows.stride, scales.data_ptr(), T, K, _code(x.dtype), _stream()), "quantize_rows")
    _count("quantize_rows")
    return rows


def quantize_matrix(w: torch.Tensor) -> BlockMatrix:
    """A weight [N, K], or a stack of them [E, N, K] (bfloat16 or float32, rows and matrices any distance apart), in blocks of 128 x 128."""
    _plain(w, (2, 3), "quantize_matrix")
    if w.get_device() != _device():
        with torch.cuda.device(w.device):
            return quantize_matrix(w)
    N, K = w.shape[-2:]
    E = w.shape[0] if w.dim() == 3 else 1
    values = _room(tuple(w.shape), w.device)
    scales = torch.empty(tuple(w.shape[:-2]) + (-(-N // BLOCK), -(-K // BLOCK)), dtype=torch.float32, device=w.device)
    matrix = BlockMatrix(values, scales)
    check(lib().rlis_quantize_matrix(w.data_ptr(), w.stride(-2), w.stride(0) if w.dim() == 3 else 0, values.data_ptr(), matrix.stride, scales.data_ptr(), E, N, K,
                                     _code(w.dtype), _stream()), "quantize_matrix")
    _count("quantize_matrix")
    return matrix


def linear_blocks(x, w: BlockMatrix, out_dtype=None, *, early: bool = False) -> torch.Tensor:
    """y = x @ w^T for a weight in blocks.  x [T, K]: plain rows (bfloat16 or float32; may be a column slice of wider rows), which are put into blocks as
    `quantize_rows` does, or BlockRows, for rows that several products read.  Every block of 128 k is summed on its own, scaled by both scales and added in
    float32; the result is rounded once, to `out_dtype` (bfloat16 or float32; None: x's, bfloat16 for BlockRows).
    `early`: w is a weight that no kernel still in flight writes, so that its first tiles may be asked for before the kernels before have finished."""
    if not isinstance(w, BlockMatrix) or w.values.dim() != 2:
        raise KernelError("linear_blocks: expected a BlockMatrix [N, K]")
    plain = not isinstance(x, BlockRows)
    if plain:
        _plain(x, (2,), "linear_blocks")
    N, K = w.values.shape
    if x.shape[1] != K or x.device != w.values.device:
        raise KernelError(f"linear_blocks: rows {tuple(x.shape)} on {x.device} and a matrix {(N, K)} on {w.device} do not go together")
    out_code = _code(out_dtype or (x.dtype if plain else torch.bfloat16))
    if w.values.get_device() != _device():
        with torch.cuda.device(w.device):
            return linear_blocks(x, w, out_dtype, early=early)
    T = x.shape[0]
    out = torch.empty((T, N), dtype=torch.bfloat16 if out_code else torch.float32, device=w.values.device)
    if plain:
        scratch = torch.empty((T * (-(-K // 16) * 16 + 4 * -(-K // BLOCK)),), dtype=torch.uint8, device=w.values.device)
        check(lib().rlis_blocks_gemm_rows(x.data_ptr(), x.stride(0), _code(x.dtype), scratch.data_ptr(), w.values.data_ptr(), w.stride, w.scales.data_ptr(), out.data_ptr(),
                                          T, N, K, out_code, _stream()), "linear_blocks")
        _count("quantize_rows")
    else:
        check(lib().rlis_blocks_gemm(x.values.data_ptr(), x.stride, x.scales.data_ptr(), w.values.data_ptr(), w.stride, w.scales.data_ptr(), out.data_ptr(), T, N, K,
                                     out_code, int(early), _stream()), "linear_blocks")
    _count("linear_blocks")
    return out
