"""Values in 8 bits with a float32 scale for each block of 128, and the ops that take them.

A block's scale is a / 448 with a = max(amax, 2^-100), and its codes are the e4m3 nearest to 448 x / a (csrc/kernels/blocks_quantize.cu).
Activations have a scale for each 128 values of a row, weights one for each 128 x 128; a matrix that a checkpoint brings in that form is
taken as it is."""

from __future__ import annotations

import ctypes

import torch

from . import _code, _count, _stream
from .library import KernelError, check, lib

BLOCK = 128                     # a block's edge
CODES = torch.float8_e4m3fn

_device = torch._C._cuda_getDevice


def _shape(t):
    return tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__


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
        if not isinstance(values, torch.Tensor) or values.dim() != 2:
            raise KernelError(f"BlockRows: expected rows [T, K], got {_shape(values)}")
        self.stride = _code_rows(values, "BlockRows")
        _scales(scales, values, (-(-values.shape[1] // BLOCK), values.shape[0]), "BlockRows")
        self.values, self.scales = values, scales

    shape = property(lambda self: self.values.shape)
    device = property(lambda self: self.values.device)

    @classmethod
    def _made(cls, values: torch.Tensor, scales: torch.Tensor, stride: int):
        """Of tensors that are known to be right."""
        new = cls.__new__(cls)
        new.values, new.scales, new.stride = values, scales, stride
        return new


class BlockMatrix:
    """A matrix [N, K], or a stack of them [E, N, K], in blocks: `values` e4m3 and `scales` float32 [.., ceil(N / 128), ceil(K / 128)]."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if not isinstance(values, torch.Tensor) or values.dim() not in (2, 3):
            raise KernelError(f"BlockMatrix: expected a matrix or a stack of them, got {_shape(values)}")
        self.stride = _code_rows(values, "BlockMatrix")
        N, K = values.shape[-2:]
        if values.dim() == 3 and values.shape[0] > 1 and values.stride(0) != N * self.stride:
            raise KernelError(f"BlockMatrix: the matrices of a stack lie one behind the other, got strides {values.stride()}")
        _scales(scales, values, tuple(values.shape[:-2]) + (-(-N // BLOCK), -(-K // BLOCK)), "BlockMatrix")
        self.values, self.scales = values, scales

    shape = property(lambda self: self.values.shape)
    device = property(lambda self: self.values.device)
    _made = classmethod(BlockRows._made.__func__)


# A new tensor on the current device.  (torch.empty takes 2.4 us, more than a small call's kernel; what it calls at the end 0.75.)
_empty = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
if _empty is None:
    def _empty(shape, stride, dtype):
        return torch.empty_strided(shape, stride, dtype=dtype, device="cuda")


def _room(N: int, K: int, E=None) -> tuple:
    """A new tensor of codes [N, K] (or [E, N, K]) whose rows start at multiples of 16 bytes, and the bytes from one to the next."""
    stride = -(-K // 16) * 16
    return (_empty((N, K), (stride, 1), CODES) if E is None else _empty((E, N, K), (N * stride, stride, 1), CODES)), stride


_FLOATS = {torch.float32: 0, torch.bfloat16: 1}


def _plain(x: torch.Tensor, dims: tuple, what: str) -> int:
    """Checks rows of plain values; their element type's code."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise KernelError(f"{what}: expected a CUDA tensor; there is no CPU path")
    code = _FLOATS.get(x.dtype)
    if code is None:
        _code(x.dtype)
    if x.dim() not in dims or x.shape[-1] < 1 or (x.stride(-1) != 1 and x.shape[-1] > 1):
        raise KernelError(f"{what}: expected rows with unit stride, got {tuple(x.shape)} with strides {x.stride()}")
    return code


def quantize_rows(x: torch.Tensor) -> BlockRows:
    """Rows x [T, K] (bfloat16 or float32; may be a column slice of wider rows) in blocks of 128 of a row."""
    code = _plain(x, (2,), "quantize_rows")
    if x.get_device() != _device():
        with torch.cuda.device(x.device):
            return quantize_rows(x)
    T, K = x.shape
    values, stride = _room(T, K)
    scales = _empty((-(-K // BLOCK), T), (T, 1), torch.float32)
    check(lib().rlis_quantize_rows(x.data_ptr(), x.stride(0), values.data_ptr(), stride, scales.data_ptr(), T, K, code, _stream()), "quantize_rows")
    _count("quantize_rows")
    return BlockRows._made(values, scales, stride)


def quantize_matrix(w: torch.Tensor) -> BlockMatrix:
    """A weight [N, K], or a stack of them [E, N, K] (bfloat16 or float32, rows and matrices any distance apart), in blocks of 128 x 128."""
    code = _plain(w, (2, 3), "quantize_matrix")
    if w.get_device() != _device():
        with torch.cuda.device(w.device):
            return quantize_matrix(w)
    N, K = w.shape[-2:]
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    stack = w.dim() == 3
    E = w.shape[0] if stack else 1
    values, stride = _room(N, K, E if stack else None)
    scales = _empty((E, nb, kb), (nb * kb, kb, 1), torch.float32) if stack else _empty((nb, kb), (kb, 1), torch.float32)
    check(lib().rlis_quantize_matrix(w.data_ptr(), w.stride(-2), w.stride(0) if stack else 0, values.data_ptr(), stride, scales.data_ptr(), E, N, K, code,
                                     _stream()), "quantize_matrix")
    _count("quantize_matrix")
    return BlockMatrix._made(values, scales, stride)


def linear_blocks(x, w: BlockMatrix, out_dtype=None, *, early: bool = False) -> torch.Tensor:
    """y = x @ w^T for a weight in blocks.  x [T, K]: plain rows (bfloat16 or float32; may be a column slice of wider rows), which are put into blocks as
    `quantize_rows` does, or BlockRows, for rows that several products read.  Every block of 128 k is summed on its own in float32, multiplied by the product of both
    scales (which should be a normal float32) and added in float32; the result is rounded once, to `out_dtype` (bfloat16 or float32; None: x's, bfloat16 for
    BlockRows).  Up to 64 rows a row's bits do not depend on the other rows of the call.
    `early`: w is a weight that no kernel still in flight writes, so that its first tiles may be asked for before the kernels before have finished."""
    if not isinstance(w, BlockMatrix) or w.values.dim() != 2:
        raise KernelError("linear_blocks: expected a BlockMatrix [N, K]")
    weight = w.values
    plain = not isinstance(x, BlockRows)
    code = _plain(x, (2,), "linear_blocks") if plain else 1
    T, K = x.shape
    N = weight.shape[0]
    device = weight.get_device()
    if weight.shape[1] != K or (x if plain else x.values).get_device() != device:
        raise KernelError(f"linear_blocks: rows {tuple(x.shape)} on {x.device} and a matrix {tuple(weight.shape)} on {w.device} do not go together")
    out_code = code if out_dtype is None else _FLOATS.get(out_dtype)
    if out_code is None:
        _code(out_dtype)
    if device != _device():
        with torch.cuda.device(device):
            return linear_blocks(x, w, out_dtype, early=early)
    out = _empty((T, N), (N, 1), torch.bfloat16 if out_code else torch.float32)
    if plain:
        kernels = lib()
        room = kernels.rlis_blocks_gemm_scratch(T, N, K)
        scratch = _empty((room,), (1,), torch.uint8) if room else None
        check(kernels.rlis_blocks_gemm_rows(x.data_ptr(), x.stride(0), code, scratch.data_ptr() if room else None, weight.data_ptr(), w.stride, w.scales.data_ptr(), out.data_ptr(), T, N, K,
                                            out_code, int(early), _stream()), "linear_blocks")
        if room:
            _count("quantize_rows")
    else:
        check(lib().rlis_blocks_gemm(x.values.data_ptr(), x.stride, x.scales.data_ptr(), weight.data_ptr(), w.stride, w.scales.data_ptr(), out.data_ptr(), T, N, K,
                                     out_code, int(early), _stream()), "linear_blocks")
    _count("linear_blocks")
    return out


MOE_LAYER_TOKENS = 16           # tokens that `moe_layer` takes
_SCORING = {"sigmoid": 0, "softmax_chosen": 1, "softmax": 2}


class _LayerMatrix(ctypes.Structure):
    _fields_ = [("w", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("row_bytes", ctypes.c_longlong), ("stack_bytes", ctypes.c_longlong)]


class _MoeLayer(ctypes.Structure):
    """A call of the layer (csrc/kernels/moe_layer.cu: RlisMoeLayer)."""
    _fields_ = ([("x", ctypes.c_void_p), ("ldx", ctypes.c_longlong), ("router", ctypes.c_void_p), ("correction", ctypes.c_void_p), ("router_bias", ctypes.c_void_p)]
                + [(n, _LayerMatrix) for n in ("up", "down", "shared_up", "shared_down")] + [("workspace", ctypes.c_void_p), ("out", ctypes.c_void_p)]
                + [(n, ctypes.c_int) for n in ("n_tokens", "width", "inner", "inner_shared", "n_experts", "n_identity", "top", "scoring", "n_groups", "keep_groups",
                                               "normalize", "shared_gate", "interleave", "interleave_shared")]
                + [(n, ctypes.c_float) for n in ("route_scale", "slope", "limit", "shift")])


def _layer_matrix(m, dims: int, rows, k, blocks: bool, device, name: str) -> _LayerMatrix:
    """A matrix of the layer (or a stack of them) of `rows` x `k` (None: any), as the launcher takes it."""
    if isinstance(m, BlockMatrix) != blocks:
        raise KernelError(f"moe_layer: {name}: the layer's matrices are all in bfloat16 or all in blocks")
    t = m.values if blocks else m
    if not isinstance(t, torch.Tensor) or t.device != device or t.dim() != dims or (rows is not None and t.shape[-2] != rows) or (k is not None and t.shape[-1] != k):
        raise KernelError(f"moe_layer: {name}: expected {'a stack of matrices' if dims == 3 else 'a matrix'} of {rows} x {k} on {device}, "
                          f"got {_shape(t)}")
    if blocks:
        return _LayerMatrix(t.data_ptr(), m.scales.data_ptr(), m.stride, t.shape[-2] * m.stride)
    if t.dtype != torch.bfloat16 or not t.is_contiguous():
        raise KernelError(f"moe_layer: {name}: expected contiguous bfloat16 or a BlockMatrix, got {t.dtype} with strides {t.stride()}")
    return _LayerMatrix(t.data_ptr(), None, 2 * t.shape[-1], 2 * t.shape[-2] * t.shape[-1])


def _layer_vector(v, n: int, device, name: str):
    if v is None:
        return None
    if not isinstance(v, torch.Tensor) or v.dtype != torch.float32 or tuple(v.shape) != (n,) or not v.is_contiguous() or v.device != device:
        raise KernelError(f"moe_layer: {name}: expected contiguous float32 [{n}] on {device}")
    return v.data_ptr()


def moe_layer(x: torch.Tensor, w_router: torch.Tensor, w_gate_up, w_down, top: int, route_scale: float = 1.0, *, correction: torch.Tensor | None = None,
              router_bias: torch.Tensor | None = None, scoring: str = "sigmoid", groups: tuple | None = None, normalize: bool = False, n_identity: int = 0,
              shared: tuple | None = None, shared_gate: bool = False, slope: float = 1.0, limit: float | None = None, up_shift: float = 0.0, interleave: int = 0,
              shared_interleave: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """A whole mixture of experts for up to `MOE_LAYER_TOKENS` tokens in two launches: what `moe_route`, `moe_up`, `moe_down`, a shared expert and `moe_combine`
    compute, every weight read once.  x [T, W] bfloat16, rows that start at multiples of 16 bytes (of a wider tensor if need be); the result [T, W] bfloat16 (`out`, or
    a new tensor).

    w_router float32 [experts + n_identity (+ 1), W] (with `shared_gate` its last row is the logit of the shared expert's gate), `correction`, `router_bias`,
    `scoring` ("sigmoid", "softmax" or "softmax_chosen"), `groups`, `normalize` and `n_identity` as `moe_route` takes them; `top` up to 16.
    w_gate_up [experts, 2 I, W] and w_down [experts, W, I], both contiguous bfloat16 or both stacks in blocks; `shared` = (gate|up [2 S, W], down [W, S]) of the
    shared expert in the same form; `interleave` (`shared_interleave`) as `moe_up` takes it (in blocks a multiple of 4); the gating of `glu_act` with
    `slope`, `limit` and `up_shift`.  W, I and S are multiples of 8, in blocks of 16, and at most 16,384; the router has up to 512 outputs.

    Scores and sums are float32; the experts' gated results go into the second product to 2^-17 of each (beside codes to 2^-22, or 2^-39 of the largest of 128 of
    them); a token's result is rounded once.  Its last bits depend on the call's other tokens, whose experts decide how the sums are cut up, and on nothing else.
    An expert's weight that is no number, or infinite, reaches only the tokens that chose it, and a token that is not finite only itself; the router's lie below 2^127."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype != torch.bfloat16 or x.dim() != 2 or x.stride(1) != 1:
        raise KernelError("moe_layer: expected bfloat16 rows [T, W] with unit stride on the device; there is no CPU path")
    dev = x.device
    if x.get_device() != _device():
        with torch.cuda.device(dev):
            return moe_layer(x, w_router, w_gate_up, w_down, top, route_scale, correction=correction, router_bias=router_bias, scoring=scoring, groups=groups,
                             normalize=normalize, n_identity=n_identity, shared=shared, shared_gate=shared_gate, slope=slope, limit=limit, up_shift=up_shift,
                             interleave=interleave, shared_interleave=shared_interleave, out=out)
    T, W = x.shape
    if x.data_ptr() % 16 or (T > 1 and x.stride(0) % 8):
        raise KernelError(f"moe_layer: rows of x start at multiples of 16 bytes, got an address of {x.data_ptr() % 16} beyond one and strides {x.stride()}")
    if T > MOE_LAYER_TOKENS:
        raise KernelError(f"moe_layer: takes up to {MOE_LAYER_TOKENS} tokens, got {T}; more go through moe_route, moe_up, moe_down and moe_combine")
    if scoring not in _SCORING:
        raise KernelError(f"moe_layer: unknown scoring {scoring!r}; known: {sorted(_SCORING)}")
    blocks = isinstance(w_gate_up, BlockMatrix)
    up = _layer_matrix(w_gate_up, 3, None, W, blocks, dev, "w_gate_up")
    E, I2 = w_gate_up.shape[:2]
    down = _layer_matrix(w_down, 3, W, I2 // 2, blocks, dev, "w_down")
    if w_down.shape[0] != E or I2 % 2:
        raise KernelError(f"moe_layer: {E} and {w_down.shape[0]} experts, {I2} rows of gate and linear branch")
    S2, shared_up, shared_down = 0, _LayerMatrix(), _LayerMatrix()
    if shared is not None:
        shared_up = _layer_matrix(shared[0], 2, None, W, blocks, dev, "shared gate|up")
        S2 = shared[0].shape[0]
        shared_down = _layer_matrix(shared[1], 2, W, S2 // 2, blocks, dev, "shared down")
        if S2 % 2 or S2 < 2:
            raise KernelError(f"moe_layer: {S2} rows of the shared expert's gate and linear branch")
    elif shared_gate:
        raise KernelError("moe_layer: a gate on the shared expert, and no shared expert")
    n_out = E + int(n_identity)
    if not isinstance(w_router, torch.Tensor) or w_router.dtype != torch.float32 or tuple(w_router.shape) != (n_out + (1 if shared_gate else 0), W) or not w_router.is_contiguous() or w_router.device != dev:
        raise KernelError(f"moe_layer: expected a contiguous float32 router [{n_out + (1 if shared_gate else 0)}, {W}] on {dev}, got {_shape(w_router)}")
    n_groups, keep = groups if groups is not None else (1, 1)
    if out is None:
        out = _empty((T, W), (W, 1), torch.bfloat16)
    elif not isinstance(out, torch.Tensor) or out.dtype != torch.bfloat16 or tuple(out.shape) != (T, W) or not out.is_contiguous() or out.device != dev:
        raise KernelError(f"moe_layer: out: expected contiguous bfloat16 {(T, W)} on {dev}")
    if T == 0:
        return out
    work = _empty((lib().rlis_moe_layer_bytes(T, int(top), W, I2 // 2, S2 // 2),), (1,), torch.uint8)
    call = _MoeLayer(x.data_ptr(), x.stride(0) if T > 1 else W, w_router.data_ptr(), _layer_vector(correction, n_out, dev, "correction"),
                     _layer_vector(router_bias, n_out, dev, "router_bias"), up, down, shared_up, shared_down, work.data_ptr(), out.data_ptr(), T, W, I2 // 2, S2 // 2, E,
                     int(n_identity), int(top), _SCORING[scoring], int(n_groups), int(keep), 1 if normalize else 0, 1 if shared_gate else 0, int(interleave),
                     int(shared_interleave), float(route_scale), float(slope), float("inf") if limit is None else float(limit), float(up_shift))
    check(lib().rlis_moe_layer(ctypes.addressof(call), _stream()), "moe_layer")
    _count("moe_layer.up" + (".blocks" if blocks else ""))
    _count("moe_layer.down" + (".blocks" if blocks else ""))
    return out
