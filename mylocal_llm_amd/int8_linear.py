"""Linear and SwiGLU products of 8-bit integer codes on the device.

Both sides are int8: weights with a scale for each output channel, activations with a scale for each
token, quantised on the way (``int8_quantize``) or given as codes.  The sum of code products is exact
in int32 and scaled in 64 bits, so a result is ``(sum q w) * s * c`` rounded to fp32 and then to the output
type; its bits depend on its own row and channel only, not on the number of tokens, the other rows or where it
lies.  The reference keeps activations in floating point (mini_llm/ops/quantized_linear.py:272-400);
these operators stand beside ``quantized_linear`` / ``quantized_swiglu``, which take an ``Int8Weight``
wherever they take a packed GGUF weight.
"""
from functools import lru_cache

import torch

from . import _lib
from .quantized_linear import _TORCH_DTYPE_ID, DevicePackedGGUFWeight

MAX_K = 131071            # 128 * 128 * K stays inside int32
_INT8 = 3                 # QMOE_DT_INT8
_MOST = 2 ** 31 - 1       # what the C entries' sizes hold


def _call(device, function, *args):
    """``function(*args, stream)`` on ``device``'s current stream, with that device current; its status."""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        return function(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return function(*args, torch._C._cuda_getCurrentRawStream(index))


@lru_cache(maxsize=4096)
def _workspace_bytes(n, k, tokens, x_dtype):
    return _lib.load().qmoe_int8_workspace_bytes(n, k, tokens, x_dtype)


def _workspace(x, n, k, tokens, x_dtype):
    """(tensor or None, address, bytes) of a product's scratch; codes that the kernels read as they are need none."""
    nbytes = _workspace_bytes(n, k, tokens, x_dtype)
    if not nbytes or (x_dtype == _INT8 and k % 256 == 0 and x.data_ptr() % 16 == 0):
        return None, None, 0
    work = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    return work, work.data_ptr(), nbytes


def _check_rows(x, what):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError(f"{what} must be a CUDA torch.Tensor")
    if x.ndim < 1 or not x.shape[-1]:
        raise ValueError(f"{what} must have rows of at least one column")
    if not x.is_contiguous():
        raise ValueError(f"{what} must be a contiguous tensor")


def int8_quantize(x):
    """Codes and scales of the rows of ``x`` [..., K] (fp32 / fp16 / bf16, contiguous, on the device).

    ``s = max|x| / 127`` in fp32, ``q = x / s`` rounded to the nearest whole number, halves to even.
    Returns int8 codes of ``x``'s shape and fp32 scales of shape ``x.shape[:-1]``.  A row of zeros has the
    scale 0; a row with a NaN or an infinity the scale NaN and codes of 0.
    """
    _check_rows(x, "Rows to quantise")
    if x.dtype not in _TORCH_DTYPE_ID:
        raise TypeError("Rows to quantise must be FP16, BF16, or FP32")
    k = x.shape[-1]
    rows = x.numel() // k
    if k > _MOST or rows > _MOST:
        raise NotImplementedError(f"Rows to quantise: at most {_MOST} rows and columns")
    codes = torch.empty_like(x, dtype=torch.int8)
    scales = x.new_empty(rows, dtype=torch.float32) if x.ndim == 2 else x.new_empty(x.shape[:-1], dtype=torch.float32)
    if rows:
        rc = _call(x.device, _lib.load().qmoe_int8_quantize, x.data_ptr(), _TORCH_DTYPE_ID[x.dtype], rows, k,
                   codes.data_ptr(), scales.data_ptr())
        if rc:
            _lib.check(rc, "Int8 quantisation")
    return codes, scales


def _tiles_of(codes, scales, dims, what):
    """Row-major codes [..., N, K] -> the kernels' tile layout, one matrix behind the other."""
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda or codes.dtype != torch.int8:
        raise TypeError(f"{what} codes must be a CUDA torch.int8 tensor")
    if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or scales.device != codes.device:
        raise TypeError(f"{what} scales must be a torch.float32 tensor on the codes' device")
    if codes.ndim != dims or min(codes.shape) < 1 or tuple(scales.shape) != tuple(codes.shape[:-1]):
        raise ValueError(f"{what} needs codes {'[E, N, K]' if dims == 3 else '[N, K]'} and a scale for each row")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{what} codes and scales must be contiguous")
    n, k = codes.shape[-2:]
    if n > _MOST:
        raise NotImplementedError(f"{what}: at most {_MOST} rows a matrix")
    if k > MAX_K:
        raise NotImplementedError(f"{what}: K beyond {MAX_K}, where an int32 sum could overflow")
    count = codes.shape[0] if dims == 3 else 1
    lib = _lib.load()
    tiles = torch.empty(count * lib.qmoe_int8_matrix_bytes(n, k), dtype=torch.uint8, device=codes.device)
    _lib.check(_call(codes.device, lib.qmoe_int8_tiles, codes.data_ptr(), count, n, k, tiles.data_ptr()), what)
    return tiles


class Int8Weight:
    """One [N, K] matrix of int8 codes with an fp32 scale for each of its N rows, on the device.

    The codes are laid out once for the kernels; the caller's ``codes`` are not kept.  ``scales`` is kept
    and read by every product.
    """

    def __init__(self, codes, scales):
        self.tiles = _tiles_of(codes, scales, 2, "Int8 weight")
        self.scales = scales
        self.shape = tuple(int(i) for i in codes.shape)
        self.device = codes.device

    @classmethod
    def quantize(cls, dense):
        """From a dense float matrix [N, K]: each row quantised as ``int8_quantize`` does."""
        if not isinstance(dense, torch.Tensor) or dense.ndim != 2:
            raise ValueError("Int8 weights are made from a dense [N, K] tensor")
        return cls(*int8_quantize(dense))

    @classmethod
    def from_packed(cls, packed):
        """From a packed GGUF matrix on the device: its dequantised rows, quantised."""
        if not isinstance(packed, DevicePackedGGUFWeight):
            raise TypeError("Expected DevicePackedGGUFWeight")
        return cls.quantize(packed.dequantize())

    @property
    def nbytes(self):
        return int(self.tiles.numel()) + 4 * self.shape[0]

    def codes(self):
        """The codes as a row-major int8 [N, K] tensor."""
        return _codes_of(self.tiles, self.shape)

    def dequantize(self):
        """Dense fp32 [N, K]."""
        return self.codes().to(torch.float32) * self.scales[:, None]


def _codes_of(tiles, shape):
    n, k = shape
    rows, cols = (n + 15) // 16, (k + 63) // 64
    blocks = tiles.view(torch.int8).reshape(rows, cols, 4, 16, 16)          # [row tile, column tile, column group, row, column]
    return blocks.permute(0, 3, 1, 2, 4).reshape(rows * 16, cols * 64)[:n, :k].contiguous()


def _activations(x, x_scales, k, device, out_dtype, what):
    """(rows, x's type id, scale address, output type) of a product's activations, checked."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError(f"{what} must be a CUDA torch.Tensor")
    if x.ndim not in (2, 3):
        raise ValueError("Expected x as [M, K] or [B, T, K]")
    if x.shape[-1] != k:
        raise ValueError("Input K does not match the weight's K")
    if not x.is_contiguous():
        raise ValueError("GPU input must be a contiguous tensor")
    if x.device != device:
        raise ValueError("all operands must be on the same device")
    m = x.numel() // k
    if m > _MOST:
        raise NotImplementedError(f"{what}: at most {_MOST} rows")
    if out_dtype is not None and out_dtype not in _TORCH_DTYPE_ID:
        raise TypeError("out_dtype must be FP16, BF16, or FP32")
    if x.dtype == torch.int8:
        if not isinstance(x_scales, torch.Tensor) or x_scales.dtype != torch.float32 or x_scales.device != device:
            raise TypeError("int8 input needs x_scales, a torch.float32 tensor on its device")
        if x_scales.shape != x.shape[:-1] or not x_scales.is_contiguous():
            raise ValueError("x_scales must be contiguous with one scale for each row of x")
        return m, _INT8, x_scales.data_ptr(), torch.float32 if out_dtype is None else out_dtype
    if x.dtype not in _TORCH_DTYPE_ID:
        raise TypeError("GPU input must be FP16, BF16, FP32 or int8 codes")
    if x_scales is not None:
        raise ValueError("x_scales belong to int8 input")
    return m, _TORCH_DTYPE_ID[x.dtype], None, x.dtype if out_dtype is None else out_dtype


def int8_linear(x, weight, *, x_scales=None, out_dtype=None):
    """``x @ weight.T`` on 8-bit codes.

    ``x`` is a contiguous [M, K] or [B, T, K] tensor, fp32 / fp16 / bf16 (its rows are quantised on the way)
    or int8 codes with ``x_scales`` (fp32, ``x.shape[:-1]``).  The result has shape ``x.shape[:-1] + (N,)`` and
    ``out_dtype`` (default: x's type, fp32 for codes).
    """
    if not isinstance(weight, Int8Weight):
        raise TypeError("Expected Int8Weight")
    n, k = weight.shape
    m, xdt, sp, odt = _activations(x, x_scales, k, weight.device, out_dtype, "Int8 linear input")
    out = x.new_empty(m, n, dtype=odt) if x.ndim == 2 else x.new_empty((*x.shape[:-1], n), dtype=odt)
    if m:
        work, at, nbytes = _workspace(x, n, k, m, xdt)
        rc = _call(x.device, _lib.load().qmoe_int8_linear, weight.tiles.data_ptr(), weight.scales.data_ptr(), n, k, x.data_ptr(), xdt, sp,
                   m, out.data_ptr(), _TORCH_DTYPE_ID[odt], at, nbytes)
        if rc:
            _lib.check(rc, "Int8 linear")
    return out


def int8_swiglu(x, gate, up, *, x_scales=None, out_dtype=None):
    """``SiLU(x @ gate.T) * (x @ up.T)`` on 8-bit codes in one product, in 64 bits up to the one rounding to fp32 (and
    then to the output type); arguments as ``int8_linear``."""
    if not isinstance(gate, Int8Weight) or not isinstance(up, Int8Weight):
        raise TypeError("gate and up must be Int8Weight")
    if gate.shape != up.shape:
        raise ValueError("gate/up must share two-dimensional [F,K] shape")
    if gate.device != up.device:
        raise ValueError("all operands must be on the same device")
    f, k = gate.shape
    m, xdt, sp, odt = _activations(x, x_scales, k, gate.device, out_dtype, "Int8 SwiGLU input")
    out = x.new_empty(m, f, dtype=odt) if x.ndim == 2 else x.new_empty((*x.shape[:-1], f), dtype=odt)
    if m:
        work, at, nbytes = _workspace(x, f, k, m, xdt)
        rc = _call(x.device, _lib.load().qmoe_int8_swiglu, gate.tiles.data_ptr(), gate.scales.data_ptr(), up.tiles.data_ptr(),
                   up.scales.data_ptr(), f, k, x.data_ptr(), xdt, sp, m, out.data_ptr(), _TORCH_DTYPE_ID[odt], at, nbytes)
        if rc:
            _lib.check(rc, "Int8 SwiGLU")
    return out
