"""Microscaled 4-bit floats (csrc/mxfp4.hip): quantisation, decoding and dense layers with both operands in that format -- inference
only, like the encoder pieces of ops_vit (`samnerf_amd.ops` re-exports everything here)."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ._opcore import ACT_GELU, ACT_NONE, DTYPE_CODE, _dev, _launch, _p, _rows, _stream_on
from .ops_vit import Planes

__all__ = ["MXFP4_BLOCK", "Mxfp4", "quantize_mxfp4", "dequantize_mxfp4", "linear_mxfp4"]

MXFP4_BLOCK = 32  # values that share a scale
MXFP4_ROWS = 16   # SNF_MXFP4_ROWS


class Mxfp4:
    """A matrix [M, K] in blocks of 32 values along K: e2m1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign), one power-of-two scale a block.

    codes uint8 [8 C, M, 16] and scales uint8 [2 C, M, 4], C = ceil(K / 256), in the order in which the product reads them (the layout
    stands in include/samnerf_hip.h); `shape` is the shape of the tensor that was quantised.  17 / 32 byte a value."""
    __slots__ = ("_data", "_codes", "_scales", "M", "K", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, K: int, shape: Optional[Tuple[int, ...]] = None):
        chunks = -(-int(K) // 256)
        if K < 1 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("Mxfp4: K >= 1, uint8 codes and uint8 scales expected")
        if codes.dim() != 3 or codes.shape[0] != 8 * chunks or codes.shape[2] != 16:
            raise ValueError(f"Mxfp4: codes of K={K} have shape [{8 * chunks}, M, 16], got {tuple(codes.shape)}")
        self.M, self.K = int(codes.shape[1]), int(K)
        if tuple(scales.shape) != (2 * chunks, self.M, 4):
            raise ValueError(f"Mxfp4: scales of [{self.M}, {K}] have shape [{2 * chunks}, {self.M}, 4], got {tuple(scales.shape)}")
        if codes.device != scales.device or not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("Mxfp4: codes and scales are contiguous and on one device")
        self.shape = tuple(shape) if shape is not None else (self.M, self.K)
        n = 1
        for d in self.shape[:-1]:
            n *= d
        if self.shape[-1] != self.K or n != self.M:
            raise ValueError(f"Mxfp4: {self.shape} is not a shape of {self.M} rows of {self.K}")
        self._data, self._codes, self._scales = codes, codes, scales

    @classmethod
    def _new(cls, M: int, K: int, device, shape) -> "Mxfp4":
        """Room for a matrix: codes and scales in one allocation, which the caller's kernel fills."""
        q = object.__new__(cls)
        q._data = torch.empty((-(-K // 256) * 136 * M,), device=device, dtype=torch.uint8)
        q._codes = q._scales = None
        q.M, q.K, q.shape = M, K, shape
        return q

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            n = -(-self.K // 256)
            self._codes = self._data[:n * 128 * self.M].view(8 * n, self.M, 16)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            n = -(-self.K // 256)
            self._scales = self._data[n * 128 * self.M:].view(2 * n, self.M, 4)
        return self._scales

    def _pointers(self) -> Tuple[int, int]:
        if self._scales is not None:
            return self.codes.data_ptr(), self._scales.data_ptr()
        p = self._data.data_ptr()
        return p, p + -(-self.K // 256) * 128 * self.M

    @property
    def device(self) -> torch.device:
        return self._data.device

    def float(self) -> torch.Tensor:
        """The values as float32, in the shape that was quantised."""
        return dequantize_mxfp4(self)


def quantize_mxfp4(x: Union[torch.Tensor, Planes]) -> Mxfp4:
    """x [..., K] (float32 / bfloat16 / float16; rows may be strided; or the encoder's operand planes) -> Mxfp4.  Per block of 32 along K the scale is
    2^max(floor(log2 max|x|) - 2, -127); values are rounded to the nearest code (halves to even), magnitudes above 6 scales become 6.
    Blocks with an infinity or a NaN become NaN as a whole.  The last block of a K that 32 does not divide is filled with zeros.  No
    gradient flows through it."""
    if isinstance(x, Planes):
        dev = _dev(x.hi, "x")
        q = Mxfp4._new(x.M, x.K, x.hi.device, (x.M, x.K))
        _launch("snf_mxfp4_quantize_planes", _p(x.hi), _p(x.lo), x.M, x.K, *q._pointers(), _stream_on(dev), units=4.0 * x.M * x.K)
        return q
    if not isinstance(x, torch.Tensor) or x.dtype not in DTYPE_CODE:
        raise TypeError(f"quantize_mxfp4: float32, bfloat16 or float16 expected, got {getattr(x, 'dtype', type(x))}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_mxfp4: rows of at least one value expected, got {tuple(x.shape)}")
    dev = _dev(x, "x")
    shape = x.shape
    K = shape[-1]
    M = x.numel() // K
    q = Mxfp4._new(M, K, x.device, shape)
    if M:
        x, ld = _rows(x.detach() if x.requires_grad else x)
        _launch("snf_mxfp4_quantize", _p(x), DTYPE_CODE[x.dtype], M, K, ld, *q._pointers(), _stream_on(dev),
                units=float(M * K * x.element_size()))
    return q


def dequantize_mxfp4(q: Mxfp4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that `q` holds, in its shape.  float32 holds every value exactly; so does the type that was quantised."""
    if not isinstance(q, Mxfp4):
        raise TypeError(f"dequantize_mxfp4: an Mxfp4 expected, got {type(q)}")
    if dtype not in DTYPE_CODE:
        raise TypeError(f"dequantize_mxfp4: float32, bfloat16 or float16 expected, got {dtype}")
    dev = _dev(q._data, "q")
    out = torch.empty(q.shape, device=q._data.device, dtype=dtype)
    if q.M:
        _launch("snf_mxfp4_dequantize", *q._pointers(), q.M, q.K, _p(out), DTYPE_CODE[dtype], _stream_on(dev),
                units=float(out.numel() * out.element_size()))
    return out


def linear_mxfp4(x: Union[torch.Tensor, Mxfp4, Planes], w: Mxfp4, bias: Optional[torch.Tensor] = None, act: int = ACT_NONE,
                 out_dtype: Optional[torch.dtype] = None, quantized: bool = False) -> Union[torch.Tensor, Mxfp4]:
    """act(x W^T + bias) with both operands in 4 bits and float32 sums: x [..., K] is quantised on the way in (rows, or the
    encoder's operand planes) or comes as an Mxfp4,
    w = quantize_mxfp4(weight [N, K]) once per checkpoint, bias [N] float32, act one of ops.ACT_*.  The result [..., N] has x's type
    (float32 for an Mxfp4 or planes) unless out_dtype says otherwise; quantized=True returns quantize_mxfp4 of the float32 result instead (an operand
    of the next layer; written by the product itself where N is a multiple of 256).  Inference only: an x that requires a gradient is
    refused under grad mode, weight and bias get none."""
    if isinstance(x, Planes):
        x = quantize_mxfp4(x)
    if not isinstance(w, Mxfp4) or len(w.shape) != 2:
        raise TypeError("linear_mxfp4: w is quantize_mxfp4(weight) of a weight [N, K]")
    if not isinstance(x, Mxfp4):
        if not isinstance(x, torch.Tensor) or x.dtype not in DTYPE_CODE:
            raise TypeError(f"linear_mxfp4: x is float32, bfloat16, float16 or an Mxfp4, got {getattr(x, 'dtype', type(x))}")
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("linear_mxfp4: x requires a gradient, and none flows through the product (torch.no_grad(), or x.detach())")
    if len(x.shape) < 1 or x.shape[-1] != w.K:
        raise ValueError(f"linear_mxfp4: x {tuple(x.shape)} does not end in the weight's {w.K} columns")
    if w.M < 1:
        raise ValueError("linear_mxfp4: a weight without rows")
    if not ACT_NONE <= int(act) <= ACT_GELU:
        raise ValueError(f"linear_mxfp4: unknown activation {act}")
    if quantized:
        if out_dtype not in (None, torch.float32):
            raise ValueError(f"linear_mxfp4: a quantized result comes from float32, not from {out_dtype}")
        out_dtype = torch.float32
    if out_dtype is None:
        out_dtype = torch.float32 if isinstance(x, Mxfp4) else x.dtype
    if out_dtype not in DTYPE_CODE:
        raise TypeError(f"linear_mxfp4: the result is float32, bfloat16 or float16, not {out_dtype}")
    dev = _dev(w._data, "w")
    _dev(x._data if isinstance(x, Mxfp4) else x, "x", dev)
    if bias is not None:
        _dev(bias, "bias", dev)
        if bias.dtype != torch.float32 or tuple(bias.shape) != (w.M,):
            raise ValueError(f"linear_mxfp4: bias is float32 [{w.M}], got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    shape, place = (*x.shape[:-1], w.M), w._data.device
    if quantized:
        q = x if isinstance(x, Mxfp4) else quantize_mxfp4(x)
        if w.M % 256:
            return quantize_mxfp4(linear_mxfp4(q, w, bias, act))
        out = Mxfp4._new(q.M, w.M, place, shape)
        _launch("snf_mxfp4_linear_quantized", *q._pointers(), *w._pointers(), _p(bias), q.M, q.K, w.M, int(act), *out._pointers(),
                _stream_on(dev), tag=f"{q.K}x{w.M}", units=2.0 * q.M * q.K * w.M)
        return out
    y = torch.empty(shape, device=place, dtype=out_dtype)
    if y.numel() == 0:
        return y
    if isinstance(x, Mxfp4):
        q = x
    elif y.numel() <= MXFP4_ROWS * w.M:  # few rows: quantised on the way into the product, one launch
        x, ld = _rows(x.detach() if x.requires_grad else x)
        _launch("snf_mxfp4_linear_rows", _p(x), DTYPE_CODE[x.dtype], ld, *w._pointers(), _p(bias), x.shape[0], w.K, w.M, int(act), _p(y),
                DTYPE_CODE[out_dtype], _stream_on(dev), tag=f"{w.K}x{w.M}", units=2.0 * y.numel() * w.K)
        return y
    else:
        q = quantize_mxfp4(x)
    _launch("snf_mxfp4_linear", *q._pointers(), *w._pointers(), _p(bias), q.M, q.K, w.M, int(act), _p(y),
            DTYPE_CODE[out_dtype], _stream_on(dev), tag=f"{q.K}x{w.M}", units=2.0 * q.M * q.K * w.M)
    return y
