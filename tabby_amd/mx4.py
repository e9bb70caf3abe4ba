"""Microscaled 4-bit floating point (MXFP4) on the GPU: conversion, the way back, and the
product of two such matrices, over the C ABI's ``tabby_mx4_*`` entries.

It stands beside ``sampler.LmHeadQ4`` (the reference's int4 lm_head, src/engine/forward.ts:
408-428, 732-770) for checkpoints whose weights are MXFP4: values of 4 bits (e2m1) in blocks
of 32 along a row, each block with a power of two of its own. ``LmHeadMx4.logits`` quantises the
hidden states as well, so that the product runs on the matrix cores' scaled 4-bit instructions.

Every call is asynchronous on the given stream (default: torch's current one) and checks its
arguments before any GPU work.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional

import torch

from .sampler import TABBY_BF16, TABBY_F16, TABBY_F32, _check, load_library

BLOCK = 32  # values to a scale
PANEL_ROWS, PANEL_COLS = 64, 128  # a panel's codes take 4,096 bytes, its scales 256

_CODES = {torch.float32: TABBY_F32, torch.float16: TABBY_F16, torch.bfloat16: TABBY_BF16}


def dtype_code(dtype) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise TypeError(f"expected float32, float16 or bfloat16, got {dtype}")
    return code


INT32_MAX = 2 ** 31 - 1  # of the C entries' sizes; ctypes would take larger ones modulo 2^32


def rows_of(x, what: str):
    """A CUDA tensor as rows: 1-D becomes one row; a row's elements must be adjacent."""
    if not x.is_cuda:
        raise ValueError(f"{what} must be a device (cuda) tensor")
    if x.dim() != 2:
        if x.dim() != 1:
            raise ValueError(f"{what} must have one or two dimensions, got {x.dim()}")
        x = x.unsqueeze(0)
    rows, cols = x.shape
    if rows < 1 or cols < 1:
        raise ValueError(f"{what} must not be empty, got {tuple(x.shape)}")
    if rows > INT32_MAX or cols > INT32_MAX:
        raise ValueError(f"{what}'s rows and columns must fit 32 bits, got {tuple(x.shape)}")
    row_stride, stride = x.stride()
    if (cols > 1 and stride != 1) or (rows > 1 and row_stride < cols):
        raise ValueError(f"{what} must hold its rows' elements adjacent and its rows apart")
    return x


def on_device(device, *tensors):
    for t in tensors:
        if t.device != device:
            raise ValueError(f"tensors lie on {device} and on {t.device}")


_HERE = contextlib.nullcontext()


@contextlib.contextmanager
def _guard(device, stream):
    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield


def _current_handle(index):
    return torch.cuda.current_stream(index).cuda_stream


# The current stream's handle without the object around it, which takes longer to make than a launch, and the
# device without the check that a tensor's existence has passed.
_current_handle = getattr(torch._C, "_cuda_getCurrentRawStream", _current_handle)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def call_on(device, stream):
    """(context, stream handle) of a call on ``device``: the device is made current where it is
    not, and what the call allocates belongs to its stream."""
    if stream is None:
        index = device.index
        if index == _current_device():
            return _HERE, _current_handle(index)
        stream = torch.cuda.current_stream(device)
    elif stream.device != device:
        raise ValueError(f"the stream belongs to {stream.device}, the tensors to {device}")
    return _guard(device, stream), stream.cuda_stream


def sizes(rows: int, cols: int):
    """Bytes of a matrix's codes and scales."""
    if rows < 2 ** 20 and cols < 2 ** 20 and rows > 0 and cols > 0:
        panels = -(-rows // PANEL_ROWS) * -(-cols // PANEL_COLS)
        return panels * 4096, panels * 256
    if rows > INT32_MAX or cols > INT32_MAX:
        raise ValueError(f"rows and columns must fit 32 bits, got {rows} x {cols}")
    code, scale = ctypes.c_int64(), ctypes.c_int64()
    _check(load_library().tabby_mx4_bytes(rows, cols, ctypes.byref(code), ctypes.byref(scale)))
    return code.value, scale.value


class Mx4Matrix:
    """A [rows, cols] matrix in MXFP4 on the device, in the library's panel layout. Its buffers may
    be written again with ``quantize(x, out=matrix)``."""

    def __init__(self, rows: int, cols: int, device="cuda"):
        self.rows, self.cols = int(rows), int(cols)
        self._code_bytes, scale = sizes(self.rows, self.cols)
        self.data = torch.empty(self._code_bytes + scale, dtype=torch.uint8, device=device)  # codes, then scales

    @property
    def codes(self):
        return self.data[:self._code_bytes]

    @property
    def scales(self):
        return self.data[self._code_bytes:]

    @classmethod
    def quantize(cls, x, out: Optional["Mx4Matrix"] = None, stream=None) -> "Mx4Matrix":
        """``x`` ([rows, cols] or [cols], float32, float16 or bfloat16) rounded to MXFP4: a block's
        power of two is floor(log2(max |x|)) - 2, values go to the nearest code (ties to even, at
        most 6); a block with a NaN or an infinity becomes NaN."""
        x = rows_of(x, "x")
        code = dtype_code(x.dtype)
        rows, cols = x.shape
        device = x.device
        if out is not None:
            if (out.rows, out.cols) != (rows, cols):
                raise ValueError(f"out is {out.rows} x {out.cols}, x is {rows} x {cols}")
            on_device(device, out.data)
        ctx, handle = call_on(device, stream)
        with ctx:
            m = cls(rows, cols, device) if out is None else out
            at = m.data.data_ptr()
            _check(load_library().tabby_mx4_quantize_device(
                x.data_ptr(), code, rows, cols, x.stride(0), at, at + m._code_bytes, handle))
        return m

    @classmethod
    def from_rowmajor(cls, codes, scales, cols: int, stream=None) -> "Mx4Matrix":
        """A checkpoint's layout, repacked once: ``codes`` uint8 [rows, ceil(cols / 32) * 16], two to a
        byte with the lower column in the low half, ``scales`` uint8 [rows, ceil(cols / 32)], the
        biased exponents."""
        blocks = -(-int(cols) // BLOCK)
        if not codes.is_cuda or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("codes and scales must be uint8 device (cuda) tensors")
        if codes.dim() != 2 or codes.shape[0] < 1 or cols < 1 or codes.shape[1] != blocks * BLOCK // 2:
            raise ValueError(f"codes must have shape (rows, {blocks * BLOCK // 2}), got {tuple(codes.shape)}")
        if tuple(scales.shape) != (codes.shape[0], blocks):
            raise ValueError(f"scales must have shape ({codes.shape[0]}, {blocks}), got {tuple(scales.shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        on_device(codes.device, scales)
        ctx, handle = call_on(codes.device, stream)
        with ctx:
            m = cls(int(codes.shape[0]), int(cols), codes.device)
            at = m.data.data_ptr()
            _check(load_library().tabby_mx4_pack_device(
                codes.data_ptr(), scales.data_ptr(), m.rows, m.cols, at, at + m._code_bytes, handle))
        return m

    def dequantize(self, dtype=None, out=None, stream=None):
        """The values that the codes stand for, [rows, cols]: exact in float32 (the default) and
        bfloat16, rounded once in float16."""
        rows, cols, device = self.rows, self.cols, self.data.device
        if out is None:
            dtype = dtype or torch.float32
            code = dtype_code(dtype)
        else:
            code = _result_code(out, dtype, rows, cols, device)
            out = rows_of(out, "out")
        ctx, handle = call_on(device, stream)
        with ctx:
            if out is None:
                out = torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)
            at = self.data.data_ptr()
            _check(load_library().tabby_mx4_dequantize_device(
                at, at + self._code_bytes, rows, cols, out.data_ptr(), code, out.stride(0), handle))
        return out


def _result_code(out, dtype, rows: int, cols: int, device) -> int:
    """The type code of a tensor that a caller has results written to, once it is seen to fit."""
    if dtype is not None and out.dtype != dtype:
        raise ValueError(f"out is {out.dtype}, asked for {dtype}")
    code = dtype_code(out.dtype)
    if tuple(rows_of(out, "out").shape) != (rows, cols):
        raise ValueError(f"out must have shape ({rows}, {cols}), got {tuple(out.shape)}")
    on_device(device, out)
    return code


def matmul(x, w: Mx4Matrix, bias=None, dtype=None, out=None, stream=None):
    """x W^T (+ bias), [rows, w.rows] of ``dtype`` (float32 by default): ``x`` is an ``Mx4Matrix``
    or a float tensor ([rows, k] or [k]), which is quantised in the call and may share memory with
    ``out``. Products of codes are exact, their sums float32, rounded once to ``dtype``."""
    device = w.data.device
    quantized = isinstance(x, Mx4Matrix)
    if not quantized:
        x = rows_of(x, "x")
        x_code = dtype_code(x.dtype)
        on_device(device, x)
    else:
        on_device(device, x.data)
    rows, k = (x.rows, x.cols) if quantized else x.shape
    if k != w.cols:
        raise ValueError(f"x has {k} columns, the weights {w.cols}")
    n = w.rows
    bias_at = None
    if bias is not None:
        on_device(device, bias)
        if bias.dtype != torch.float32 or not bias.is_contiguous() or tuple(bias.shape) != (n,):
            raise ValueError(f"bias must be a contiguous float32 tensor of {n} entries")
        bias_at = bias.data_ptr()
    if out is None:
        dtype = dtype or torch.float32
        code = dtype_code(dtype)
    else:
        code = _result_code(out, dtype, rows, n, device)
        out = rows_of(out, "out")
    lib = load_library()
    w_at = w.data.data_ptr()
    ctx, handle = call_on(device, stream)
    with ctx:
        if out is None:
            out = torch.empty_strided((rows, n), (n, 1), dtype=dtype, device=device)
        if quantized:
            x_at = x.data.data_ptr()
            _check(lib.tabby_mx4_matmul_device(
                x_at, x_at + x._code_bytes, rows, w_at, w_at + w._code_bytes, bias_at, n, k, out.data_ptr(), code,
                out.stride(0), handle))
        else:
            size = sum(sizes(rows, k))
            space = torch.empty(size, dtype=torch.uint8, device=device)
            _check(lib.tabby_mx4_linear_device(
                x.data_ptr(), x_code, x.stride(0), rows, w_at, w_at + w._code_bytes, bias_at, n, k, out.data_ptr(),
                code, out.stride(0), space.data_ptr(), size, handle))
    return out


class LmHeadMx4:
    """An lm_head with MXFP4 weights [vocab, hidden] and an optional float32 bias [vocab]."""

    def __init__(self, weight: Mx4Matrix, bias=None):
        self.weight, self.bias = weight, bias
        self.vocab, self.hidden = weight.rows, weight.cols

    def logits(self, hidden_states, dtype=None, out=None, stream=None):
        """Logits [rows, vocab] (float32 by default) of hidden states [rows, hidden] or [hidden]."""
        return matmul(hidden_states, self.weight, self.bias, dtype=dtype, out=out, stream=stream)
