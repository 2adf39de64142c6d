"""Linear layers in 8-bit floating point with a scale for every block of 128 values.

Values are e4m3 codes times a power of two: ``k = min {k : max |x| <= 448 * 2^k}`` over the block, ``code = e4m3(x * 2^-k)``.
The division is exact, so a value is rounded once, at most half a step (2^-4 relative to it, for what is not below
2^-14.8 of the block's maximum).  Activations and gradients have a scale for every 128 values along the contraction of
the product that reads them, weights one for every 128 x 128 tile, so that a weight and its transpose share their codes:

    y = Q(x) Q(w)^T          dx = Q(dy) Q(w)          dw = Q(dy^T) Q(x^T)^T

with sums in fp32, on the GPU those of its matrix units: 32 products at a time are added to a 32-bit sum, which is cut off, not
rounded (so are products some 2^25 below the sum): 8192 products of one sign come out low by 4e-6 of their sum on average in
the kernel for many rows, by 2e-7 in that for few, by nothing in that for up to eight tokens.  A NaN or an infinity becomes
the NaN code (it reaches every output that reads it) and leaves its block's scale alone.  The reference project has no
counterpart.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from maester_b200.ops import reference as ref
from maester_b200.ops.functional import _C

_TYPES = (torch.bfloat16, torch.float32)


class Fp8Blocks:
    """A matrix [rows, cols] as e4m3 codes with power-of-two block scales.

    ``data``: float8_e4m3fn [rows, cols rounded up to 128], zeros past ``cols``; ``scales``: uint8
    [ceil(rows / 128), ceil(blocks / 4), 32, 4, 4], the biased exponent of row ``128 t + 32 i + j`` and block ``4 u + b`` at
    [t, u, j, i, b] (the order in which the matrix unit reads them), zeros past the end."""

    __slots__ = ("data", "scales", "cols")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, cols: int):
        if data.dtype != torch.float8_e4m3fn or data.dim() != 2 or not data.is_contiguous():
            raise TypeError("codes have to be a contiguous float8_e4m3fn matrix")
        blocks = data.shape[1] // ref.FP8_BLOCK
        if data.shape[1] % ref.FP8_BLOCK or not 0 <= data.shape[1] - cols < ref.FP8_BLOCK:
            raise ValueError(f"{cols} columns need codes of {-(-cols // 128) * 128} columns, got {data.shape[1]}")
        want = (-(-data.shape[0] // 128), -(-blocks // 4), 32, 4, 4)
        if scales.dtype != torch.uint8 or tuple(scales.shape) != want or not scales.is_contiguous():
            raise ValueError(f"scales have to be contiguous uint8 {want}, got {scales.dtype} {tuple(scales.shape)}")
        if scales.device != data.device:
            raise ValueError(f"scales are on {scales.device}, codes on {data.device}")
        if data.is_cuda and (data.data_ptr() | scales.data_ptr()) & 15:
            raise ValueError("codes and scales have to start on a 16-byte boundary (parts of a larger buffer may not)")
        self.data, self.scales, self.cols = data, scales, cols

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def shape(self) -> tuple[int, int]:
        return self.data.shape[0], self.cols

    @property
    def device(self) -> torch.device:
        return self.data.device

    def exponents(self) -> torch.Tensor:
        """uint8 [rows, blocks]: the scale of block b of row r is ``2^(exponents[r, b] - 127)``."""
        return ref.fp8_unpack_exponents(self.scales, self.rows, self.data.shape[1] // ref.FP8_BLOCK)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return ref.fp8_dequantize(self.data, self.exponents())[:, :self.cols].to(dtype)


def _quantized(x: torch.Tensor, square: bool = False) -> torch.Tensor:
    """On the CPU: what the codes of a matrix (blocks along its rows) stand for."""
    return ref.fp8_dequantize(*ref.fp8_quantize(x, square))[:, :x.shape[1]]


def _forward(x: torch.Tensor, w: torch.Tensor, keep_x: bool, keep_w: bool):
    """(y, x^T | None, w^T | None) with the transposes in the form that ``_backward`` takes."""
    if x.is_cuda:
        return _C().fp8_linear_fwd(x, w, keep_x, keep_w)
    y = (_quantized(x) @ _quantized(w, True).T).to(x.dtype)
    return y, _quantized(x.T) if keep_x else None, _quantized(w.T, True) if keep_w else None


def _backward(dy: torch.Tensor, K: int, x_t, w_t, dw: torch.Tensor | None, accumulate: bool) -> torch.Tensor | None:
    """dx | None; the weight's gradient goes into ``dw``."""
    if dy.is_cuda:
        return _C().fp8_linear_bwd(dy, K, x_t, w_t, dw, accumulate)
    if x_t is not None:
        value = _quantized(dy.T) @ x_t.T
        dw.add_(value) if accumulate else dw.copy_(value)
    return None if w_t is None else (_quantized(dy) @ w_t.T).to(dy.dtype)


def _as_matrix(x: torch.Tensor) -> torch.Tensor:
    x2 = x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    return x2 if x2.stride(1) == 1 or x2.shape[1] == 1 else x2.contiguous()


def quantize_fp8(x: torch.Tensor, *, square: bool = False, transpose: bool = False) -> Fp8Blocks:
    """Codes of a matrix (bf16 or fp32): one scale for every 128 values of a row, or (``square``) for every 128 x 128 tile.
    ``transpose``: codes of ``x.T`` instead, from the same single pass over ``x``."""
    if x.dim() != 2 or 0 in x.shape:
        raise ValueError(f"a matrix that is not empty is wanted, got {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise TypeError(f"bf16 or fp32 is wanted, got {x.dtype}")
    x = x.detach()
    x = x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()
    if x.is_cuda:
        codes, scales = _C().fp8_quantize(x, not transpose, transpose, square)[int(transpose)]
    else:
        codes, exps = ref.fp8_quantize(x.T if transpose else x, square)
        scales = ref.fp8_pack_exponents(exps)
    return Fp8Blocks(codes, scales, x.shape[0] if transpose else x.shape[1])


def matmul_fp8(a: Fp8Blocks, b: Fp8Blocks, *, out_dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """``a @ b.T`` [a.rows, b.rows] with fp32 sums, rounded once to ``out_dtype`` (bf16 or fp32).  ``out``: row-major result
    buffer; with ``accumulate`` (fp32 only) the product is added to it."""
    if a.cols != b.cols:
        raise ValueError(f"contraction of {a.cols} with {b.cols} values")
    if a.device != b.device:
        raise ValueError(f"operands on {a.device} and {b.device}")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        if out_dtype not in _TYPES:
            raise TypeError(f"bf16 or fp32 output is wanted, got {out_dtype}")
        out = torch.empty(a.rows, b.rows, device=a.device, dtype=out_dtype)
    elif tuple(out.shape) != (a.rows, b.rows) or out.device != a.device or (out.stride(1) != 1 and out.shape[1] > 1) or (
            out.stride(0) < out.shape[1] and out.shape[0] > 1):
        raise ValueError(f"out has to be a row-major {(a.rows, b.rows)} matrix on {a.device}")
    elif out.dtype not in _TYPES or (accumulate and out.dtype != torch.float32):
        raise TypeError(f"out is {out.dtype}: bf16 or fp32 is wanted, fp32 to accumulate")
    if out.is_cuda:
        _C().fp8_gemm(a.data, a.scales, b.data, b.scales, out, accumulate)
        increment_version(out)
        return out
    value = a.dequantize() @ b.dequantize().T
    return out.add_(value) if accumulate else out.copy_(value)


class _LinearFp8(Function):
    """What backward needs is kept as codes (1 byte a value): x^T for dw and w^T for dx, written by the passes that
    quantise x and w for the forward product."""

    @staticmethod
    def forward(ctx, x, w):
        need_x, need_w = ctx.needs_input_grad
        x2 = _as_matrix(x)
        w2 = w if w.stride(1) == 1 or w.shape[1] == 1 else w.contiguous()
        y, xt, wt = _forward(x2, w2, need_w, need_x)
        ctx.save_for_backward(w, xt, wt)
        ctx.x_shape = x.shape
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, xt, wt = ctx.saved_tensors
        dw = mg = None
        if xt is not None:
            mg = getattr(w, "main_grad", None)
            dw = torch.empty(w.shape, device=w.device, dtype=w.dtype) if mg is None else mg
        dx = _backward(_as_matrix(dy), w.shape[1], xt, wt, dw, mg is not None)
        return None if dx is None else dx.view(ctx.x_shape), None if mg is not None else dw


def linear_fp8(x: torch.Tensor, w: torch.Tensor | Fp8Blocks) -> torch.Tensor:
    """``x @ w.T`` for ``x`` [..., K] (bf16 or fp32, the type of the result) and ``w`` [N, K]: a bf16 or fp32 weight, which is
    quantised in the call and gets its gradient (into ``w.main_grad`` where there is one), or ``Fp8Blocks`` that were laid
    out once (``quantize_fp8(w, square=True)``), for inference."""
    if x.dim() < 1 or x.dtype not in _TYPES:
        raise TypeError(f"x has to be bf16 or fp32, got {x.dtype}")
    held = isinstance(w, Fp8Blocks)
    if not held and (w.dim() != 2 or w.dtype not in _TYPES):
        raise TypeError("w has to be Fp8Blocks or a bf16 or fp32 matrix")
    N, K = w.shape
    if x.shape[-1] != K:
        raise ValueError(f"x {tuple(x.shape)} does not fit the weight {(N, K)}")
    if w.device != x.device:
        raise ValueError(f"the weight is on {w.device}, x on {x.device}")
    grad = torch.is_grad_enabled() and (x.requires_grad or (not held and w.requires_grad))
    if held and grad:
        raise RuntimeError("a weight that is held as codes has no gradient and passes none on: use the weight itself, "
                           "or torch.no_grad()")
    if x.numel() == 0 or N == 0 or K == 0:
        if not held and grad:
            return x @ w.T.to(x.dtype)
        return torch.zeros(*x.shape[:-1], N, device=x.device, dtype=x.dtype)
    if grad:
        return _LinearFp8.apply(x, w)
    x2 = _as_matrix(x)
    if not held:
        y = _forward(x2, w if w.stride(1) == 1 or K == 1 else w.contiguous(), False, False)[0]
    elif x.is_cuda:
        y = _C().fp8_linear(x2, w.data, w.scales)
    else:
        y = matmul_fp8(quantize_fp8(x2), w, out_dtype=x.dtype)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)
