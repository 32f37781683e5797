"""Matrix products in 8-bit integers with a scale per token and per output channel: the
projections around the batched attention (tinygiant_b200/paged.py) and the logits of a batch,
where the reference multiplies one row at a time (csrc/libtinygiant.c:173-318).

    lin = Int8Linear.quantize(W)                       # W: cuda [N][K]
    y = lin(x)                                         # x: cuda [M][K]
    y = lin(x, norm=w, eps=1e-6, residual=h, out=h)    # h += RMSNorm(x) * w @ W^T
"""
from __future__ import annotations

import torch

from ._lib import TGX_FROM_F32, check, get_lib
from .paged import DTYPES, dtype_code, on_stream, stream_handle


def _matrix(t, cols, device, name):
    """(pointer, row stride) of a matrix with dense rows."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[1] != cols or (stride[1] != 1 and cols > 1 and t.numel()):
        raise ValueError(f"{name}: expected rows of {cols}, dense in a row, got {tuple(shape)} with strides {stride}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t.data_ptr(), stride[0] if shape[0] > 1 else cols


def _norm(norm, cols, device):
    if norm is None:
        return None
    if norm.shape != (cols,) or norm.dtype != torch.float32 or norm.device != device or not norm.is_contiguous():
        raise ValueError(f"norm: expected contiguous float32 [{cols}] on {device}")
    return norm.data_ptr()


def quantize_rows(x, norm=None, eps: float = 1e-6, stream=None):
    """(codes int8 [M][K rounded up to 16], scales float32 [M]) of the rows of x, or of their
    RMSNorm times `norm`."""
    if x.dim() != 2 or not x.is_cuda:
        raise ValueError("x: expected a cuda matrix")
    if stream is not None:
        with on_stream(stream, x.device):
            return quantize_rows(x, norm, eps)
    lib = get_lib()
    m, k = x.shape
    px, sx = _matrix(x, k, x.device, "x")
    rb = int(lib.tgx_i8_row_bytes(k))
    if not rb:
        raise ValueError(f"rows of {k}: expected 1 .. 131072")
    codes = torch.empty((m, rb), dtype=torch.int8, device=x.device)
    scales = torch.empty(m, dtype=torch.float32, device=x.device)
    if m:
        check(lib.tgx_i8_quantize_rows(dtype_code(x), px, sx, m, k, _norm(norm, k, x.device), eps, codes.data_ptr(),
                                       scales.data_ptr(), stream_handle(x.device)), lib)
    return codes, scales


class Int8Linear:
    """W [N][K] as int8 codes [N][K rounded up to 16] (zeros behind K) and a float32 scale per row."""

    def __init__(self, codes, scales, in_features: int):
        self.lib = get_lib()
        n = codes.shape[0]
        if codes.dtype != torch.int8 or not codes.is_cuda or not codes.is_contiguous() or codes.dim() != 2 or n < 1 or \
                codes.shape[1] != int(self.lib.tgx_i8_row_bytes(in_features)):
            raise ValueError("codes: expected a contiguous int8 cuda tensor [N][K rounded up to 16]")
        if scales.dtype != torch.float32 or scales.device != codes.device or scales.shape != (n,) or \
                not scales.is_contiguous():
            raise ValueError(f"scales: expected contiguous float32 [{n}] on {codes.device}")
        self.codes, self.scales, self.in_features, self.out_features = codes, scales, in_features, n
        self.device = codes.device

    @classmethod
    def quantize(cls, weight, stream=None):
        """From float32, bfloat16 or float16 weights [N][K] on the device."""
        return cls(*quantize_rows(weight, stream=stream), weight.shape[1])

    def __call__(self, x, out=None, norm=None, eps: float = 1e-6, residual=None, stream=None, dtype=None):
        """x [M][K] W^T (+ residual) -> out [M][N] of x's type, x quantised per row, behind its
        RMSNorm when `norm` is given.  out may be residual.  dtype: a 16-bit type for out and
        residual with a float32 x, which is rounded to it as x.to(dtype) would, but keeps finite
        values beyond its range."""
        if stream is not None:
            with on_stream(stream, self.device):
                return self(x, out, norm, eps, residual, None, dtype)
        dev, k, n = self.device, self.in_features, self.out_features
        code, dtype = dtype_code(x), dtype or x.dtype
        if dtype != x.dtype:
            if x.dtype != torch.float32 or dtype not in DTYPES:
                raise TypeError(f"no product of {x.dtype} rows to {dtype}")
            code = DTYPES[dtype] | TGX_FROM_F32
        px, sx = _matrix(x, k, dev, "x")
        m = x.shape[0]
        if out is None:
            out = x.new_empty((m, n), dtype=dtype)
            po, so = out.data_ptr(), n
        else:
            po, so = _matrix(out, n, dev, "out")
            if out.dtype != dtype or out.shape[0] != m:
                raise ValueError(f"out: expected {m} rows of {dtype}")
        pr, sr = None, 0
        if residual is not None:
            pr, sr = _matrix(residual, n, dev, "residual")
            if residual.dtype != dtype or residual.shape[0] != m:
                raise ValueError(f"residual: expected {m} rows of {dtype}")
        if not m:
            return out
        size = self.lib.tgx_i8_matmul_scratch_bytes(m, n, k)
        scratch = self.codes.new_empty(size)
        check(self.lib.tgx_i8_matmul(code, px, sx, m, k, _norm(norm, k, dev), eps, self.codes.data_ptr(),
                                     self.scales.data_ptr(), n, pr, sr, po, so, scratch.data_ptr(), size,
                                     stream_handle(dev)), self.lib)
        return out
