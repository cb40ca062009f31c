"""Block-scaled 8-bit and 4-bit storage on the kernels of libhmx.so (csrc/norm.hip, csrc/mx4.hip): a norm whose output is
stored in 8 bits, tables and layers in 4 bits, and the products that read them.

Formats (32 consecutive values of a row share one scale byte b, standing for 2^(b - 127)): "mx8" holds a value as e4m3,
"mx4" as e2m1, the value with the even index in the low half of its byte.  A row of d values takes dp = 32 ceil(d / 32)
codes, zeros past d.  The scale is the least power of two that cuts no value of the block off, values are rounded to
nearest even, and a block that holds a NaN or an infinity stands for NaN (scale byte 255).

CUDA tensors only, no gradients; no CPU fallback.
"""
import torch

from . import hmx
from .enc_ops import _norm_operands
from .ops import _launch, _one_device, _rows

BLOCK = 32


def padded(d):
    """Codes of a row of d values."""
    return -(-d // BLOCK) * BLOCK


def add_rmsnorm_mx8(x, residual, scale, eps=1e-6):
    """enc_ops.add_rmsnorm with y in mx8 -> (codes float8_e4m3fn (..., dp), scales uint8 (..., dp / 32), s); residual
    None: s is x.  Statistics and y are float64, and y is rounded once, to its code; no gradient."""
    device, x2, r2, bf16 = _norm_operands("add_rmsnorm_mx8", x, residual, scale, eps)
    T, d = x2.shape
    dp = padded(d)
    lead = x.shape[:-1]
    s = torch.empty(x.shape, dtype=x.dtype, device=device) if r2 is not None else None
    codes = torch.empty(*lead, dp, dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty(*lead, dp // BLOCK, dtype=torch.uint8, device=device)
    _launch("hmx_add_rmsnorm_mx8", device, x2.data_ptr(), x2.stride(0), hmx.ptr(r2), 0 if r2 is None else r2.stride(0),
            scale.contiguous().data_ptr(), T, d, eps, bf16, hmx.ptr(s), codes.data_ptr(), scales.data_ptr())
    return codes, scales, (x if s is None else s)


def _checked(what, codes, scales, code_dtype, per_block):
    """-> device, rows, blocks of a row, contiguous codes and scales."""
    device = _one_device(what, codes, scales)
    if codes.dtype != code_dtype or scales.dtype != torch.uint8:
        raise hmx.HmxError(f"{what}: codes are {code_dtype} and scales uint8, got {codes.dtype} and {scales.dtype}")
    if codes.dim() < 1 or codes.shape[:-1] != scales.shape[:-1] or scales.shape[-1] < 1 or \
            codes.shape[-1] != scales.shape[-1] * per_block:
        raise hmx.HmxError(f"{what}: codes {tuple(codes.shape)} need one scale per {per_block} along the last dimension, "
                           f"got {tuple(scales.shape)}")
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 16:                  # a view that starts inside another tensor's storage
        codes = codes.clone()
    return device, scales.numel() // scales.shape[-1], scales.shape[-1], codes, scales


def _dequantize(what, bits, codes, scales, d, dtype):
    device, n, blocks, codes, scales = _checked(what, codes, scales, torch.uint8 if bits == 4 else torch.float8_e4m3fn,
                                                BLOCK * bits // 8)
    d = blocks * BLOCK if d is None else int(d)
    if padded(d) != blocks * BLOCK or d < 1:
        raise hmx.HmxError(f"{what}: rows of {d} values do not take {blocks} blocks")
    if dtype not in (torch.float32, torch.bfloat16):
        raise hmx.HmxError(f"{what}: values are float32 or bfloat16, not {dtype}")
    out = torch.empty(*scales.shape[:-1], d, dtype=dtype, device=device)
    _launch("hmx_mx_dequantize", device, codes.data_ptr(), scales.data_ptr(), n, d, bits, int(dtype == torch.bfloat16),
            out.data_ptr())
    return out


def dequantize_mx8(codes, scales, d=None, dtype=torch.bfloat16):
    """The values that mx8 codes stand for, (..., d); d None: all dp of them.  float32 holds each exactly, bfloat16 from
    2^-126 up (it rounds to multiples of 2^-133 below)."""
    return _dequantize("dequantize_mx8", 8, codes, scales, d, dtype)


def dequantize_mx4(codes, scales, d=None, dtype=torch.bfloat16):
    """The values that mx4 codes stand for, (..., d); d None: all dp of them.  bfloat16 holds each exactly."""
    return _dequantize("dequantize_mx4", 4, codes, scales, d, dtype)


def quantize_mx4(table, out=None):
    """table (..., d) float32 or bfloat16 -> (codes uint8 (..., dp / 2), scales uint8 (..., dp / 32)).  Run it again
    after the table's weights changed; out (codes, scales): it is written there, for captured graphs that read it."""
    device = _one_device("quantize_mx4", table)
    if table.dtype not in (torch.float32, torch.bfloat16) or table.dim() < 1 or table.shape[-1] < 1:
        raise hmx.HmxError(f"quantize_mx4: a float32 or bfloat16 table of rows, got {table.dtype} {tuple(table.shape)}")
    t2 = _rows(table)
    n, d = t2.shape
    dp = padded(d)
    shapes = (*table.shape[:-1], dp // 2), (*table.shape[:-1], dp // BLOCK)
    if out is None:
        codes, scales = (torch.empty(s, dtype=torch.uint8, device=device) for s in shapes)
    else:
        codes, scales = out
        if any(t.shape != s or t.dtype != torch.uint8 or t.device != device or not t.is_contiguous()
               for t, s in zip(out, shapes)):
            raise hmx.HmxError(f"quantize_mx4: out is contiguous uint8 {shapes[0]} and {shapes[1]} on {device}")
    _launch("hmx_mx4_quantize", device, t2.data_ptr(), t2.stride(0), n, d, int(table.dtype == torch.bfloat16),
            codes.data_ptr(), scales.data_ptr())
    return codes, scales


_X_KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float8_e4m3fn: 2}


def linear_mx4(x, codes, scales, x_scales=None, out_dtype=torch.float32):
    """out (..., N) = x (..., K) times the transposed mx4 table (codes (N, dp / 2), scales (N, dp / 32)), dp = padded(K).

    x is float32 (all 24 bits take part), bfloat16, or mx8 codes (..., dp) with x_scales (..., dp / 32); bits of x below
    2^-133 are left out, and table values from 2^128 on count as infinite.  Sums are float32, out is float32 or bfloat16;
    no gradient.  Made for few rows of x: the scores of a batch of users over an item table, a layer for single tokens.  More
    rows re-read the table once per 16 (K <= 128), or 32 (10 where x is float32)."""
    device, n, blocks, codes, scales = _checked("linear_mx4", codes, scales, torch.uint8, BLOCK // 2)
    if scales.dim() != 2:
        raise hmx.HmxError(f"linear_mx4: the table is a matrix, got codes {tuple(codes.shape)}")
    kind = _X_KINDS.get(x.dtype)
    if kind is None or x.dim() < 1 or (kind == 2) != (x_scales is not None):
        raise hmx.HmxError("linear_mx4: x is float32, bfloat16, or float8_e4m3fn codes with x_scales; got "
                           f"{x.dtype}, x_scales {'missing' if x_scales is None else 'given'}")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise hmx.HmxError(f"linear_mx4: out is float32 or bfloat16, not {out_dtype}")
    if kind == 2:
        xdev, m, xblocks, x2, x_scales = _checked("linear_mx4 (x)", x, x_scales, torch.float8_e4m3fn, BLOCK)
        k = xblocks * BLOCK
        x2 = x2.view(m, k)
    else:
        xdev = _one_device("linear_mx4", x)
        x2 = _rows(x)
        m, k = x2.shape
    if xdev != device:
        raise hmx.HmxError(f"linear_mx4: x lies on {xdev}, the table on {device}")
    if padded(k) != blocks * BLOCK:
        raise hmx.HmxError(f"linear_mx4: rows of {k} values do not match a table of {blocks} blocks of {BLOCK}")
    out = torch.empty(*x.shape[:-1], n, dtype=out_dtype, device=device)
    nbytes = 0 if k <= 128 else hmx.lib().hmx_linear_mx4_workspace_bytes(kind, m, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _launch("hmx_linear_mx4", device, x2.data_ptr(), x2.stride(0), hmx.ptr(x_scales), kind, m, codes.data_ptr(),
            scales.data_ptr(), n, k, int(out_dtype == torch.bfloat16), out.data_ptr(), hmx.ptr(ws), nbytes)
    return out
