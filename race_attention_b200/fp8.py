"""8-bit operators around RACE attention: quantisation in blocks of 128, the
product of such operands, a linear layer trained through it, and a
root-mean-square norm that can hand its result on in 8 bits.

The reference runs the layers around its attention as torch modules in 32
bits (nn.LayerNorm and nn.Linear of RACEBlock, misc/vit.py:1040-1068 and
misc/race.py:176-206); nothing here replaces those by default.

A held value is an e4m3 code (``torch.float8_e4m3fn``) times the float32 scale
of its block, ``scale = max(amax / 448, 2^-126)``.  Rows of activations and
gradients carry a scale for each 128 columns, weights one for each 128 x 128
block.  A block that holds an infinity or a NaN gets a non-finite scale.

All calls run on the current stream of the inputs' device, allocate through
torch's caching allocator, never synchronise and can be captured in a CUDA graph
(after a first call outside the capture).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import nn

from . import _lib
from ._lib import RaceBlocks, RaceMatmulDesc, RaceNormDesc, RaceRows, check
from .functional import _SUPPORTED, host_status

BLOCK = 128
F8 = torch.float8_e4m3fn
_NO_ROWS = RaceRows(None, 0)
_NO_BLOCKS = RaceBlocks(None, 0, None, 0, 0)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _blocks_of(n: int) -> int:
    return -(-n // BLOCK)


def _code(dtype: torch.dtype) -> int:
    return _lib.RACE_F32 if dtype == torch.float32 else _lib.RACE_BF16


def _cuda(x: torch.Tensor, what: str) -> torch.Tensor:
    if not x.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA devices only (no CPU fallback)")
    return x


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, columns] of a supported type with contiguous columns."""
    if x.dtype not in _SUPPORTED:
        x = x.to(torch.float32)
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _rr(x: Optional[torch.Tensor]) -> RaceRows:
    return _NO_ROWS if x is None else RaceRows(x.data_ptr(), x.stride(0))


class _on:
    """Makes the tensor's device current for the call when it is not."""
    __slots__ = ("guard",)

    def __init__(self, device: torch.device):
        self.guard = (None if device.index == torch.cuda.current_device()
                      else torch.cuda.device(device))

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


class BlockFp8:
    """8-bit codes [R, K] with their scales: [R, ceil(K/128)] (one for each 128
    columns of a row) or [ceil(R/128), ceil(K/128)] (one for each 128 x 128
    block, ``square``).

    Codes made by ``quantize_fp8`` and ``rms_norm`` have rows that start on
    16-byte boundaries and scales whose first axis is contiguous, which the
    product reads in place; codes of another layout are copied by it."""

    __slots__ = ("codes", "scales", "square")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != F8 or codes.dim() != 2:
            raise ValueError("codes must be a 2-D torch.float8_e4m3fn tensor")
        r, k = codes.shape
        if scales.dtype != torch.float32 or scales.device != codes.device:
            raise ValueError("scales must be float32 on the codes' device")
        shape = tuple(scales.shape)
        if shape == (r, _blocks_of(k)):
            self.square = False
        elif shape == (_blocks_of(r), _blocks_of(k)):
            self.square = True
        else:
            raise ValueError(f"scales of codes [{r}, {k}] must be [{r}, {_blocks_of(k)}] or "
                             f"[{_blocks_of(r)}, {_blocks_of(k)}], got {list(shape)}")
        self.codes, self.scales = codes, scales

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def dequantize(self) -> torch.Tensor:
        """The values in float32 (for inspection and tests)."""
        s = self.scales.repeat_interleave(BLOCK, 1)[:, :self.codes.shape[1]]
        if self.square and self.codes.shape[0] != self.scales.shape[0]:
            s = s.repeat_interleave(BLOCK, 0)[:self.codes.shape[0]]
        return self.codes.float() * s


def _new_codes(rows: int, cols: int, device) -> torch.Tensor:
    pitch = -(-cols // 16) * 16
    c = torch.empty((rows, pitch), dtype=F8, device=device)
    return c if pitch == cols else c[:, :cols]


def _new_scales(rows: int, cols: int, device) -> torch.Tensor:
    return torch.empty_strided((rows, _blocks_of(cols)), (1, max(rows, 1)), dtype=torch.float32,
                               device=device)


def _pitch(codes: torch.Tensor) -> int:
    """Bytes between rows; a single row has any pitch that is a multiple of 16."""
    return codes.stride(0) if codes.shape[0] > 1 else -(-codes.shape[1] // 16) * 16


def _rb(b: Optional[BlockFp8]) -> RaceBlocks:
    if b is None:
        return _NO_BLOCKS
    s = b.scales
    return RaceBlocks(b.codes.data_ptr(), _pitch(b.codes), s.data_ptr(), s.stride(0), s.stride(1))


def _in_place(b: BlockFp8) -> BlockFp8:
    """b itself if the copy engine can walk its codes, else a copy that it can."""
    c = b.codes
    r, k = c.shape
    if ((k <= 1 or c.stride(1) == 1) and c.data_ptr() % 16 == 0
            and (r <= 1 or (c.stride(0) % 16 == 0 and c.stride(0) >= k))):
        return b
    n = _new_codes(r, k, c.device)
    n.view(torch.uint8).copy_(c.view(torch.uint8))
    return BlockFp8(n, b.scales)


def quantize_fp8(x: torch.Tensor, square: bool = False,
                 transposed: Union[bool, str] = False):
    """x [..., K] (float32 or bfloat16; leading axes are flattened) in 8 bits.

    square=False: one scale for each 128 columns of a row; square=True: one for
    each 128 x 128 block (weights).  transposed=True returns a pair, x and its
    transpose [K, R], from one reading of x: with square=False the transpose
    has its own codes, a scale for each 128 rows of a column; with square=True
    it has the same codes and scales.  transposed="only" returns the transpose
    alone.  Not differentiable."""
    if transposed not in (False, True, "only"):
        raise ValueError(f"transposed must be False, True or 'only', got {transposed!r}")
    x = _rows(_cuda(x.detach(), "quantize_fp8"))
    r, k = x.shape
    dev = x.device
    by_rows = by_cols = None
    if square:
        scales = torch.empty((_blocks_of(r), _blocks_of(k)), dtype=torch.float32, device=dev)
    if transposed != "only":
        by_rows = BlockFp8(_new_codes(r, k, dev), scales if square else _new_scales(r, k, dev))
    if transposed:
        by_cols = BlockFp8(_new_codes(k, r, dev), scales.t() if square else _new_scales(k, r, dev))
    with _on(dev):
        check(_lib.load().race_quantize(_rr(x), _code(x.dtype), r, k, int(square), _rb(by_rows),
                                        _rb(by_cols), _raw_stream(dev.index)))
    if transposed == "only":
        return by_cols
    return (by_rows, by_cols) if transposed else by_rows


def fp8_matmul(a: BlockFp8, b: BlockFp8, out_dtype: torch.dtype = torch.bfloat16,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a [M, K] times b [N, K] transposed: [M, N] in float32 or bfloat16.

    a has a scale for each 128 columns of a row; b the same or one for each
    128 x 128 block.  Each 128-long partial product is scaled and summed in 32
    bits, in an order that depends on the shape alone.  out: a [M, N] tensor to
    write (any row stride, contiguous columns), of the result's type."""
    if a.square and a.codes.shape[0] != a.scales.shape[0]:
        raise ValueError("a must have a scale for each row; only b may have square blocks")
    m, k = a.codes.shape
    n, kb = b.codes.shape
    if kb != k:
        raise ValueError(f"a [{m}, {k}] and b [{n}, {kb}] must have the same number of columns")
    dev = a.codes.device
    if b.codes.device != dev:
        raise ValueError("a and b must be on the same device")
    if out_dtype not in _SUPPORTED:
        raise ValueError("out_dtype must be float32 or bfloat16")
    _cuda(a.codes, "fp8_matmul")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=dev)
    elif (out.shape != (m, n) or out.dtype != out_dtype or out.device != dev
          or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n)):
        raise ValueError(f"out must be a [{m}, {n}] {out_dtype} tensor with contiguous columns")
    a, b = _in_place(a), _in_place(b)
    desc = RaceMatmulDesc(_code(out_dtype), int(b.square), m, n, k, 0, 0)
    lib = _lib.load()
    with _on(dev):
        status = host_status.word(dev)
        need = lib.race_scaled_matmul_workspace(desc)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        check(lib.race_scaled_matmul(desc, _rb(a), _rb(b), _rr(out), status,
                                     ws.data_ptr() if need else None, need,
                                     _raw_stream(dev.index)))
    return out


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, held, out_dtype):
        # x [R, K]; weight [N, K], or None with ``held``, its 8-bit form (and its
        # transpose's, where x needs a gradient)
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        xr, xc = quantize_fp8(x, transposed=True) if need_w else (quantize_fp8(x), None)
        if weight is not None:
            held = (quantize_fp8(weight, square=True, transposed=True) if need_x
                    else (quantize_fp8(weight, square=True), None))
        y = fp8_matmul(xr, held[0], out_dtype)
        ctx.x_dtype, ctx.w_dtype = x.dtype, None if weight is None else weight.dtype
        saved = []
        for b in (xc if need_w else None, held[1] if need_x else None):
            saved += [None, None] if b is None else [b.codes, b.scales]
        ctx.save_for_backward(*saved)
        return y

    @staticmethod
    def backward(ctx, dy):
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        xc, xs, wc, ws = ctx.saved_tensors
        if need_x and need_w:
            dyr, dyc = quantize_fp8(dy, transposed=True)
        else:
            dyr = quantize_fp8(dy) if need_x else None
            dyc = quantize_fp8(dy, transposed="only") if need_w else None
        dx = dw = None
        if need_x:
            t = ctx.x_dtype if ctx.x_dtype in _SUPPORTED else torch.float32
            dx = fp8_matmul(dyr, BlockFp8(wc, ws), t).to(ctx.x_dtype)
        if need_w:
            t = ctx.w_dtype if ctx.w_dtype in _SUPPORTED else torch.float32
            dw = fp8_matmul(dyc, BlockFp8(xc, xs), t).to(ctx.w_dtype)
        return dx, dw, None, None


Weight = Union[torch.Tensor, BlockFp8, Tuple[BlockFp8, BlockFp8]]


def fp8_linear(x: Union[torch.Tensor, BlockFp8], weight: Weight,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [..., K] times weight [N, K] transposed with both in 8 bits: [..., N].

    Training: x and weight are float32 or bfloat16 tensors.  The forward pass
    quantises both, rows of x by 128 columns and the weight by 128 x 128
    blocks; the backward pass quantises dy along the output features for dx =
    dy W and along the tokens for dW = dy^T x.  Between the passes x is kept in
    8 bits.  Gradients have the types of x and weight.

    Serving: weight may be held as ``quantize_fp8(w, square=True)`` (add
    transposed=True for gradients of x with a frozen weight), and x may be a
    BlockFp8 as ``rms_norm(..., quantize=True)`` returns it; nothing is
    quantised twice then.

    out_dtype: float32 or bfloat16; by default x's type (bfloat16 where x comes
    in 8 bits)."""
    held = weight if isinstance(weight, tuple) else (weight, None)
    if not isinstance(held[0], BlockFp8):
        held = None
    if isinstance(x, BlockFp8):
        if held is None:
            if torch.is_grad_enabled() and weight.requires_grad:
                raise ValueError("x in 8 bits has no gradient: pass the tensor itself to train")
            held = (quantize_fp8(weight, square=True), None)
        return fp8_matmul(x, held[0], torch.bfloat16 if out_dtype is None else out_dtype)
    _cuda(x, "fp8_linear")
    n, k = held[0].shape if held is not None else weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, weight [{n}, {k}] needs {k}")
    if out_dtype is None:
        out_dtype = x.dtype if x.dtype in _SUPPORTED else torch.float32
    x2 = x.reshape(-1, k)
    if held is None:
        y = _Linear.apply(x2, weight, None, out_dtype)
    elif not (torch.is_grad_enabled() and x.requires_grad):
        y = fp8_matmul(quantize_fp8(x2), held[0], out_dtype)
    else:
        if held[1] is None:
            raise ValueError("gradients of x need the weight's transpose too: "
                             "quantize_fp8(w, square=True, transposed=True)")
        y = _Linear.apply(x2, None, held, out_dtype)
    return y.view(*x.shape[:-1], n)


def _norm_desc(x: torch.Tensor, weight: torch.Tensor, eps: float) -> RaceNormDesc:
    return RaceNormDesc(_code(x.dtype), _code(weight.dtype), x.shape[0], x.shape[1], eps)


def _norm_weight(weight: torch.Tensor) -> torch.Tensor:
    w = weight.detach()
    if w.dtype not in _SUPPORTED:
        w = w.to(torch.float32)
    return w.contiguous()


def _norm_forward(x, weight, residual, eps, quantize, want_rstd):
    """(y or BlockFp8, h, rstd) of [R, K] rows."""
    r, k = x.shape
    dev = x.device
    h = torch.empty((r, k), dtype=x.dtype, device=dev) if residual is not None else None
    y = None if quantize else torch.empty((r, k), dtype=x.dtype, device=dev)
    y8 = BlockFp8(_new_codes(r, k, dev), _new_scales(r, k, dev)) if quantize else None
    rstd = torch.empty(r, dtype=torch.float32, device=dev) if want_rstd else None
    with _on(dev):
        check(_lib.load().race_rms_norm(
            _norm_desc(x, weight, eps), _rr(x), _rr(residual), weight.data_ptr(), _rr(y), _rb(y8),
            _rr(h), None if rstd is None else rstd.data_ptr(), _raw_stream(dev.index)))
    return (y8 if quantize else y), h, rstd


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        shape = x.shape
        ctx.dtypes = (x.dtype, weight.dtype, None if residual is None else residual.dtype)
        x2, w = _rows(x), _norm_weight(weight)
        r2 = None if residual is None else _rows(residual)
        y, h, rstd = _norm_forward(x2, w, r2, eps, False, True)
        ctx.save_for_backward(x2 if h is None else h, w, rstd)
        ctx.eps = eps
        y = y.view(shape)
        return y if h is None else (y, h.view(shape))

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, w, rstd = ctx.saved_tensors
        xt, wt, rt = ctx.dtypes
        shape = None if dy is None else dy.shape
        if dy is None:                      # y was not used: the norm passes dh through
            if dh is None:
                return None, None, None, None
            return dh.to(xt), torch.zeros_like(w).to(wt), None if rt is None else dh.to(rt), None
        dy2 = _rows(dy.to(h.dtype))
        dh2 = None if dh is None else _rows(dh.to(h.dtype))
        dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
        dw = torch.empty_like(w)
        desc = _norm_desc(h, w, ctx.eps)
        lib = _lib.load()
        with _on(h.device):
            need = lib.race_rms_norm_workspace(desc)
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=h.device)
            check(lib.race_rms_norm_backward(desc, _rr(dy2), _rr(dh2), _rr(h), w.data_ptr(),
                                             rstd.data_ptr(), _rr(dx), dw.data_ptr(),
                                             ws.data_ptr(), ws.numel(),
                                             _raw_stream(h.device.index)))
        dx = dx.view(shape)
        return dx.to(xt), dw.to(wt), None if rt is None else dx.to(rt), None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6, quantize: bool = False):
    """Root-mean-square norm over the last axis with the residual's addition:
    h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight.

    Returns y, or (y, h) where a residual is given (h is the residual of the
    next layer).  Both have x's type (float32 or bfloat16); y is computed in 32
    bits from the sum before it is rounded to h.  weight: [K], float32 or
    bfloat16.  Gradients flow to x, residual and weight.

    quantize=True returns y as a BlockFp8 [R, K] (leading axes flattened) for
    ``fp8_linear``, without its higher-precision form ever being written; it is
    for serving, under torch.no_grad()."""
    _cuda(x, "rms_norm")
    if weight.dim() != 1 or x.dim() < 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"weight must be [{x.shape[-1] if x.dim() else 0}], got {list(weight.shape)}")
    if weight.device != x.device:
        raise ValueError("x and weight must be on the same device")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError("residual must have x's shape, type and device")
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                        (residual is not None and residual.requires_grad))
    if quantize:
        if grad:
            raise ValueError("quantize=True has no gradient: call it under torch.no_grad(), or "
                             "pass the plain result to fp8_linear to train")
        y, h, _ = _norm_forward(_rows(x), _norm_weight(weight),
                                None if residual is None else _rows(residual), eps, True, False)
        return y if h is None else (y, h.view(x.shape))
    if grad:
        return _Norm.apply(x, weight, residual, eps)
    y, h, _ = _norm_forward(_rows(x), _norm_weight(weight),
                            None if residual is None else _rows(residual), eps, False, False)
    return y.view(x.shape) if h is None else (y.view(x.shape), h.view(x.shape))


class RMSNorm(nn.Module):
    """``rms_norm`` with its weight."""

    def __init__(self, width: int, eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(width, device=device, dtype=dtype))

    def forward(self, x, residual=None, quantize: bool = False):
        return rms_norm(x, self.weight, residual, self.eps, quantize)


class Fp8Linear(nn.Module):
    """A linear layer without bias whose products run in 8 bits.

    The parameter ``weight`` [out_features, in_features] stays in float32 or
    bfloat16 and is quantised on each training pass.  ``hold()`` quantises it
    once for serving; ``release()`` drops that copy.  A held copy does not
    follow later changes of ``weight``: training mode ignores it."""

    def __init__(self, in_features: int, out_features: int, device=None, dtype=None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.weight = nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        nn.init.kaiming_uniform_(self.weight, a=5 ** 0.5)
        self.held: Optional[BlockFp8] = None

    def hold(self) -> "Fp8Linear":
        self.held = quantize_fp8(self.weight, square=True)
        return self

    def release(self) -> "Fp8Linear":
        self.held = None
        return self

    def forward(self, x, out_dtype: Optional[torch.dtype] = None):
        if self.held is not None and not self.training:
            return fp8_linear(x, self.held, out_dtype)
        return fp8_linear(x, self.weight, out_dtype)
