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
(after a first call outside the capture); the optimizer's step cannot.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import nn

from . import _lib
from .functional import _SUPPORTED, host_status

_lib.load()                       # the bindings below link to it
from . import _race_torch as _ops  # noqa: E402

BLOCK = 128
F8 = torch.float8_e4m3fn


def _blocks_of(n: int) -> int:
    return -(-n // BLOCK)


def _cuda(x: torch.Tensor, what: str) -> torch.Tensor:
    """x on a GPU, in a type the kernels read."""
    if not x.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA devices only (no CPU fallback)")
    return x if x.dtype in _SUPPORTED else x.to(torch.float32)


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
        if scales.dtype != torch.float32 or scales.device != codes.device or scales.dim() != 2:
            raise ValueError("scales must be a 2-D float32 tensor on the codes' device")
        r, k = codes.shape
        sr, sk = scales.shape
        if sk != -(-k // BLOCK) or (sr != r and sr != -(-r // BLOCK)):
            raise ValueError(f"scales of codes [{r}, {k}] must be [{r}, {_blocks_of(k)}] or "
                             f"[{_blocks_of(r)}, {_blocks_of(k)}], got {list(scales.shape)}")
        self.square = sr != r
        self.codes, self.scales = codes, scales

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def _by_square(self) -> bool:
        """Whether the scales serve as those of square blocks: one row's are both kinds."""
        return self.square or self.codes.shape[0] <= 1

    def dequantize(self) -> torch.Tensor:
        """The values in float32 (for inspection and tests)."""
        s = self.scales.repeat_interleave(BLOCK, 1)[:, :self.codes.shape[1]]
        if self.square and self.codes.shape[0] != self.scales.shape[0]:
            s = s.repeat_interleave(BLOCK, 0)[:self.codes.shape[0]]
        return self.codes.float() * s


def _held(codes: torch.Tensor, scales: torch.Tensor, square: bool) -> BlockFp8:
    """A BlockFp8 of tensors that fit by construction."""
    b = BlockFp8.__new__(BlockFp8)
    b.codes, b.scales, b.square = codes, scales, square
    return b


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
    x = _cuda(x, "quantize_fp8")
    mode = 0 if transposed is False else 1 if transposed is True else 2
    c, s, ct, st = _ops.quantize(x, square, mode)
    if mode == 0:
        return _held(c, s, square)
    t = _held(ct, st, square)
    return t if mode == 2 else (_held(c, s, square), t)


def fp8_matmul(a: BlockFp8, b: BlockFp8, out_dtype: torch.dtype = torch.bfloat16,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a [M, K] times b [N, K] transposed: [M, N] in float32 or bfloat16.

    a has a scale for each 128 columns of a row; b the same or one for each
    128 x 128 block.  Each 128-long partial product is scaled and summed in 32
    bits, in an order that depends on the shape alone.  out: a [M, N] tensor to
    write (any row stride, contiguous columns), of the result's type."""
    if out_dtype not in _SUPPORTED:
        raise ValueError("out_dtype must be float32 or bfloat16")
    codes = a.codes
    if not codes.is_cuda:
        raise RuntimeError("fp8_matmul runs on CUDA devices only (no CPU fallback)")
    return _ops.matmul(codes, a.scales, a.square and codes.shape[0] > 1, b.codes, b.scales, b.square, out_dtype == torch.float32,
                       out, host_status.word(codes.device))


def _check_pair(w: BlockFp8, t: BlockFp8) -> None:
    """t as the transpose of the held weight w: what can be seen without reading the codes."""
    c, d = w.codes, t.codes
    n, k = c.shape
    if not t._by_square() or d.device != c.device or d.shape != (k, n):
        raise ValueError(f"the transpose that goes with a held weight [{n}, {k}] needs square blocks, "
                         f"[{k}, {n}], on the weight's device")
    if n > 1 and d.data_ptr() == c.data_ptr() and d.stride() == c.stride():
        raise ValueError("the weight itself stands in its transpose's place: "
                         "quantize_fp8(w, square=True, transposed=True) returns both")


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
    held = None
    if isinstance(weight, BlockFp8):
        held = (weight, None)
    elif not isinstance(weight, torch.Tensor):
        if len(weight) != 2 or not all(isinstance(b, BlockFp8) for b in weight):
            raise ValueError("weight must be a tensor, a BlockFp8, or the pair of a BlockFp8 and its transpose")
        held = weight
        _check_pair(*held)
    if isinstance(x, BlockFp8):
        if held is None:
            if (torch.is_grad_enabled() and weight.requires_grad) or _ops.has_tangent(weight):
                raise ValueError("x in 8 bits has no gradient: pass the tensor itself to train")
            held = (quantize_fp8(weight, square=True), None)
        return fp8_matmul(x, held[0], torch.bfloat16 if out_dtype is None else out_dtype)
    x = _cuda(x, "fp8_linear")
    n, k = held[0].codes.shape if held is not None else weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, weight [{n}, {k}] needs {k}")
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype not in _SUPPORTED:
        raise ValueError("out_dtype must be float32 or bfloat16")
    f32 = out_dtype == torch.float32
    status = host_status.word(x.device)
    if held is None:
        if weight.dtype not in _SUPPORTED:
            weight = weight.to(torch.float32)
        if weight.device != x.device:
            raise ValueError("x and weight must be on the same device")
        return _ops.linear(x, weight, None, None, None, None, f32, status)
    w, t = held
    if not w._by_square() or w.codes.device != x.device:
        raise ValueError("a held weight needs square blocks, on x's device")
    if t is None:
        if torch.is_grad_enabled() and x.requires_grad:
            raise ValueError("gradients of x need the weight's transpose too: "
                             "quantize_fp8(w, square=True, transposed=True)")
        return _ops.linear(x, None, w.codes, w.scales, None, None, f32, status)
    return _ops.linear(x, None, w.codes, w.scales, t.codes, t.scales, f32, status)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6, quantize: bool = False):
    """Root-mean-square norm over the last axis with the residual's addition:
    h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight.

    Returns y, or (y, h) where a residual is given (h is the residual of the
    next layer).  Both have x's type, float32 or bfloat16 (another type computes
    and returns in float32); y is computed in 32 bits from the sum before it is
    rounded to h.  weight: [K], float32 or bfloat16.  Gradients flow to x,
    residual and weight.

    quantize=True returns y as a BlockFp8 [R, K] (leading axes flattened) for
    ``fp8_linear``, without its higher-precision form ever being written; it is
    for serving, under torch.no_grad()."""
    if weight.dim() != 1 or x.dim() < 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"weight must be [{x.shape[-1] if x.dim() else 0}], got {list(weight.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError("residual must have x's shape, type and device")
    if x.dtype not in _SUPPORTED and residual is not None:
        residual = residual.to(torch.float32)
    x = _cuda(x, "rms_norm")
    if weight.device != x.device:
        raise ValueError("x and weight must be on the same device")
    if weight.dtype not in _SUPPORTED:
        weight = weight.to(torch.float32)
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                        (residual is not None and residual.requires_grad))
    if not quantize:
        y, _, h = _ops.norm(x, weight, residual, eps, False, grad)
        return y if residual is None else (y, h)
    if grad:
        raise ValueError("quantize=True has no gradient: call it under torch.no_grad(), or "
                         "pass the plain result to fp8_linear to train")
    c, s, h = _ops.norm(x, weight, residual, eps, True, False)
    return _held(c, s, False) if residual is None else (_held(c, s, False), h)


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
    once for serving; ``release()`` drops that copy.  Training mode ignores it,
    and where the weight has changed since (a loaded state, an optimizer's step,
    another device or type) the next serving call quantises it again.  Writes
    through ``weight.data`` cannot be seen: call ``hold()`` after them.  Inputs
    that ask for a gradient go through the weight itself, in eval mode too; others
    are served, and the weight gets no gradient from them."""

    def __init__(self, in_features: int, out_features: int, device=None, dtype=None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.weight = nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        nn.init.kaiming_uniform_(self.weight, a=5 ** 0.5)
        self.held: Optional[BlockFp8] = None

    def hold(self) -> "Fp8Linear":
        self.held = quantize_fp8(self.weight, square=True)
        self._held_at = self._version()
        return self

    def release(self) -> "Fp8Linear":
        self.held = None
        return self

    def _version(self) -> int:
        """Counts the writes into the weight that torch knows of."""
        return -1 if self.weight.is_inference() else self.weight._version

    def __setattr__(self, name, value):
        if name == "weight":
            self.__dict__["_held_at"] = None       # another tensor, another count
        super().__setattr__(name, value)

    def __setstate__(self, state):                 # a copy's weight is another tensor too
        super().__setstate__(state)
        self._held_at = None

    def _apply(self, fn, recurse=True):            # .to(), .bfloat16(), ...
        super()._apply(fn, recurse)
        self._held_at = None
        return self

    def forward(self, x, out_dtype: Optional[torch.dtype] = None):
        if self.held is not None and not self.training and not (
                torch.is_grad_enabled() and isinstance(x, torch.Tensor) and x.requires_grad):
            if self._held_at != self._version():
                self.hold()
            return fp8_linear(x, self.held, out_dtype)
        return fp8_linear(x, self.weight, out_dtype)
