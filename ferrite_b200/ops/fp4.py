"""Block-scaled 4-bit matrices on the device: quantiser, expander, products and an expert layer for a few tokens
(``csrc/kernels/fp4.cu``, ``fp4_gemm.cu``, ``fp4_moe.cu``).

A value is an e2m1 code times the scale of its block of consecutive columns:

* ``"mxfp4"``: blocks of 32, the scale a power of two (ue8m0): ``2^ceil(log2(amax / 6))``, the form of the expert weights
  (``ops/quant.py::quant_fp4_weight``);
* ``"nvfp4"``: blocks of 16, the scale an e4m3 number (``amax / 6`` rounded, ``ops/quant.py::fp4_act_roundtrip`` with
  ``scale="e4m3"``), and optionally one f32 ``tensor_scale`` by which the values are divided first.

A block that holds an infinity or a NaN gets the NaN scale: all of its values, and every product that meets it, read NaN.

All functions launch on the current stream of their operands' device, allocate with torch's allocator (nothing is kept
between calls, so calls may overlap on several streams and be captured) and raise ``ValueError`` / ``TypeError`` for
arguments they do not take and ``KernelError`` when CUDA refuses a launch.

A wait inside a product or an expert layer that ran out leaves the output unwritten and is reported in four int32 words
``[code, block, kernel, split]``: in the ``status`` tensor that the call was given (a slice of a
:class:`~ferrite_b200.parallel.status.StatusArena`, say, which an engine checks after every step), else in words that all
such calls on a device share and :func:`check` reads.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from .. import _lib
from .quant import e2m1_unpack

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_F32_MAX = torch.finfo(torch.float32).max
LINEAR_INSIDE = 32   # 128-column groups of one row that fb_fp4_linear always quantises inside the product


class Fp4Tensor:
    """A 4-bit tensor ``[..., rows, cols]``: ``codes`` [..., rows, 64 * ceil(cols / 128)] uint8 (the even column in the low
    nibble, zero codes behind the last column) and ``scales`` [..., ceil(rows / 128), C, 512] uint8 with C =
    ceil(cols / 128) (mxfp4) or twice that (nvfp4): byte ``16 i + 4 g + s`` of a chunk is the scale of row ``32 g + i`` and
    block ``s`` of the chunk's four.  Scales are not negative (an nvfp4 byte has no sign bit); scale bytes of rows and blocks that
    do not exist are never NaN codes.

    ``tensor_scale`` (a float, nvfp4 only) multiplies every value."""

    __slots__ = ("codes", "scales", "fmt", "shape", "tensor_scale")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str, shape, tensor_scale: Optional[float] = None):
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        shape = tuple(shape)
        if len(shape) < 2 or shape[-1] < 1 or min(shape) < 0:
            raise ValueError(f"a 4-bit tensor has a shape [..., rows, cols >= 1], got {shape}")
        if tensor_scale is not None:
            _check_scale(tensor_scale, fmt)
        g = (shape[-1] + 127) >> 7
        if codes.shape != (*shape[:-1], 64 * g) or scales.shape != (*shape[:-2], (shape[-2] + 127) >> 7, g if fmt == "mxfp4" else 2 * g, 512):
            raise ValueError(f"codes {tuple(codes.shape)} / scales {tuple(scales.shape)} do not belong to a {fmt} tensor of shape {shape}")
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
            raise TypeError("codes and scales are uint8")
        if codes.device != scales.device:
            raise ValueError("codes and scales are on different devices")
        if not (codes.is_contiguous() and scales.is_contiguous()) or codes.data_ptr() & 31 or scales.data_ptr() & 15:
            raise ValueError("codes and scales are contiguous, codes on a 32-byte and scales on a 16-byte boundary")
        self.codes, self.scales, self.fmt, self.shape, self.tensor_scale = codes, scales, fmt, shape, tensor_scale

    @classmethod
    def _of(cls, codes, scales, fmt, shape, tensor_scale):
        """Without the checks, for parts that were made here."""
        t = cls.__new__(cls)
        t.codes, t.scales, t.fmt, t.shape, t.tensor_scale = codes, scales, fmt, shape, tensor_scale
        return t

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, device, non_blocking: bool = False) -> "Fp4Tensor":
        """The same tensor on another device."""
        move = lambda t: t.to(device, non_blocking=non_blocking)
        return Fp4Tensor(move(self.codes), move(self.scales), self.fmt, self.shape, self.tensor_scale)

    def __repr__(self) -> str:
        return f"Fp4Tensor({self.fmt}, shape={self.shape}, tensor_scale={self.tensor_scale}, device={self.device})"

    @staticmethod
    def from_rows(packed: torch.Tensor, scale: torch.Tensor, fmt: str = "mxfp4", tensor_scale: Optional[float] = None) -> "Fp4Tensor":
        """From checkpoint order: ``packed`` [..., rows, cols / 2] codes (cols a whole number of blocks) and ``scale`` bytes
        [..., rows, cols / block], as ``ops/quant.py::quant_fp4_weight`` returns them.  Copies; done once at load time."""
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        if packed.dim() < 2 or not packed.shape[-1]:
            raise ValueError(f"packed has a shape [..., rows, cols / 2], got {tuple(packed.shape)}")
        if packed.device != scale.device:
            raise ValueError(f"packed is on {packed.device}, scale on {scale.device}")
        rows, cols = packed.shape[-2], 2 * packed.shape[-1]
        if tuple(scale.shape) != (*packed.shape[:-1], cols // BLOCK[fmt]) or cols % BLOCK[fmt]:
            raise ValueError(f"packed {tuple(packed.shape)} and scale {tuple(scale.shape)} do not match for {fmt}")
        if packed.dtype != torch.uint8 or scale.dtype != torch.uint8:
            raise TypeError("packed codes and scale bytes are uint8")
        g = (cols + 127) // 128
        codes = torch.nn.functional.pad(packed, (0, 64 * g - cols // 2)).contiguous()
        if codes.data_ptr() == packed.data_ptr():   # nothing was padded: the caller's bytes, on whatever boundary
            codes = codes.clone()
        return Fp4Tensor(codes, pack_scales(scale, 128 * g // BLOCK[fmt]), fmt, (*packed.shape[:-1], cols), tensor_scale)


def pack_scales(scale: torch.Tensor, blocks: Optional[int] = None) -> torch.Tensor:
    """Scale bytes [..., rows, n] in row order -> chunks [..., ceil(rows / 128), ceil(blocks / 4), 512]; missing bytes are 0
    (a valid exponent, and a zero in e4m3)."""
    rows, n = scale.shape[-2:]
    blocks = max(n, blocks or 0)
    s = torch.nn.functional.pad(scale, (0, blocks - n + -blocks % 4, 0, -rows % 128))
    lead = s.shape[:-2]
    s = s.reshape(*lead, s.shape[-2] // 128, 4, 32, s.shape[-1] // 4, 4)
    k = len(lead)
    out = s.permute(*range(k), k, k + 3, k + 2, k + 1, k + 4)
    return out.reshape(*lead, s.shape[k], s.shape[k + 3], 512).contiguous()


def unpack_scales(chunks: torch.Tensor, rows: int, blocks: int) -> torch.Tensor:
    """The inverse of :func:`pack_scales`: bytes [..., rows, blocks]."""
    lead = chunks.shape[:-3]
    k = len(lead)
    s = chunks.reshape(*lead, chunks.shape[k], chunks.shape[k + 1], 32, 4, 4).permute(*range(k), k, k + 3, k + 2, k + 1, k + 4)
    return s.reshape(*lead, chunks.shape[k] * 128, -1)[..., :rows, :blocks]


def _check_scale(ts: float, fmt: str) -> None:
    if fmt != "nvfp4":
        raise ValueError("tensor_scale belongs to nvfp4")
    if not (isinstance(ts, (int, float)) and 2.0 ** -100 <= ts <= 2.0 ** 100):
        raise ValueError(f"tensor_scale is a number in [2^-100, 2^100], got {ts!r}")


def _alpha(xs: Optional[float], ws: Optional[float]) -> float:
    """The factor of a product's sums.  (The scales of an ordinary pair multiply to something near one; out of this range the
    factor itself would overflow f32 or lose bits.)"""
    if xs is None and ws is None:
        return 1.0
    alpha = (xs or 1.0) * (ws or 1.0)
    if not 2.0 ** -100 <= alpha <= 2.0 ** 100:
        raise ValueError(f"the product of the tensor scales must be in [2^-100, 2^100], got {alpha!r}")
    return float(alpha)


def _call(device: torch.device, name: str, *args) -> None:
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        _lib.lib().call(name, *args, stream=stream)
    else:
        with torch.cuda.device(index):
            _lib.lib().call(name, *args, stream=stream)


def _matrix(x: torch.Tensor, what: str) -> Tuple[int, int, int, int, int]:
    """(batch, rows, cols, batch stride, row stride) of a tensor whose leading dimensions form one stride."""
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what} is float32, bfloat16 or float16, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{what} is not on a CUDA device")
    shape = x.shape
    if len(shape) < 2:
        raise ValueError(f"{what} has a shape [..., rows, cols], got {tuple(shape)}")
    rows, cols = shape[-2:]
    if cols < 1:
        raise ValueError(f"{what} has no columns")
    if len(shape) == 2 and x.is_contiguous():
        return 1, rows, cols, 0, cols
    ld = x.stride(-2) if rows > 1 else cols
    if (cols > 1 and x.stride(-1) != 1) or ld < cols:
        raise ValueError(f"{what} has rows of consecutive values that do not overlap, got strides {x.stride()}")
    if x.dim() == 2:
        return 1, rows, cols, 0, ld
    if x.numel() == 0:
        return 0, rows, cols, 0, ld
    batch, bs = 1, rows * ld
    for n, s in zip(reversed(x.shape[:-2]), reversed(x.stride()[:-2])):   # innermost first
        if n == 1:
            continue
        if batch == 1:
            bs = s
        elif s != bs * batch:
            raise ValueError(f"the leading dimensions of {what} have no common stride: {tuple(x.shape)} {x.stride()}")
        batch *= n
    return batch, rows, cols, bs, ld


def quantize(x: torch.Tensor, fmt: str = "mxfp4", tensor_scale: Optional[float] = None) -> Fp4Tensor:
    """Quantise ``x`` [..., rows, cols] (f32, bf16 or f16; rows may be strided) along its last dimension."""
    if fmt not in FORMATS:
        raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
    if tensor_scale is not None:
        _check_scale(tensor_scale, fmt)
    batch, rows, cols, bs, ld = _matrix(x, "x")
    g = (cols + 127) // 128
    lead, dev = x.shape[:-2], x.device
    codes = torch.empty(*lead, rows, 64 * g, dtype=torch.uint8, device=dev)
    scales = torch.empty(*lead, (rows + 127) // 128, g if fmt == "mxfp4" else 2 * g, 512, dtype=torch.uint8, device=dev)
    if batch * rows:
        _call(dev, "fb_fp4_quantize", x, _DTYPES[x.dtype], ld, bs, codes, scales, batch, rows, cols, FORMATS[fmt],
              float(tensor_scale or 0.0))
    return Fp4Tensor._of(codes, scales, fmt, tuple(x.shape), tensor_scale)


def _extent(t: torch.Tensor) -> int:
    """Bytes from the first to behind the last element."""
    n = t.numel()
    if n and not t.is_contiguous():
        n = 1 + sum((k - 1) * s for k, s in zip(t.shape, t.stride()))
    return n * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of consecutive last dimensions may share memory: the spans between their first and last elements
    meet, and they are not columns of one buffer that lie beside each other."""
    a0, b0 = a.data_ptr(), b.data_ptr()
    if b0 >= a0 + _extent(a) or a0 >= b0 + _extent(b):
        return False
    if a.dim() == b.dim() == 2 and a.shape[0] > 1 and b.shape[0] > 1:
        pitch = a.stride(0) * a.element_size()
        if pitch and pitch == b.stride(0) * b.element_size():
            d = (b0 - a0) % pitch
            return d < a.shape[1] * a.element_size() or d + b.shape[1] * b.element_size() > pitch
    return True


def _out(out: Optional[torch.Tensor], shape, dtype: torch.dtype, device: torch.device, *operands: torch.Tensor):
    """``out`` (which must not meet itself or an operand) or a new tensor of ``shape``, and its :func:`_matrix`."""
    if out is None:
        if dtype not in _DTYPES:
            raise TypeError(f"out is float32, bfloat16 or float16, got {dtype}")
        out = torch.empty(*shape, dtype=dtype, device=device)
        rows, cols = shape[-2:]
        return out, (math.prod(shape[:-2]), rows, cols, rows * cols, cols)
    if tuple(out.shape) != tuple(shape) or out.device != device:
        raise ValueError(f"out must be {tuple(shape)} on {device}, got {tuple(out.shape)} on {out.device}")
    if not out.numel():
        return out, (0, 0, 0, 0, 0)
    batch, rows, cols, bs, ld = m = _matrix(out, "out")
    if batch > 1 and bs < (rows - 1) * ld + cols and not (bs >= cols and (batch - 1) * bs + cols <= ld):
        raise ValueError(f"the matrices of out overlap: strides {out.stride()}")
    if any(_overlap(out, t) for t in operands):
        raise ValueError("out and an operand share memory")
    return out, m


def _status(status: Optional[torch.Tensor], device: torch.device) -> Optional[torch.Tensor]:
    if status is not None and (status.dtype is not torch.int32 or status.dim() != 1 or status.numel() < 4 or status.stride(0) != 1
                               or status.device != device):
        raise ValueError(f"status must be four consecutive int32 words on {device}, got {status.dtype} {tuple(status.shape)} on {status.device}")
    return status


def dequantize(q: Fp4Tensor, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values of ``q``, rounded to ``dtype`` (or into ``out``, whose rows may be strided): once without a tensor scale
    (code times block scale is exact in f32); with one, their f32 product with the scale, rounded to f32, is."""
    if not q.codes.is_cuda:
        raise ValueError("q is not on a CUDA device")
    out, (batch, rows, cols, bs, ld) = _out(out, q.shape, dtype, q.device, q.codes, q.scales)
    if batch * rows:
        _call(q.device, "fb_fp4_dequantize", q.codes, q.scales, out, _DTYPES[out.dtype], ld, bs, batch, rows, cols,
              FORMATS[q.fmt], float(q.tensor_scale or 0.0))
    return out


def matmul(x: Fp4Tensor, w: Fp4Tensor, out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None,
           status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T`` of two 4-bit matrices [M, K] and [N, K] of one format: products of the values they stand for, summed in
    f32, multiplied in f32 by the product of their tensor scales (itself rounded to f32) and rounded to ``out_dtype``, or to the
    type of a given ``out``.  ``status``: see the module."""
    if len(x.shape) != 2 or len(w.shape) != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"matmul takes [M, K] and [N, K], got {x.shape} and {w.shape}")
    if x.fmt != w.fmt:
        raise ValueError(f"matmul takes two tensors of one format, got {x.fmt} and {w.fmt}")
    if not x.codes.is_cuda or x.device != w.device:
        raise ValueError(f"matmul takes tensors of one CUDA device, got {x.device} and {w.device}")
    M, N, K = x.shape[0], w.shape[0], x.shape[1]
    alpha = _alpha(x.tensor_scale, w.tensor_scale)
    status = _status(status, x.device)
    out, (_, _, _, _, ldo) = _out(out, (M, N), out_dtype, x.device, x.codes, x.scales, w.codes, w.scales)
    if M and N:
        _call(x.device, "fb_fp4_matmul", x.codes, x.scales, w.codes, w.scales, out, _DTYPES[out.dtype], ldo, M, N, K,
              FORMATS[x.fmt], alpha, status)
    return out


def linear(x: torch.Tensor, w: Fp4Tensor, out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
           x_scale: Optional[float] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``quantize(x, w.fmt, x_scale) @ w.T`` for ``x`` [M, K] (f32, bf16, f16) and 4-bit weights [N, K], in one call
    (a few short rows in one launch, else two).  ``out_dtype`` defaults to x's; a given ``out`` keeps its own type and must
    not share memory with an operand.  ``status``: see the module."""
    if x.dim() != 2 or len(w.shape) != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"linear takes [M, K] and 4-bit [N, K], got {tuple(x.shape)} and {w.shape}")
    if x_scale is not None:
        _check_scale(x_scale, w.fmt)
    alpha = _alpha(x_scale, w.tensor_scale)
    _, M, K, _, ldx = _matrix(x, "x")
    dev = x.device
    if dev != w.device:
        raise ValueError(f"x is on {dev}, w on {w.device}")
    status = _status(status, dev)
    N = w.shape[0]
    if out is None:
        out, ldo = torch.empty(M, N, dtype=out_dtype or x.dtype, device=dev), N
        if out.dtype not in _DTYPES:
            raise TypeError(f"out is float32, bfloat16 or float16, got {out.dtype}")
    else:
        out, (_, _, _, _, ldo) = _out(out, (M, N), out.dtype, dev, x, w.codes, w.scales)
    if M and N:
        g = (K + 127) // 128
        work = None
        if M > 1 or g > LINEAR_INSIDE:   # (one row of up to so many groups is quantised inside the product)
            work = torch.empty((M * 64 * g + 511) // 512 * 512 + (M + 127) // 128 * (g if w.fmt == "mxfp4" else 2 * g) * 512,
                               dtype=torch.uint8, device=dev)
        _call(dev, "fb_fp4_linear", x, _DTYPES[x.dtype], ldx, work, w.codes, w.scales, out, _DTYPES[out.dtype], ldo, M, N, K,
              FORMATS[w.fmt], float(x_scale or 0.0), alpha, status)
    return out


SCORES = {"sqrtsoftplus": 0, "sigmoid": 1, "softmax": 2}
MOE_MAX_TOKENS, MOE_MAX_EXPERTS, MOE_MAX_TOPK, MOE_MAX_DIM = 32, 512, 32, 8192


def moe(x: torch.Tensor, logits: torch.Tensor, w13: Fp4Tensor, w2: Fp4Tensor, topk: int, *, bias: Optional[torch.Tensor] = None,
        score: str = "sqrtsoftplus", norm: bool = True, scale: float = 1.0, limit: float = 0.0,
        out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None, accumulate: bool = False,
        status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The routed experts of a layer for up to 32 tokens, in two kernels.

    ``x`` [T, D] (f32, bf16, f16), ``logits`` [T, E] f32 of the router, ``w13`` mxfp4 [E, 2, I, D] (gate, up), ``w2`` mxfp4
    [E, D, I] (I a multiple of 32).  Every token takes the ``topk`` experts of largest ``score(logits) + bias``, computed and
    added in f32 (ties and equal logits to the lower index; NaN below every number; without a bias the logits decide), weighted by
    ``scale * score``, with ``norm`` divided by the sum of the chosen scores (scores that are all zero in f32 stay zero).  Activations meet the weights as e4m3 with a
    power-of-two scale per 32 values (``ops/quant.py::fp8_act_roundtrip``): x before the gate and up products, and
    ``silu(min(g, limit)) * clamp(u, -limit, limit) * weight`` before the down product (``limit`` 0: no clamp).  The
    result, summed in f32, is rounded once to ``out_dtype`` (default: x's) or, with ``accumulate``, added to ``out``, which
    may be x.  A NaN in a token stays in that token's row; a NaN scale in ``w2`` reaches every row of a call in which any token
    takes that expert (all experts share one accumulator), so ``w2`` should hold none.  ``status``: see the module."""
    if score not in SCORES:
        raise ValueError(f"score must be one of {sorted(SCORES)}, got {score!r}")
    if w13.fmt != "mxfp4" or w2.fmt != "mxfp4":
        raise ValueError("moe takes mxfp4 experts")
    if len(w13.shape) != 4 or w13.shape[1] != 2 or len(w2.shape) != 3:
        raise ValueError(f"moe takes w13 [E, 2, I, D] and w2 [E, D, I], got {w13.shape} and {w2.shape}")
    E, _, I, D = w13.shape
    if w2.shape != (E, D, I):
        raise ValueError(f"w13 {w13.shape} asks for w2 {(E, D, I)}, got {w2.shape}")
    if I % 32 or I < 32:
        raise ValueError(f"moe takes experts of a multiple of 32 columns, got {I}")
    if x.dim() != 2 or x.shape[1] != D:
        raise ValueError(f"x must be [T, {D}], got {tuple(x.shape)}")
    T = x.shape[0]
    if T > MOE_MAX_TOKENS or not 1 <= E <= MOE_MAX_EXPERTS or not 1 <= topk <= min(E, MOE_MAX_TOPK):
        raise ValueError(f"moe takes up to {MOE_MAX_TOKENS} tokens, {MOE_MAX_EXPERTS} experts and topk {MOE_MAX_TOPK}, "
                         f"got {T}, {E}, {topk}")
    if D > MOE_MAX_DIM:
        raise ValueError(f"moe takes rows of up to {MOE_MAX_DIM} values, got {D}")
    if not (limit >= 0.0) or not abs(scale) <= _F32_MAX:
        raise ValueError(f"limit must not be negative and scale must be finite in f32, got {limit}, {scale}")
    if logits.dtype != torch.float32 or tuple(logits.shape) != (T, E) or (E > 1 and logits.stride(1) != 1) or (T > 1 and logits.stride(0) < E):
        raise ValueError(f"logits must be f32 {(T, E)} with rows of consecutive values, got {logits.dtype} {tuple(logits.shape)} {logits.stride()}")
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (E,) or not bias.is_contiguous()):
        raise ValueError(f"bias must be contiguous f32 {(E,)}, got {bias.dtype} {tuple(bias.shape)}")
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    dev = w13.device
    if any(t is not None and t.device != dev for t in (x, logits, bias, w2.codes)):
        raise ValueError("moe takes tensors of one device")
    status = _status(status, dev)
    _, _, _, _, ldx = _matrix(x, "x")
    out, (_, _, _, _, ldo) = _out(out, (T, D), out_dtype or x.dtype, dev, w13.codes, w13.scales, w2.codes, w2.scales)
    if T:
        tile = 128 * (8 if T <= 8 else 16 if T <= 16 else 32) + 512
        work = torch.empty(4096 + min(E, T * topk) * ((I + 127) // 128) * tile, dtype=torch.uint8, device=dev)
        _call(dev, "fb_fp4_moe", x, _DTYPES[x.dtype], ldx, logits, logits.stride(0) if T > 1 else E, bias, w13.codes, w13.scales,
              w2.codes, w2.scales, out, _DTYPES[out.dtype], ldo, int(accumulate), work, T, E, topk, D, I, SCORES[score], int(norm),
              float(scale), float(limit) if limit else math.inf, status)
    return out


def check(device=None) -> None:
    """Raise ``KernelError`` if a wait inside one of this module's kernels on ``device`` (default: the current one) that was
    given no ``status`` ran out since the last check.  Waits for the current stream alone, and clears the words for every
    caller on the device: calls that have to be told apart get a ``status`` of their own."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    host = (ctypes.c_int * 4)()
    with torch.cuda.device(dev):
        _lib.lib().call("fb_fp4_status", ctypes.cast(host, ctypes.POINTER(ctypes.c_int)), 1)
    if host[0]:
        raise _lib.KernelError(f"a wait of a 4-bit kernel ran out (block {host[1]}, {host[2]}, {host[3]}): its output is not valid")


def reference_dequantize(q: Fp4Tensor) -> torch.Tensor:
    """The values of ``q`` as f64, in plain torch (CPU or GPU): the statement that the kernels are tested against."""
    from .quant import e2m1_decode, ue8m0_decode
    rows, cols = q.shape[-2:]
    v = e2m1_decode(e2m1_unpack(q.codes)).double()
    b = BLOCK[q.fmt]
    s = unpack_scales(q.scales, rows, v.shape[-1] // b)
    if q.fmt == "mxfp4":
        f = torch.where(s == 255, torch.full((), math.nan, dtype=torch.float64, device=s.device), ue8m0_decode(s).double())
        f = torch.where(s == 0, torch.full((), 2.0 ** -127, dtype=torch.float64, device=s.device), f)
    else:
        f = s.contiguous().view(torch.float8_e4m3fn).double()
    return (v.unflatten(-1, (-1, b)) * f.unsqueeze(-1)).flatten(-2)[..., :cols] * (q.tensor_scale or 1.0)
