"""A causal language model's last steps on the GPU: final norm, vocabulary product
in microscaled floating point, log probabilities.

The reference re-ranks with the log probabilities that its inference engine
returns for answer tokens (pipeline/utils/vllm_handler.py:109-144); rerank.py does
it with these operators behind a decoder whose body stays a PyTorch(-ROCm)
forward, as the encoder's does.

    mx_quantize(x, format)                  -> MxRows        rows in blocks of 32 with a shared power-of-two scale
    mx_dequantize(rows, dtype)              -> (n, d) tensor
    rms_norm_mx(x, weight, eps, residual)   -> (MxRows, updated residual)
    mx_matmul(a, b, dtype)                  -> (m, n) tensor, a's rows times b's
    token_logprobs(logits, tokens, top_k)   -> TokenLogprobs

Everything is enqueued on torch's current stream of the tensors' GPU without
waiting, allocates through torch, and can be captured into a HIP graph.  The
operators have no derivatives: they refuse inputs that record a backward pass or
carry a forward-mode tangent.
"""
from __future__ import annotations

from collections import namedtuple

import torch
from torch.autograd import forward_ad

from . import _native

__all__ = ["MxRows", "TokenLogprobs", "mx_quantize", "mx_dequantize", "rms_norm_mx", "mx_matmul", "token_logprobs"]

FORMATS = {"mxfp4": _native.MTR_MX_FP4, "mxfp8": _native.MTR_MX_FP8}
BLOCK, PAD = _native.MTR_MX_BLOCK, _native.MTR_MX_PAD
MOST = (1 << 31) - 1        # what the library's 32-bit numbers hold: ctypes would cut off the rest without a word

TokenLogprobs = namedtuple("TokenLogprobs", "logprobs entropy top_ids top_logprobs")
TokenLogprobs.__doc__ = """What token_logprobs returns: logprobs (n, g) and entropy (n,) float32, top_ids (n, top_k)
int64, top_logprobs (n, top_k) float32."""

_CODES = {torch.float32: _native.MTR_F32, torch.bfloat16: _native.MTR_BF16, torch.float16: _native.MTR_F16}
# The handle of the current stream alone: building a Stream object around it costs as much as a launch.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _code(dtype, what):
    """The library's code of a torch dtype it takes."""
    code = _CODES.get(dtype)
    if code is None:
        raise TypeError(f"{what}: unsupported dtype {dtype}")
    return code


def _no_derivative(t, what):
    """Refuses a tensor whose derivatives would be lost without a word."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} has no backward pass: detach its inputs or call it under torch.no_grad()")
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what} has no forward derivative: pass the primal of its dual tensors")


def _rows(x, what):
    """A (n, d) GPU tensor with dense rows (copied if its last dimension is strided, or if it stands for
    the negative of what its memory holds, as the imaginary part of a conjugate does)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() != 2:
        raise ValueError(f"{what} wants a 2-D GPU tensor")
    _no_derivative(x, what)
    if x.is_neg():
        x = x.resolve_neg()
    return x if x.stride(1) == 1 or x.shape[1] < 2 else x.contiguous()


def _into(out, what):
    """Checks `out` of an operator without derivatives."""
    if not isinstance(out, torch.Tensor) or not out.is_cuda:
        raise ValueError(f"{what}: out must be a GPU tensor")
    if out.is_neg():
        raise ValueError(f"{what}: out stands for the negative of its memory")
    _no_derivative(out, what)


def _written(out):
    """Tells autograd that `out` has been overwritten: not before, as a refused call leaves it as it was."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def _width(d, format):
    """(element bytes, scale bytes) of a stored row."""
    padded = (d + PAD - 1) // PAD * PAD
    return (padded // 2 if format == "mxfp4" else padded), padded // BLOCK


class MxRows:
    """Rows in microscaled floating point, as include/medtutor_retrieval.h lays them
    out: `values` (n, element bytes) and `scales` (n, scale bytes), uint8 tensors on
    one GPU with dense rows, the number `d` of elements of a row, and the `format`,
    "mxfp4" or "mxfp8"."""

    __slots__ = ("_values", "_scales", "_both", "_n", "_at", "d", "format", "device")

    def __init__(self, values, scales, d: int, format: str = "mxfp4"):
        if format not in FORMATS:
            raise ValueError(f"format must be one of {sorted(FORMATS)}")
        if not 1 <= d <= MOST:
            raise ValueError(f"rows of {d} elements: at least one, at most {MOST}")
        for t in (values, scales):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.uint8 or t.dim() != 2 or not t.is_contiguous():
                raise ValueError("MxRows wants contiguous 2-D uint8 GPU tensors")
        if values.device != scales.device:
            raise ValueError(f"values are on {values.device}, scales on {scales.device}")
        want = _width(d, format)
        if (values.shape[1], scales.shape[1]) != want or values.shape[0] != scales.shape[0]:
            raise ValueError(f"{format} rows of {d} elements have {want[0]} element and {want[1]} scale bytes, "
                             f"got {tuple(values.shape)} and {tuple(scales.shape)}")
        self._values, self._scales, self._both = values, scales, None
        self._n, self._at = values.shape[0], (values.data_ptr(), scales.data_ptr())
        self.d, self.format, self.device = int(d), format, values.device

    @classmethod
    def empty(cls, n, d, format, device):
        """Room for n rows, values and scales in one allocation."""
        if format not in FORMATS:
            raise ValueError(f"format must be one of {sorted(FORMATS)}")
        if not 1 <= d <= MOST:
            raise ValueError(f"rows of {d} elements: at least one, at most {MOST}")
        width, blocks = _width(d, format)
        rows = cls.__new__(cls)
        both = torch.empty_strided((n * (width + blocks),), (1,), dtype=torch.uint8, device=device)
        start = both.data_ptr()
        rows._both, rows._values, rows._scales = both, None, None
        rows._n, rows._at = n, (start, start + n * width)
        rows.d, rows.format, rows.device = d, format, both.device
        return rows

    @property
    def values(self):
        if self._values is None:
            width = _width(self.d, self.format)[0]
            self._values = self._both[:self._n * width].view(self._n, width)
        return self._values

    @property
    def scales(self):
        if self._scales is None:
            width, blocks = _width(self.d, self.format)
            self._scales = self._both[self._n * width:].view(self._n, blocks)
        return self._scales

    def __len__(self):
        return self._n

    @property
    def nbytes(self):
        return self._n * sum(_width(self.d, self.format))

    def rows(self, lo, hi):
        """Rows [lo, hi) as a view."""
        return MxRows(self.values[lo:hi], self.scales[lo:hi], self.d, self.format)

    def __reduce__(self):       # copies and pickles hold their own tensors' addresses
        return MxRows, (self.values, self.scales, self.d, self.format)

    def __repr__(self):
        return f"MxRows({len(self)} x {self.d}, {self.format}, {self.device})"


def mx_quantize(x, format: str = "mxfp4") -> MxRows:
    """(n, d) float32 / bfloat16 / float16 rows to microscaled floating point: blocks
    of 32 with the smallest power-of-two scale under which the block's largest
    magnitude rounds to the largest element or less, elements rounded to nearest,
    ties to even.  A block that holds a NaN or infinity reads back as NaN."""
    x = _rows(x, "mx_quantize")
    n, d = x.shape
    code = _code(x.dtype, "mx_quantize")
    device = x.device
    out = MxRows.empty(n, d, format, device)
    values, scales = out._at
    rc = _native.lib().mtr_mx_quantize(x.data_ptr(), code, n, d, x.stride(0), FORMATS[format], values, scales, device.index,
                                       _stream(device.index))
    if rc:
        _native.check(rc)
    return out


def mx_dequantize(rows: MxRows, dtype=None, out=None):
    """What microscaled rows stand for, as a (n, d) tensor of `dtype` (bfloat16, which
    holds every value exactly but the very smallest, unless given) or into `out`, a
    (n, d) GPU tensor with dense rows that do not overlap."""
    n, d, device, given = rows._n, rows.d, rows.device, out is not None
    if not given:
        dtype = dtype or torch.bfloat16
        code = _code(dtype, "mx_dequantize")
        out = torch.empty_strided((n, d), (d, 1), dtype=dtype, device=device)
    else:
        _into(out, "mx_dequantize")
        code = _code(out.dtype, "mx_dequantize")
        if out.shape != (n, d) or out.device != device or (d > 1 and out.stride(1) != 1) or (dtype is not None and dtype != out.dtype):
            raise ValueError("out must be a (n, d) tensor of the dtype on the rows' GPU, its rows dense")
    values, scales = rows._at
    rc = _native.lib().mtr_mx_dequantize(values, scales, FORMATS[rows.format], n, d, out.data_ptr(), code, out.stride(0), device.index,
                                         _stream(device.index))
    if rc:
        _native.check(rc)
    if given:
        _written(out)
    return out


def rms_norm_mx(x, weight, eps: float = 1e-6, residual=None, format: str = "mxfp8"):
    """Root-mean-square norm of x + residual, as microscaled rows: (MxRows, h) with
    h = x + residual in their dtype (None without a residual), the rows
    h / sqrt(mean(h^2) + eps) * weight.  x, residual: (n, d), one dtype; weight: (d,)
    of that dtype or float32.  Sums are in 32 bits: a row whose squares add up to more
    than float32 holds comes back as zeros (one whose squares are less than it holds does
    not).  A zero row gives zeros, with eps 0 too.  d up to 65536."""
    x = _rows(x, "rms_norm_mx")
    n, d = x.shape
    dtype, device = x.dtype, x.device
    code = _code(dtype, "rms_norm_mx")
    if (not isinstance(weight, torch.Tensor) or weight.shape != (d,) or weight.device != device
            or weight.dtype not in (dtype, torch.float32)):
        raise ValueError(f"rms_norm_mx wants a ({d},) weight of the rows' dtype or float32 on their GPU")
    _no_derivative(weight, "rms_norm_mx")
    if weight.is_neg():
        weight = weight.resolve_neg()
    if weight.stride(0) != 1:
        weight = weight.contiguous()
    h = None
    if residual is not None:
        residual = _rows(residual, "rms_norm_mx")
        if residual.shape != x.shape or residual.dtype != dtype or residual.device != device:
            raise ValueError("rms_norm_mx wants a residual of the rows' shape and dtype on their GPU")
        h = torch.empty_strided((n, d), (d, 1), dtype=dtype, device=device)
    out = MxRows.empty(n, d, format, device)
    values, scales = out._at
    rc = _native.lib().mtr_rms_norm_mx(
        x.data_ptr(), None if h is None else residual.data_ptr(), weight.data_ptr(), code, _CODES[weight.dtype], n, d, x.stride(0),
        0 if h is None else residual.stride(0), eps, FORMATS[format], None if h is None else h.data_ptr(), values, scales, device.index,
        _stream(device.index))
    if rc:
        _native.check(rc)
    return out, h


def mx_matmul(a: MxRows, b: MxRows, dtype=None, out=None):
    """(m, n) products of a's m rows (either format) with b's n rows (mxfp4), summed in
    32 bits; float32 unless `dtype` says bfloat16, or into `out`, a (m, n) GPU tensor
    with dense rows that do not overlap.  Rows of 1024 results and more start on 128
    bytes, as an index's rows do: where n is no multiple of that, the result is not
    contiguous (its stride(0) is larger than n).  Sums are held in 32 bits whatever the
    sizes and the result's type, and rounded once."""
    if b.format != "mxfp4":
        raise ValueError("mx_matmul wants its second operand in mxfp4")
    if a.d != b.d:
        raise ValueError(f"rows of {a.d} and of {b.d} elements")
    device = a.device
    if device != b.device:
        raise ValueError(f"operands are on {device} and {b.device}")
    m, n, given = a._n, b._n, out is not None
    if not given:
        dtype = dtype or torch.float32
        line = 32 if dtype == torch.float32 else 64
        out = torch.empty_strided((m, n), (n if n < 1024 else (n + line - 1) // line * line, 1), dtype=dtype, device=device)
    else:
        _into(out, "mx_matmul")
        if out.shape != (m, n) or out.device != device or (n > 1 and out.stride(1) != 1) or (dtype is not None and dtype != out.dtype):
            raise ValueError("out must be a (m, n) tensor of the dtype on the operands' GPU, its rows dense")
    if out.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"mx_matmul: unsupported dtype {out.dtype}")
    lib = _native.lib()
    need = lib.mtr_mx_matmul_workspace(m, n, a.d)
    workspace = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device) if need else None
    rc = lib.mtr_mx_matmul(*a._at, FORMATS[a.format], m, *b._at, n, a.d, out.data_ptr(), _CODES[out.dtype], out.stride(0),
                           workspace.data_ptr() if need else None, need, device.index, _stream(device.index))
    if rc:
        _native.check(rc)
    if given:
        _written(out)
    return out


def token_logprobs(logits, tokens=None, top_k: int = 0) -> TokenLogprobs:
    """Of (n, v) float32 / bfloat16 / float16 logits: the log probabilities of the given
    tokens, (n,) or (n, g) int64, the entropy in nats, and the top_k (up to 64) best
    tokens with theirs, ordered by (logit descending, id ascending).

    Logits of -inf are excluded tokens: their log probability is -inf and they are no
    alternatives; slots beyond the tokens that are left hold id -1 and -inf.  A row
    with nothing left has entropy 0; one that holds a NaN or +inf has NaN everywhere.
    A negative token is padding, its log probability 0; one >= v gives NaN (the call
    does not wait for the GPU and so cannot raise)."""
    logits = _rows(logits, "token_logprobs")
    n, v = logits.shape
    code = _code(logits.dtype, "token_logprobs")
    device = logits.device
    if tokens is None:
        g = 0
    else:
        if not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int64 or tokens.device != device:
            raise ValueError("token_logprobs wants int64 tokens on the logits' GPU")
        if tokens.dim() == 1:
            tokens = tokens[:, None]
        if tokens.dim() != 2 or tokens.shape[0] != n:
            raise ValueError(f"token_logprobs wants ({n},) or ({n}, g) tokens, got {tuple(tokens.shape)}")
        tokens = tokens.contiguous()
        g = tokens.shape[1]
        if g > MOST:
            raise ValueError(f"{g} tokens a row: at most {MOST}")
    if not 0 <= top_k <= _native.MTR_MAX_ALTERNATIVES:
        raise ValueError(f"top_k must be in [0, {_native.MTR_MAX_ALTERNATIVES}]")
    lib = _native.lib()
    empty = torch.empty_strided
    logprobs = empty((n, g), (g, 1), dtype=torch.float32, device=device)
    entropy = empty((n,), (1,), dtype=torch.float32, device=device)
    top_ids = empty((n, top_k), (top_k, 1), dtype=torch.int64, device=device)
    top_logprobs = empty((n, top_k), (top_k, 1), dtype=torch.float32, device=device)
    need = lib.mtr_token_logprobs_workspace(n, v, top_k)
    workspace = empty((need,), (1,), dtype=torch.uint8, device=device) if need else None
    rc = lib.mtr_token_logprobs(
        logits.data_ptr(), code, n, v, logits.stride(0), tokens.data_ptr() if g else None, g, top_k, logprobs.data_ptr(), entropy.data_ptr(),
        top_ids.data_ptr(), top_logprobs.data_ptr(), workspace.data_ptr() if need else None, need, device.index, _stream(device.index))
    if rc:
        _native.check(rc)
    return TokenLogprobs(logprobs, entropy, top_ids, top_logprobs)
