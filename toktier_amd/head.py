"""The answering end: from a model's last hidden states to the next token ids.

Three operators of ``libtoktier_head.so`` (``include/toktier_head.h``), hand
written for gfx950, and ``OutputHead``, which runs them one after another:

- ``rms_norm_fp8``: root-mean-square norm of ``x + residual``, its output in
  8-bit floats (e4m3) with a power-of-two scale (e8m0) per 128 values;
- ``matmul_fp8``: product of such rows with weights held the same way;
- ``sample``: one token a row by temperature, top-k, top-p and min-p from a
  given random number.

Inputs and outputs are torch tensors on one GPU. Calls queue on torch's
current stream of that device, never synchronize and can be captured into a
graph. There is no CPU fallback: a refused call raises ``EngineError`` with
the library's status and message, a tensor that does not fit raises
``ValueError`` or ``TypeError`` before anything is queued. There is no
backward pass: where an input requires grad so do the outputs, and a backward
pass that reaches them raises; what would have to be written into ``out`` or
``residual_out`` is refused there.

    head = OutputHead(norm_weight, *quantize_fp8(lm_head))
    out = head.next_ids(hidden, u, residual=residual, temperature=0.7, top_p=0.9)
    out.ids        # int32 on the device: rows of the projection, a tokenizer's ids
"""

from __future__ import annotations

import ctypes as C
import operator
import struct
import warnings
from pathlib import Path
from typing import NamedTuple

import torch
from torch.autograd.graph import increment_version as _written

from ._build import HEAD_LIB, verify_head
from ._ffi import EngineError

__all__ = ["rms_norm_fp8", "matmul_fp8", "sample", "quantize_fp8",
           "OutputHead", "NormOutput", "Sampled", "EngineError", "BLOCK"]

BLOCK = 128  # values that share a scale

TKH_F32, TKH_BF16, TKH_F16 = 0, 1, 2
_DTYPES = {torch.float32: TKH_F32, torch.bfloat16: TKH_BF16,
           torch.float16: TKH_F16}
_FP8, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_INF = float("inf")

#: every entry point include/toktier_head.h declares
SYMBOLS = ("tk_head_norm", "tk_head_matmul", "tk_head_sample",
           "tk_head_sample_workspace", "tk_head_last_error",
           "tk_head_abi_version", "tk_head_sources")

#: TKH_ABI_VERSION of the structs packed below
ABI_VERSION = 1

# The argument structs of include/toktier_head.h, packed in one step: a call
# of a single token lasts a few microseconds, and so would filling a
# ctypes.Structure field by field.
_NORM = struct.Struct("6Q7qf3i")
_MATMUL = struct.Struct("5Q8q2i")
_SAMPLE = struct.Struct("11Q4qfi2f2i")

_lib: C.CDLL | None = None


def lib(path: Path | None = None) -> C.CDLL:
    """Load the library (``RuntimeError`` if it was never built or takes other
    arguments; a ``RuntimeWarning`` if its sources have changed since)."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else HEAD_LIB
    if not p.exists():
        raise RuntimeError(
            f"{p} is missing: build it with toktier_amd._build.build_head() "
            "(hipcc --offload-arch=gfx950); there is no CPU fallback")
    L = C.CDLL(str(p))
    # an older library would read the packed arguments by other fields
    version = L.tk_head_abi_version() if hasattr(L, "tk_head_abi_version") else 0
    if version != ABI_VERSION:
        raise RuntimeError(f"{p} takes arguments of version {version}, not {ABI_VERSION}: "
                           "build it again with toktier_amd._build.build_head()")
    stale = verify_head(p)
    if stale:
        warnings.warn(f"{p}: {stale}", RuntimeWarning, stacklevel=2)
    for name in ("tk_head_norm", "tk_head_matmul", "tk_head_sample"):
        f = getattr(L, name)
        f.restype = C.c_int
        f.argtypes = [C.c_char_p, C.c_void_p]
    L.tk_head_sample_workspace.restype = C.c_uint64
    L.tk_head_sample_workspace.argtypes = [C.c_int64, C.c_int64, C.c_int32]
    L.tk_head_last_error.restype = C.c_char_p
    L.tk_head_last_error.argtypes = []
    if path is None:
        _lib = L
    return L


def _fail(status: int, call: str) -> None:
    detail = (lib().tk_head_last_error() or b"").decode("utf-8", "replace")
    raise EngineError(status, call, detail)


# the current stream's handle without the Stream object around it, which
# takes a microsecond to make
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """``t`` as rows of a dense last axis, without copying."""
    if t.dim() != 2:
        if t.dim() == 0:
            raise ValueError(f"{name} has no axis")
        k = t.shape[-1]
        try:
            t = t.view(t.numel() // k if k else 0, k)
        except RuntimeError:
            raise ValueError(f"the leading axes of {name} do not lie at one "
                             "stride: make it contiguous") from None
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"the last axis of {name} is not dense")
    return t


def _on(t: torch.Tensor, device: torch.device, name: str) -> None:
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")


def _gpu(t: torch.Tensor, name: str) -> torch.device:
    device = t.device
    if device.type != "cuda":
        raise ValueError(f"{name} is on {device}: these operators run on a GPU")
    return device


class _NoBackward(torch.autograd.Function):
    """A call's outputs, as they are, where an input of it requires grad: a
    backward pass that reaches them raises instead of passing them over."""

    @staticmethod
    def forward(ctx, call, outputs, *inputs):
        ctx.call = call
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in outputs if not t.is_floating_point()])
        return outputs

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(f"{ctx.call} has no backward pass")


def _untracked(call: str, outputs: tuple, *inputs) -> tuple:
    """``outputs`` of inputs some of which may require grad."""
    if not torch.is_grad_enabled():
        return outputs
    inputs = [t for t in inputs if isinstance(t, torch.Tensor) and t.requires_grad]
    return _NoBackward.apply(call, outputs, *inputs) if inputs else outputs


def _given(t: torch.Tensor, name: str, *inputs) -> None:
    """Refuses to write into ``t`` what autograd would have to follow."""
    if torch.is_grad_enabled() and (t.requires_grad or any(i.requires_grad for i in inputs)):
        raise ValueError(f"{name} where a tensor requires grad: there is no backward pass")


class NormOutput(NamedTuple):
    q: torch.Tensor            # float8_e4m3fn, rows padded to 128 in memory
    scale: torch.Tensor        # float8_e8m0fnu, one for 128 values
    residual: torch.Tensor | None  # x + residual in x's type


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *,
                 residual: torch.Tensor | None = None, eps: float = 1e-6,
                 residual_out: torch.Tensor | None = None) -> NormOutput:
    """``(x + residual) * rsqrt(mean((x + residual)**2) + eps) * weight`` over
    the last axis, computed in 32 bits, as 8-bit values and scales that
    ``matmul_fp8`` reads.

    ``x``: ``[..., k]`` of float32, bfloat16 or float16; ``residual`` like it;
    ``weight``: ``[k]`` of x's type or float32. With a residual, the sum comes
    back in x's type as ``residual`` (into ``residual_out``, which may be
    ``residual`` itself); the norm reads the sum before that rounding. ``q``
    and ``scale`` have x's leading axes; q's rows are padded in memory to a
    multiple of 128 with zeros. Values that are not finite become NaN."""
    device = _gpu(x, "x")
    if not hasattr(eps, "__float__"):
        raise TypeError(f"eps is {eps!r}: a number is wanted")
    kind = x.dtype
    dtype = _DTYPES.get(kind)
    if dtype is None:
        raise TypeError(f"x is {kind}: float32, bfloat16 or float16 is wanted")
    x2 = _rows(x, "x")
    rows, k = x2.shape
    if weight.shape != (k,) or (k > 1 and weight.stride(0) != 1):
        raise ValueError(f"weight has shape {tuple(weight.shape)}: ({k},), dense, is wanted")
    weight_kind = weight.dtype
    if weight_kind != kind and weight_kind != torch.float32:
        raise TypeError(f"weight is {weight_kind}: {kind} or float32 is wanted")
    _on(weight, device, "weight")
    res_ptr = res_stride = out_ptr = out_stride = 0
    given = residual_out is not None
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != kind:
            raise ValueError("residual does not have x's shape and type")
        _on(residual, device, "residual")
        res = _rows(residual, "residual")
        res_ptr, res_stride = res.data_ptr(), res.stride(0)
        if residual_out is None:
            residual_out = x.new_empty(x.shape)
        elif residual_out.shape != x.shape or residual_out.dtype != kind:
            raise ValueError("residual_out does not have x's shape and type")
        else:
            _on(residual_out, device, "residual_out")
            _given(residual_out, "residual_out", x, residual)
        out = _rows(residual_out, "residual_out")
        out_ptr, out_stride = out.data_ptr(), out.stride(0)
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    blocks = (k + BLOCK - 1) // BLOCK
    padded = blocks * BLOCK
    q = x.new_empty((rows, padded), dtype=_FP8)
    scale = x.new_empty((rows, blocks), dtype=_E8M0)
    status = (_lib or lib()).tk_head_norm(_NORM.pack(
        x2.data_ptr(), res_ptr, weight.data_ptr(), q.data_ptr(),
        scale.data_ptr(), out_ptr, rows, k, x2.stride(0), res_stride, padded,
        blocks, out_stride, eps, dtype, _DTYPES[weight_kind], device.index),
        _raw_stream(device.index))
    if status:
        _fail(status, "tk_head_norm")
    if given:
        _written(residual_out)
    if padded != k:
        q = q[:, :k]
    if x.dim() != 2:
        q = q.view(x.shape)
        scale = scale.view(x.shape[:-1] + (blocks,))
    if x.requires_grad or (residual is not None and residual.requires_grad):
        outputs = (q, scale) if residual is None else (q, scale, residual_out)
        q, scale, *rest = _untracked("rms_norm_fp8", outputs, x, weight, residual)
        return NormOutput(q, scale, *(rest or [None]))
    if weight.requires_grad:  # of which the sum knows nothing
        q, scale = _untracked("rms_norm_fp8", (q, scale), weight)
    return NormOutput(q, scale, residual_out)


def _eight(t: torch.Tensor, scale: torch.Tensor, name: str):
    if t.dtype != _FP8:
        raise TypeError(f"{name} is {t.dtype}: {_FP8} is wanted")
    if scale.dtype != _E8M0 and scale.dtype != torch.uint8:
        raise TypeError(f"{name}_scale is {scale.dtype}: {_E8M0} or uint8 is wanted")
    t, s = _rows(t, name), _rows(scale, name + "_scale")
    rows, k = t.shape
    if s.shape != (rows, (k + BLOCK - 1) // BLOCK):
        raise ValueError(f"{name}_scale has shape {tuple(scale.shape)} for rows of {t.shape[1]}")
    return t, s


def matmul_fp8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor,
               w_scale: torch.Tensor, *, out_dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``a @ w.T`` of 8-bit floats with a power-of-two scale for each block of
    128 of the summed axis, rounded once to ``out_dtype`` (bfloat16 or
    float16). The matrix unit cuts each product of 8 neighbours along k to
    about 2**-13 of the largest of them before it adds them up: some 2**-21 of
    the sum of ``|a w|`` on ordinary rows, up to 2**-10 of it where very unequal
    products stand side by side (``include/toktier_head.h``).

    ``a``: ``[..., k]``, ``w``: ``[n, k]`` of float8_e4m3fn, their scales
    ``[..., ceil(k / 128)]`` of float8_e8m0fnu (or its bytes as uint8). Rows
    start at multiples of 16 bytes (``rms_norm_fp8`` and ``quantize_fp8`` give
    such rows for any k; of a single row only the address counts). The result
    is ``[..., n]``, its rows at a multiple of 16 bytes in memory, or ``out``.
    How many rows a has decides the order of the sums: a row's values may
    differ by a rounding from those that it has beside other rows."""
    device = _gpu(a, "a")
    dtype = _DTYPES.get(out_dtype if out is None else out.dtype)
    if dtype is None or dtype == TKH_F32:
        raise TypeError("the product comes in bfloat16 or float16")
    a2, as2 = _eight(a, a_scale, "a")
    if w.dim() != 2:
        raise ValueError("w has two axes")
    w2, ws2 = _eight(w, w_scale, "w")
    m, k = a2.shape
    n = w2.shape[0]
    if w2.shape[1] != k:
        raise ValueError(f"rows of {k} and of {w2.shape[1]}")
    _on(a_scale, device, "a_scale")
    _on(w, device, "w")
    _on(w_scale, device, "w_scale")
    given = out is not None
    if not given:
        c = a.new_empty((m, (n + 7) // 8 * 8), dtype=out_dtype)
        if n % 8:
            c = c[:, :n]
        out = c if a.dim() == 2 else c.view(a.shape[:-1] + (n,))
    else:
        _given(out, "out", a, a_scale, w, w_scale)
        if out.shape != a.shape[:-1] + (n,):
            raise ValueError(f"out has shape {tuple(out.shape)}")
        _on(out, device, "out")
        c = _rows(out, "out")
    status = (_lib or lib()).tk_head_matmul(_MATMUL.pack(
        a2.data_ptr(), as2.data_ptr(), w2.data_ptr(), ws2.data_ptr(),
        c.data_ptr(), m, n, k, a2.stride(0), as2.stride(0), w2.stride(0),
        ws2.stride(0), c.stride(0), dtype, device.index),
        _raw_stream(device.index))
    if status:
        _fail(status, "tk_head_matmul")
    if given:
        _written(out)
    if a.requires_grad or w.requires_grad or a_scale.requires_grad or w_scale.requires_grad:
        out, = _untracked("matmul_fp8", (out,), a, a_scale, w, w_scale)
    return out


class Sampled(NamedTuple):
    ids: torch.Tensor      # int32
    logprob: torch.Tensor  # float32


def _setting(v, rows: int, dtype: torch.dtype, device: torch.device, name: str,
             low, high):
    """``(pointer, value)`` of a sampler's setting: a number for every row, or
    a tensor of one a row."""
    if isinstance(v, torch.Tensor):
        if v.shape != (rows,) or v.dtype != dtype or (rows > 1 and v.stride(0) != 1):
            raise ValueError(f"{name} is a number or a dense {dtype} tensor of {rows}")
        _on(v, device, name)
        return v.data_ptr(), 0
    try:
        fits = low <= v <= high
        if dtype is torch.int32:
            v = operator.index(v)
    except TypeError:
        raise TypeError(f"{name} is {v!r}: a number or a {dtype} tensor is wanted") from None
    if not fits:
        raise ValueError(f"{name} is {v}: {low} to {high} is wanted")
    return 0, v


def sample(logits: torch.Tensor, u: torch.Tensor, *,
           temperature: float | torch.Tensor = 1.0,
           top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0,
           min_p: float | torch.Tensor = 0.0,
           allowed: torch.Tensor | None = None) -> Sampled:
    """One token a row of ``logits`` (``[rows, vocab]`` of float32, bfloat16
    or float16) from ``u``, one float32 in [0, 1) a row.

    A token weighs ``2**((x - max) * log2(e) / temperature)``, counted in whole
    2**-40ths, so that what a row's logits give does not depend on the batch
    that they are in. In the order of falling logits, equal ones by rising index, ``top_k`` keeps
    that many (0: all); of them ``top_p`` keeps each that has less than its
    share of their weight before it; of those ``min_p`` keeps the ones of at
    least that share of the largest's weight. The token is the first by index
    at which the running weight of what stays passes ``u`` of it. Temperature
    0 takes the largest logit. Settings are numbers, or device tensors of one
    a row (float32; int32 for top_k): there temperature <= 0 is greedy, top_k
    <= 0 and top_p >= 1 keep all, top_p <= 0 keeps the first.

    ``allowed``: int32 words ``[rows or 1, ceil(vocab / 32)]``, bit i % 32 of
    word i // 32 set where token i may be drawn. NaN and -inf are never drawn.
    A row that leaves nothing gives id -1 and logprob -inf; else ``logprob``
    is the natural logarithm of the token's share of what stays."""
    device = _gpu(logits, "logits")
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None:
        raise TypeError(f"logits are {logits.dtype}: float32, bfloat16 or float16 is wanted")
    if logits.dim() != 2:
        raise ValueError("logits have two axes")
    x = _rows(logits, "logits")
    rows, vocab = x.shape
    if u.shape != (rows,) or u.dtype != torch.float32 or (rows > 1 and u.stride(0) != 1):
        raise ValueError(f"u is a dense float32 tensor of {rows}")
    dev = device
    _on(u, dev, "u")
    t_ptr, t = _setting(temperature, rows, torch.float32, dev, "temperature", 0.0, _INF)
    k_ptr, k = _setting(top_k, rows, torch.int32, dev, "top_k", 0, 2 ** 31 - 1)
    p_ptr, p = _setting(top_p, rows, torch.float32, dev, "top_p", 0.0, 1.0)
    f_ptr, f = _setting(min_p, rows, torch.float32, dev, "min_p", 0.0, 1.0)
    mask, mask_stride = 0, 0
    if allowed is not None:
        words = (vocab + 31) // 32
        if (allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[1] != words
                or allowed.shape[0] not in (1, rows)):
            raise ValueError(f"allowed is an int32 tensor of ({rows} or 1, {words})")
        _on(allowed, dev, "allowed")
        allowed = _rows(allowed, "allowed")
        mask = allowed.data_ptr()
        mask_stride = allowed.stride(0) if allowed.shape[0] > 1 else 0
    L = _lib or lib()
    size = L.tk_head_sample_workspace(rows, vocab, dtype)
    work = u.new_empty(size, dtype=torch.uint8)
    ids = u.new_empty(rows, dtype=torch.int32)
    logprob = u.new_empty(rows)
    status = L.tk_head_sample(_SAMPLE.pack(
        x.data_ptr(), u.data_ptr(), t_ptr, k_ptr, p_ptr, f_ptr, mask,
        ids.data_ptr(), logprob.data_ptr(), work.data_ptr(), size, rows, vocab,
        x.stride(0), mask_stride, t, k, p, f, dtype, device.index),
        _raw_stream(device.index))
    if status:
        _fail(status, "tk_head_sample")
    if logits.requires_grad or u.requires_grad or t_ptr or p_ptr or f_ptr:
        ids, logprob = _untracked("sample", (ids, logprob), logits, u, temperature, top_p, min_p)
    return Sampled(ids, logprob)


def quantize_fp8(x: torch.Tensor, chunk: int = 16384
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of a float tensor ``[n, k]`` as ``matmul_fp8`` reads them: e4m3
    values and, for each 128, the least power of two that holds their largest
    below e4m3's largest value. Done once when weights are loaded, in plain
    torch operations over ``chunk`` rows at a time. Rows are padded in memory
    to a multiple of 128 with zeros. The result does not require grad, whether
    or not x does."""
    if x.dim() != 2 or not x.is_floating_point():
        raise ValueError("rows of floats are wanted")
    n, k = x.shape
    if k < 1:
        raise ValueError("rows of no values")
    blocks = (k + BLOCK - 1) // BLOCK
    q = torch.zeros((n, blocks * BLOCK), dtype=torch.uint8, device=x.device)
    scale = torch.empty((n, blocks), dtype=torch.uint8, device=x.device)
    for r in range(0, n, chunk):
        y = torch.nn.functional.pad(x[r:r + chunk].float(), (0, blocks * BLOCK - k))
        y = y.view(y.shape[0], blocks, BLOCK)
        a = y.abs()
        frac, e = torch.frexp(torch.where(a.isfinite(), a, 0.0).amax(-1))
        # 448 = 0.875 * 2^9
        e = torch.where(frac > 0, e - 9 + (frac > 0.875).int(), 0).clamp(-127, 127)
        q[r:r + chunk] = torch.ldexp(y, -e[..., None]).to(_FP8).view(torch.uint8).flatten(1)
        scale[r:r + chunk] = (e + 127).to(torch.uint8)
    return q.view(_FP8)[:, :k], scale.view(_E8M0)


class OutputHead:
    """The last steps of a model over a tokenizer's vocabulary: final norm,
    vocabulary projection, next token.

    ``norm_weight``: ``[k]``; ``w``, ``w_scale``: the projection ``[n, k]`` in
    8 bits (``quantize_fp8``); all three are held detached. ``vocab``: the
    tokens that may be drawn, where the projection's rows are padded beyond the
    tokenizer's ids (its vocabulary with the added tokens)."""

    def __init__(self, norm_weight: torch.Tensor, w: torch.Tensor,
                 w_scale: torch.Tensor, *, eps: float = 1e-6,
                 vocab: int | None = None,
                 logits_dtype: torch.dtype = torch.bfloat16):
        if w.dim() != 2 or norm_weight.shape != (w.shape[1],):
            raise ValueError("norm_weight and w do not fit each other")
        if vocab is not None and not 1 <= vocab <= w.shape[0]:
            raise ValueError(f"vocab {vocab} of {w.shape[0]} rows")
        if logits_dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("logits come in bfloat16 or float16")
        self.norm_weight = norm_weight.detach()
        self.w, self.w_scale = _eight(w.detach(), w_scale.detach(), "w")
        if vocab is not None:
            self.w, self.w_scale = self.w[:vocab], self.w_scale[:vocab]
        self.eps = eps
        self.logits_dtype = logits_dtype

    def logits(self, x: torch.Tensor, *, residual: torch.Tensor | None = None
               ) -> torch.Tensor:
        """``[..., n]`` logits of the hidden states ``[..., k]``."""
        y = rms_norm_fp8(x, self.norm_weight, residual=residual, eps=self.eps)
        return matmul_fp8(y.q, y.scale, self.w, self.w_scale,
                          out_dtype=self.logits_dtype)

    def next_ids(self, x: torch.Tensor, u: torch.Tensor, *,
                 residual: torch.Tensor | None = None, **settings) -> Sampled:
        """One token for each of the hidden states ``[rows, k]``; settings as
        in ``sample``. The same call gives the same tokens; a row may get
        another beside other rows, whose number decides how the product is
        split and so the order of its 32-bit sums."""
        if x.dim() != 2:
            raise ValueError("hidden states have two axes")
        return sample(self.logits(x, residual=residual), u, **settings)
