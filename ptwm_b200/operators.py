"""Operators that apply decoded weights on CUDA: ``rms_norm`` and ``matvec``.

What a container decodes to includes norm vectors and, for microscaled models, matrices of 4-bit values with a scale per
group, which torch cannot multiply by.  ``ScaledWeight`` is a handle on such a matrix where it lies, ``matvec`` multiplies
it with one token or many, and ``rms_norm`` is the norm in front of it, with the residual's addition and, if asked for, an
output in 8 bits with scales (``ScaledActivations``) that ``matvec`` reads.  ``Projection`` is a norm and the matrices that
read it.

Every call runs on the current stream of its tensors' device, allocates its results with torch, waits for nothing and can be
captured into a CUDA graph; a backward pass (of any operator) only while no graph of the same leaves that was recorded
outside the capture is still alive, since torch adds to their gradients on the stream that had them first.

The waits inside the kernels are bounded.  None is expected to run out; a kernel in which one did writes NaN, and ``operator_status`` says so.
"""
from __future__ import annotations

import ctypes as C
from typing import Any, Callable, Mapping, Optional, Sequence, Union

import torch

from torch._C import _cuda_getCurrentRawStream as _stream  # what torch.cuda.current_stream() wraps, a microsecond faster
from torch.autograd import forward_ad

from . import _lib
from .container import _check

__all__ = ["Projection", "ScaledActivations", "ScaledWeight", "matvec", "operator_status", "rms_norm"]

_PLAIN = {torch.float32: 1, torch.float16: 4, torch.bfloat16: 6}
_E4M3, _BF16 = 29, 6
_TOO_SMALL = -2
_QUANT = {None: 0, "row": 1, "block": 2}
_U8 = (torch.uint8,) + ((torch.float4_e2m1fn_x2,) if hasattr(torch, "float4_e2m1fn_x2") else ())
_E8M0 = torch.float8_e8m0fnu


def _on_cuda(what: str, t: Any, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{what} lives in host memory; move it to CUDA first")
    if device is not None and t.device != device:
        raise ValueError(f"{what} lives on {t.device}, the others on {device}")


def operator_status(device: Union[None, int, str, torch.device] = None) -> int:
    """0, or 1 from when on a wait inside a kernel of these operators has given up on the device (the current one where it is None).
    Waits for the device."""
    if device is None or isinstance(device, int):
        index = device
    else:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"{device} is no CUDA device")
        index = device.index
    return _check(_lib.lib().ptwm_b200_operator_status(torch.cuda.current_device() if index is None else index))


class ScaledActivations:
    """Rows of E4M3 values with their scales: fp32 per row (``scales`` has the rows' leading dimensions) or E8M0 per 32
    values (one more dimension, a 32nd of the columns)."""

    __slots__ = ("values", "scales", "quant")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor) -> None:
        _on_cuda("values", values)
        _on_cuda("scales", scales, values.device)
        if values.dtype != torch.float8_e4m3fn or values.dim() < 1:
            raise TypeError(f"values are rows of float8_e4m3fn, got {values.dtype} with {values.dim()} dimensions")
        if scales.dtype == torch.uint8:
            scales = scales.view(_E8M0)
        if scales.dtype == torch.float32:
            quant, want = "row", values.shape[:-1]
        elif scales.dtype == _E8M0:
            quant, want = "block", (*values.shape[:-1], values.shape[-1] // 32)
            if values.shape[-1] % 32:
                raise ValueError(f"block scales need whole blocks of 32 values, got rows of {values.shape[-1]}")
        else:
            raise TypeError(f"scales are float32 per row or float8_e8m0fnu (uint8) per 32 values, got {scales.dtype}")
        if tuple(scales.shape) != tuple(want):
            raise ValueError(f"scales have shape {tuple(scales.shape)}, expected {tuple(want)}")
        self.values, self.scales, self.quant = values, scales, quant

    @classmethod
    def _of(cls, values: torch.Tensor, scales: torch.Tensor, quant: str) -> "ScaledActivations":
        self = object.__new__(cls)
        self.values, self.scales, self.quant = values, scales, quant
        return self

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    def __repr__(self) -> str:
        return f"ScaledActivations(shape={tuple(self.shape)}, quant={self.quant!r}, device={self.device})"


def scaled_names(name: str, has: Callable[[str], bool]) -> tuple[str, str, Optional[str]]:
    """The tensors that make up the microscaled matrix ``name``: values, scales and fp32 scale, as ModelOpt names them
    (``name.weight``, ``.weight_scale``, ``.weight_scale_2``), as gpt-oss does (``name_blocks``, ``name_scales``), or
    ``name``, ``name_scale``, ``name_scale_2``.  Raises KeyError where no such set is there."""
    for values, scales, top in ((f"{name}.weight", f"{name}.weight_scale", f"{name}.weight_scale_2"), (f"{name}_blocks", f"{name}_scales", None),
                                (name, f"{name}_scale", f"{name}_scale_2")):
        if has(values) and has(scales):
            return values, scales, top if top is not None and has(top) else None
    raise KeyError(name)


class ScaledWeight:
    """A matrix of 4-bit values with group scales, where it lies in device memory.

    ``values``: E2M1 codes, two to a byte with the even column in the low nibble: uint8 or float4_e2m1fn_x2 of shape
    [rows, cols / 2], or [rows, cols / 32, 16].  ``scales``: E8M0 (uint8 or float8_e8m0fnu) of shape [rows, cols / 32], which
    is MXFP4, or float8_e4m3fn of shape [rows, cols / 16], NVFP4, with ``global_scale`` as one fp32 number in device memory
    (1 where it is None).  ``expert`` picks one matrix of a stack of them.

    The tensors are kept and read in place; only one whose rows are not contiguous or do not start at multiples of 16
    bytes is copied, once, here."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, global_scale: Optional[torch.Tensor] = None, *, expert: Optional[int] = None) -> None:
        _on_cuda("values", values)
        _on_cuda("scales", scales, values.device)
        if values.dtype not in _U8:
            raise TypeError(f"values are packed nibbles (uint8 or float4_e2m1fn_x2), got {values.dtype}")
        if scales.dtype in (torch.uint8, _E8M0):
            self.kind, self.group = "mxfp4", 32
        elif scales.dtype == torch.float8_e4m3fn:
            self.kind, self.group = "nvfp4", 16
        else:
            raise TypeError(f"scales are E8M0 (uint8 or float8_e8m0fnu) or float8_e4m3fn, got {scales.dtype}")
        values, scales = values.view(torch.uint8), scales.view(torch.uint8)
        if expert is not None:
            values, scales = values[expert], scales[expert]
        if values.dim() == 3 and values.shape[-1] == 16 and scales.dim() == 2:
            values = values.reshape(values.shape[0], -1)
        if values.dim() != 2 or scales.dim() != 2:
            raise ValueError(f"one matrix of values and one of scales are wanted, got shapes {tuple(values.shape)} and {tuple(scales.shape)}"
                             + ("; pick one of a stack with expert=" if values.dim() > 2 else ""))
        self.rows, self.cols = values.shape[0], 2 * values.shape[1]
        if not self.rows or not self.cols or self.cols % self.group or tuple(scales.shape) != (self.rows, self.cols // self.group):
            raise ValueError(f"{self.kind}: values of {self.rows} x {self.cols} want scales of {self.rows} x {self.cols}/{self.group}, got {tuple(scales.shape)}")
        if global_scale is not None:
            _on_cuda("global_scale", global_scale, values.device)
            if self.kind != "nvfp4":
                raise ValueError("only NVFP4 matrices have a global scale")
            if global_scale.dtype != torch.float32 or global_scale.numel() != 1:
                raise TypeError(f"global_scale is one float32 number, got {global_scale.dtype} of shape {tuple(global_scale.shape)}")
        self.device = values.device
        self._values, self._scales, self._global = self._aligned(values), self._aligned(scales), global_scale
        self._args = _lib.ScaledWeightArgs(self._values.data_ptr(), self._scales.data_ptr(), 0 if global_scale is None else global_scale.data_ptr(),
                                           self.rows, self.cols, self._values.stride(0), self._scales.stride(0), self.group, 0)
        self._ref = C.addressof(self._args)
        self._ordinal = self.device.index

    @staticmethod
    def _aligned(t: torch.Tensor) -> torch.Tensor:
        """``t`` where its rows can be read as they lie, else a copy whose rows start at multiples of 16 bytes."""
        wide = t.shape[0] == 1 or (t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1])
        if wide and (t.shape[1] == 1 or t.stride(1) == 1) and t.data_ptr() % 16 == 0 and t.stride(0) < 1 << 32:
            if t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1]:
                return t
        pitch = (t.shape[1] + 15) // 16 * 16
        copy = torch.zeros(t.shape[0], pitch, dtype=torch.uint8, device=t.device)
        copy[:, :t.shape[1]] = t
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(t.device).synchronize()  # the handle may be used on another stream next
        return copy[:, :t.shape[1]]

    @classmethod
    def from_state(cls, state: Mapping[str, torch.Tensor], name: str, *, expert: Optional[int] = None) -> "ScaledWeight":
        """The matrix ``name`` of a state dict (``load_file``, ``dict(handle.decode_model())``); see ``scaled_names``."""
        values, scales, top = scaled_names(name, state.__contains__)
        return cls(state[values], state[scales], None if top is None else state[top], expert=expert)

    # Copies and pickles are made of the tensors: the addresses kept beside them are this object's own.
    def __getstate__(self) -> tuple:
        return self._values, self._scales, self._global, self.kind  # (bytes: plain pickle does not take float8 storages)

    def __setstate__(self, state: tuple) -> None:
        values, scales, top, kind = state
        self.__init__(values, scales if kind == "mxfp4" else scales.view(torch.float8_e4m3fn), top)

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    def __repr__(self) -> str:
        return f"ScaledWeight({self.kind}, {self.rows} x {self.cols}, device={self.device})"


# ---- rms_norm -------------------------------------------------------------------------------------
def _norm(x, weight, residual, eps: float, quant: Optional[str]):
    """(y or ScaledActivations, h) of checked, contiguous tensors."""
    shape = x.shape
    cols = shape[-1]
    device = x.get_device()
    if residual is None:
        h, h_at, residual_at = x, 0, 0
    else:
        h = torch.empty_like(x)
        h_at, residual_at = h.data_ptr(), residual.data_ptr()
    if quant is None:
        out = torch.empty_like(x)
        y_at, scales_at = out.data_ptr(), 0
    else:
        values = torch.empty_like(x, dtype=torch.float8_e4m3fn)
        scales = _new(shape[:-1], torch.float32, x.device) if quant == "row" else _new((*shape[:-1], cols // 32), _E8M0, x.device)
        out = ScaledActivations._of(values, scales, quant)
        y_at, scales_at = values.data_ptr(), scales.data_ptr()
    rc = _lib.lib().ptwm_b200_rms_norm(x.data_ptr(), residual_at, weight.data_ptr(), h_at, y_at, scales_at, x.numel() // cols, cols, _PLAIN[x.dtype], _PLAIN[weight.dtype],
                                       _QUANT[quant], eps, device, _stream(device))
    if rc < 0:
        _check(rc)
    return out, h


def _new(shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """torch.empty; its quickest form for the usual two dimensions."""
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _refuse_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """A dual tensor does not require a gradient, so nothing else would notice it."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("rms_norm and matvec have no forward-mode derivatives; unpack their dual tensors first")


def _once(*grads: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():  # as it is in a backward pass with create_graph
        raise RuntimeError("rms_norm and matvec have first derivatives only: their backward passes cannot be differentiated")
    _refuse_tangents(*grads)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h = _norm(x, weight, residual, eps, None)
        ctx.save_for_backward(h, weight)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return (y, h) if residual is not None else y

    @staticmethod
    def backward(ctx, dy, dh=None):
        _once(dy, dh)
        h, weight = ctx.saved_tensors
        for_x, need_w, for_residual, _ = ctx.needs_input_grad
        need_x = for_x or for_residual
        if dy is None:  # only the residual stream was used
            dx = dh
            dw = torch.zeros_like(weight) if need_w and dh is not None else None
        else:
            dy = dy.contiguous()
            dh = None if dh is None else dh.contiguous()
            cols, device = h.shape[-1], h.get_device()
            rows = h.numel() // cols
            dx = torch.empty_like(h) if need_x else None
            dw = torch.empty_like(weight) if need_w else None
            L = _lib.lib()
            size = L.ptwm_b200_rms_norm_grad_scratch_bytes(rows, cols) if need_w else 0
            scratch = _new((size,), torch.uint8, h.device) if size else None
            _check(L.ptwm_b200_rms_norm_grad(h.data_ptr(), weight.data_ptr(), dy.data_ptr(), 0 if dh is None else dh.data_ptr(), 0 if dx is None else dx.data_ptr(),
                                             0 if dw is None else dw.data_ptr(), 0 if scratch is None else scratch.data_ptr(), size, rows, cols, _PLAIN[h.dtype],
                                             _PLAIN[weight.dtype], ctx.eps, device, _stream(device)))
        return (dx if for_x else None), dw, (dx if for_residual else None), None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, residual: Optional[torch.Tensor] = None, quant: Optional[str] = None):
    """Root-mean-square norm over the last dimension, with the residual's addition.

    ``h = x + residual`` (rounded to x's type; without a residual ``h = x``), then
    ``y = h / sqrt(mean(h^2) + eps) * weight`` with fp32 sums and one rounding.  x and residual are fp32, fp16 or bf16 of one
    shape and type, weight is a vector of any of these types.  Returns ``y``, or ``(y, h)`` with a residual.

    ``quant``: None for y in x's type; "row" or "block" for ``ScaledActivations``, E4M3 values with a fp32 scale per row
    (max|y| / 448) or an E8M0 scale per 32 values (the smallest power of two that keeps them within 448).  A row or block
    that is not finite has NaN for scale and values.  Squares are summed in fp32: a row whose squares pass its range, with values of some 10^19, has an infinite
    root mean square, and y is zero.

    Without ``quant`` there are gradients for x, residual and weight: first ones, backwards."""
    try:
        device, dtype, shape = x.get_device(), x.dtype, x.shape
        fine = (device >= 0 and weight.get_device() == device and dtype in _PLAIN and weight.dtype in _PLAIN and weight.shape == shape[-1:] and shape[-1] > 0
                and quant in _QUANT and (quant != "block" or shape[-1] % 32 == 0)
                and (residual is None or (residual.get_device() == device and residual.dtype is dtype and residual.shape == shape)))
    except (AttributeError, IndexError, TypeError):
        fine = False
    if not fine:
        _refuse_norm(x, weight, residual, quant)
    _refuse_tangents(x, weight, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        if quant is not None:
            raise ValueError("an 8-bit output has no gradient: call under torch.no_grad() or detach the inputs")
        return _RmsNorm.apply(x.contiguous(), weight.contiguous(), None if residual is None else residual.contiguous(), float(eps))
    y, h = _norm(x.contiguous(), weight.contiguous(), None if residual is None else residual.contiguous(), eps, quant)
    return y if residual is None else (y, h)


def _refuse_norm(x, weight, residual, quant) -> None:
    """What is wrong with the arguments of ``rms_norm``."""
    _on_cuda("x", x)
    _on_cuda("weight", weight, x.device)
    if x.dtype not in _PLAIN or weight.dtype not in _PLAIN:
        raise TypeError(f"x and weight are float32, float16 or bfloat16, got {x.dtype} and {weight.dtype}")
    if quant not in _QUANT:
        raise ValueError(f"quant is None, 'row' or 'block', got {quant!r}")
    if not x.shape or x.shape[-1] == 0 or weight.shape != x.shape[-1:]:
        raise ValueError(f"weight of shape {tuple(weight.shape)} does not fit rows of x, shape {tuple(x.shape)}")
    if quant == "block" and x.shape[-1] % 32:
        raise ValueError(f"block scales need whole blocks of 32 values, got rows of {x.shape[-1]}")
    if residual is not None:
        _on_cuda("residual", residual, x.device)
        raise ValueError(f"residual is {residual.dtype} {tuple(residual.shape)}, x {x.dtype} {tuple(x.shape)}; they have to be alike")
    raise TypeError("rms_norm: unsuitable arguments")


# ---- matvec ---------------------------------------------------------------------------------------
def _product(x, scales, quant, weight: ScaledWeight, out_dtype: torch.dtype) -> torch.Tensor:
    device, tokens, shape = weight._ordinal, x.numel() // weight.cols, x.shape
    if scales is None:
        code, scales_at = _PLAIN[x.dtype], 0
    else:
        code, scales_at = _E4M3, scales.data_ptr()
    y = _new((shape[0], weight.rows) if len(shape) == 2 else (*shape[:-1], weight.rows), out_dtype, weight.device)
    _with_scratch(_lib.lib().ptwm_b200_matvec, (weight._ref, x.data_ptr(), scales_at, y.data_ptr(), tokens, code, _QUANT[quant], _PLAIN[out_dtype]), (weight,), x, tokens, code, 0)
    return y


def _with_scratch(call, args: tuple, weights: Sequence[ScaledWeight], x: torch.Tensor, tokens: int, code: int, grad: int) -> None:
    """A product's call.  Few tokens, and bf16 ones that lie well, need no scratch: it is not asked for unless the call says so."""
    device = weights[0]._ordinal
    rc = _TOO_SMALL if code != _BF16 and (grad or tokens > 16) else call(*args, 0, 0, device, _stream(device))
    if rc == _TOO_SMALL:
        # (one of several matrices may want some where another does not)
        size = max(_lib.lib().ptwm_b200_matvec_scratch_bytes(w._ref, x.data_ptr(), tokens, code, grad) for w in weights)
        scratch = _new((size,), torch.uint8, x.device)
        rc = call(*args, scratch.data_ptr(), size, device, _stream(device))
    if rc < 0:
        _check(rc)


class _Matvec(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, out_dtype):
        ctx.weight, ctx.dtype = weight, x.dtype
        return _product(x, None, None, weight, out_dtype)

    @staticmethod
    def backward(ctx, dy):
        _once(dy)
        w = ctx.weight
        dy = dy.contiguous()
        dx = torch.empty((*dy.shape[:-1], w.cols), dtype=ctx.dtype, device=dy.device)
        tokens, code = dy.numel() // w.rows, _PLAIN[dy.dtype]  # the output's type
        _with_scratch(_lib.lib().ptwm_b200_matvec_grad_of, (w._ref, dy.data_ptr(), dx.data_ptr(), tokens, code, _PLAIN[ctx.dtype]), (w,), dy, tokens, code, 1)
        return dx, None, None


def matvec(x, weight: ScaledWeight, *, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``y[..., n] = sum_k x[..., k] W[n, k]`` with a 4-bit matrix, for one token or many.

    x is fp32, fp16 or bf16 of shape [..., cols], or ``ScaledActivations``, at most 2^19 tokens.  Sums are fp32, rounded once to ``out_dtype``
    (x's type; bf16 for ScaledActivations); tensor cores cut, in them, what fp32 does not hold: fp32 results are within some 1e-6 of their norm.  fp32 tokens
    are taken to 2^-23 of their value where they are few, and whole otherwise.  Where tokens are few, values beyond 2^28 (fp32) or 2^31 (bf16) apart cost
    another pass over the matrix.  The gradient goes back to a plain x, from the output's type and rounded once to x's: the
    first one, backwards.  ScaledActivations and the matrix have none."""
    if not isinstance(weight, ScaledWeight):
        raise TypeError(f"weight is a ScaledWeight, got {type(weight).__name__}")
    if type(x) is ScaledActivations:
        scales, quant, x = x.scales, x.quant, x.values
        if (scales.requires_grad or x.requires_grad) and torch.is_grad_enabled():
            raise ValueError("8-bit tokens have no gradient: call under torch.no_grad() or detach their values and scales")
        out_dtype = out_dtype or torch.bfloat16
        if not scales.is_contiguous():
            scales = scales.contiguous()
    else:
        scales = quant = None
        _on_cuda("x", x)
        if x.dtype not in _PLAIN:
            raise TypeError(f"x is float32, float16, bfloat16 or ScaledActivations, got {x.dtype}")
        out_dtype = out_dtype or x.dtype
    if out_dtype not in _PLAIN:
        raise TypeError(f"out_dtype is float32, float16 or bfloat16, got {out_dtype}")
    if x.get_device() != weight._ordinal:
        raise ValueError(f"x lives on {x.device}, the weight on {weight.device}")
    shape = x.shape
    if not shape or shape[-1] != weight.cols:
        raise ValueError(f"x of shape {tuple(shape)} does not fit a matrix of {weight.rows} x {weight.cols}")
    _refuse_tangents(x, scales)
    if not x.is_contiguous():
        x = x.contiguous()
    if scales is None and x.requires_grad and torch.is_grad_enabled():
        return _Matvec.apply(x, weight, out_dtype)
    return _product(x, scales, quant, weight, out_dtype)


class Projection:
    """A norm and the matrices that read its output, such as the gate and up projections of a feed-forward block.

    ``projection(x, residual)`` returns ``([W x' for W in weights], h)`` with ``x', h = rms_norm(x, norm, eps,
    residual=residual, quant=quant)``; ``h`` is x where there is no residual.  The matrices' products are one launch where tokens are few.
    ``norm`` and ``weights`` are checked against one another once, here, and stay as they are; others want another ``Projection``."""

    def __init__(self, norm: torch.Tensor, weights: Sequence[ScaledWeight], *, eps: float = 1e-6, quant: Optional[str] = None) -> None:
        self._norm, self._weights, self.eps, self.quant = norm, tuple(weights), eps, quant
        _on_cuda("norm", norm)
        if quant not in _QUANT:
            raise ValueError(f"quant is None, 'row' or 'block', got {quant!r}")
        if norm.dim() != 1:
            raise ValueError(f"norm is a vector, got shape {tuple(norm.shape)}")
        for w in self.weights:
            if not isinstance(w, ScaledWeight):
                raise TypeError(f"weights are ScaledWeights, got {type(w).__name__}")
            if w.cols != norm.shape[0] or w.device != norm.device:
                raise ValueError(f"a norm of {norm.shape[0]} on {norm.device} does not fit {w!r}")
        parts = [self.weights[i:i + 4] for i in range(0, len(self.weights), 4)]
        self._calls = [((C.c_uint64 * len(p))(*[w._ref for w in p]), p) for p in parts]

    @property
    def norm(self) -> torch.Tensor:
        return self._norm

    @property
    def weights(self) -> tuple[ScaledWeight, ...]:
        return self._weights

    def __getstate__(self) -> tuple:  # a copy refers to its own matrices
        return self.norm, self.weights, self.eps, self.quant

    def __setstate__(self, state: tuple) -> None:
        norm, weights, eps, quant = state
        self.__init__(norm, weights, eps=eps, quant=quant)

    def __call__(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> tuple[list[torch.Tensor], torch.Tensor]:
        got = rms_norm(x, self.norm, self.eps, residual=residual, quant=self.quant)
        y, h = (got, x) if residual is None else got
        if self.quant is not None:  # checked, contiguous and without a gradient
            return self._products(y.values, y.scales, x.dtype), h
        if y.requires_grad and torch.is_grad_enabled():
            return [matvec(y, w) for w in self.weights], h
        return self._products(y, None, x.dtype), h

    def _products(self, x: torch.Tensor, scales: Optional[torch.Tensor], out_dtype: torch.dtype) -> list[torch.Tensor]:
        """The products of all matrices, four to a call."""
        out = []
        tokens, head = x.numel() // self.norm.shape[0], tuple(x.shape[:-1])
        code, scales_at = (_PLAIN[x.dtype], 0) if scales is None else (_E4M3, scales.data_ptr())
        for refs, weights in self._calls:
            ys = [_new((*head, w.rows), out_dtype, x.device) for w in weights]
            at = (C.c_uint64 * len(ys))(*[y.data_ptr() for y in ys])
            _with_scratch(_lib.lib().ptwm_b200_matvec_group, (refs, at, len(ys), x.data_ptr(), scales_at, tokens, code, _QUANT[self.quant], _PLAIN[out_dtype]), weights, x, tokens, code, 0)
            out += ys
        return out
