"""Operators around the experts, on torch tensors: the router on given logits, the dense product with bias, activation
and residual, and the log probabilities of given tokens.

Thin wrappers over the C ABI (include/promoe_b200.h: pm_k_route, pm_k_linear, pm_k_token_logprobs): they check shapes and types,
allocate results where the caller brings none and launch on torch's current stream of the tensors' device. They
hold no state besides what a caller hands to their constructors, run without scratch memory and can be captured into a CUDA graph.
No gradients: tensors that require one are refused while autograd records, and so are those with a forward-mode tangent and calls
that torch.jit traces.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_SCORING = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}
_DROPPED = {"out": 0, "zero": 16}


# The stream as an integer, without the Stream object that torch.cuda.current_stream makes (1 us of a call that takes 5). A torch
# built without CUDA has neither; it has no CUDA tensors to call these operators with either.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_tracing = torch._C._get_tracing_state
_I32, _F32 = torch.int32, torch.float32


def _elsewhere(index: int, fn, *args) -> int:
    """fn(*args, stream) with device `index` current, on its current stream."""
    with torch.cuda.device(index):
        return fn(*args, _raw_stream(index))


def _matrix(t: torch.Tensor, what: str, width: int | None = None, dtypes=_DTYPES) -> tuple[int, int, int, int]:
    """(device index, rows, width, pitch) of a CUDA matrix with dense rows, none over another."""
    index, shape = t.get_device(), t.shape
    if index < 0 or len(shape) != 2 or t.dtype not in dtypes:
        raise ValueError(f"{what} must be a 2-D CUDA tensor of {', '.join(str(d) for d in dtypes)}")
    rows, n = shape
    if rows > 0x7fffffff or n > 0x7fffffff:  # ctypes would cut them off
        raise ValueError(f"{what} has too many rows or columns")
    if width is not None and n != width:
        raise ValueError(f"{what} must have rows of {width} values, not {n}")
    pitch, inner = t.stride()
    if inner != 1 and n > 1:
        raise ValueError(f"the rows of {what} must be dense")
    if rows <= 1:
        pitch = n  # the stride of a single row says nothing
    elif pitch < n:
        raise ValueError(f"the rows of {what} must not overlap (expanded tensors: call contiguous())")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient: these operators have no backward pass")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what} has a forward-mode tangent: these operators have no derivative")
    return index, rows, n, pitch


def _fixed(name: str):
    """An attribute that is set once: the launch arguments made from it would not follow."""
    return property(lambda self: getattr(self, "_" + name))


def _refuse_tracing():
    raise ValueError("torch.jit cannot trace these operators")


class Router:
    """Chooses top_k of num_expert experts per token from router logits (pm_k_route states the rule).

    scoring: "softmax" or "sigmoid". bias: [num_expert] float32 on the device, added to the scores for the choice only (a
    load-balancing correction). n_group / topk_group / group_score ("max" or "top2"): choose among the best groups
    only; dropped: what becomes of the others' experts, "out" (they cannot be chosen) or, with a bias, "zero" (their score + bias
    counts as 0, which passes by negative ones). norm_topk: weights divided by their sum. routed_scale: multiplies the weights.
    The bias is used in place, not copied."""

    num_expert, top_k, bias, device_index = (_fixed(n) for n in ("num_expert", "top_k", "bias", "device_index"))

    def __init__(self, num_expert: int, top_k: int, scoring: str = "softmax", bias: torch.Tensor | None = None, n_group: int = 1,
                 topk_group: int = 1, group_score: str = "max", norm_topk: bool = False, routed_scale: float = 1.0,
                 dropped: str = "out"):
        if scoring not in _SCORING:
            raise ValueError(f"scoring must be one of {sorted(_SCORING)}")
        if group_score not in _GROUP_SCORE:
            raise ValueError(f"group_score must be one of {sorted(_GROUP_SCORE)}")
        if dropped not in _DROPPED:
            raise ValueError(f"dropped must be one of {sorted(_DROPPED)}")
        if not all(-0x80000000 <= n <= 0x7fffffff for n in (num_expert, top_k, n_group, topk_group)):  # ctypes would cut them off
            raise ValueError("num_expert, top_k, n_group and topk_group must be 32-bit numbers")
        if bias is not None:
            if not bias.is_cuda or bias.dtype != torch.float32 or bias.shape != (num_expert,) or not bias.is_contiguous():
                raise ValueError("bias must be a contiguous float32 CUDA tensor of shape [num_expert]")
            bias = bias.detach()  # keeps the memory, whatever becomes of the caller's tensor
        self._num_expert, self._top_k, self._bias = num_expert, top_k, bias
        self._device_index = None if bias is None else bias.get_device()
        self.rule = _lib.pm_router(num_expert, top_k, _SCORING[scoring], n_group, topk_group, _GROUP_SCORE[group_score] + _DROPPED[dropped],
                                   int(norm_topk), routed_scale, None if bias is None else bias.data_ptr())
        self._ref = C.byref(self.rule)
        self._fn = _lib.load().pm_k_route
        # the rule's own checks, without a token
        _lib.check(self._fn(self._ref, None, 0, num_expert, 0, None, None, None))

    def __call__(self, logits: torch.Tensor, out: tuple[torch.Tensor, torch.Tensor] | None = None):
        """logits [T, num_expert] float32 / bf16 / fp16 -> (ids [T, top_k] int32, weights [T, top_k] float32)."""
        if _tracing() is not None:
            _refuse_tracing()
        index, T, _, pitch = _matrix(logits, "logits", self._num_expert)
        if self._device_index is not None and self._device_index != index:
            raise ValueError(f"logits must be on cuda:{self._device_index}, where the bias is")
        shape = (T, self._top_k)
        if out is None:
            device = logits.device
            ids, w = torch.empty(shape, dtype=_I32, device=device), torch.empty(shape, dtype=_F32, device=device)
        else:
            ids, w = out
            try:
                fits = (ids.shape == shape == w.shape and ids.dtype is _I32 and w.dtype is _F32 and ids.get_device() == index
                        and w.get_device() == index and ids.is_contiguous() and w.is_contiguous())
            except AttributeError:  # no tensors
                fits = False
            if not fits:
                raise ValueError(f"out must be contiguous int32 and float32 tensors of shape {shape} on cuda:{index}")
        if index == _current_device():
            rc = self._fn(self._ref, logits.data_ptr(), _DTYPES[logits.dtype], pitch, T, ids.data_ptr(), w.data_ptr(), _raw_stream(index))
        else:
            rc = _elsewhere(index, self._fn, self._ref, logits.data_ptr(), _DTYPES[logits.dtype], pitch, T, ids.data_ptr(), w.data_ptr())
        if rc:
            _lib.check(rc)
        return ids, w


# struct pm_linear as bytes, in one step: filling the ctypes structure takes 0.5 us more
_PM_LINEAR = struct.Struct("@5P4q7iP").pack


class Linear:
    """y = activation(x weight^T + bias) + residual in one kernel (pm_k_linear).

    weight [N, K] bf16 or fp16 with dense rows, bias [N] of the same type or float32, activation None / "relu" / "silu" /
    "gelu" / "gelu_tanh", out_dtype the weight's type (default) or float32. The tensors are used in place, not copied.
    A row of y depends on no other row; its last bits depend on the number of rows, which the order of the sums follows."""

    weight, bias, out_dtype, device_index, N, K = (_fixed(n) for n in ("weight", "bias", "out_dtype", "device_index", "N", "K"))

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
                 out_dtype: torch.dtype | None = None):
        self._learns = weight.requires_grad or (bias is not None and bias.requires_grad)
        weight = weight.detach()
        index, N, K, pitch = _matrix(weight, "weight", dtypes=(torch.bfloat16, torch.float16))
        if activation not in _ACTS:
            raise ValueError(f"activation must be one of {[a for a in _ACTS if a]} or None")
        out_dtype = weight.dtype if out_dtype is None else out_dtype
        if out_dtype not in (torch.float32, weight.dtype):
            raise ValueError(f"out_dtype must be float32 or {weight.dtype}")
        if bias is not None:
            bias = bias.detach()
            if bias.shape != (N,) or bias.dtype not in (torch.float32, weight.dtype) or not bias.is_contiguous():
                raise ValueError(f"bias must be a contiguous tensor of shape [{N}], float32 or {weight.dtype}")
            if bias.get_device() != index:
                raise ValueError(f"bias must be on cuda:{index}, not on {bias.device}")
        self._weight, self._bias, self._out_dtype, self._device_index, self._N, self._K = weight, bias, out_dtype, index, N, K
        self._x_dtypes, self._y_dtypes = (weight.dtype,), (out_dtype,)
        self._ld_w = pitch
        self._kind = (N, K, _DTYPES[weight.dtype], _DTYPES[out_dtype], 0 if bias is None else _DTYPES[bias.dtype], _ACTS[activation], 0)
        self._fn = _lib.load().pm_k_linear

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """x [M, K] of the weight's type, residual [M, N] of out_dtype (dense rows, any pitch) -> y [M, N]. out may be the
        residual itself; otherwise it must not overlap it, nor ever x, the weight or the bias."""
        index = self._device_index
        if _tracing() is not None:
            _refuse_tracing()
        if self._learns and torch.is_grad_enabled():
            raise ValueError("the weight or the bias requires a gradient: these operators have no backward pass")
        on, M, _, ld_x = _matrix(x, "x", self._K, self._x_dtypes)
        if out is None:
            out = torch.empty((M, self._N), dtype=self._out_dtype, device=x.device)
        on_y, rows, _, ld_y = _matrix(out, "out", self._N, self._y_dtypes)
        if rows != M:
            raise ValueError(f"out must have {M} rows, not {rows}")
        res, ld_r = 0, 0
        if residual is not None:
            on_r, rows, _, ld_r = _matrix(residual, "residual", self._N, self._y_dtypes)
            if rows != M:
                raise ValueError(f"residual must have {M} rows, not {rows}")
            if on_r != index:
                raise ValueError(f"residual must be on cuda:{index}, where the weight is")
            res = residual.data_ptr()
        if on != index or on_y != index:
            raise ValueError(f"x and out must be on cuda:{index}, where the weight is")
        a = _PM_LINEAR(x.data_ptr(), self._weight.data_ptr(), 0 if self._bias is None else self._bias.data_ptr(), res, out.data_ptr(), ld_x, self._ld_w, ld_r, ld_y, M, *self._kind)
        rc = self._fn(a, _raw_stream(index)) if index == _current_device() else _elsewhere(index, self._fn, a)
        if rc:
            _lib.check(rc)
        return out

    def _without_memory(self) -> "Linear":
        """For a caller that keeps the weight and the bias itself and says at each call (_dense) where they are."""
        self._weight = self._bias = None
        return self

    def _dense(self, x: torch.Tensor, M: int, weight: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor:
        """x [..., K] -> [..., N] for a caller that has looked: x is contiguous, of the weight's type and device, M rows; weight and bias
        are laid out like those this product was made from."""
        index = self._device_index
        out = torch.empty((*x.shape[:-1], self._N), dtype=self._out_dtype, device=x.device)
        a = _PM_LINEAR(x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), 0, out.data_ptr(), self._K,
                       self._ld_w, 0, self._N, M, *self._kind)
        rc = self._fn(a, _raw_stream(index)) if index == _current_device() else _elsewhere(index, self._fn, a)
        if rc:
            _lib.check(rc)
        return out


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_n: int = 0, out=None):
    """Log probability of targets[t] under softmax(logits[t]), the entropy of that distribution and its top_n best
    alternatives, for every row: (logp [T], entropy [T], top_ids [T, top_n] int32, top_logp [T, top_n]), all but the ids float32.

    logits [T, V] float32 / bf16 / fp16, targets [T] int64; a negative target names no token (logp 0). Masked logits (-inf)
    have probability 0; pm_k_token_logprobs states what rows without a distribution give. out: the four results to fill."""
    if _tracing() is not None:
        _refuse_tracing()
    index, T, V, pitch = _matrix(logits, "logits")
    if top_n < 0:
        raise ValueError("top_n must not be negative")
    if targets.shape != (T,) or targets.dtype != torch.int64 or targets.get_device() != index or not targets.is_contiguous():
        raise ValueError(f"targets must be a contiguous int64 tensor of shape [{T}] on cuda:{index}")
    if out is None:
        new = lambda shape, dtype: torch.empty(shape, dtype=dtype, device=logits.device)  # noqa: E731
        logp, entropy, ids, best = new((T,), _F32), new((T,), _F32), new((T, top_n), _I32), new((T, top_n), _F32)
    else:
        logp, entropy, ids, best = out
        row, wide = (T,), (T, top_n)
        try:
            fits = (logp.shape == row == entropy.shape and ids.shape == wide == best.shape and ids.dtype is _I32
                    and logp.dtype is entropy.dtype is best.dtype is _F32 and logp.get_device() == index and entropy.get_device() == index
                    and ids.get_device() == index and best.get_device() == index and logp.is_contiguous() and entropy.is_contiguous()
                    and ids.is_contiguous() and best.is_contiguous())
        except AttributeError:  # no tensors
            fits = False
        if not fits:
            raise ValueError(f"out must be contiguous tensors on cuda:{index}: float32 {row} twice, int32 and float32 {wide}")
    args = (logits.data_ptr(), _DTYPES[logits.dtype], pitch, T, V, targets.data_ptr(), top_n, logp.data_ptr(), entropy.data_ptr(),
            ids.data_ptr(), best.data_ptr())
    fn = _lib.load().pm_k_token_logprobs
    rc = fn(*args, _raw_stream(index)) if index == _current_device() else _elsewhere(index, fn, *args)
    if rc:
        _lib.check(rc)
    return logp, entropy, ids, best
