"""Operators around the experts, on torch tensors: the router on given logits, the dense product with bias, activation
and residual, and the log probabilities of given tokens.

Thin wrappers over the C ABI (include/promoe_b200.h: pm_k_route, pm_k_linear, pm_k_token_logprobs): they check shapes and types,
allocate results where the caller brings none and launch on torch's current stream of the tensors' device. They
hold no state besides what a caller hands to their constructors, run without scratch memory and can be captured into a CUDA graph.
No gradients: tensors that require one are refused while autograd records.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_SCORING = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}


def _call(device: torch.device, fn, *args) -> None:
    """fn(*args, stream) with `device` current, on its current stream."""
    if device.index == torch.cuda.current_device():
        _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))


def _rows(t: torch.Tensor, what: str, width: int | None = None, dtypes=_DTYPES) -> torch.Tensor:
    """A CUDA matrix with dense rows of `width` values."""
    if not t.is_cuda or t.dim() != 2 or t.dtype not in dtypes:
        raise ValueError(f"{what} must be a 2-D CUDA tensor of {', '.join(str(d) for d in dtypes)}")
    if width is not None and t.shape[1] != width:
        raise ValueError(f"{what} must have rows of {width} values, not {t.shape[1]}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"the rows of {what} must be dense")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient: these operators have no backward pass")
    return t


def _pitch(t: torch.Tensor) -> int:
    """Distance of two rows; rows that lie over one another (a broadcast) are no matrix that the kernels take."""
    if t.shape[0] <= 1:
        return max(t.shape[1], 1)
    if t.stride(0) < t.shape[1]:
        raise ValueError("rows must not overlap (expanded tensors: call contiguous())")
    return t.stride(0)


def _result(out, shape, dtype, device, what: str) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if out.shape != shape or out.dtype != dtype or out.device != device or not out.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")
    return out


def _same_device(device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device}, not on {t.device}")


class Router:
    """Chooses top_k of num_expert experts per token from router logits (pm_k_route states the rule).

    scoring: "softmax" or "sigmoid". bias: [num_expert] float32 on the device, added to the scores for the choice only (a
    load-balancing correction). n_group / topk_group / group_score ("max" or "top2"): choose among the best groups
    only. norm_topk: weights divided by their sum. routed_scale: multiplies the weights."""

    def __init__(self, num_expert: int, top_k: int, scoring: str = "softmax", bias: torch.Tensor | None = None, n_group: int = 1,
                 topk_group: int = 1, group_score: str = "max", norm_topk: bool = False, routed_scale: float = 1.0):
        if scoring not in _SCORING:
            raise ValueError(f"scoring must be one of {sorted(_SCORING)}")
        if group_score not in _GROUP_SCORE:
            raise ValueError(f"group_score must be one of {sorted(_GROUP_SCORE)}")
        if bias is not None:
            if not bias.is_cuda or bias.dtype != torch.float32 or bias.shape != (num_expert,) or not bias.is_contiguous():
                raise ValueError("bias must be a contiguous float32 CUDA tensor of shape [num_expert]")
        self.num_expert, self.top_k, self.bias = num_expert, top_k, bias
        self.rule = _lib.pm_router(num_expert, top_k, _SCORING[scoring], n_group, topk_group, _GROUP_SCORE[group_score],
                                   int(norm_topk), routed_scale, None if bias is None else bias.data_ptr())
        self._ref = C.byref(self.rule)
        self._fn = _lib.load().pm_k_route
        # the rule's own checks, without a token
        _lib.check(self._fn(self._ref, None, 0, num_expert, 0, None, None, None))

    def __call__(self, logits: torch.Tensor, out: tuple[torch.Tensor, torch.Tensor] | None = None):
        """logits [T, num_expert] float32 / bf16 / fp16 -> (ids [T, top_k] int32, weights [T, top_k] float32)."""
        _rows(logits, "logits", self.num_expert)
        dev, T = logits.device, logits.shape[0]
        _same_device(dev, bias=self.bias)
        shape = (T, self.top_k)
        ids, w = out if out is not None else (None, None)
        ids, w = _result(ids, shape, torch.int32, dev, "ids"), _result(w, shape, torch.float32, dev, "weights")
        _call(dev, self._fn, self._ref, logits.data_ptr(), _DTYPES[logits.dtype], _pitch(logits) if T > 1 else self.num_expert, T,
              ids.data_ptr(), w.data_ptr())
        return ids, w


class Linear:
    """y = activation(x weight^T + bias) + residual in one kernel (pm_k_linear).

    weight [N, K] bf16 or fp16 with dense rows, bias [N] of the same type or float32, activation None / "relu" / "silu" /
    "gelu" / "gelu_tanh", out_dtype the weight's type (default) or float32. The tensors are used in place, not copied."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
                 out_dtype: torch.dtype | None = None):
        weight = weight.detach()
        _rows(weight, "weight", dtypes=(torch.bfloat16, torch.float16))
        if activation not in _ACTS:
            raise ValueError(f"activation must be one of {[a for a in _ACTS if a]} or None")
        out_dtype = weight.dtype if out_dtype is None else out_dtype
        if out_dtype not in (torch.float32, weight.dtype):
            raise ValueError(f"out_dtype must be float32 or {weight.dtype}")
        if bias is not None:
            bias = bias.detach()
            if bias.shape != (weight.shape[0],) or bias.dtype not in (torch.float32, weight.dtype) or not bias.is_contiguous():
                raise ValueError(f"bias must be a contiguous tensor of shape [{weight.shape[0]}], float32 or {weight.dtype}")
            _same_device(weight.device, bias=bias)
        self.weight, self.bias, self.out_dtype, self.device = weight, bias, out_dtype, weight.device
        self.N, self.K = weight.shape
        self._fixed = dict(w=weight.data_ptr(), bias=None if bias is None else bias.data_ptr(), ld_w=_pitch(weight),
                           N=self.N, K=self.K, dtype=_DTYPES[weight.dtype], out_dtype=_DTYPES[out_dtype],
                           bias_dtype=0 if bias is None else _DTYPES[bias.dtype], act=_ACTS[activation])
        self._fn = _lib.load().pm_k_linear

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """x [M, K] of the weight's type, residual [M, N] of out_dtype (dense rows, any pitch) -> y [M, N]. out may be the
        residual itself; it must not overlap x, the weight or the bias."""
        _rows(x, "x", self.K, (self.weight.dtype,))
        M, dev = x.shape[0], self.device
        _same_device(dev, x=x, residual=residual, out=out)
        if residual is not None:
            _rows(residual, "residual", self.N, (self.out_dtype,))
            if residual.shape[0] != M:
                raise ValueError(f"residual must have {M} rows, not {residual.shape[0]}")
        if out is None:
            out = torch.empty((M, self.N), dtype=self.out_dtype, device=dev)
        else:
            _rows(out, "out", self.N, (self.out_dtype,))
            if out.shape[0] != M:
                raise ValueError(f"out must have {M} rows, not {out.shape[0]}")
        a = _lib.pm_linear(x=x.data_ptr(), y=out.data_ptr(), residual=None if residual is None else residual.data_ptr(),
                           ld_x=_pitch(x), ld_y=_pitch(out), ld_residual=0 if residual is None else _pitch(residual), M=M, **self._fixed)
        _call(dev, self._fn, C.byref(a))
        return out


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_n: int = 0, out=None):
    """Log probability of targets[t] under softmax(logits[t]), the entropy of that distribution and its top_n best
    alternatives, for every row: (logp [T], entropy [T], top_ids [T, top_n] int32, top_logp [T, top_n]), all but the ids float32.

    logits [T, V] float32 / bf16 / fp16, targets [T] int64; a negative target names no token (logp 0). Masked logits (-inf)
    have probability 0; pm_k_token_logprobs states what rows without a distribution give. out: the four results to fill."""
    _rows(logits, "logits")
    T, V = logits.shape
    dev = logits.device
    if targets.shape != (T,) or targets.dtype != torch.int64 or targets.device != dev or not targets.is_contiguous():
        raise ValueError(f"targets must be a contiguous int64 tensor of shape [{T}] on {dev}")
    logp, entropy, ids, best = out if out is not None else (None, None, None, None)
    logp, entropy = _result(logp, (T,), torch.float32, dev, "logp"), _result(entropy, (T,), torch.float32, dev, "entropy")
    ids, best = _result(ids, (T, top_n), torch.int32, dev, "top_ids"), _result(best, (T, top_n), torch.float32, dev, "top_logp")
    _call(dev, _lib.load().pm_k_token_logprobs, logits.data_ptr(), _DTYPES[logits.dtype], _pitch(logits), T, V,
          targets.data_ptr(), top_n, logp.data_ptr(), entropy.data_ptr(), ids.data_ptr(), best.data_ptr())
    return logp, entropy, ids, best
