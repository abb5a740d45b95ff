"""Mixture-of-experts operators over the C-ABI: routing rows to experts.

Device memory and streams come from torch; all compute is the HIP library's.
Tensors on the CPU are rejected: there is no CPU path.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

_SCORES = {"softmax": _lib.CKAN_SCORE_SOFTMAX, "sigmoid": _lib.CKAN_SCORE_SIGMOID}
_DTYPES = {torch.float32: _lib.CKAN_DTYPE_F32, torch.bfloat16: _lib.CKAN_DTYPE_BF16}


def _require_device(*tensors) -> None:
    first = tensors[0]
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("kan_amd's mixture operators run only on a ROCm device (MI355X); "
                               f"got a tensor on {t.device}")
        if t.device != first.device:
            raise RuntimeError(f"tensors on {first.device} and {t.device}: one device is needed")


def _dtype_code(t: torch.Tensor, name: str) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise RuntimeError(f"{name} must be float32 or bfloat16, got {t.dtype}") from None


class RouteFunction(torch.autograd.Function):
    """(weights, indices) of ``route``; differentiable in the logits."""

    @staticmethod
    def forward(ctx, logits: torch.Tensor, bias: Optional[torch.Tensor], desc):
        rows = logits.shape[0]
        w = torch.empty(rows, desc.top_k, dtype=torch.float32, device=logits.device)
        idx = torch.empty(rows, desc.top_k, dtype=torch.int64, device=logits.device)
        with torch.cuda.device(logits.device):
            _lib.check(_lib.load().ckan_route(desc, logits.data_ptr(), _lib.ptr(bias), w.data_ptr(),
                                              idx.data_ptr(), _lib.stream_ptr(logits.device)))
        ctx.save_for_backward(logits, idx)
        ctx.mark_non_differentiable(idx)
        ctx.desc = desc
        return w, idx

    @staticmethod
    def backward(ctx, dw: torch.Tensor, _didx):
        logits, idx = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            return None, None, None
        dw = dw.to(torch.float32).contiguous()
        dl = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with torch.cuda.device(logits.device):
            _lib.check(_lib.load().ckan_route_backward(
                ctx.desc, logits.data_ptr(), idx.data_ptr(), dw.data_ptr(), dl.data_ptr(),
                _lib.stream_ptr(logits.device)))
        return dl, None, None


def route(logits: torch.Tensor, top_k: int, *, score: str = "softmax",
          bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: int = 1,
          renormalize: bool = True, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Each row's ``top_k`` experts: (weights [rows, top_k] fp32, indices [rows, top_k] int64).

    ``logits`` [rows, experts] (fp32 or bf16; up to 512 experts) give the scores by
    ``score``: 'softmax' over the experts or 'sigmoid' of each.  The choice goes by
    score + ``bias`` ([experts] fp32, a balance correction that moves no weight);
    with ``groups`` > 1 only the ``top_groups`` groups of consecutive experts stay
    whose two largest keys sum highest.  Equal keys go to the lowest index.  The
    weights are the chosen scores, over their sum with ``renormalize``, times
    ``scale``.  An expert whose logit is -inf or NaN is never chosen; a row that
    has fewer than ``top_k`` others fills up with index -1 and weight 0.

    Differentiable in ``logits`` (through the weights, not through the choice)."""
    if score not in _SCORES:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
    if logits.dim() != 2:
        raise RuntimeError(f"logits must be [rows, experts], got {tuple(logits.shape)}")
    _require_device(logits, bias)
    code = _dtype_code(logits, "logits")
    experts = logits.shape[1]
    if bias is not None:
        if tuple(bias.shape) != (experts,):
            raise RuntimeError(f"bias must be [{experts}], got {tuple(bias.shape)}")
        bias = bias.detach().to(torch.float32).contiguous()
    if logits.stride(1) != 1 or logits.stride(0) < experts:
        logits = logits.contiguous()
    desc = _lib.CkanRouteDesc(logits.shape[0], max(logits.stride(0), experts), experts, int(top_k),
                              _SCORES[score], int(groups), int(top_groups), int(bool(renormalize)),
                              code, float(scale))
    return RouteFunction.apply(logits, bias, desc)
