"""Mixture-of-experts operators over the C-ABI: routing rows to experts and the
products of ChebyKAN experts.

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


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous at a 16-byte aligned address, as the library's vector loads need it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


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


def _experts_forward(x, coeffs, indices, weights, desc, keep):
    """(y, saved): saved is None without ``keep``."""
    lib, dev = _lib.load(), x.device
    y = torch.empty(desc.rows, desc.out_dim, dtype=x.dtype, device=dev)
    nbytes = lib.ckan_experts_workspace_bytes(desc, 0, int(not keep))
    with torch.cuda.device(dev):
        # both from torch's allocator on the current stream: reused by it in stream order
        saved = (torch.empty(max(lib.ckan_experts_saved_bytes(desc), 256), dtype=torch.uint8, device=dev)
                 if keep else None)
        ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dev)
        _lib.check(lib.ckan_experts_forward(desc, x.data_ptr(), coeffs.data_ptr(), indices.data_ptr(),
                                            weights.data_ptr(), y.data_ptr(), _lib.ptr(saved), ws.data_ptr(), nbytes,
                                            _lib.stream_ptr(dev)))
    return y, saved


class ExpertsFunction(torch.autograd.Function):
    """``kan_experts`` with its gradients in x, coeffs and weights."""

    @staticmethod
    def forward(ctx, x, coeffs, weights, indices, desc):
        y, saved = _experts_forward(x, coeffs, indices, weights, desc, keep=True)
        ctx.save_for_backward(saved, indices, weights)
        ctx.desc = desc
        ctx.shapes = (x.shape, coeffs.shape, x.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        saved, indices, weights = ctx.saved_tensors
        desc = ctx.desc
        xs, cs, dtype = ctx.shapes
        need_x, need_c, need_w = ctx.needs_input_grad[:3]
        if not (need_x or need_c or need_w):
            return None, None, None, None, None
        dev = dy.device
        dy = _aligned(dy.to(dtype))
        dx = torch.empty(xs, dtype=dtype, device=dev) if need_x else None
        dw = torch.empty(weights.shape, dtype=weights.dtype, device=dev) if need_w else None
        if desc.rows == 0:
            return dx, torch.zeros(cs, dtype=dtype, device=dev) if need_c else None, dw, None, None
        dc = torch.empty(cs, dtype=dtype, device=dev) if need_c else None
        lib = _lib.load()
        nbytes = lib.ckan_experts_workspace_bytes(desc, 1, 0)
        with torch.cuda.device(dev):
            ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dev)
            _lib.check(lib.ckan_experts_backward(desc, indices.data_ptr(), weights.data_ptr(), saved.data_ptr(),
                                                 dy.data_ptr(), _lib.ptr(dx), _lib.ptr(dc), _lib.ptr(dw), ws.data_ptr(),
                                                 nbytes, _lib.stream_ptr(dev)))
        return dx, dc, dw, None, None


def kan_experts(x: torch.Tensor, coeffs: torch.Tensor, indices: torch.Tensor,
                weights: torch.Tensor) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] f_e(x[t]) with e = indices[t, j], f_e the ChebyKAN layer
    of coefficients coeffs[e] (kan/layers/chebykan.py:64-67).

    ``x`` [rows, in] and ``coeffs`` [experts, in, out, degree+1] are both fp32 or both
    bf16 (y [rows, out] likewise); ``indices`` [rows, top_k] int64 and ``weights`` [rows,
    top_k] (fp32 or bf16) as ``route`` returns them.  A slot whose index lies outside
    [0, experts) has no expert: a row of such slots gives zeros.  Degrees 1 to 16,
    up to 512 experts.  fp32 results carry fp32 accuracy (operands of 22 bits), bf16
    ones are rounded once from fp32 sums of 11-bit basis values.

    Differentiable in x, coeffs and weights; sums run in a fixed order, so a call
    repeats bit for bit."""
    _require_device(x, coeffs, indices, weights)
    code = _dtype_code(x, "x")
    if coeffs.dtype != x.dtype:
        raise RuntimeError(f"x and coeffs must have one dtype, got {x.dtype} and {coeffs.dtype}")
    wcode = _dtype_code(weights, "weights")
    if indices.dtype != torch.int64:
        raise RuntimeError(f"indices must be int64, got {indices.dtype}")
    if coeffs.dim() != 4:
        raise RuntimeError(f"coeffs must be [experts, in, out, degree+1], got {tuple(coeffs.shape)}")
    experts, in_dim, out_dim, dd = coeffs.shape
    if x.dim() != 2 or x.shape[1] != in_dim:
        raise RuntimeError(f"x must be [rows, {in_dim}], got {tuple(x.shape)}")
    if indices.dim() != 2 or indices.shape[0] != x.shape[0] or weights.shape != indices.shape:
        raise RuntimeError(f"indices and weights must be [{x.shape[0]}, top_k], got {tuple(indices.shape)} and "
                           f"{tuple(weights.shape)}")
    desc = _lib.CkanExpertsDesc(x.shape[0], experts, indices.shape[1], in_dim, out_dim, dd - 1, code, wcode)
    x, coeffs, indices, weights = _aligned(x), _aligned(coeffs), indices.contiguous(), weights.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or coeffs.requires_grad or weights.requires_grad):
        return ExpertsFunction.apply(x, coeffs, weights, indices, desc)
    return _experts_forward(x, coeffs, indices, weights, desc, keep=False)[0]
