"""Mixture-of-experts operators over the C-ABI: routing rows to experts and the
products of ChebyKAN experts.

Device memory and streams come from torch; all compute is the HIP library's.
Tensors on the CPU are rejected: there is no CPU path.
"""
from __future__ import annotations

from contextlib import nullcontext
from functools import lru_cache
from typing import Any, Dict, Optional, Tuple

import torch
import torch.nn as nn

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


_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _stream(device: torch.device) -> int:
    """hipStream_t of torch's current stream, without building a Stream object (2 us)."""
    return _raw_stream(device.index) if _raw_stream is not None else _lib.stream_ptr(device)


def _on(device: torch.device):
    """Makes ``device`` current for the library's launches; nothing to do when it is."""
    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous at a 16-byte aligned address, as the library's vector loads need it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _route_forward(logits, bias, desc):
    dev = logits.device
    w = torch.empty(desc.rows, desc.top_k, dtype=torch.float32, device=dev)
    idx = torch.empty(desc.rows, desc.top_k, dtype=torch.int64, device=dev)
    with _on(dev):
        _lib.check(_lib.load().ckan_route(desc, logits.data_ptr(), _lib.ptr(bias), w.data_ptr(), idx.data_ptr(),
                                          _stream(dev)))
    return w, idx


def _once(name: str) -> None:
    """Refuses a backward that is to be differentiated again: it would be a constant."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name} is differentiable once (create_graph is not supported)")


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A saved tensor as its kernel reads it, whatever layout a hook returned it in."""
    return t if t is None or t.is_contiguous() else t.contiguous()


def _pitched(desc, **pitches):
    """desc with these row pitches: a hook on saved tensors may have returned them in another layout
    than they were saved in."""
    if all(getattr(desc, name) == pitch for name, pitch in pitches.items()):
        return desc
    desc = type(desc).from_buffer_copy(desc)
    for name, pitch in pitches.items():
        setattr(desc, name, pitch)
    return desc


def _logit_rows(logits: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """logits with contiguous rows, and their pitch."""
    experts = logits.shape[1]
    if logits.stride(1) != 1 or logits.stride(0) < experts:
        logits = logits.contiguous()
    return logits, max(logits.stride(0), experts)


class RouteFunction(torch.autograd.Function):
    """The weights of ``route``, differentiable in the logits; the indices go by the
    side (``out``): an output more costs the autograd engine 4 us a step."""

    @staticmethod
    def forward(ctx, logits: torch.Tensor, bias: Optional[torch.Tensor], desc, out: list):
        w, idx = _route_forward(logits, bias, desc)
        ctx.save_for_backward(logits)
        ctx.desc, ctx.idx, ctx.idx_version = desc, idx, idx._version
        out.append(idx)
        return w

    @staticmethod
    def backward(ctx, dw: torch.Tensor):
        _once("route")
        logits, = ctx.saved_tensors
        if ctx.idx._version != ctx.idx_version:
            raise RuntimeError("route's indices were modified in place before its backward; change a clone")
        if dw.dtype != torch.float32 or not dw.is_contiguous():
            dw = dw.to(torch.float32).contiguous()
        dl = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        logits, ld = _logit_rows(logits)
        # the engine runs a node on its device and stream
        _lib.check(_lib.load().ckan_route_backward(_pitched(ctx.desc, logits_ld=ld), logits.data_ptr(), ctx.idx.data_ptr(),
                                                   dw.data_ptr(), dl.data_ptr(), _stream(dl.device)))
        return dl, None, None, None


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
    ``scale``.  An expert whose logit is -inf or NaN is never chosen and scores 0 (+inf
    counts as the largest finite logit), one whose bias is -inf or NaN is never chosen and
    keeps its score; a row that has fewer than ``top_k`` others fills up with index -1 and weight 0.

    Differentiable once in ``logits`` (through the weights, not through the choice);
    the indices are not to be changed in place before the backward."""
    if score not in _SCORES:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
    if logits.dim() != 2:
        raise RuntimeError(f"logits must be [rows, experts], got {tuple(logits.shape)}")
    _lib.refuse_tangents("route", logits)
    _require_device(logits, bias)
    code = _dtype_code(logits, "logits")
    experts = logits.shape[1]
    if bias is not None:
        if tuple(bias.shape) != (experts,):
            raise RuntimeError(f"bias must be [{experts}], got {tuple(bias.shape)}")
        bias = bias.detach().to(torch.float32).contiguous()
    logits, ld = _logit_rows(logits)
    desc = _lib.CkanRouteDesc(logits.shape[0], ld, experts, int(top_k),
                              _SCORES[score], int(groups), int(top_groups), int(bool(renormalize)),
                              code, float(scale))
    if torch.is_grad_enabled() and logits.requires_grad:
        out: list = []
        return RouteFunction.apply(logits, bias, desc, out), out[0]
    return _route_forward(logits, bias, desc)


def _experts_forward(x, coeffs, indices, weights, desc, keep):
    """(y, saved): saved is None without ``keep``."""
    lib, dev = _lib.load(), x.device
    y = torch.empty(desc.rows, desc.out_dim, dtype=x.dtype, device=dev)
    nbytes = lib.ckan_experts_workspace_bytes(desc, 0, int(not keep))
    with _on(dev):
        # both from torch's allocator on the current stream: reused by it in stream order
        saved = (torch.empty(max(lib.ckan_experts_saved_bytes(desc), 256), dtype=torch.uint8, device=dev)
                 if keep else None)
        ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dev)
        _lib.check(lib.ckan_experts_forward(desc, x.data_ptr(), coeffs.data_ptr(), indices.data_ptr(),
                                            weights.data_ptr(), y.data_ptr(), _lib.ptr(saved), ws.data_ptr(), nbytes,
                                            _stream(dev)))
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
        _once("kan_experts")
        saved, indices, weights = map(_dense, ctx.saved_tensors)
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
        ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dev)
        # the engine runs a node on its device and stream
        _lib.check(lib.ckan_experts_backward(desc, indices.data_ptr(), weights.data_ptr(), saved.data_ptr(),
                                             dy.data_ptr(), _lib.ptr(dx), _lib.ptr(dc), _lib.ptr(dw), ws.data_ptr(),
                                             nbytes, _stream(dev)))
        return dx, dc, dw, None, None


def kan_experts(x: torch.Tensor, coeffs: torch.Tensor, indices: torch.Tensor,
                weights: torch.Tensor) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] f_e(x[t]) with e = indices[t, j], f_e the ChebyKAN layer
    of coefficients coeffs[e] (kan/layers/chebykan.py:64-67).

    ``x`` [rows, in] and ``coeffs`` [experts, in, out, degree+1] are both fp32 or both
    bf16 (y [rows, out] likewise); ``indices`` [rows, top_k] int64 and ``weights`` [rows,
    top_k] (fp32 or bf16) as ``route`` returns them.  A slot whose index lies outside
    [0, experts) has no expert: a row of such slots gives zeros.  Degrees 1 to 16,
    up to 512 experts.  fp32 results carry fp32 accuracy: operands of 22 bits, coefficients
    down to 2^-13 of their expert's largest (an error of 2^-35 of that below), gradients of
    any size for x; for the coefficients' gradient those down to 2^-16 of the largest among
    the expert's rows (an error of 2^-38 of that below).  bf16 results are rounded once from
    fp32 sums of 11-bit basis values.

    Differentiable once in x, coeffs and weights; sums run in a fixed order, so a call
    repeats bit for bit."""
    _lib.refuse_tangents("kan_experts", x, coeffs, weights)
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


def _gate_logits(x: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
    """x gate^T in fp32, inside autocast too: the choice hangs on it."""
    if not torch.is_autocast_enabled(x.device.type):
        return x @ gate.t()
    with torch.autocast(x.device.type, enabled=False):
        return x @ gate.t()


def kan_mixture(x: torch.Tensor, gate: torch.Tensor, coeffs: torch.Tensor, top_k: int, *, score: str = "softmax",
                bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: int = 1, renormalize: bool = True,
                scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A whole mixture layer: (y, weights, indices) with ``route``'s choice among the experts by
    the logits x gate^T and y[t] = sum_j weights[t, j] f_e(x[t]) as ``kan_experts``'.

    ``x`` [rows, in], ``gate`` [experts, in] and ``coeffs`` [experts, in, out, degree+1] are fp32 or
    bf16 each; y [rows, out] has x's dtype, weights and indices are ``route``'s.  Few rows without a
    gradient (up to 1024 slots, fewer than 64 an expert on average; of many fp32 coefficients of degree
    9 and more up to 8 rows of 64 slots, or from 8 slots an expert on) take a form of their own: the gate's sums in
    64 bits, the chosen experts' coefficients read as they lie, x unrounded.  Otherwise the gate's
    product is torch's in fp32 and the rest is ``route`` and ``kan_experts`` (in fp32 unless x and coeffs
    are both bf16), differentiable as they are in x, gate and coeffs."""
    if score not in _SCORES:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
    _lib.refuse_tangents("kan_mixture", x, gate, coeffs)
    _require_device(x, gate, coeffs, bias)
    codes = [_dtype_code(t, name) for t, name in ((x, "x"), (gate, "gate"), (coeffs, "coeffs"))]
    if coeffs.dim() != 4:
        raise RuntimeError(f"coeffs must be [experts, in, out, degree+1], got {tuple(coeffs.shape)}")
    experts, in_dim, out_dim, dd = coeffs.shape
    if x.dim() != 2 or x.shape[1] != in_dim:
        raise RuntimeError(f"x must be [rows, {in_dim}], got {tuple(x.shape)}")
    if tuple(gate.shape) != (experts, in_dim):
        raise RuntimeError(f"gate must be [{experts}, {in_dim}], got {tuple(gate.shape)}")
    if bias is not None and tuple(bias.shape) != (experts,):
        raise RuntimeError(f"bias must be [{experts}], got {tuple(bias.shape)}")
    for name, v in (("in_dim", in_dim), ("out_dim", out_dim), ("degree", dd - 1), ("top_k", top_k), ("groups", groups),
                    ("top_groups", top_groups)):
        if not -1 <= v < 1 << 31:  # the descriptor's 32 bits would take another number for it
            raise RuntimeError(f"{name} is out of range: {v}")
    rows, lib = x.shape[0], _lib.load()
    desc = _lib.CkanMixtureDesc(rows, experts, int(top_k), in_dim, out_dim, dd - 1, _SCORES[score], int(groups),
                                int(top_groups), int(bool(renormalize)), *codes, float(scale))
    trains = torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or coeffs.requires_grad)
    if trains or not lib.ckan_mixture_few(desc):
        weights, indices = route(_gate_logits(x.to(torch.float32), gate.to(torch.float32)), top_k, score=score, bias=bias,
                                 groups=groups, top_groups=top_groups, renormalize=renormalize, scale=scale)
        # in the wider of the two types, so that fp32 rows keep fp32's accuracy on bf16 coefficients in either form
        dtype = torch.promote_types(x.dtype, coeffs.dtype)
        return kan_experts(x.to(dtype), coeffs.to(dtype), indices, weights).to(x.dtype), weights, indices
    dev = x.device
    x, gate, coeffs = _aligned(x), _aligned(gate), _aligned(coeffs)
    if bias is not None:
        bias = bias.detach().to(torch.float32).contiguous()
    y = torch.empty(rows, out_dim, dtype=x.dtype, device=dev)
    weights = torch.empty(rows, desc.top_k, dtype=torch.float32, device=dev)
    indices = torch.empty(rows, desc.top_k, dtype=torch.int64, device=dev)
    nbytes = lib.ckan_mixture_workspace_bytes(desc)
    # from torch's allocator on the current stream: reused by it in stream order
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with _on(dev):
        _lib.check(lib.ckan_mixture_forward(desc, x.data_ptr(), gate.data_ptr(), coeffs.data_ptr(), _lib.ptr(bias),
                                            y.data_ptr(), weights.data_ptr(), indices.data_ptr(), ws.data_ptr(), nbytes,
                                            _stream(dev)))
    return y, weights, indices


@lru_cache(maxsize=4096)
def _few_rows(rows, experts, top_k, in_dim, out_dim, degree, score, groups, top_groups, coeff_code) -> bool:
    """The library's rule by sizes; asking it takes 4 us."""
    desc = _lib.CkanMixtureDesc(rows, experts, top_k, in_dim, out_dim, degree, score, groups, top_groups, 1, 0, 0, coeff_code,
                                1.0)
    return bool(_lib.load().ckan_mixture_few(desc))


class MixtureKANLayer(nn.Module):
    """A mixture of ChebyKAN layers: each row goes to ``top_k`` of ``experts`` layers of
    ``ChebyKANLayer(input_dim, output_dim, degree)`` (kan/layers/chebykan.py:21-51), chosen
    and weighted by a linear gate through ``route``, computed by ``kan_experts``.

    Parameters: ``gate`` [experts, input_dim] and ``cheby_coeffs`` [experts, input_dim,
    output_dim, degree+1], each expert initialised as the layer is.  ``compute``: 'fp32'
    or 'bf16' (the experts' operands and outputs are bf16, the gate, the choice and the
    weights stay fp32; the output is fp32, as a ChebyKANLayer's).  Few rows without a
    gradient go through ``kan_mixture`` on the fp32 parameters in either mode; otherwise 'bf16' casts the
    coefficients of all experts in every forward.  To serve rows from bf16 coefficients, call
    ``kan_mixture`` on coefficients cast once.

    With ``balance``, a per-expert bias steers the choice, not the weights:
    ``update_balance`` moves it towards experts that got fewer rows than the mean."""

    def __init__(self, input_dim: int, output_dim: int, degree: int, experts: int, top_k: int = 2, *,
                 score: str = "softmax", groups: int = 1, top_groups: int = 1, renormalize: bool = True,
                 scale: float = 1.0, balance: bool = False, init_scale: Optional[float] = None,
                 compute: str = "fp32"):
        super().__init__()
        if score not in _SCORES:
            raise ValueError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
        if compute not in ("fp32", "bf16"):
            raise ValueError(f"compute must be 'fp32' or 'bf16', got {compute!r}")
        if not 1 <= degree <= 16:
            raise ValueError(f"experts have degree 1 to 16, got {degree}")
        if groups < 1 or experts % groups or not 1 <= top_groups <= groups:
            raise ValueError(f"groups must divide experts and hold top_groups: got {experts} experts, {groups} "
                             f"groups, {top_groups} kept")
        if not 1 <= top_k <= experts // groups * top_groups:
            raise ValueError(f"top_k must lie in [1, {experts // groups * top_groups}], got {top_k}")
        self.input_dim, self.output_dim, self.degree = input_dim, output_dim, degree
        self.experts, self.top_k, self.score = experts, top_k, score
        self.groups, self.top_groups = groups, top_groups
        self.renormalize, self.scale, self.compute = renormalize, scale, compute
        self.gate = nn.Parameter(torch.empty(experts, input_dim))
        self.cheby_coeffs = nn.Parameter(torch.empty(experts, input_dim, output_dim, degree + 1))
        nn.init.normal_(self.gate, mean=0.0, std=input_dim ** -0.5)
        nn.init.normal_(self.cheby_coeffs, mean=0.0, std=init_scale or 1.0 / (input_dim * (degree + 1)))
        self.register_buffer("balance_bias", torch.zeros(experts) if balance else None)
        self._last_indices: Optional[torch.Tensor] = None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = x.reshape(-1, self.input_dim).to(torch.float32)
        how = dict(score=self.score, bias=self.balance_bias, groups=self.groups, top_groups=self.top_groups,
                   renormalize=self.renormalize, scale=self.scale)
        if self._few(x):
            y, _, indices = kan_mixture(x, self.gate, self.cheby_coeffs, self.top_k, **how)
        elif self.compute == "fp32":  # what kan_mixture does, without its checks (10 us of the host's time)
            weights, indices = route(_gate_logits(x, self.gate.to(torch.float32)), self.top_k, **how)
            y = kan_experts(x, self.cheby_coeffs.to(torch.float32), indices, weights)
        else:
            weights, indices = route(_gate_logits(x, self.gate), self.top_k, **how)
            y = kan_experts(x.bfloat16(), self.cheby_coeffs.bfloat16(), indices, weights).to(torch.float32)
        self._last_indices = indices if self.balance_bias is not None else None
        return y

    def _few(self, x: torch.Tensor) -> bool:
        """Whether x is for ``kan_mixture``. In bf16 mode by its rule for bf16 coefficients, which has no limit for high degrees: past
        that one its parts run in fp32 too, and casting all coefficients takes longer."""
        if torch.is_grad_enabled() and (x.requires_grad or self.gate.requires_grad or self.cheby_coeffs.requires_grad):
            return False
        code = _lib.CKAN_DTYPE_F32 if self.compute == "fp32" else _lib.CKAN_DTYPE_BF16
        return _few_rows(x.shape[0], self.experts, self.top_k, self.input_dim, self.output_dim, self.degree,
                         _SCORES[self.score], self.groups, self.top_groups, code)

    @torch.no_grad()
    def update_balance(self, speed: float = 1e-3) -> None:
        """Moves the balance bias of each expert by ``speed``, up where the last forward
        gave it fewer rows than the mean and down where more."""
        if self.balance_bias is None:
            raise RuntimeError("the layer was built without balance=True")
        if self._last_indices is None:
            raise RuntimeError("update_balance needs a forward first")
        idx = self._last_indices.reshape(-1)
        load = torch.zeros(self.experts + 1, device=idx.device)
        load.scatter_add_(0, torch.where(idx >= 0, idx, self.experts), torch.ones_like(idx, dtype=load.dtype))
        load = load[:-1]
        self.balance_bias.add_(speed * torch.sign(load.mean() - load))

    def get_coefficients(self) -> torch.Tensor:
        return self.cheby_coeffs

    def get_analytical_form(self) -> Dict[str, Any]:
        return {"type": "MixtureKANLayer", "input_dim": self.input_dim, "output_dim": self.output_dim,
                "degree": self.degree, "experts": self.experts, "top_k": self.top_k, "basis": "chebyshev",
                "gate": self.gate.detach().cpu().numpy(),
                "coefficients": self.cheby_coeffs.detach().cpu().numpy()}

    def extra_repr(self) -> str:
        return (f"input_dim={self.input_dim}, output_dim={self.output_dim}, degree={self.degree}, "
                f"experts={self.experts}, top_k={self.top_k}, score={self.score}")
