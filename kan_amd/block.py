"""What stands around the layers of a deep KAN, over the C-ABI: the norms, gate, dropout and
sum of a residual block, the stack of such blocks, dropout by itself, and the log
probabilities at a network's end.

Device memory and streams come from torch; all compute is the HIP library's.
Tensors on the CPU are rejected: there is no CPU path.
"""
from __future__ import annotations

from typing import Iterable, NamedTuple, Optional, Tuple, Union

import torch
import torch.nn as nn

from . import _lib
from .mixture import _dense, _on, _once, _pitched, _stream

_NORMS = {"rms": _lib.CKAN_NORM_RMS, "layer": _lib.CKAN_NORM_LAYER}
_DTYPES = {torch.float32: _lib.CKAN_DTYPE_F32, torch.bfloat16: _lib.CKAN_DTYPE_BF16}


def _check(name: str, device: torch.device, t: torch.Tensor) -> None:
    if t.is_cuda and t.device == device and t.dtype in _DTYPES:
        return
    if not t.is_cuda:
        raise RuntimeError(f"kan_amd's block operators run only on a ROCm device (MI355X); {name} is on {t.device}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, another tensor on {device}: one device is needed")
    raise RuntimeError(f"{name} must be float32 or bfloat16, got {t.dtype}")


def _rows(t: torch.Tensor, dim: int) -> torch.Tensor:
    """t as [rows, dim], its rows contiguous; itself where it has that form (a view would cost
    a node of the graph), a copy only where no view has it."""
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    return t if (t.stride(1) == 1 or dim == 1) and t.stride(0) >= 0 else t.contiguous()


def _pitch(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.stride(0)


def _like(t: torch.Tensor) -> torch.Tensor:
    """Dense memory of t's shape and type (empty_like takes a third less host time than empty)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _shaped(t: Optional[torch.Tensor], shape) -> Optional[torch.Tensor]:
    return t if t is None or len(shape) == 2 else t.view(shape)


def _drop_state(p: float, state, call: int, device: torch.device):
    """(device tensor or None, seed, offset) of a dropout's ``state`` and ``call``."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the dropout probability must lie in [0, 1], got {p}")
    if not 0 <= call < 1 << 63:
        raise ValueError(f"the dropout call must lie in [0, 2^63), got {call}")
    if p == 0.0:
        return None, 0, 0
    if isinstance(state, torch.Tensor):
        if state.dtype != torch.int64 or state.numel() != 2 or not state.is_contiguous() or state.device != device:
            raise RuntimeError(f"the dropout state must be a contiguous int64 tensor of (seed, offset) on {device}, got "
                               f"{state.dtype} {tuple(state.shape)} on {state.device}")
        return state, 0, call
    if isinstance(state, int):
        return None, state & (1 << 64) - 1, call
    raise ValueError("dropout needs its state: an int seed, or an int64 tensor of (seed, offset) on the device")


# ---- norms around a residual block ---------------------------------------------

class ResidualFunction(torch.autograd.Function):
    """``residual_norm`` and ``row_norm`` with their gradients; outputs (out, h), absent
    ones None."""

    @staticmethod
    def forward(ctx, x, y, gate, post_weight, post_bias, next_weight, next_bias, call):
        tensors = (x, y, gate, post_weight, post_bias, next_weight, next_bias)
        out, h, stats = _residual_forward(tensors, call, keep=True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*tensors, stats)
        ctx.desc, ctx.h_dtype = call.desc, call.h_dtype
        return out, h

    @staticmethod
    def backward(ctx, dout, dh):
        _once("residual_norm")
        need = ctx.needs_input_grad
        if dout is None and dh is None:
            return (None,) * 8
        x, y, gate, *vectors, stats = ctx.saved_tensors
        post_weight, post_bias, next_weight, next_bias, stats = map(_dense, (*vectors, stats))
        desc, dev = ctx.desc, x.device
        if dout is not None:
            dout = _rows(dout if dout.dtype == x.dtype else dout.to(x.dtype), desc.dim)
        if dh is not None:
            dh = _rows(dh if dh.dtype == ctx.h_dtype else dh.to(ctx.h_dtype), desc.dim)
        x, y = _rows(x, desc.dim), y if y is None else _rows(y, desc.dim)
        gate = _rows(gate, desc.dim) if desc.gate_rows else _dense(gate)
        desc = _pitched(desc, x_ld=x.stride(0), y_ld=_pitch(y), gate_ld=gate.stride(0) if desc.gate_rows else 0)
        inputs = (x, y, gate, post_weight, post_bias, next_weight, next_bias)
        grads = [_like(t) if n else None for t, n in zip(inputs, need)]
        if desc.rows == 0:
            return (*(None if g is None else g.zero_() for g in grads), None)
        lib = _lib.load()
        nbytes = lib.ckan_residual_workspace_bytes(desc)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        ptr = _lib.ptr
        buffers = _lib.CkanResidualBuffers(
            x.data_ptr(), ptr(y), ptr(gate), ptr(post_weight), ptr(post_bias), ptr(next_weight), ptr(next_bias), 0, 0, 0,
            stats.data_ptr(), ptr(dout), ptr(dh), *map(ptr, grads), _pitch(dout), _pitch(dh))
        # the engine runs a node on its device and stream
        _lib.check(lib.ckan_residual_backward(desc, buffers, ws.data_ptr(), nbytes, _stream(dev)))
        return (*grads, None)


class _ResidualCall(NamedTuple):
    """What a call takes besides its tensors."""
    desc: "_lib.CkanResidualDesc"
    state: Optional[torch.Tensor]
    seed: int
    offset: int
    h_dtype: torch.dtype


def _residual_forward(tensors, call, keep):
    """(out, h, stats); the tensors are [rows, dim] and [dim]."""
    x, y, gate, post_weight, post_bias, next_weight, next_bias = tensors
    desc, dev, ptr = call.desc, x.device, _lib.ptr
    rows, dim = desc.rows, desc.dim
    out = _like(x) if y is not None else None
    h = None
    if next_weight is not None:  # of y's type where there is a y
        h = _like(y) if y is not None else torch.empty(rows, dim, dtype=call.h_dtype, device=dev)
    stats = torch.empty(rows * 4 + 4, dtype=torch.float32, device=dev) if keep else None
    buffers = _lib.CkanResidualBuffers(
        x.data_ptr(), ptr(y), ptr(gate), ptr(post_weight), ptr(post_bias), ptr(next_weight), ptr(next_bias),
        ptr(call.state), ptr(out), ptr(h), ptr(stats), dropout_seed=call.seed, dropout_offset=call.offset)
    with _on(dev):
        _lib.check(_lib.load().ckan_residual_forward(desc, buffers, _stream(dev)))
    return out, h, stats


# Descriptors by their fields: a structure of this size costs microseconds to build.
_residual_descs = {}


def _residual_desc(*fields) -> "_lib.CkanResidualDesc":
    desc = _residual_descs.get(fields)
    if desc is None:
        if len(_residual_descs) > 4096:
            _residual_descs.clear()
        desc = _residual_descs[fields] = _lib.CkanResidualDesc(*fields)
    return desc


def _code(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else _DTYPES[t.dtype]


def _residual(x, y, gate, post_weight, post_bias, next_weight, next_bias, norm, eps, scale, dropout, state, call,
              h_dtype):
    if norm not in _NORMS:
        raise ValueError(f"norm must be one of {sorted(_NORMS)}, got {norm!r}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"x must be [..., dim] with dim >= 1, got {tuple(x.shape)}")
    shape, dev = x.shape, x.device
    dim = shape[-1]
    if dim > 1 << 20:  # the descriptor's 32 bits would take a larger one for another
        raise RuntimeError(f"dim above 2^20 is not supported, got {dim}")
    _lib.refuse_tangents("residual_norm", x, y, gate, post_weight, post_bias, next_weight, next_bias)
    _check("x", dev, x)
    for name, t in (("post_weight", post_weight), ("post_bias", post_bias), ("next_weight", next_weight),
                    ("next_bias", next_bias)):
        if t is not None:
            _check(name, dev, t)
            if t.dim() != 1 or t.shape[0] != dim:
                raise RuntimeError(f"{name} must be [{dim}], got {tuple(t.shape)}")
    if (post_bias is not None and post_weight is None) or (next_bias is not None and next_weight is None):
        raise RuntimeError("a norm's bias needs its weight")
    if h_dtype not in _DTYPES:
        raise RuntimeError(f"a norm's result is float32 or bfloat16, not {h_dtype}")
    gate_rows = False
    if gate is not None:
        _check("gate", dev, gate)
        gate_rows = gate.dim() > 1 and gate.shape == shape
        if not gate_rows and tuple(gate.shape) != (dim,):
            raise RuntimeError(f"gate must be [{dim}] or {tuple(shape)}, got {tuple(gate.shape)}")
    if y is not None:
        _check("y", dev, y)
        if y.shape != shape:
            raise RuntimeError(f"y must be of x's shape {tuple(shape)}, got {tuple(y.shape)}")
    drop_state, seed, offset = _drop_state(dropout, state, call, dev)
    x = _rows(x, dim)
    if y is not None:
        y = _rows(y, dim)
    if gate is not None:
        gate = _rows(gate, dim) if gate_rows else gate.contiguous()
    post_weight, post_bias, next_weight, next_bias = (
        t if t is None or t.is_contiguous() else t.contiguous() for t in (post_weight, post_bias, next_weight, next_bias))
    desc = _residual_desc(x.shape[0], x.stride(0), _pitch(y), gate.stride(0) if gate_rows else 0, dim, _DTYPES[x.dtype],
                          _DTYPES[h_dtype if y is None else y.dtype], _code(gate), _code(post_weight), _code(post_bias),
                          _code(next_weight), _code(next_bias), _NORMS[norm], int(gate_rows), float(eps), float(scale),
                          float(dropout))
    tensors = (x, y, gate, post_weight, post_bias, next_weight, next_bias)
    how = _ResidualCall(desc, drop_state, seed, offset, h_dtype)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        out, h = ResidualFunction.apply(*tensors, how)
    else:
        out, h, _ = _residual_forward(tensors, how, keep=False)
    return _shaped(out, shape), _shaped(h, shape)


def row_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, norm: str = "rms",
             eps: float = 1e-6, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The norm before a block: each row of x [..., dim] as (v - mean) / sqrt(mean((v -
    mean)^2) + eps) * weight + bias, with mean 0 for norm='rms' ('layer' takes it out).

    x, weight and bias [dim] are fp32 or bf16 each; the result has ``dtype``, x's by
    default.  fp32 arithmetic, rounded once.  Differentiable once in x, weight and bias."""
    return _residual(x, None, None, None, None, weight, bias, norm, eps, 1.0, 0.0, None, 0, dtype or x.dtype)[1]


def residual_norm(x: torch.Tensor, y: torch.Tensor, *, norm: str = "rms", eps: float = 1e-6,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, scale: float = 1.0, dropout: float = 0.0,
                  dropout_state: Union[int, torch.Tensor, None] = None, dropout_call: int = 0,
                  next_weight: Optional[torch.Tensor] = None, next_bias: Optional[torch.Tensor] = None
                  ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """What follows a block: out = x + scale * gate * drop(post(y)), and with ``next_weight``
    also h = next(out), the norm before the block that comes after: (out, h).

    ``x`` [..., dim] is the residual stream, ``y`` of its shape the block's result; each is fp32 or
    bf16.  ``post`` and ``next`` are ``row_norm``'s norms with their own weights [dim] and
    biases, absent without a weight.  ``gate`` is [dim] or of x's shape, 1 without one.
    ``dropout`` draws ``functional.dropout``'s mask for y's shape from ``dropout_state`` and
    ``dropout_call``.  out has x's dtype, h has y's and comes from out before its rounding;
    arithmetic is in fp32.

    Differentiable once in x, y, gate, weights and biases; sums run in a fixed order, so
    a call repeats bit for bit."""
    out, h = _residual(x, y, gate, post_weight, post_bias, next_weight, next_bias, norm, eps, scale, dropout,
                       dropout_state, dropout_call, y.dtype)
    return out if next_weight is None else (out, h)


# ---- dropout -----------------------------------------------------------------------

def _dropout_launch(x, p, state, seed, offset, keep):
    """(y, used) of x [rows, dim]."""
    dev = x.device
    y = _like(x)
    used = torch.empty(2, dtype=torch.int64, device=dev) if keep else None
    desc = _lib.CkanDropoutDesc(x.shape[0], max(x.shape[1], 1), x.stride(0), p, seed, offset, _DTYPES[x.dtype])
    with _on(dev):
        _lib.check(_lib.load().ckan_dropout(desc, _lib.ptr(state), x.data_ptr(), y.data_ptr(), _lib.ptr(used),
                                            _stream(dev)))
    return y, used


class DropoutFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, state, seed, offset):
        y, used = _dropout_launch(x, p, state, seed, offset, keep=True)
        ctx.p, ctx.used, ctx.dtype = p, used, x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        _once("dropout")
        dy = _rows(dy if dy.dtype == ctx.dtype else dy.to(ctx.dtype), dy.shape[-1])
        dx, _ = _dropout_launch(dy, ctx.p, ctx.used, 0, 0, keep=False)
        return dx, None, None, None, None


def dropout(x: torch.Tensor, p: float, state: Union[int, torch.Tensor], call: int = 0) -> torch.Tensor:
    """x [..., dim] (fp32 or bf16) with each element kept with probability 1 - p and divided by it, else 0.

    The mask is a function of the seed, the call's number, the row and the column, by a
    counter-based generator (Philox 4x32-10), and never stored.  ``state`` is the seed, or a
    device tensor int64[2] of (seed, offset), to whose offset ``call`` is added: a captured graph that
    adds to the tensor between its calls draws new masks at every replay.  Equal state and
    call give equal masks.  Differentiable once in x, with the state as the forward read it."""
    if x.dim() < 1:
        raise RuntimeError("x must be [..., dim], got a scalar")
    _lib.refuse_tangents("dropout", x)
    _check("x", x.device, x)
    state, seed, offset = _drop_state(float(p), state, int(call), x.device)
    if x.numel() == 0:
        return x.clone()
    rows = _rows(x, x.shape[-1])
    if torch.is_grad_enabled() and rows.requires_grad:
        return _shaped(DropoutFunction.apply(rows, float(p), state, seed, offset), x.shape)
    return _shaped(_dropout_launch(rows, float(p), state, seed, offset, keep=False)[0], x.shape)


# ---- log probabilities ----------------------------------------------------------------

class LogProbs(NamedTuple):
    """What ``log_probs`` returns; the last two are None without ``top``."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def _log_probs_forward(logits, targets, desc, keep):
    lib, dev, rows = _lib.load(), logits.device, desc.rows
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    top_logp = torch.empty(rows, desc.top, dtype=torch.float32, device=dev) if desc.top else None
    top_idx = torch.empty(rows, desc.top, dtype=torch.int64, device=dev) if desc.top else None
    stats = torch.empty(rows, 3, dtype=torch.float32, device=dev) if keep else None
    nbytes = lib.ckan_log_probs_workspace_bytes(desc)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _on(dev):
        _lib.check(lib.ckan_log_probs(desc, logits.data_ptr(), targets.data_ptr(), logp.data_ptr(), entropy.data_ptr(),
                                      _lib.ptr(top_logp), _lib.ptr(top_idx), _lib.ptr(stats), _lib.ptr(ws), nbytes,
                                      _stream(dev)))
    return logp, entropy, top_logp, top_idx, stats


class LogProbsFunction(torch.autograd.Function):
    """logp and entropy, differentiable in the logits; the likeliest classes go by the side."""

    @staticmethod
    def forward(ctx, logits, targets, desc, out: list):
        logp, entropy, top_logp, top_idx, stats = _log_probs_forward(logits, targets, desc, keep=True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, targets, stats)
        ctx.desc = desc
        out += [top_logp, top_idx]
        return logp, entropy

    @staticmethod
    def backward(ctx, dlogp, dentropy):
        _once("log_probs")
        if dlogp is None and dentropy is None:
            return None, None, None, None
        logits, targets, stats = ctx.saved_tensors
        logits, targets, stats = _rows(logits, ctx.desc.classes), _dense(targets), _dense(stats)
        desc = _pitched(ctx.desc, logits_ld=logits.stride(0))
        dlogp, dentropy = (g if g is None or (g.dtype == torch.float32 and g.is_contiguous())
                           else g.to(torch.float32).contiguous() for g in (dlogp, dentropy))
        dl = _like(logits)
        _lib.check(_lib.load().ckan_log_probs_backward(desc, logits.data_ptr(), targets.data_ptr(), stats.data_ptr(),
                                                       _lib.ptr(dlogp), _lib.ptr(dentropy), dl.data_ptr(),
                                                       _stream(dl.device)))
        return dl, None, None, None


def log_probs(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0) -> LogProbs:
    """Log probabilities of given classes under softmax(logits): (logp, entropy, top_logp,
    top_indices), the first two fp32 of ``targets``' shape, the last two [..., top] or None.

    ``logits`` [..., classes] fp32 or bf16, ``targets`` [...] int64.  A target outside [0,
    classes) is none: logp 0, no gradient.  ``entropy`` is the row's, in nats.  ``top`` (up to 64)
    asks for the likeliest classes in falling order, equal logits by the lower index.  A class
    whose logit is -inf has no probability and is not listed (index -1 and -inf fill up); a
    row of such classes only has logp -inf, entropy 0 and no gradient.  NaN or +inf makes a row's
    numbers NaN.

    -logp.mean() is the cross entropy.  Differentiable once in the logits through logp and
    entropy."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError(f"logits must be [..., classes], got {tuple(logits.shape)}")
    if targets.shape != logits.shape[:-1]:
        raise RuntimeError(f"targets must be {tuple(logits.shape[:-1])}, got {tuple(targets.shape)}")
    if targets.dtype != torch.int64:
        raise RuntimeError(f"targets must be int64, got {targets.dtype}")
    shape, classes = targets.shape, logits.shape[-1]
    if classes > 1 << 30 or not 0 <= top <= 64:  # the descriptor's 32 bits would take others for these
        raise RuntimeError(f"log_probs takes up to 2^30 classes and top from 0 to 64, got {classes} and {top}")
    _lib.refuse_tangents("log_probs", logits)
    _check("logits", logits.device, logits)
    if targets.device != logits.device:
        raise RuntimeError(f"targets are on {targets.device}, logits on {logits.device}: one device is needed")
    logits = _rows(logits, classes)
    if len(shape) != 1 or not targets.is_contiguous():
        targets = targets.reshape(-1).contiguous()
    desc = _lib.CkanLogProbsDesc(logits.shape[0], logits.stride(0), classes, int(top), _DTYPES[logits.dtype])
    if torch.is_grad_enabled() and logits.requires_grad:
        out: list = []
        got = (*LogProbsFunction.apply(logits, targets, desc, out), *out)
    else:
        got = _log_probs_forward(logits, targets, desc, keep=False)[:4]
    if len(shape) == 1:
        return LogProbs(*got)
    return LogProbs(*(None if t is None else t.view(shape + t.shape[1:]) for t in got))


# ---- a stack of residual blocks ----------------------------------------------------------

class ResidualKAN(nn.Module):
    """KAN layers of one width as a stack of residual blocks:

        h = norm_0(x);  for each layer i:  x = x + scale gate_i drop(post_i(layer_i(h))),  h = norm_{i+1}(x)

    ``layers`` map [rows, dim] to [rows, dim] (ChebyKANLayer, MixtureKANLayer, ...); their tanh saturates
    where a deep stack's values grow, which the norms before them keep in place.  ``row_norm`` opens the
    stack, one ``residual_norm`` closes each block together with the next one's norm.  ``norm``: 'rms', or
    'layer' with biases; ``post``: a norm after each layer too; ``gate``: the initial value of a
    learned gate [dim] a block, None for none.  The last norm's h is the result with
    ``final_norm``, else x.

    ``dropout`` is drawn in training mode from the buffer ``dropout_state`` (seed, offset): a forward uses one
    call a layer and moves the offset on, on the device, so that replays of a captured step draw anew. A forward
    made again for its backward (activation checkpointing) would draw other masks: checkpoint the layers, not the
    stack. Ranks of a data-parallel run draw different masks only if their buffers are not broadcast."""

    def __init__(self, layers: Iterable[nn.Module], dim: int, *, norm: str = "rms", post: bool = True,
                 gate: Optional[float] = 0.1, scale: float = 1.0, dropout: float = 0.0, eps: float = 1e-6,
                 final_norm: bool = True):
        super().__init__()
        if norm not in _NORMS:
            raise ValueError(f"norm must be one of {sorted(_NORMS)}, got {norm!r}")
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"the dropout probability must lie in [0, 1], got {dropout}")
        self.layers = nn.ModuleList(layers)
        for i, layer in enumerate(self.layers):
            width = getattr(layer, "input_dim", dim), getattr(layer, "output_dim", dim)
            if width != (dim, dim):
                raise ValueError(f"layer {i} maps {width[0]} to {width[1]} values, the stack has {dim}")
        self.dim, self.norm, self.scale, self.dropout, self.eps = dim, norm, scale, dropout, eps
        n = len(self.layers)
        norms = n + 1 if final_norm else n

        def vectors(count, value):
            return nn.ParameterList([nn.Parameter(torch.full((dim,), float(value))) for _ in range(count)])

        self.pre_weight = vectors(norms, 1)
        self.pre_bias = vectors(norms if norm == "layer" else 0, 0)
        self.post_weight = vectors(n if post else 0, 1)
        self.post_bias = vectors(n if post and norm == "layer" else 0, 0)
        self.gate = vectors(0 if gate is None else n, gate or 0)
        self.register_buffer("dropout_state", torch.tensor([int(torch.randint(0, 2 ** 62, ())), 0]))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        def at(vectors, i):
            return vectors[i] if i < len(vectors) else None

        x = x.reshape(-1, self.dim)
        n, drop = len(self.layers), self.dropout if self.training else 0.0
        if not len(self.pre_weight):
            return x
        h = row_norm(x, self.pre_weight[0], at(self.pre_bias, 0), norm=self.norm, eps=self.eps)
        for i, layer in enumerate(self.layers):
            got = residual_norm(x, layer(h), norm=self.norm, eps=self.eps, post_weight=at(self.post_weight, i),
                                post_bias=at(self.post_bias, i), gate=at(self.gate, i), scale=self.scale, dropout=drop,
                                dropout_state=self.dropout_state if drop else None, dropout_call=i,
                                next_weight=at(self.pre_weight, i + 1), next_bias=at(self.pre_bias, i + 1))
            x, h = got if isinstance(got, tuple) else (got, got)
        if drop:
            with torch.no_grad():
                self.dropout_state[1:].add_(n)
        return h

    def extra_repr(self) -> str:
        return f"dim={self.dim}, norm={self.norm}, scale={self.scale}, dropout={self.dropout}"
