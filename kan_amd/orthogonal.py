"""Newton-Schulz orthogonalisation over the C-ABI, and the Muon step built on it.

Device memory and streams come from torch; all compute is the HIP library's.
Tensors on the CPU are rejected: there is no CPU path.
"""
from __future__ import annotations

import math
from typing import Tuple

import torch

from . import _lib

# The quintic's coefficients: singular values in (0, 1] go to about [0.7, 1.2] in five
# steps, small ones growing by 3.4445 a step.
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_DTYPES = {torch.float32: _lib.CKAN_DTYPE_F32, torch.bfloat16: _lib.CKAN_DTYPE_BF16}


def _workspace(desc, device: torch.device):
    lib = _lib.load()
    nbytes = lib.ckan_orthogonalize_workspace_bytes(desc)
    # from torch's allocator on the current stream: reused by it in stream order
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device), nbytes


def orthogonalize(g: torch.Tensor, steps: int = 5,
                  coefficients: Tuple[float, float, float] = NS_COEFFICIENTS,
                  eps: float = 1e-7) -> torch.Tensor:
    """The matrices ``g`` [..., rows, cols] (fp32 or bf16) brought near U V^T of their
    singular value decompositions: X = g / (|g|_F + eps), then ``steps`` times
    X = a X + (b A + c A^2) X with A = X X^T (X^T X where rows > cols).

    Sums are in fp32 over operands of 22 bits, so fp32 matrices come out as from
    fp32 products (with a side of at most 64 in fp64); bf16 ones carry an error of at
    most 2^-9 besides their rounding.  The result has g's dtype.  Not differentiable."""
    if g.dim() < 2:
        raise RuntimeError(f"g must be [..., rows, cols], got {tuple(g.shape)}")
    _lib.refuse_tangents("orthogonalize", g)
    if not g.is_cuda:
        raise RuntimeError("kan_amd's orthogonalisation runs only on a ROCm device (MI355X); "
                           f"got a tensor on {g.device}")
    if g.dtype not in _DTYPES:
        raise RuntimeError(f"g must be float32 or bfloat16, got {g.dtype}")
    g = g.detach()
    rows, cols = g.shape[-2:]
    if g.numel() == 0:
        return torch.empty_like(g)
    x = g.reshape(-1, rows, cols)
    if x.is_contiguous() or not x.transpose(1, 2).is_contiguous():
        x, strides = x.contiguous(), (rows * cols, cols, 1)
    else:
        strides = (rows * cols, 1, rows)
    # not x.stride(): a dimension of one may have any
    out = torch.empty_strided(x.shape, strides, dtype=x.dtype, device=x.device)
    a, b, c = (float(v) for v in coefficients)
    desc = _lib.CkanOrthoDesc(*strides, 0, x.shape[0], rows, cols, 1, int(steps), _DTYPES[g.dtype], a, b, c, float(eps))
    with torch.cuda.device(x.device):
        ws, nbytes = _workspace(desc, x.device)
        _lib.check(_lib.load().ckan_orthogonalize(desc, x.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                                  nbytes, _lib.stream_ptr(x.device)))
    return out.reshape(g.shape)


def matrix_shape(shape) -> Tuple[int, int, int, int]:
    """(batch, rows, cols, inner) of a parameter as matrices: a [rows, cols] weight;
    a ChebyKAN layer's [in, out, D] coefficients as [out, in D], the matrix that
    acts on the basis values; experts' [E, in, out, D] as E of those."""
    if len(shape) == 2:
        return 1, shape[0], shape[1], 1
    if len(shape) == 3:
        return 1, shape[1], shape[0] * shape[2], shape[2]
    if len(shape) == 4:
        return shape[0], shape[2], shape[1] * shape[3], shape[3]
    raise ValueError("Muon takes matrices: [rows, cols] weights, [in, out, degree+1] coefficients or "
                     f"[experts, in, out, degree+1] ones, got {tuple(shape)}")


@torch.no_grad()
def muon_step_(p: torch.Tensor, g: torch.Tensor, buf: torch.Tensor, *, lr: float,
               momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
               steps: int = 5, coefficients: Tuple[float, float, float] = NS_COEFFICIENTS,
               eps: float = 1e-7) -> None:
    """One Muon step in place on parameters ``p`` with gradient ``g`` and momentum ``buf``:

        buf = momentum buf + (1 - momentum) g
        u = (1 - momentum) g + momentum buf  (buf without ``nesterov``)
        p = (1 - lr weight_decay) p - lr sqrt(max(1, rows / cols)) orthogonalize(u)

    with p, g and buf of one shape that ``matrix_shape`` takes as matrices, fp32 and
    contiguous on a ROCm device."""
    batch, rows, cols, inner = matrix_shape(p.shape)
    for t, name in ((p, "p"), (g, "g"), (buf, "buf")):
        if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
            raise RuntimeError(f"muon_step_: {name} must be fp32, contiguous and on a ROCm device")
        if t.shape != p.shape or t.device != p.device:
            raise RuntimeError(f"muon_step_: {name} is {tuple(t.shape)} on {t.device}, "
                               f"p {tuple(p.shape)} on {p.device}")
    if p.numel() == 0:
        return
    a, b, c = (float(v) for v in coefficients)
    if inner == 1:
        strides = (rows * cols, cols, 1, 0)
    else:  # [.., in, out, D]: row o, column (i, d)
        strides = (rows * cols, inner, rows * inner, 1)
    if len(p.shape) > 2 and inner == 1:  # degree 0: [.., in, out, 1]
        strides = (rows * cols, 1, rows, 0)
    desc = _lib.CkanOrthoDesc(*strides, batch, rows, cols, inner, int(steps), _lib.CKAN_DTYPE_F32, a, b, c,
                              float(eps))
    with torch.cuda.device(p.device):
        ws, nbytes = _workspace(desc, p.device)
        _lib.check(_lib.load().ckan_muon_step(
            desc, p.data_ptr(), g.data_ptr(), buf.data_ptr(), float(lr), float(momentum),
            float(weight_decay), math.sqrt(max(1.0, rows / cols)), int(bool(nesterov)), ws.data_ptr(), nbytes,
            _lib.stream_ptr(p.device)))
    for t in (p, buf):  # written through their pointers
        torch.autograd.graph.increment_version(t)
