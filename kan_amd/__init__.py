"""kan_amd: the ChebyKAN layer hot path of 0xEodum/KAN, MI355X (gfx950) native.

Public surface (mirrors the reference's names for this path):
    ChebyKANLayer, JacobiKANLayer, HermiteKANLayer, KANLayer, KANSequential,
    get_layer, LAYER_REGISTRY
    ChebyshevBasis, JacobiBasis, HermiteBasis, BasisFunction, get_basis, BASIS_REGISTRY
    optim.SGD, optim.Adam (fused HIP steps), optim.Muon (orthogonalised momentum)
    MixtureKANLayer (rows routed to ChebyKAN experts)
    ResidualKAN (layers as residual blocks: norms, gate, dropout and sum in one launch)
    ResidentExecutor (whole training steps of a layer stack, resident on one GPU)
    functional.chebykan (autograd op), functional.route, functional.kan_experts,
    functional.kan_mixture, functional.orthogonalize, functional.row_norm,
    functional.residual_norm, functional.dropout, functional.log_probs

All compute runs in the in-tree HIP library ``libckan_gfx950.so`` (C-ABI in
include/chebykan.h); there is no CPU fallback.
"""
from .basis import (BASIS_REGISTRY, BasisFunction, ChebyshevBasis, HermiteBasis, JacobiBasis,
                    get_basis)
from .layers import (LAYER_REGISTRY, ChebyKANLayer, HermiteKANLayer, JacobiKANLayer, KANLayer,
                     KANSequential, get_layer)
from .mixture import MixtureKANLayer
from .block import ResidualKAN
from . import functional, optim
from .executor import ResidentExecutor

__version__ = "0.1.0"

__all__ = [
    "ChebyKANLayer", "JacobiKANLayer", "HermiteKANLayer", "KANLayer", "KANSequential",
    "MixtureKANLayer", "ResidualKAN", "get_layer", "LAYER_REGISTRY",
    "ChebyshevBasis", "JacobiBasis", "HermiteBasis", "BasisFunction", "get_basis",
    "BASIS_REGISTRY",
    "functional", "optim", "ResidentExecutor", "__version__",
]
