"""kan_b200 — the ChebyKAN layer hot path of 0xEodum/KAN on NVIDIA B200 (sm_100a).

Public surface: ``ChebyKANLayer`` (drop-in for kan.layers.chebykan.ChebyKANLayer),
``install_into_reference`` (swap it into the reference's layer registry), ``JacobiKANLayer`` and
``HermiteKANLayer`` (the reference's other recurrence-based layers on the same fp32 kernels), the
functional ``ops``, the kernel-backed ``optim.SGD`` / ``optim.Adam`` / ``optim.Muon``, the
8-bit inference layer (``quantize_int8``) and the data-parallel helpers in ``dp``.  Everything computes in hand-written CUDA
behind the C ABI of ``include/chebykan_b200.h``; there is no CPU fallback.
"""
from .layer import ChebyKANLayer, ChebyshevBasis, KANLayer, chebykan_apply, install_into_reference
from .poly import HermiteBasis, HermiteKANLayer, JacobiBasis, JacobiKANLayer
from .stack import FusedChebyKANStack, fuse_layernorm
from .int8 import Int8ChebyKANLayer, quantize_int8
from .loss import MSELoss, mse_loss
from . import ops, optim, dp, workloads, graph, poly, small

__all__ = ["MSELoss", "mse_loss", "FusedChebyKANStack", "fuse_layernorm", "Int8ChebyKANLayer", "quantize_int8", "ChebyKANLayer", "ChebyshevBasis", "KANLayer",
           "JacobiKANLayer", "HermiteKANLayer", "JacobiBasis", "HermiteBasis", "chebykan_apply", "install_into_reference",
           "ops", "optim", "dp", "workloads", "graph", "poly", "small"]
__version__ = "0.1.0"
