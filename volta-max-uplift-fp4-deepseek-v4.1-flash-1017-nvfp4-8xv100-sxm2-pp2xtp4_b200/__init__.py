"""B200-native (sm_100a) routed-expert MoE layer: the drop-in for the reference
build's routed-expert FusedMoE quant-method plugin.

Import name: ``b200moe`` (see ``__graft_entry__.load_package``).  Modules:
``moe`` (the plugin: B200NativeMoe, B200NativeMoEMethod), ``packing`` (device
packing and the reference route plan), ``tiers`` (tier map -> slot maps,
expert-parallel placement), ``ep`` (expert-parallel dispatch / combine),
``permute`` and ``fp8`` (stateless operators: tokens sorted by expert and back,
E4M3 products with a scale per block of 128, their quantizers and gradients),
``experts`` (FP8 experts built of them), ``_lib`` (ctypes binding of
libb200moe.so, and the operators' torch binding), ``build`` (nvcc and g++ build).
"""

from . import _lib, tiers  # noqa: F401

__all__ = ["_lib", "tiers"]
