"""fermix_amd: batched fp32 slogdet / slogpf / det / pf on AMD Instinct MI355X
(gfx950) with hand-written HIP kernels behind a C ABI (include/fermix.h), keeping the
Python interface of ChenAo-Phys/fermix; and the operators of the network in front of the
determinants (attention with a relative position bias, its one-token step, residual norms)."""

from .api import FermixDeviceError, FermixFallbackWarning, FermixTuneWarning, det, pf, slogdet, slogpf
from .network import attention, attention_step, distance_buckets, relative_bias, residual_norm

__all__ = [
    "slogdet",
    "slogpf",
    "det",
    "pf",
    "distance_buckets",
    "relative_bias",
    "attention",
    "attention_step",
    "residual_norm",
    "FermixFallbackWarning",
    "FermixDeviceError",
    "FermixTuneWarning",
]
