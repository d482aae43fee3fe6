"""vit_amd: MI355X-native (gfx950, HIP) engine for the VTCNN train / predict hot path.

The compute lives in libvtcnn_hip.so (hand-written HIP kernels behind the C ABI declared in
include/vtcnn_hip.h); this package is the thin host-side mirror of the reference's
Model / Trainer / DataLoader interface on top of it.  There is no CPU fallback: importing
`vit_amd.engine` without the built library raises.
"""
from . import _lib  # noqa: F401
from .engine import VTCNN, Dims, DataLoader, Trainer, SelfAttention, load_dataset  # noqa: F401

from .ops import block_norms_bwd, block_norms_fwd, distill_bwd, distill_fwd, distill_fwd_bwd  # noqa: F401
from .ops import relpos_attention_bwd, relpos_attention_fwd, relpos_buckets  # noqa: F401

__all__ = ["VTCNN", "Dims", "DataLoader", "Trainer", "SelfAttention", "load_dataset",
           "distill_fwd", "distill_bwd", "distill_fwd_bwd", "block_norms_fwd", "block_norms_bwd",
           "relpos_buckets", "relpos_attention_fwd", "relpos_attention_bwd"]
