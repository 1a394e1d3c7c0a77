"""omarchy-mac-torch's convolution hot path on AMD Instinct MI355X (gfx950), as hand-written HIP.

    import omarchy_mac_torch                 # registers the "omarchy_mac_torch" device
    model = model.to("omarchy_mac_torch")
    omarchy_mac_torch.accelerate(model)      # optional: fused conv/BN/ReLU/pool stacks
    torch.compile(model, backend="omarchy_mac_torch")

The same API as the reference package (omarchy_mac_torch/__init__.py): DEVICE, FALLBACKS, accelerate,
FusedSequential, synchronize, empty_cache, memory_allocated, memory_reserved, set_queue_depth, validate_kernels.
`hip_ops` exposes the tensor-level entry points over libomt_hip.so's C ABI directly; `graphs` replays captured steps
as HIP graphs; `ffn` is the feed-forward sublayer of a language model (residual RMS norm, gated block with 8-bit
checkpoints, 8-bit serving); `lm` both ends of its training step (embedding, preference and policy losses on logits), with
`optim.AdamW` (states in 8 bits or 32) at the end.
"""

from omarchy_mac_torch import _lib  # noqa: F401  (libomt_hip.so; ImportError when it is not built)
from omarchy_mac_torch import hip_ops  # noqa: F401
from omarchy_mac_torch import native as _native  # noqa: F401  (registers the device)
from omarchy_mac_torch import compile as _compile  # noqa: F401  (torch.compile backend "omarchy_mac_torch")
from omarchy_mac_torch import optim  # noqa: F401  (fused SGD / Adam / AdamW by default on the device; AdamW in 8 bits)
from omarchy_mac_torch import graphs  # noqa: F401  (captured steps replayed as HIP graphs)
from omarchy_mac_torch import ffn  # noqa: F401  (the feed-forward sublayer: norm, gated block, 8-bit serving)
from omarchy_mac_torch import lm  # noqa: F401  (embedding, losses on logits)
from omarchy_mac_torch.native import (DEVICE, FALLBACKS, empty_cache, memory_allocated, memory_reserved,
                                      set_queue_depth, synchronize, validate_kernels)
from omarchy_mac_torch.stacks import FusedSequential, accelerate

__version__ = "0.2.0"
__all__ = ["DEVICE", "FALLBACKS", "FusedSequential", "accelerate", "empty_cache", "ffn", "graphs", "hip_ops", "lm", "memory_allocated",
           "memory_reserved", "optim", "set_queue_depth", "synchronize", "validate_kernels"]
