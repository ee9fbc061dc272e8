"""B200 (sm_100a) product-key memory layer of KumarDev7/model.

``MemoryPool`` / ``MemoryLayer`` mirror the reference's Flax module and its
caller block, ``MemoryPoolLM`` / ``Generator`` the language model and its
decoder around them; ``layer_norm``, ``linear_cross_entropy``, their
gradients and ``orthogonalize`` are the operators of a training step around
them.  Every step runs
in the CUDA library ``libmemlayer.so`` behind the C ABI of
``include/memlayer.h``.
"""

from .memory import MemoryLayer, MemoryPool  # noqa: F401
from .model import Generator, MemoryPoolLM, ModelConfig  # noqa: F401
from .train_ops import (layer_norm, layer_norm_backward, linear_cross_entropy,  # noqa: F401
                        linear_cross_entropy_backward, orthogonalize)

__all__ = ["MemoryPool", "MemoryLayer", "MemoryPoolLM", "ModelConfig", "Generator", "layer_norm",
           "layer_norm_backward", "linear_cross_entropy", "linear_cross_entropy_backward", "orthogonalize"]
