"""MI355X-native flash attention for the CudaTransformer FlashAttentionLayer path.

Layers of this package
  * ``libctattn.so``   -- HIP kernels for gfx950 behind a C-ABI (``include/ctattn.h``).
  * ``cuda_transformer`` -- C++ host module (pybind11) mirroring the reference's
    ``Tensor`` / ``FlashAttentionLayer`` API on top of that C-ABI.
  * ``packed``         -- attention on packed sequences of different lengths.
  * ``paged``          -- a paged key / value cache and attention of requests that share a prompt.
  * ``sampling``       -- next tokens by temperature, top-k, top-p and min-p.
  * ``embedding``      -- scaled token lookup with a reproducible gradient.
  * ``muon``           -- Newton-Schulz orthogonalisation and the Muon step.
  * ``_capi``          -- ctypes binding of the same C-ABI over torch device tensors
    (torch is plumbing: memory and streams).

torch is imported first so every native library here binds to the HIP runtime torch
loaded (one runtime per process).
"""
import torch  # noqa: F401  (must precede loading the native libraries)

from ._capi import (  # noqa: E402
    BF16,
    F32,
    POLICY_AUTO,
    POLICY_DETERMINISTIC,
    POLICY_GENERIC,
    FlashAttentionFunction,
    bwd_workspace_bytes,
    flash_attention,
    flash_attn_bwd,
    flash_attn_fwd,
    last_error,
    out_proj_bwd,
    out_proj_fwd,
    qkv_proj_bwd,
    qkv_proj_fwd,
    set_policy,
    sgd_update,
)
from .embedding import (  # noqa: E402
    EmbeddingLookupFunction,
    embedding,
    embedding_grad,
    embedding_grad_workspace_bytes,
    embedding_lookup,
)
from .muon import Muon, muon_update, newton_schulz, newton_schulz_workspace_bytes  # noqa: E402
from .packed import (  # noqa: E402
    PackedAttentionFunction,
    PackedPlan,
    flash_attention_packed,
    flash_attn_packed_bwd,
    flash_attn_packed_fwd,
    packed_bwd_workspace_bytes,
    packed_plan,
)
from .paged import (  # noqa: E402
    cache_write,
    flash_attn_shared_prefix,
    page_pool,
    page_release,
    page_reserve,
    shared_prefix_workspace_bytes,
)
from .sampling import sample_tokens, sample_workspace_bytes  # noqa: E402

__all__ = [
    "BF16",
    "F32",
    "POLICY_AUTO",
    "POLICY_DETERMINISTIC",
    "POLICY_GENERIC",
    "EmbeddingLookupFunction",
    "FlashAttentionFunction",
    "Muon",
    "PackedAttentionFunction",
    "PackedPlan",
    "bwd_workspace_bytes",
    "cache_write",
    "embedding",
    "embedding_grad",
    "embedding_grad_workspace_bytes",
    "embedding_lookup",
    "flash_attention",
    "flash_attention_packed",
    "flash_attn_bwd",
    "flash_attn_fwd",
    "flash_attn_packed_bwd",
    "flash_attn_packed_fwd",
    "flash_attn_shared_prefix",
    "muon_update",
    "newton_schulz",
    "newton_schulz_workspace_bytes",
    "packed_bwd_workspace_bytes",
    "packed_plan",
    "page_pool",
    "page_release",
    "page_reserve",
    "sample_tokens",
    "sample_workspace_bytes",
    "shared_prefix_workspace_bytes",
    "out_proj_bwd",
    "out_proj_fwd",
    "qkv_proj_bwd",
    "qkv_proj_fwd",
    "sgd_update",
    "last_error",
    "set_policy",
]
