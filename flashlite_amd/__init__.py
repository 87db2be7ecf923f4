"""flashlite_amd -- FlashAttention-2 forward for AMD Instinct MI355X (gfx950).

Drop-in for the ``flash_attn_wmma`` extension of thebigblender/FlashLite:

    from flashlite_amd import forward_flash2, forward_naive
    out = forward_flash2(q, k, v, sm_scale=0.0, is_causal=False, out=None)

(``import flash_attn_wmma`` works too, from the repository root.)  The
functions are the torch binding built from ``csrc/flash_attn.cpp``; the
kernels are hand-written HIP for gfx950 in ``csrc/*.hip`` behind the C ABI
declared in ``include/flashlite_attn.h``.  There is no fallback: if the
extension is not built, importing raises ImportError.
"""

from __future__ import annotations

import os

import torch  # noqa: F401  (loads libtorch/libc10 before the extension)

_PKG_DIR = os.path.dirname(os.path.abspath(__file__))

try:
    from . import flash_attn_wmma as _ext
except ImportError as exc:  # pragma: no cover - exercised only without a build
    raise ImportError(
        "flashlite_amd: the HIP extension is not built. Run `python flashlite_amd/build.py` "
        "(or `python -c 'import __graft_entry__ as g; g.build()'`) from the repository root."
    ) from exc

forward_flash2 = _ext.forward_flash2
forward_naive = _ext.forward_naive
# Beyond the reference surface: strided [B, H, N, 64] views (a [B, N, H, 64]
# tensor passes as x.transpose(1, 2)), N_k != N_q with the causal diagonal
# aligned bottom-right, and the fp32 log-sum-exp with return_lse=True.
# num_splits / workspace select split-KV for few query rows over many keys.
forward_flash2_ex = _ext.forward_flash2_ex
splitkv_workspace_bytes = _ext.splitkv_workspace_bytes

# Serving over a paged cache: a step's blocks and slots, its drafts' ancestors,
# rotary positions (and their gradient) with the cache's writes, attention for
# trees of drafted tokens or one token.
plan_cache = _ext.plan_cache
plan_tree = _ext.plan_tree
forward_rotary = _ext.forward_rotary
backward_rotary = _ext.backward_rotary
rotary_to_cache = _ext.rotary_to_cache
forward_tree = _ext.forward_tree
tree_workspace_bytes = _ext.tree_workspace_bytes

# Norms of q and k for each head with the rotary positions (of one or several
# axes) in the same pass, their gradients, and the form that stores k and v.
forward_norm_rotary = _ext.forward_norm_rotary
backward_norm_rotary = _ext.backward_norm_rotary
norm_rotary_to_cache = _ext.norm_rotary_to_cache
norm_rotary_workspace_bytes = _ext.norm_rotary_workspace_bytes

# Attention over packed sequences of different lengths, and its gradients.
forward_packed = _ext.forward_packed
backward_packed = _ext.backward_packed
packed_workspace_bytes = _ext.packed_workspace_bytes

from .rotary import rotary_axes, rotary_frequencies  # noqa: E402

__all__ = ["forward_flash2", "forward_naive", "forward_flash2_ex", "splitkv_workspace_bytes",
           "plan_cache", "plan_tree", "forward_rotary", "backward_rotary", "rotary_to_cache",
           "rotary_frequencies", "forward_tree", "tree_workspace_bytes", "forward_norm_rotary",
           "backward_norm_rotary", "norm_rotary_to_cache", "norm_rotary_workspace_bytes",
           "rotary_axes", "forward_packed", "backward_packed", "packed_workspace_bytes"]
