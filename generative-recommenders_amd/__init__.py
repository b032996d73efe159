"""MI355X-native HSTU jagged attention (forward): ``hstu_mha`` and ``delta_hstu_mha``, the jagged
concatenation / split that feeds the cached form (``concat_2D_jagged``, ``split_2D_jagged``, ``write_kv_tail``),
the dense steps either side of the attention (``hstu_compute_uqvk``, ``hstu_compute_output``,
``hstu_preprocess_and_attention``), rotated positions with a paged K/V cache in 4 bits (``qk_norm_rope``, ``append_paged_kv``,
``read_paged_kv``, ``delta_hstu_mha_paged``), and a gated recurrence in the attention's place with what stands between two layers
(``gated_recurrence``, ``gated_recurrence_step``, ``gated_residual_norm``).

Drop-in for ``generative_recommenders.ops.hstu_attention`` of the reference, backed by
hand-written gfx950 HIP kernels behind a C ABI (``csrc/``, ``include/hstu_hip.h``).
The directory name contains a hyphen, so load it with ``importlib`` under the module name
``generative_recommenders_amd`` (``__graft_entry__.load_package()`` does exactly that).
"""

from .common import HammerKernel  # noqa: F401
from .ops.hstu_attention import delta_hstu_mha, hstu_mha  # noqa: F401
from .ops.hstu_compute import hstu_compute_output, hstu_compute_uqvk, hstu_preprocess_and_attention  # noqa: F401
from .ops.jagged_tensors import concat_2D_jagged, split_2D_jagged, write_kv_tail  # noqa: F401
from .ops.paged_cache import (  # noqa: F401
    PagedKVCache, allocate_paged_kv_cache, append_paged_kv, delta_hstu_mha_paged, make_rotary_table, qk_norm_rope, read_paged_kv,
)
from .ops.recurrent import gated_recurrence, gated_recurrence_step, gated_residual_norm  # noqa: F401
from .ops import native_op  # noqa: F401  (defines torch.ops.hstu.hstu_mha / hstu_mha_fwd on these kernels)

__all__ = [
    "HammerKernel", "hstu_mha", "delta_hstu_mha", "concat_2D_jagged", "split_2D_jagged", "write_kv_tail", "hstu_compute_uqvk",
    "hstu_compute_output", "hstu_preprocess_and_attention", "PagedKVCache", "allocate_paged_kv_cache", "append_paged_kv",
    "delta_hstu_mha_paged", "make_rotary_table", "qk_norm_rope", "read_paged_kv", "gated_recurrence", "gated_recurrence_step",
    "gated_residual_norm",
]
