"""MI355X (gfx950) DeepSeek Sparse Attention path: lightning indexer -> top-k -> sparse MLA.

Hand-written HIP kernels behind the C ABI of ``include/dsa_mi355x.h``; this
package is the host-side mirror of the reference's Python operator interface
(examples/lightning_indexer, examples/topk_selector,
examples/sparse_flash_attention and examples/deepseek_v4 of tilelang-ascend,
including the V4 ``sparse_flash_mla`` operator).  Around it, the dense attention
layer's operators: the 8-bit projection behind ``act_quant``, head norms with
rotation into a paged cache, and the attention of new tokens over that cache; and
a decoding step over trees of drafted tokens: the pages' plan, the attention of the
nodes, their acceptance and the order of the cache rows.
"""
from ._lib import DSAError, library_path, load_library, load_torch_ops
from .act_quant import act_quant
from .lightning_indexer import indexer, indexer_logits, lightning_indexer
from .norm_rope import qk_norm_rope, qk_norm_rope_paged
from .paged_gqa import paged_gqa_fwd
from .paged_plan import PagedPlan, paged_free, paged_plan
from .paged_tree import paged_commit, paged_tree_fwd, tree_accept
from .quant_matmul import quant_matmul
from .sparse_flash_mla import sparse_attn, sparse_attn_kernel, sparse_flash_mla
from .sparse_mla import sparse_attention_fwd, sparse_attn_tilelang, sparse_gqa_fwd, sparse_mla_fwd
from .topk_selector import simple_topk_selector, topk_selector

__all__ = [
    "DSAError",
    "PagedPlan",
    "act_quant",
    "indexer",
    "indexer_logits",
    "library_path",
    "lightning_indexer",
    "load_library",
    "load_torch_ops",
    "paged_commit",
    "paged_free",
    "paged_gqa_fwd",
    "paged_plan",
    "paged_tree_fwd",
    "qk_norm_rope",
    "qk_norm_rope_paged",
    "quant_matmul",
    "simple_topk_selector",
    "sparse_attention_fwd",
    "sparse_attn",
    "sparse_attn_kernel",
    "sparse_attn_tilelang",
    "sparse_flash_mla",
    "sparse_gqa_fwd",
    "sparse_mla_fwd",
    "topk_selector",
    "tree_accept",
]
