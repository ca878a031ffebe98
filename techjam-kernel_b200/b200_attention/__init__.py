"""B200 (sm_100a) fused attention forward behind the reference's attention API.

- ``b200_fused_attention``: functional operator (reference: triton_fused_attention)
- ``attention_dispatch``: planner (reference: model/attention_dispatch.py)
- ``B200FusedSelfAttention``: module adapter (reference: TritonFusedSelfAttention)
- ``b200_linear``: the block's linear layers with their elementwise epilogues
  (bias, exact GELU, residual add, padded-row zeroing) fused into one kernel
- ``b200_attention_softmax`` / ``B200SoftmaxSelfAttention``: the row softmax
  over materialised scores (reference: triton_attention_softmax /
  TritonSelfAttention, also exported under those names)
- ``b200_tree_attention``, ``b200_cache_*`` / ``PagedKVCache``: attention for drafted
  tokens (or one token) over a paged key/value cache of 16 or 32 bits or of 4, and the
  cache's page operations
- ``b200_verify_drafts``: which drafted tokens the target keeps, and the next one
"""

from .fused_attention import (DeviceError, b200_fused_attention, check_device_errors,  # noqa: F401
                              clear_device_errors, read_device_errors)
from .linear import b200_linear  # noqa: F401
from .paged_cache import (PagedKVCache, b200_cache_accept, b200_cache_append,  # noqa: F401
                          b200_cache_compact, b200_cache_fork, b200_cache_free,
                          b200_cache_read, b200_cache_reserve, b200_tree_attention)
from .softmax import (B200SoftmaxSelfAttention, TritonSelfAttention,  # noqa: F401
                      b200_attention_softmax, triton_attention_softmax)
from .verify import b200_verify_drafts  # noqa: F401
