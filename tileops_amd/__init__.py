"""MI355X (gfx950) paged GQA decode attention behind the TileOPs operator contract.

Public surface: the attention ops, the ops of a serving step around the cache, the backend seam, the manifest loader.  The HIP library is opened lazily on
the first kernel build; importing this package touches no device.
"""

from .backend import (  # noqa: F401
    BUILTIN, AmbiguousTargetError, BackendError, OpNotAvailableError, TensorSpec, UnknownTargetError,
    default_target, load_failures, register_detector, register_kernel_builder, registered_targets, set_default_target,
)
from .ops import (  # noqa: F401
    GroupedQueryAttentionDecodeWithKVCacheFwdOp,
    GroupedQueryAttentionDecodePagedWithKVCacheFwdOp,
    GroupedQueryAttentionMultiTokenDecodePagedWithKVCacheFwdOp,
    GroupedQueryAttentionPrefillPagedWithKVCacheFwdOp,
)
from .serving_ops import (  # noqa: F401
    GroupedQueryAttentionDecodePagedWithFP4KVCacheFwdOp,
    PagedFP4KVCacheGatherFwdOp,
    PagedKVCacheAllocFwdOp,
    PagedKVCacheReleaseFwdOp,
    QKNormRopePagedKVAppendFwdOp,
)

__all__ = [
    "GroupedQueryAttentionDecodePagedWithFP4KVCacheFwdOp",
    "PagedFP4KVCacheGatherFwdOp",
    "PagedKVCacheAllocFwdOp",
    "PagedKVCacheReleaseFwdOp",
    "QKNormRopePagedKVAppendFwdOp",
    "GroupedQueryAttentionDecodeWithKVCacheFwdOp",
    "GroupedQueryAttentionDecodePagedWithKVCacheFwdOp",
    "GroupedQueryAttentionMultiTokenDecodePagedWithKVCacheFwdOp",
    "GroupedQueryAttentionPrefillPagedWithKVCacheFwdOp",
]
__version__ = "0.1.0"
