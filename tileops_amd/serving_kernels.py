"""L1 host wrappers of the serving-step kernels: pages, append, 4-bit rows, attention over a 4-bit cache.

Each class states the calls that it serves (``applies`` / ``refusal``, like every kernel class of the package); ``forward`` is one
registered operator, which enqueues one library call on the current stream.  Nothing is read back.  The reference has no counterpart
of these.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Optional

import torch

from . import custom_ops as _custom_ops  # noqa: F401 - registers torch.ops.tileops_amd.*
from . import native
from .kernels import GFX950_ARCH, Kernel

__all__ = [
    "GQADecodePagedFP4Kernel", "PagedFP4KVCacheGatherKernel", "PagedKVCacheAllocKernel", "PagedKVCacheReleaseKernel",
    "QKNormRopePagedKVAppendKernel", "ServingCall",
]

FP4 = torch.float4_e2m1fn_x2
FP8 = torch.float8_e4m3fn
HEAD_DIMS = (64, 128, 256)


@dataclass(frozen=True)
class ServingCall:
    """Facts of one call that kernel selection filters on (``dim`` 0 where no rows are touched)."""

    dim: int = 0
    page_size: int = 0
    dtype: Optional[torch.dtype] = None
    arch: Optional[int] = None


class _ServingKernel(Kernel):
    supported_archs = [GFX950_ARCH]
    general = True

    def __init__(self, op: Any, *, device_index: Optional[int] = None) -> None:
        super().__init__(device_index=device_index)
        self.op = op
        self.init_config()

    @classmethod
    def applies(cls, call: ServingCall) -> bool:
        return call.dim == 0 or call.dim in HEAD_DIMS


class PagedKVCacheAllocKernel(_ServingKernel):
    """Pages, slots and positions of a step's new tokens."""

    def forward(self, cache_seqlens, block_table, free_pages, free_count, cu_seqlens_q, total_q):
        return torch.ops.tileops_amd.kv_alloc(cache_seqlens, block_table, free_pages, free_count, cu_seqlens_q, total_q, self.op.page_size)


class PagedKVCacheReleaseKernel(_ServingKernel):
    """Pages of finished sequences back onto the list."""

    def forward(self, finished, seqlens, block_table, free_pages, free_count):
        return torch.ops.tileops_amd.kv_release(finished, seqlens, block_table, free_pages, free_count, self.op.page_size)


class QKNormRopePagedKVAppendKernel(_ServingKernel):
    """Norm and rotation of query and key rows with the append of keys and values."""

    def forward(self, q, k, v, q_weight, k_weight, cos_table, sin_table, positions, slot_mapping, k_cache, v_cache, k_scale, v_scale):
        op = self.op
        code = {FP4: native.DT_FP4_E2M1, FP8: native.DT_FP8_E4M3FN}.get(op.cache_dtype)
        if code is None:
            code = native.dtype_code(q.dtype)
        return torch.ops.tileops_amd.qk_norm_rope_append(
            q, k, v, q_weight, k_weight, cos_table, sin_table, positions, slot_mapping, k_cache, v_cache, k_scale, v_scale,
            op.rotary_dim, op.interleaved, op.eps, op.page_size, code)


class PagedFP4KVCacheGatherKernel(_ServingKernel):
    """Rows of a 4-bit cache as 16-bit values."""

    def forward(self, k, v, k_scale, v_scale, slot_mapping):
        return torch.ops.tileops_amd.kv_gather_fp4(k, v, k_scale, v_scale, slot_mapping, self.op.dtype)


class GQADecodePagedFP4Kernel(_ServingKernel):
    """Paged GQA decode over a 4-bit cache (MFMA, K codes on the 4-bit matrix path)."""

    @classmethod
    def applies(cls, call: ServingCall) -> bool:
        return call.dim in HEAD_DIMS and call.page_size % 16 == 0 and call.dtype in (torch.float16, torch.bfloat16)

    def forward(self, q, k, v, k_scale, v_scale, real_seqlen_kv, block_table):
        op = self.op
        return torch.ops.tileops_amd.gqa_paged_decode_fp4(
            q, k, v, k_scale, v_scale, real_seqlen_kv, block_table, op.q_len, op.heads, op.heads_kv, op.dim, op.page_size,
            float(op.sm_scale), float(op.softcap), op.is_causal)
