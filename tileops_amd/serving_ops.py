"""L2 ops of a serving step around a paged KV cache, 4-bit, FP8 or 16-bit.

One step of a serving program: ``PagedKVCacheAllocFwdOp`` takes pages for the new tokens and says where each goes,
``QKNormRopePagedKVAppendFwdOp`` norms and rotates the projected rows and appends keys and values there, an attention op reads the
cache -- for a 4-bit cache ``GroupedQueryAttentionDecodePagedWithFP4KVCacheFwdOp``, for the others the decode ops of ``ops.py`` --
and ``PagedKVCacheReleaseFwdOp`` gives the pages of finished sequences back.  ``PagedFP4KVCacheGatherFwdOp`` reads 4-bit rows back as
16-bit values (to move a sequence to another cache).  No call reads device memory on the host, so a step can be captured in a graph.

4-bit cache: blocks of 32 head elements as e2m1 codes (two to a byte, lower nibble first) and one scale byte, ``code * 2 ** (byte - 127)``;
codes ``[n_pages, heads_kv, page_size, dim // 2]``, scales ``[n_pages, heads_kv, page_size, dim // 32]``, both ``uint8``.  A slot is
``page * page_size + offset`` in every cache.

The reference has none of these ops; arguments, checks and messages follow its paged ops (src/tileops/ops/attention/gqa.py:57-90, :897-1046).
"""

from __future__ import annotations

from typing import Dict, Optional

import torch

from . import native
from .backend import Target
from .kernels import get_arch
from .op_base import _UNRESOLVED, Op
from .ops import _attention_scale, _score_softcap, _validate_attention_dtype, _validate_gqa_dims, _validate_positive
from .serving_kernels import (
    FP4, FP8, GQADecodePagedFP4Kernel, PagedFP4KVCacheGatherKernel, PagedKVCacheAllocKernel, PagedKVCacheReleaseKernel,
    QKNormRopePagedKVAppendKernel, ServingCall,
)

__all__ = [
    "GroupedQueryAttentionDecodePagedWithFP4KVCacheFwdOp",
    "PagedFP4KVCacheGatherFwdOp",
    "PagedKVCacheAllocFwdOp",
    "PagedKVCacheReleaseFwdOp",
    "QKNormRopePagedKVAppendFwdOp",
]


def _check(name: str, t: torch.Tensor, device: torch.device, dtype: torch.dtype, shape: tuple) -> None:
    """A contiguous tensor of this shape and dtype on *device*, or a ``ValueError`` that says what is not."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise ValueError(f"Expected {name}.dtype {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"Expected {name}.shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"Expected {name} on {device}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_table(t: torch.Tensor, device: torch.device, batch: int, width: Optional[int] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"block_table must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype != torch.int32:
        raise ValueError(f"Expected block_table.dtype {torch.int32}, got {t.dtype}")
    if t.dim() != 2 or t.shape[0] != batch or t.shape[1] < 1 or (width is not None and t.shape[1] != width):
        raise ValueError(f"Expected block_table.shape ({batch}, {'num_pages' if width is None else width}), got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"Expected block_table on {device}, got {t.device}")
    if t.stride(1) != 1 or (batch > 1 and t.stride(0) < t.shape[1]):
        raise ValueError("block_table rows must be contiguous (stride(1) == 1) and must not overlap")


class _ServingOp(Op):
    """What the ops of this module share: one kernel class per op, and the native host path.

    A call goes the long way -- the checks below, kernel selection, the registered operator -- the first time, on any other device than
    that one, under a tracer, a dispatch mode or a function mode, with gradients or an external target, and whenever something is wrong with it.  Otherwise
    ``hostcall`` (csrc/hostcall.cpp) does the same checks and the launch in one native call, or answers None: then the long way is taken.
    """

    _key: str = ""
    _kernel_class: type = PagedKVCacheAllocKernel

    @property
    def default_kernel_map(self) -> Dict[str, type]:
        return {self._key: self._kernel_class}

    def _install(self, kernel_map: Optional[Dict[str, type]], target: Target) -> None:
        if target is not None:
            self.target = target
        self._selected: dict = {}
        self._device: Optional[int] = None  # a device on which the shipped kernel has served this instance
        self.dispatch_kernel(kernel_map)

    def _native(self) -> bool:
        return (self._device is not None and native._hostcall is not None and self._builder is None and self.kernel_map[self._key] is self._kernel_class
                and not torch.compiler.is_compiling())

    @staticmethod
    def _checked(result):
        if result.__class__ is int:
            native._check(result)
        return result

    def _kernel(self, inputs: tuple, dtype: Optional[torch.dtype] = None):
        if self._builder is not None and self._builder is not _UNRESOLVED:
            return self.get_or_build_kernel(self._key, inputs)  # an external target serves this instance
        device = inputs[0].device
        memo = (device, dtype, self.kernel_map[self._key])
        kernel = self._selected.get(memo)
        if kernel is None:
            index = device.index if device.type == "cuda" else None
            call = ServingCall(dim=getattr(self, "dim", 0), page_size=self.page_size, dtype=dtype, arch=get_arch(index))
            key = self.select_kernel_key((self._key,), call)
            kernel = self.get_or_build_kernel(key, inputs, key=(device, dtype, self.kernel_map[key]),
                                              build=lambda: self.kernel_map[key](self, device_index=index))
            self._selected[memo] = kernel
        if ((self._device is None or native._hostcall is None) and device.type == "cuda" and device.index is not None
                and not torch.compiler.is_compiling()):  # (no module: the instance comes from another process)
            native.hostcall()
            self._device = device.index
        return kernel


class PagedKVCacheAllocFwdOp(_ServingOp):
    """Pages for a step's new tokens.

    ``forward(cache_seqlens [batch], block_table [batch, max_pages_per_req], free_pages [num_pages], free_count [1], cu_seqlens_q=None,
    total_q=None)``, all ``int32``, returns ``(slot_mapping [total_q] int64, positions [total_q] int32, real_seqlen_kv [batch] int32,
    refused [batch] bool, free_count_out [1] int32)`` and writes the block-table entries of the pages that it takes.

    Sequence ``b`` gets the tokens ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1]`` of the packed step (one each without ``cu_seqlens_q``, whose
    entries do not decrease); ``total_q`` is the step's length, which may be padded behind the last sequence.  ``free_pages[:free_count]`` is
    a stack of free pages.  Sequences are served in batch order; one that would outgrow its row, whose tokens do not all lie below
    ``total_q``, or for which the pages do not last, is ``refused``: its ``real_seqlen_kv`` stays ``cache_seqlens[b]``, and its tokens -- like padding -- have slot and position -1.  ``free_count`` is not
    written (a repeated call gives the same answer): pass ``free_count_out`` to the next step.  The outputs may share one allocation.
    """

    _key = "paged_kv_cache_alloc_kernel"
    _kernel_class = PagedKVCacheAllocKernel
    compile_op_names = ("tileops_amd::kv_alloc",)

    def __init__(self, batch: int, max_pages_per_req: int, page_size: int, num_pages: int, kernel_map: Optional[Dict[str, type]] = None, *,
                 target: Target = None) -> None:
        _validate_positive(batch=batch, max_pages_per_req=max_pages_per_req, page_size=page_size, num_pages=num_pages)
        self.batch, self.max_pages_per_req, self.page_size, self.num_pages = batch, max_pages_per_req, page_size, num_pages
        self._install(kernel_map, target)

    def _infer_output_shapes(self, cache_seqlens_shape, block_table_shape, free_pages_shape, free_count_shape, cu_seqlens_q_shape=None,
                             total_q=None) -> dict[str, tuple[int, ...]]:
        n = self.batch if total_q is None else total_q
        return {"slot_mapping": (n,), "positions": (n,), "real_seqlen_kv": (self.batch,), "refused": (self.batch,), "free_count_out": (1,)}

    def forward(self, cache_seqlens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                cu_seqlens_q: Optional[torch.Tensor] = None, total_q: Optional[int] = None):
        if self._native():
            outs = native._hostcall.kv_alloc(cache_seqlens, block_table, free_pages, free_count, cu_seqlens_q, total_q, self.batch,
                                             self.max_pages_per_req, self.num_pages, self.page_size, self._device,
                                             torch._C._cuda_getCurrentRawStream(self._device))
            if outs is not None:
                return self._checked(outs)
        if not isinstance(block_table, torch.Tensor):
            raise ValueError(f"block_table must be a torch.Tensor, got {type(block_table).__name__}")
        device = block_table.device
        _check_table(block_table, device, self.batch, self.max_pages_per_req)
        _check("cache_seqlens", cache_seqlens, device, torch.int32, (self.batch,))
        _check("free_pages", free_pages, device, torch.int32, (self.num_pages,))
        _check("free_count", free_count, device, torch.int32, (1,))
        if cu_seqlens_q is None:
            if total_q is not None and total_q != self.batch:
                raise ValueError(f"total_q must be batch ({self.batch}) without cu_seqlens_q, got {total_q}")
            total_q = self.batch
        else:
            _check("cu_seqlens_q", cu_seqlens_q, device, torch.int32, (self.batch + 1,))
            if total_q is None:
                raise ValueError("total_q is required with cu_seqlens_q")
            if total_q < 0:
                raise ValueError(f"total_q must be non-negative, got {total_q}")
        kernel = self._kernel((cache_seqlens, block_table, free_pages, free_count, cu_seqlens_q))
        return kernel(cache_seqlens, block_table, free_pages, free_count, cu_seqlens_q, total_q)


class PagedKVCacheReleaseFwdOp(_ServingOp):
    """Pages of finished sequences back onto the list of free ones.

    ``forward(finished [batch] bool, seqlens [batch] int32, block_table [batch, max_pages_per_req] int32, free_pages [num_pages] int32,
    free_count [1] int32)`` writes the pages of the finished sequences' rows behind ``free_pages[:free_count]``, in batch order, and
    returns ``(seqlens_out, free_count_out)``: lengths with 0 for the finished, and the new count.  ``seqlens``, ``free_count`` and the
    table are not written.  The outputs may share one allocation.
    """

    _key = "paged_kv_cache_release_kernel"
    _kernel_class = PagedKVCacheReleaseKernel
    compile_op_names = ("tileops_amd::kv_release",)

    def __init__(self, batch: int, max_pages_per_req: int, page_size: int, num_pages: int, kernel_map: Optional[Dict[str, type]] = None, *,
                 target: Target = None) -> None:
        _validate_positive(batch=batch, max_pages_per_req=max_pages_per_req, page_size=page_size, num_pages=num_pages)
        self.batch, self.max_pages_per_req, self.page_size, self.num_pages = batch, max_pages_per_req, page_size, num_pages
        self._install(kernel_map, target)

    def _infer_output_shapes(self, finished_shape, seqlens_shape, block_table_shape, free_pages_shape, free_count_shape) -> dict[str, tuple[int, ...]]:
        return {"seqlens_out": (self.batch,), "free_count_out": (1,)}

    def forward(self, finished: torch.Tensor, seqlens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor):
        if self._native():
            outs = native._hostcall.kv_release(finished, seqlens, block_table, free_pages, free_count, self.batch, self.max_pages_per_req,
                                               self.num_pages, self.page_size, self._device, torch._C._cuda_getCurrentRawStream(self._device))
            if outs is not None:
                return self._checked(outs)
        if not isinstance(block_table, torch.Tensor):
            raise ValueError(f"block_table must be a torch.Tensor, got {type(block_table).__name__}")
        device = block_table.device
        _check_table(block_table, device, self.batch, self.max_pages_per_req)
        _check("finished", finished, device, torch.bool, (self.batch,))
        _check("seqlens", seqlens, device, torch.int32, (self.batch,))
        _check("free_pages", free_pages, device, torch.int32, (self.num_pages,))
        _check("free_count", free_count, device, torch.int32, (1,))
        return self._kernel((finished, seqlens, block_table, free_pages, free_count))(finished, seqlens, block_table, free_pages, free_count)


class QKNormRopePagedKVAppendFwdOp(_ServingOp):
    """RMS norm of query and key rows per head, rotary embedding, and the append of keys and values to a paged cache, in one pass.

    ``forward(q [tokens, heads, dim], k, v [tokens, heads_kv, dim], q_weight, k_weight [dim], cos_table, sin_table [max_position,
    rotary_dim // 2], positions [tokens] int32, slot_mapping [tokens] int64, k_cache, v_cache, k_scale=None, v_scale=None)`` returns the
    query rows, normed and rotated; keys (likewise) and values go to their slots of the cache.

    * ``q``, ``k``, ``v`` fp16 or bf16; heads contiguous, any token stride (slices of one projection are taken as they are);
    * ``q_weight`` / ``k_weight`` of that dtype or fp32, or None: no norm of these rows.  ``y = x / sqrt(mean(x ** 2) + eps) * weight``;
    * ``rotary_dim`` (default ``dim``; 0: no rotation, tables and positions None): the first elements of a head, in halves or, if
      ``interleaved``, in neighbouring pairs; tables of ``q``'s dtype or fp32; a position outside the tables is read as the nearest row;
    * ``cache_dtype`` None: ``k_cache``, ``v_cache [n_tokens, heads_kv, dim]`` of ``q``'s dtype; ``torch.float8_e4m3fn``: the same with
      ``k_scale``, ``v_scale [n_tokens, heads_kv]`` fp32, as the decode ops read it; ``torch.float4_e2m1fn_x2``: the 4-bit cache;
    * a token with a slot outside the pool (-1: padding, a refused sequence) is not appended.  No slot may occur twice.
    """

    _key = "qk_norm_rope_paged_kv_append_kernel"
    _kernel_class = QKNormRopePagedKVAppendKernel
    compile_op_names = ("tileops_amd::qk_norm_rope_append",)

    def __init__(self, heads: int, heads_kv: int, dim: int, page_size: int, rotary_dim: Optional[int] = None, eps: float = 1e-6,
                 interleaved: bool = False, cache_dtype: Optional[torch.dtype] = None, kernel_map: Optional[Dict[str, type]] = None, *,
                 target: Target = None) -> None:
        _validate_gqa_dims(heads, heads_kv, dim)
        _validate_positive(page_size=page_size)
        rotary_dim = dim if rotary_dim is None else rotary_dim
        if rotary_dim < 0 or rotary_dim % 2 != 0 or rotary_dim > dim:
            raise ValueError("rotary_dim must be an even number between 0 and dim")
        if not eps >= 0:
            raise ValueError("eps must be non-negative")
        if cache_dtype is not None and cache_dtype not in (FP4, FP8):
            _validate_attention_dtype(cache_dtype)
        self.heads, self.heads_kv, self.dim, self.page_size = heads, heads_kv, dim, page_size
        self.rotary_dim, self.eps, self.interleaved, self.cache_dtype = rotary_dim, float(eps), bool(interleaved), cache_dtype
        self._install(kernel_map, target)

    def _infer_output_shapes(self, q_shape, *other_shapes) -> dict[str, tuple[int, ...]]:
        return {"q_out": tuple(q_shape)}

    def _check_rows(self, name: str, t: torch.Tensor, device: torch.device, dtype: torch.dtype, shape: tuple) -> None:
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
        if t.dtype != dtype:
            raise ValueError(f"Expected {name}.dtype {dtype}, got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"Expected {name}.shape {tuple(shape)}, got {tuple(t.shape)}")
        if t.device != device:
            raise ValueError(f"Expected {name} on {device}, got {t.device}")
        token, head, element = t.stride()
        if (element != 1 or (head != self.dim and shape[1] > 1) or token % 2 != 0) and t.numel() > 0:
            raise ValueError(f"the heads of {name} must be contiguous and its token stride even, got strides {t.stride()}")
        if not torch.compiler.is_compiling() and t.data_ptr() % 4 != 0:
            raise ValueError(f"{name} must be 4-byte aligned")

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                cos_table: Optional[torch.Tensor], sin_table: Optional[torch.Tensor], positions: Optional[torch.Tensor],
                slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self._native():
            out = native._hostcall.qk_norm_rope_append(
                q, k, v, q_weight, k_weight, cos_table, sin_table, positions, slot_mapping, k_cache, v_cache, k_scale, v_scale, self.heads,
                self.heads_kv, self.dim, self.page_size, self.rotary_dim, self.interleaved, self._cache_code(q), self.eps, self._device,
                torch._C._cuda_getCurrentRawStream(self._device))
            if out is not None:
                return self._checked(out)
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError(f"q must be a tensor of shape [tokens, {self.heads}, {self.dim}]")
        device, dtype, tokens = q.device, q.dtype, q.shape[0]
        _validate_attention_dtype(dtype)
        self._check_rows("q", q, device, dtype, (tokens, self.heads, self.dim))
        self._check_rows("k", k, device, dtype, (tokens, self.heads_kv, self.dim))
        self._check_rows("v", v, device, dtype, (tokens, self.heads_kv, self.dim))
        _check("slot_mapping", slot_mapping, device, torch.int64, (tokens,))
        weight_dtype = None
        for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
            if t is None:
                continue
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{name} must be a torch.Tensor or None, got {type(t).__name__}")
            if t.dtype not in (dtype, torch.float32) or (weight_dtype or t.dtype) != t.dtype:
                raise ValueError(f"q_weight and k_weight must both be {dtype} or both torch.float32, got {t.dtype} for {name}")
            weight_dtype = t.dtype
            _check(name, t, device, t.dtype, (self.dim,))
        if self.rotary_dim:
            if cos_table is None or sin_table is None or positions is None:
                raise ValueError("cos_table, sin_table and positions are required with rotary_dim > 0")
            if not isinstance(cos_table, torch.Tensor):
                raise ValueError(f"cos_table must be a torch.Tensor, got {type(cos_table).__name__}")
            if cos_table.dtype not in (dtype, torch.float32):
                raise ValueError(f"cos_table must be {dtype} or torch.float32, got {cos_table.dtype}")
            if cos_table.dim() != 2 or cos_table.shape[0] < 1:
                raise ValueError(f"cos_table must have shape [max_position, {self.rotary_dim // 2}], got {tuple(cos_table.shape)}")
            _check("cos_table", cos_table, device, cos_table.dtype, (cos_table.shape[0], self.rotary_dim // 2))
            _check("sin_table", sin_table, device, cos_table.dtype, cos_table.shape)
            _check("positions", positions, device, torch.int32, (tokens,))
        elif cos_table is not None or sin_table is not None:
            raise ValueError("cos_table and sin_table must be None with rotary_dim 0")
        self._check_caches(device, dtype, k_cache, v_cache, k_scale, v_scale)
        if not self.rotary_dim:
            positions = None
        kernel = self._kernel((q, k, v, q_weight, k_weight, cos_table, sin_table, positions, slot_mapping, k_cache, v_cache, k_scale, v_scale), dtype)
        return kernel(q, k, v, q_weight, k_weight, cos_table, sin_table, positions, slot_mapping, k_cache, v_cache, k_scale, v_scale)

    def _cache_code(self, q) -> int:
        """Type code of the cache for the native path: 0 for a cache of ``q``'s type, -1 (taken by no call) for one of another 16-bit type."""
        if self.cache_dtype is None:
            return 0
        if self.cache_dtype == FP4:
            return native.DT_FP4_E2M1
        if self.cache_dtype == FP8:
            return native.DT_FP8_E4M3FN
        return 0 if getattr(q, "dtype", None) == self.cache_dtype else -1

    def _check_caches(self, device, dtype, k_cache, v_cache, k_scale, v_scale) -> None:
        if not isinstance(k_cache, torch.Tensor) or k_cache.dim() < 1 or k_cache.shape[0] < 1:
            raise ValueError("k_cache must be a tensor that holds at least one page")
        n = k_cache.shape[0]
        if self.cache_dtype == FP4:
            _check_fp4_cache(device, n, self.heads_kv, self.page_size, self.dim, k_cache, v_cache, k_scale, v_scale, "_cache")
            return
        if n % self.page_size != 0:
            raise ValueError("k_cache token dimension must be divisible by page_size")
        want = dtype if self.cache_dtype is None else self.cache_dtype
        if want != FP8 and want != dtype:
            raise ValueError(f"cache_dtype must be the dtype of q ({dtype}), torch.float8_e4m3fn or torch.float4_e2m1fn_x2, got {want}")
        _check("k_cache", k_cache, device, want, (n, self.heads_kv, self.dim))
        _check("v_cache", v_cache, device, want, (n, self.heads_kv, self.dim))
        if want == FP8:
            if k_scale is None or v_scale is None:
                raise ValueError("k_scale and v_scale are required when the KV cache is float8_e4m3fn")
            _check("k_scale", k_scale, device, torch.float32, (n, self.heads_kv))
            _check("v_scale", v_scale, device, torch.float32, (n, self.heads_kv))
        elif k_scale is not None or v_scale is not None:
            raise ValueError("k_scale and v_scale must be None with a 16-bit KV cache")


def _check_fp4_cache(device, pages, heads_kv, page_size, dim, k, v, k_scale, v_scale, suffix="") -> None:
    if k_scale is None or v_scale is None:
        raise ValueError("k_scale and v_scale are required with a 4-bit KV cache")
    codes, scales = (pages, heads_kv, page_size, dim // 2), (pages, heads_kv, page_size, dim // 32)
    _check("k" + suffix, k, device, torch.uint8, codes)
    _check("v" + suffix, v, device, torch.uint8, codes)
    _check("k_scale", k_scale, device, torch.uint8, scales)
    _check("v_scale", v_scale, device, torch.uint8, scales)


class PagedFP4KVCacheGatherFwdOp(_ServingOp):
    """Rows of a 4-bit cache as 16-bit values: ``forward(k, v, k_scale, v_scale, slot_mapping [tokens] int64)`` returns ``k, v [tokens,
    heads_kv, dim]`` of ``dtype`` (bf16: exact; fp16: rounded), zeros for slots outside the pool."""

    _key = "paged_fp4_kv_cache_gather_kernel"
    _kernel_class = PagedFP4KVCacheGatherKernel
    compile_op_names = ("tileops_amd::kv_gather_fp4",)

    def __init__(self, heads_kv: int, dim: int, page_size: int, dtype: torch.dtype = torch.bfloat16, kernel_map: Optional[Dict[str, type]] = None,
                 *, target: Target = None) -> None:
        _validate_positive(heads_kv=heads_kv, dim=dim, page_size=page_size)
        _validate_attention_dtype(dtype)
        self.heads_kv, self.dim, self.page_size, self.dtype = heads_kv, dim, page_size, dtype
        self._install(kernel_map, target)

    def _infer_output_shapes(self, k_shape, v_shape, k_scale_shape, v_scale_shape, slot_mapping_shape) -> dict[str, tuple[int, ...]]:
        shape = (slot_mapping_shape[0], self.heads_kv, self.dim)
        return {"k_out": shape, "v_out": shape}

    def forward(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor):
        if self._native():
            outs = native._hostcall.kv_gather_fp4(k, v, k_scale, v_scale, slot_mapping, self.heads_kv, self.dim, self.page_size,
                                                  native.DT_BF16 if self.dtype == torch.bfloat16 else native.DT_FP16, self._device,
                                                  torch._C._cuda_getCurrentRawStream(self._device))
            if outs is not None:
                return self._checked(outs)
        if not isinstance(k, torch.Tensor) or k.dim() != 4 or k.shape[0] < 1:
            raise ValueError(f"k must have shape [n_pages, {self.heads_kv}, {self.page_size}, {self.dim // 2}]")
        _check_fp4_cache(k.device, k.shape[0], self.heads_kv, self.page_size, self.dim, k, v, k_scale, v_scale)
        if not isinstance(slot_mapping, torch.Tensor) or slot_mapping.dim() != 1:
            raise ValueError("slot_mapping must have shape [tokens]")
        _check("slot_mapping", slot_mapping, k.device, torch.int64, slot_mapping.shape)
        return self._kernel((k, v, k_scale, v_scale, slot_mapping), self.dtype)(k, v, k_scale, v_scale, slot_mapping)


class GroupedQueryAttentionDecodePagedWithFP4KVCacheFwdOp(_ServingOp):
    """Paged GQA decode over a 4-bit KV cache.  Layout: Q ``[batch, heads, dim]``, or ``[batch, q_len, heads, dim]`` with ``q_len`` > 1
    (speculative verify, short prefill chunks: the cache already holds the ``q_len`` new tokens, ``real_seqlen_kv`` counts them, and the
    causal mask is bottom-right aligned); K, V codes ``[n_pages, heads_kv, page_size, dim // 2]`` and scale bytes
    ``[n_pages, heads_kv, page_size, dim // 32]`` with ``seqlen_kv = n_pages * page_size``; ``real_seqlen_kv [batch]``;
    ``block_table [batch, num_pages]``.  ``page_size`` is a multiple of 16.  A query row that sees no token is zeros.

    Arguments otherwise as ``GroupedQueryAttentionDecodePagedWithKVCacheFwdOp``.
    """

    _key = "gqa_decode_paged_fp4_kernel"
    _kernel_class = GQADecodePagedFP4Kernel
    compile_op_names = ("tileops_amd::gqa_paged_decode_fp4",)
    _seen_call: Optional[dict] = None

    def __init__(self, batch: int, heads: int, heads_kv: int, seqlen_kv: int, dim: int, page_size: int, q_len: int = 1, is_causal: bool = True,
                 sm_scale: Optional[float] = None, softcap: Optional[float] = None, kernel_map: Optional[Dict[str, type]] = None, *,
                 target: Target = None) -> None:
        _validate_gqa_dims(heads, heads_kv, dim)
        _validate_positive(batch=batch, seqlen_kv=seqlen_kv, page_size=page_size, q_len=q_len)
        if page_size % 16 != 0:
            raise ValueError("page_size must be a multiple of 16 with a 4-bit KV cache")
        if seqlen_kv % page_size != 0:
            raise ValueError("seqlen_kv must be divisible by page_size")
        self.batch, self.heads, self.heads_kv, self.seqlen_kv, self.dim = batch, heads, heads_kv, seqlen_kv, dim
        self.page_size, self.q_len, self.is_causal = page_size, q_len, bool(is_causal)
        self.sm_scale, self.softcap = float(_attention_scale(dim, sm_scale)), float(_score_softcap(softcap))
        self._plans: dict = {}
        self._install(kernel_map, target)

    def _infer_output_shapes(self, q_shape, k_shape, v_shape, k_scale_shape, v_scale_shape, real_seqlen_kv_shape,
                             block_table_shape) -> dict[str, tuple[int, ...]]:
        return {"o": tuple(q_shape)}

    def observe_call(self, real_seqlen_kv: torch.Tensor) -> None:
        """Record the context lengths of a call so that ``eval_roofline`` prices the bytes actually addressed."""
        lens = real_seqlen_kv.to("cpu", torch.int64)
        self._seen_call = {"sum_len": int(lens.sum()), "sum_pages": int(((lens + self.page_size - 1) // self.page_size).sum())}

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                real_seqlen_kv: torch.Tensor, block_table: torch.Tensor) -> torch.Tensor:
        if self._native():
            dtype = getattr(q, "dtype", None)
            plan = self._plans.get(dtype)  # workspace bytes and type code
            if plan is not None:
                out = native._hostcall.decode_fp4(
                    k, v, k_scale, v_scale, q, real_seqlen_kv, block_table, self.batch, self.q_len, self.heads, self.heads_kv,
                    self.seqlen_kv // self.page_size, self.dim, self.page_size, self.is_causal, self.sm_scale, self.softcap, *plan, self._device,
                    torch._C._cuda_getCurrentRawStream(self._device))
                if out is not None:
                    self.dtype = dtype
                    return self._checked(out)
        if not isinstance(q, torch.Tensor):
            raise ValueError(f"q must be a torch.Tensor, got {type(q).__name__}")
        device, dtype = q.device, q.dtype
        _validate_attention_dtype(dtype)
        _check("q", q, device, dtype, (self.batch, self.heads, self.dim) if self.q_len == 1 else (self.batch, self.q_len, self.heads, self.dim))
        _check_fp4_cache(device, self.seqlen_kv // self.page_size, self.heads_kv, self.page_size, self.dim, k, v, k_scale, v_scale)
        _check("real_seqlen_kv", real_seqlen_kv, device, torch.int32, (self.batch,))
        _check_table(block_table, device, self.batch)
        self.dtype = dtype
        kernel = self._kernel((q, k, v, k_scale, v_scale, real_seqlen_kv, block_table), dtype)
        if self._device is not None and dtype not in self._plans:
            self._plans[dtype] = (native.decode_fp4_workspace(self.batch, self.q_len, self.heads, self.heads_kv, self.dim, self.page_size, dtype),
                                  native.dtype_code(dtype))
        return kernel(q, k, v, k_scale, v_scale, real_seqlen_kv, block_table)
