"""Torch-tensor wrappers over the C ABI (one function per entry point of include/triattn_b200.h).

PyTorch is used for device memory and streams only; all arithmetic happens in
the CUDA kernels of ``libtriattn_b200.so``.  Every wrapper launches on the
current torch stream and does not synchronise.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _native
from ._native import PagedLayout


def _ptr(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream():
    # raw handle of torch's current stream on the current device (the public current_stream() object costs ~15 us)
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()))


def split_kv_axes(kv_cache: torch.Tensor, kv_axis: Optional[int] = None):
    """(key_cache, value_cache) views ``[nb, bs, H, D]`` of a 5-D paged cache.

    Same disambiguation rule as the reference's ``_split_kv_axes``
    (runtime/kv_compaction.py:94-117): the axis of size 2 among the first two
    is the K/V axis; if both are 2 an explicit ``kv_axis`` hint is required.
    """
    if kv_cache.ndim != 5:
        raise ValueError(f"Unsupported kv_cache ndim={kv_cache.ndim}, expect 5")
    d0 = int(kv_cache.shape[0]) == 2
    d1 = int(kv_cache.shape[1]) == 2
    if d0 and d1:
        if kv_axis not in (0, 1):
            raise ValueError(
                "Ambiguous KV layout for compaction: both dim0 and dim1 have size 2. "
                "Register an explicit layout hint via register_kv_layout_axis_hint(...)."
            )
        d0, d1 = kv_axis == 0, kv_axis == 1
    if d0:
        return kv_cache[0], kv_cache[1]
    if d1:
        return kv_cache[:, 0], kv_cache[:, 1]
    raise ValueError("Unsupported KV layout for compaction: expected a dimension with size 2")


_VIEW_CACHE: dict = {}


@dataclass
class PagedCacheView:
    """Device-side description of the layers of one KV-cache group (shared block table)."""

    k_ptrs: torch.Tensor   # [L] int64 on device
    v_ptrs: torch.Tensor   # [L] int64 on device
    num_layers: int
    num_blocks: int
    block_size: int
    num_kv_heads: int
    head_dim: int
    block_stride: int
    token_stride: int
    head_stride: int
    device: torch.device
    dtype: torch.dtype

    @classmethod
    def from_layers(cls, kv_caches: Sequence[torch.Tensor], kv_axis: Optional[int] = None) -> "PagedCacheView":
        if not kv_caches:
            raise ValueError("no kv cache layers")
        # An engine keeps the same cache tensors for its whole life: remember the view (device pointer arrays
        # included) per set of layers, so a compression step costs no per-layer Python and no pointer upload.
        key = (kv_axis, tuple(int(c.data_ptr()) for c in kv_caches), tuple(kv_caches[0].shape),
               tuple(kv_caches[0].stride()), kv_caches[0].dtype, str(kv_caches[0].device))
        hit = _VIEW_CACHE.get(key)
        if hit is not None:
            return hit
        view = cls._build(kv_caches, kv_axis)
        if len(_VIEW_CACHE) >= 64:
            _VIEW_CACHE.clear()
        _VIEW_CACHE[key] = view
        return view

    @classmethod
    def _build(cls, kv_caches: Sequence[torch.Tensor], kv_axis: Optional[int]) -> "PagedCacheView":
        k0, v0 = split_kv_axes(kv_caches[0], kv_axis)
        if k0.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"paged cache must be 16-bit, got {k0.dtype}")
        if k0.dtype != torch.bfloat16:
            raise ValueError("the scorer reads bf16 keys; fp16 caches are not supported")
        if k0.stride(3) != 1:
            raise ValueError("head_dim axis of the paged cache must be contiguous")
        kp, vp = [], []
        for c in kv_caches:
            k, v = split_kv_axes(c, kv_axis)
            if k.shape != k0.shape or k.stride() != k0.stride() or v.stride() != k0.stride():
                raise ValueError("all layers of a KV-cache group must share shape and strides")
            if k.data_ptr() % 16 or v.data_ptr() % 16:
                raise ValueError("paged cache base pointers must be 16-byte aligned")
            kp.append(k.data_ptr())
            vp.append(v.data_ptr())
        dev = k0.device
        return cls(
            k_ptrs=torch.tensor(kp, dtype=torch.int64, device=dev),
            v_ptrs=torch.tensor(vp, dtype=torch.int64, device=dev),
            num_layers=len(kv_caches),
            num_blocks=int(k0.shape[0]),
            block_size=int(k0.shape[1]),
            num_kv_heads=int(k0.shape[2]),
            head_dim=int(k0.shape[3]),
            block_stride=int(k0.stride(0)),
            token_stride=int(k0.stride(1)),
            head_stride=int(k0.stride(2)),
            device=dev,
            dtype=k0.dtype,
        )

    def layout(self, num_reqs: int, group_size: int, max_blocks_per_req: int, rope_interleaved: bool = False) -> PagedLayout:
        return PagedLayout(
            num_layers=self.num_layers, num_reqs=int(num_reqs), num_kv_heads=self.num_kv_heads,
            group_size=int(group_size), head_dim=self.head_dim, block_size=self.block_size,
            num_blocks=self.num_blocks, max_blocks_per_req=int(max_blocks_per_req),
            block_stride=self.block_stride, token_stride=self.token_stride, head_stride=self.head_stride,
            rope_interleaved=1 if rope_interleaved else 0, reserved=0,
        )


@dataclass
class DeviceStats:
    """Calibrated statistics packed for the kernels: ``[L, Hq, F]`` fp32 each, plus omega and offsets."""

    q_mean_real: torch.Tensor
    q_mean_imag: torch.Tensor
    q_abs_mean: torch.Tensor
    freq_scale_sq: torch.Tensor
    omega: torch.Tensor
    offsets: torch.Tensor
    rope_interleaved: bool = False

    @property
    def num_layers(self) -> int:
        return int(self.q_mean_real.shape[0])

    @property
    def num_heads(self) -> int:
        return int(self.q_mean_real.shape[1])

    @property
    def num_freqs(self) -> int:
        return int(self.q_mean_real.shape[2])

    def select_layers(self, layer_indices: Sequence[int]) -> "DeviceStats":
        idx = torch.as_tensor(list(layer_indices), dtype=torch.long, device=self.q_mean_real.device)
        return DeviceStats(
            self.q_mean_real.index_select(0, idx).contiguous(), self.q_mean_imag.index_select(0, idx).contiguous(),
            self.q_abs_mean.index_select(0, idx).contiguous(), self.freq_scale_sq.index_select(0, idx).contiguous(),
            self.omega, self.offsets, self.rope_interleaved)

    def slice_heads(self, start: int, end: int) -> "DeviceStats":
        """Statistics rows of query heads [start, end): the shard a tensor-parallel rank owns."""
        return DeviceStats(
            self.q_mean_real[:, start:end].contiguous(), self.q_mean_imag[:, start:end].contiguous(),
            self.q_abs_mean[:, start:end].contiguous(), self.freq_scale_sq[:, start:end].contiguous(),
            self.omega, self.offsets, self.rope_interleaved)


def _i32(x, device) -> torch.Tensor:
    if isinstance(x, torch.Tensor):
        return x.to(device=device, dtype=torch.int32).contiguous()
    return torch.as_tensor(list(x), dtype=torch.int32, device=device)


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise _native.NativeLibraryError(
            f"{_native.TRITON_SCORING_REQUIRED_MARKER}:tensor_not_on_cuda:{name} (there is no CPU path)")


def prep_weights(stats: DeviceStats, round_start: torch.Tensor, offset_agg: int = _native.OFFSETS_MEAN,
                 flags: int = 0) -> torch.Tensor:
    """``[L, B, Hq, rows, F]`` fp32 folded weights (``triattn_prep_weights``)."""
    lib = _native.load()
    _require_cuda(stats.q_mean_real, "stats")
    dev = stats.q_mean_real.device
    rs = _i32(round_start, dev)
    L, Hq, F = stats.num_layers, stats.num_heads, stats.num_freqs
    B, O = int(rs.numel()), int(stats.offsets.numel())
    rows = lib.triattn_weight_rows(offset_agg, O)
    scratch = torch.empty(lib.triattn_prep_scratch_floats(B, F, O, offset_agg), dtype=torch.float32, device=dev)
    out = torch.empty((L, B, Hq, rows, F), dtype=torch.float32, device=dev)
    _native.check(lib.triattn_prep_weights(
        _ptr(stats.q_mean_real), _ptr(stats.q_mean_imag), _ptr(stats.q_abs_mean), _ptr(stats.freq_scale_sq),
        _ptr(stats.omega), _ptr(stats.offsets), _ptr(rs), L, B, Hq, F, O, offset_agg, flags,
        _ptr(scratch), _ptr(out), _stream()), "prep_weights")
    return out


def prep_weights_fused(stats: DeviceStats, round_start: torch.Tensor, offset_agg: int = _native.OFFSETS_MEAN,
                       flags: int = 0, moments_to_clear: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``triattn_prep_weights`` in one launch, no scratch (``triattn_prep_weights_fused``); optionally zeroes
    the ``[L, B, Hq, 2]`` fp64 moments array the scorer accumulates into."""
    lib = _native.load()
    _require_cuda(stats.q_mean_real, "stats")
    dev = stats.q_mean_real.device
    rs = _i32(round_start, dev)
    L, Hq, F = stats.num_layers, stats.num_heads, stats.num_freqs
    B, O = int(rs.numel()), int(stats.offsets.numel())
    out = torch.empty((L, B, Hq, lib.triattn_weight_rows(offset_agg, O), F), dtype=torch.float32, device=dev)
    _native.check(lib.triattn_prep_weights_fused(
        _ptr(stats.q_mean_real), _ptr(stats.q_mean_imag), _ptr(stats.q_abs_mean), _ptr(stats.freq_scale_sq),
        _ptr(stats.omega), _ptr(stats.offsets), _ptr(rs), L, B, Hq, F, O, offset_agg, flags, _ptr(out),
        _ptr(moments_to_clear), _stream()), "prep_weights_fused")
    return out


def score_paged(view: PagedCacheView, layout: PagedLayout, block_table: torch.Tensor, seq_lens: torch.Tensor,
                weights: torch.Tensor, offset_agg: int = _native.OFFSETS_MEAN, num_offsets: int = 17,
                status: Optional[torch.Tensor] = None, raw: Optional[torch.Tensor] = None,
                moments: Optional[torch.Tensor] = None, cuda_cores: bool = False):
    """Raw scores ``[L, B, Hkv, t_pad, Gp]`` fp32 and moments ``[L, B, Hq, 2]`` fp64 (``triattn_score_paged``;
    ``cuda_cores=True`` calls the all-fp32 cross-check ``triattn_score_paged_cuda_cores``)."""
    lib = _native.load()
    gp = lib.triattn_padded_group(layout.group_size)
    if gp == 0:
        _native.check(2, "score_paged:group_size")
    L, B, Hkv = layout.num_layers, layout.num_reqs, layout.num_kv_heads
    t_pad = layout.max_blocks_per_req * layout.block_size
    dev = view.device
    if raw is None:
        raw = torch.empty((L, B, Hkv, t_pad, gp), dtype=torch.float32, device=dev)
    if moments is None:
        moments = torch.empty((L, B, Hkv * layout.group_size, 2), dtype=torch.float64, device=dev)
    fn = lib.triattn_score_paged_cuda_cores if cuda_cores else lib.triattn_score_paged
    _native.check(fn(
        ctypes.byref(layout), _ptr(view.k_ptrs), _ptr(block_table), _ptr(seq_lens), _ptr(weights),
        offset_agg, num_offsets, _ptr(raw), _ptr(moments), _ptr(status), _stream()), "score_paged")
    return raw, moments


def finalize_scores(layout: PagedLayout, raw: torch.Tensor, moments: torch.Tensor, seq_lens: torch.Tensor,
                    prefill_lens: Optional[torch.Tensor], window: int, normalize: bool = True,
                    group_reduce: int = _native.REDUCE_MAX, head_reduce: int = _native.REDUCE_NONE,
                    layer_reduce: int = _native.REDUCE_MEAN) -> torch.Tensor:
    """Scores for the top-k ``[Lo, B, Ho, t_pad]`` fp32 (``triattn_finalize_scores``).

    Entries at or beyond a request's length are not written (left as -inf).
    """
    lib = _native.load()
    L, B, Hkv = layout.num_layers, layout.num_reqs, layout.num_kv_heads
    t_pad = layout.max_blocks_per_req * layout.block_size
    Lo = L if layer_reduce == _native.REDUCE_NONE else 1
    Ho = Hkv if head_reduce == _native.REDUCE_NONE else 1
    dev = raw.device
    out = torch.full((Lo, B, Ho, t_pad), float("-inf"), dtype=torch.float32, device=dev)
    _native.check(lib.triattn_finalize_scores(
        ctypes.byref(layout), _ptr(raw), _ptr(moments), _ptr(seq_lens), _ptr(prefill_lens), int(window),
        1 if normalize else 0, group_reduce, head_reduce, layer_reduce, _ptr(out), _stream()),
        "finalize_scores")
    return out


def finalize_scores_scatter(layout: PagedLayout, raw: torch.Tensor, moments: torch.Tensor, seq_lens: torch.Tensor,
                            prefill_lens: Optional[torch.Tensor], window: int, normalize: bool, group_reduce: int,
                            head_reduce: int, recv_ptrs: torch.Tensor, rank: int) -> None:
    """Per-layer score rows, each stored into the receive buffer of the rank that owns it
    (``triattn_finalize_scores_scatter``).  ``recv_ptrs``: int64 device tensor with one pointer per rank to that
    rank's ``[ranks, rows / ranks, t_pad]`` fp32 buffer, valid on this device (peer mappings; the own buffer
    included)."""
    lib = _native.load()
    _require_cuda(recv_ptrs, "recv_ptrs")
    if recv_ptrs.dtype != torch.int64 or not recv_ptrs.is_contiguous():
        raise ValueError("recv_ptrs must be a contiguous int64 tensor of device pointers")
    _native.check(lib.triattn_finalize_scores_scatter(
        ctypes.byref(layout), _ptr(raw), _ptr(moments), _ptr(seq_lens), _ptr(prefill_lens), int(window),
        1 if normalize else 0, group_reduce, head_reduce, _ptr(recv_ptrs), int(recv_ptrs.numel()), int(rank), _stream()),
        "finalize_scores_scatter")


def max_over_slots(slots: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``slots`` ``[S, ...]`` fp32 -> elementwise maximum over the first axis (``triattn_max_over_slots``)."""
    lib = _native.load()
    _require_cuda(slots, "slots")
    if slots.dtype != torch.float32 or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous fp32 tensor")
    if out is None:
        out = torch.empty(slots.shape[1:], dtype=torch.float32, device=slots.device)
    _native.check(lib.triattn_max_over_slots(_ptr(slots), int(slots.shape[0]), int(out.numel()), _ptr(out), _stream()),
                  "max_over_slots")
    return out


def select_topk(scores: torch.Tensor, seq_lens: torch.Tensor, keep_counts: torch.Tensor, num_reqs: int,
                rows_per_req_inner: int, keep_pitch: int, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Ascending keep indices ``[rows, keep_pitch]`` int32 (``triattn_select_topk``); ``scores`` is ``[rows, stride]``."""
    lib = _native.load()
    _require_cuda(scores, "scores")
    rows = int(scores.shape[0])
    if scores.stride(1) != 1:
        raise ValueError("score rows must be contiguous")
    out = torch.empty((rows, keep_pitch), dtype=torch.int32, device=scores.device)
    _native.check(lib.triattn_select_topk(
        _ptr(scores), rows, int(scores.stride(0)), _ptr(seq_lens), _ptr(keep_counts), int(num_reqs),
        int(rows_per_req_inner), _ptr(out), int(keep_pitch), _ptr(status), _stream()), "select_topk")
    return out


def compact_paged(view: PagedCacheView, layout: PagedLayout, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  keep: torch.Tensor, keep_strides: tuple, keep_counts: torch.Tensor,
                  status: Optional[torch.Tensor] = None, preserve_dropped: bool = False,
                  max_dropped_rows: int = 0) -> None:
    """In-place compaction of K and V (``triattn_compact_paged`` / ``triattn_compact_paged_preserve``).

    ``keep_strides`` = (layer, request, head) strides of ``keep`` in elements; 0 shares a row.
    """
    lib = _native.load()
    ls, rs, hs = (int(s) for s in keep_strides)
    if not preserve_dropped:
        _native.check(lib.triattn_compact_paged(
            ctypes.byref(layout), _ptr(view.k_ptrs), _ptr(view.v_ptrs), _ptr(block_table), _ptr(seq_lens),
            _ptr(keep), ls, rs, hs, _ptr(keep_counts), _ptr(status), _stream()), "compact_paged")
        return
    nbytes = lib.triattn_compact_preserve_scratch_bytes(ctypes.byref(layout), int(max_dropped_rows))
    scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=view.device)
    _native.check(lib.triattn_compact_paged_preserve(
        ctypes.byref(layout), _ptr(view.k_ptrs), _ptr(view.v_ptrs), _ptr(block_table), _ptr(seq_lens),
        _ptr(keep), ls, rs, hs, _ptr(keep_counts), int(max_dropped_rows), _ptr(scratch), nbytes, _ptr(status),
        _stream()), "compact_paged_preserve")


def compress_workspace_bytes(layout: PagedLayout, num_offsets: int, offset_agg: int, keep_pitch: int) -> int:
    """Workspace with which the fused step scores all layers in one launch."""
    return int(_native.load().triattn_compress_workspace_bytes(ctypes.byref(layout), num_offsets, offset_agg, keep_pitch))


def compress_workspace_bytes_min(layout: PagedLayout, num_offsets: int, offset_agg: int, keep_pitch: int) -> int:
    """Smallest workspace the fused step accepts (raw scores of one layer at a time)."""
    return int(_native.load().triattn_compress_workspace_bytes_min(ctypes.byref(layout), num_offsets, offset_agg, keep_pitch))


def compress_paged(view: PagedCacheView, layout: PagedLayout, stats: DeviceStats, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, round_start: torch.Tensor, prefill_lens: Optional[torch.Tensor],
                   keep_counts: torch.Tensor, keep_pitch: int, window: int, normalize: bool = True,
                   offset_agg: int = _native.OFFSETS_MEAN, flags: int = 0,
                   layer_reduce: int = _native.REDUCE_MEAN, workspace: Optional[torch.Tensor] = None,
                   keep_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The fused default-mode step (``triattn_compress_paged``); returns keep ``[B, Hkv, keep_pitch]`` int32."""
    lib = _native.load()
    O = int(stats.offsets.numel())
    if workspace is None:
        workspace = torch.empty(compress_workspace_bytes(layout, O, offset_agg, keep_pitch), dtype=torch.uint8,
                                device=view.device)
    if keep_out is None:
        keep_out = torch.empty((layout.num_reqs, layout.num_kv_heads, keep_pitch), dtype=torch.int32, device=view.device)
    _native.check(lib.triattn_compress_paged(
        ctypes.byref(layout), _ptr(view.k_ptrs), _ptr(view.v_ptrs), _ptr(block_table), _ptr(seq_lens),
        _ptr(round_start), _ptr(prefill_lens), _ptr(keep_counts), _ptr(stats.q_mean_real), _ptr(stats.q_mean_imag),
        _ptr(stats.q_abs_mean), _ptr(stats.freq_scale_sq), _ptr(stats.omega), _ptr(stats.offsets), O, offset_agg,
        flags, int(window), 1 if normalize else 0, layer_reduce, _ptr(workspace), workspace.numel(),
        _ptr(keep_out), int(keep_pitch), _ptr(status), _stream()), "compress_paged")
    return keep_out


def rewrite_block_tables(block_table: torch.Tensor, blocks_before: torch.Tensor, lens_after: torch.Tensor,
                         block_size: int, freed_capacity: Optional[int] = None, fill_value: int = 0,
                         status: Optional[torch.Tensor] = None):
    """Shrink every row of a device block table to ``ceil(lens_after / block_size)`` entries in place
    (``triattn_rewrite_block_tables``).

    Returns ``(blocks_after [B] int32, freed_ids [capacity] int32, freed_count [1] int32)``, all on the device;
    the freed ids are ordered by request, then by position in the row, like the concatenation of the
    ``removed_block_ids`` lists of layout_engine.truncate_tail_reclaim_group.
    """
    lib = _native.load()
    _require_cuda(block_table, "block_table")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 [B, max_blocks] tensor")
    B, width = int(block_table.shape[0]), int(block_table.shape[1])
    dev = block_table.device
    cap = B * width if freed_capacity is None else int(freed_capacity)
    blocks_after = torch.empty(B, dtype=torch.int32, device=dev)
    freed = torch.empty(max(cap, 1), dtype=torch.int32, device=dev)
    count = torch.zeros(1, dtype=torch.int32, device=dev)
    _native.check(lib.triattn_rewrite_block_tables(
        _ptr(block_table), B, width, int(block_size), _ptr(blocks_before), _ptr(lens_after), _ptr(blocks_after),
        _ptr(freed), cap, _ptr(count), int(fill_value), _ptr(status), _stream()), "rewrite_block_tables")
    return blocks_after, freed, count


# ------------------------------------------------------------------------------------------ attention over the cache
# These run once per layer and decode step, so their checks avoid creating tensor views and device objects.
_NO_GUARD = contextlib.nullcontext()


def _on_device(index: int):
    """Makes the device current for the launches inside (nothing to do when it already is)."""
    return _NO_GUARD if index == torch.cuda.current_device() else torch.cuda.device(index)


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _expect(t: torch.Tensor, name: str, dtype: torch.dtype, index: int, shape: tuple) -> int:
    """Address of ``t``, a contiguous ``dtype`` tensor of ``shape`` on CUDA device ``index``."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on cuda:{index}, "
                         f"got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _status_ptr(status: Optional[torch.Tensor], index: int):
    if status is None:
        return None
    if status.dtype is not torch.int32 or status.get_device() != index or status.numel() < 1 or not status.is_contiguous():
        raise ValueError(f"status must be an int32 tensor on cuda:{index}")
    return status.data_ptr()


def _workspace(t: Optional[torch.Tensor], nbytes: int, like: torch.Tensor):
    """(tensor, address, bytes) of the caller's workspace or a new one."""
    if t is None:
        t = like.new_empty(max(nbytes, 16), dtype=torch.uint8)
    elif t.get_device() != like.get_device() or not t.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on {like.device}")
    return t, t.data_ptr(), t.numel() * t.element_size()


def _cache_geometry(kv_cache: torch.Tensor, kv_axis: Optional[int]):
    """(K address, V address, blocks, block size, KV heads, head_dim, block / token / head stride) of one layer's
    5-D tensor, the K/V axis found as in :func:`split_kv_axes`."""
    shape, st = kv_cache.shape, kv_cache.stride()
    if len(shape) != 5:
        raise ValueError(f"Unsupported kv_cache ndim={len(shape)}, expect 5")
    first, second = shape[0] == 2, shape[1] == 2
    if first and second:
        if kv_axis not in (0, 1):
            raise ValueError("Ambiguous KV layout: both dim0 and dim1 have size 2; pass kv_axis")
        first = kv_axis == 0
    elif not (first or second):
        raise ValueError("Unsupported KV layout: expected a dimension with size 2")
    if kv_cache.dtype is not torch.bfloat16 or st[4] != 1:
        raise ValueError("kv_cache must be a bf16 tensor with a contiguous head_dim axis")
    k = kv_cache.data_ptr()
    if first:
        return k, k + 2 * st[0], shape[1], shape[2], shape[3], shape[4], st[1], st[2], st[3]
    return k, k + 2 * st[1], shape[0], shape[2], shape[3], shape[4], st[0], st[2], st[3]


def _check_queries(q: torch.Tensor, num_kv_heads: int, head_dim: int) -> int:
    """Query heads per KV head of ``q`` [N, Hq, D]."""
    if q.dtype is not torch.bfloat16 or q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("q must be a bf16 [N, Hq, D] tensor with a contiguous last axis")
    if q.shape[2] != head_dim:
        raise ValueError(f"q has head_dim {q.shape[2]}, the cache has {head_dim}")
    g, rem = divmod(q.shape[1], num_kv_heads)
    if rem or g <= 0:
        raise ValueError(f"q has {q.shape[1]} heads, not a multiple of the cache's {num_kv_heads} KV heads")
    return g


@functools.lru_cache(maxsize=1024)
def _layer_layout(B, H, g, D, bs, nb, width, block_stride, token_stride, head_stride):
    """One layer's geometry as the library takes it (kept alive by the reference next to it)."""
    layout = PagedLayout(1, B, H, g, D, bs, nb, width, block_stride, token_stride, head_stride, 0, 0)
    return ctypes.byref(layout), layout


@functools.lru_cache(maxsize=1024)
def _attend_bytes(B, H, g, D, bs, nb, width, block_stride, token_stride, head_stride, max_query_len, num_listed):
    ref, _ = _layer_layout(B, H, g, D, bs, nb, width, block_stride, token_stride, head_stride)
    return int(_native.load().triattn_attend_workspace_bytes(ref, max_query_len, num_listed))


def attend_paged(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 query_start_loc: torch.Tensor, max_query_len: int, *, scale: Optional[float] = None,
                 tree_mask: Optional[torch.Tensor] = None, block_list: Optional[torch.Tensor] = None,
                 weight_sums: Optional[torch.Tensor] = None, reset_weight_sums: bool = False,
                 kv_axis: Optional[int] = None, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
    """Attention of a step's query tokens over one layer's paged cache (``triattn_attend_paged``); returns ``(out, lse)``.

    ``q`` ``[N, Hq, D]`` bf16, request ``b`` owning rows ``query_start_loc[b] .. query_start_loc[b + 1] - 1`` (at most
    ``max_query_len`` <= 64); the keys and values of these tokens are already in the cache, in the last slots of the
    request's ``seq_lens[b]`` tokens.  ``max_query_len`` times the group size chooses the kernel: up to 8 rows the
    probabilities enter the product with V in two bf16 parts, above in one, and above 16 a row tile is 128 rows; pass the
    step's own maximum, not the largest there may be.  ``kv_cache`` is the layer's 5-D tensor (see :func:`split_kv_axes`), ``block_table``
    ``[B, width]`` int32.  Every query token sees all earlier tokens; among the request's own tokens it sees token ``j`` if
    bit ``j`` of its ``tree_mask`` word (``[N]`` int64) is set, without a mask the tokens up to itself.

    ``block_list`` ``[B, Hkv, S]`` int32 (:func:`select_blocks`) restricts each KV head to the listed blocks: distinct logical
    indices in any order, negative ones unused, of which the first ``min(S, blocks of the request)`` count.
    ``weight_sums`` ``[num_blocks, Hkv, block_size]`` fp32 receives, per cached token and KV head, the attention weight the
    token got from this call's rows: added to what older tokens have (``reset_weight_sums``: starting anew, for all requests of the
    call - one whose blocks had another owner and others that go on take calls of their own), while the
    request's own tokens always start anew, whatever their slots held (the requests of such a call share no cache
    blocks).  ``out`` ``[N, Hq, D]`` bf16, ``lse`` ``[N, Hq]`` fp32
    (natural log); rows that no request owns are left as they are, and so are the rows of a request with bad lengths, which is
    skipped: in an ``out`` and ``lse`` that this call allocates they hold anything.  ``status`` (int32) collects what
    was skipped, as ``DEV_*`` bits; without it nobody learns of it.  ``workspace``: at least
    :func:`attend_workspace_bytes` bytes that no overlapping call uses.
    """
    lib = _native.load()
    _require_cuda(q, "q")
    index = q.get_device()
    k, v, nb, bs, H, D, s0, s1, s2 = _cache_geometry(kv_cache, kv_axis)
    if kv_cache.get_device() != index:
        raise ValueError(f"kv_cache is on {kv_cache.device}, q on {q.device}")
    g = _check_queries(q, H, D)
    B, N, S = seq_lens.numel(), q.shape[0], 0
    width = block_table.shape[1] if block_table.dim() == 2 else -1
    if B == 0 or width == 0:
        raise ValueError("seq_lens and block_table must not be empty")
    p_lens = _expect(seq_lens, "seq_lens", torch.int32, index, (B,))
    p_table = _expect(block_table, "block_table", torch.int32, index, (B, width))
    p_start = _expect(query_start_loc, "query_start_loc", torch.int32, index, (B + 1,))
    p_tree = None if tree_mask is None else _expect(tree_mask, "tree_mask", torch.int64, index, (N,))
    p_list = None
    if block_list is not None:
        S = block_list.shape[-1] if block_list.dim() == 3 else 0
        if S == 0:
            raise ValueError("block_list must be a [B, Hkv, S] tensor with S > 0")
        p_list = _expect(block_list, "block_list", torch.int32, index, (B, H, S))
    p_sums = None if weight_sums is None else _expect(weight_sums, "weight_sums", torch.float32, index, (nb, H, bs))
    p_status = _status_ptr(status, index)
    geometry = (B, H, g, D, bs, nb, width, s0, s1, s2)
    with _on_device(index):
        if out is None:
            out = q.new_empty(q.shape)
        elif out.dtype is not torch.bfloat16 or out.get_device() != index or out.shape != q.shape or out.stride(2) != 1:
            raise ValueError("out must be a bf16 tensor of q's shape on q's device with a contiguous last axis")
        elif out.data_ptr() == q.data_ptr() and N > 0:
            raise ValueError("out must not be q")
        if lse is None:
            lse = q.new_empty((N, H * g), dtype=torch.float32)
            p_lse = lse.data_ptr()
        else:
            p_lse = _expect(lse, "lse", torch.float32, index, (N, H * g))
        if N == 0:
            return out, lse
        workspace, p_ws, ws_bytes = _workspace(workspace, _attend_bytes(*geometry, max_query_len, S), q)
        _native.check(lib.triattn_attend_paged(
            _layer_layout(*geometry)[0], k, v, p_table, p_lens, p_start, q.data_ptr(), q.stride(0), q.stride(1), N,
            max_query_len, 1.0 / math.sqrt(D) if scale is None else scale, p_tree, p_list, S, p_sums,
            1 if reset_weight_sums else 0, out.data_ptr(), out.stride(0), out.stride(1), p_lse, p_ws, ws_bytes, p_status,
            _raw_stream(index)), "attend_paged")
    return out, lse


def attend_workspace_bytes(layout: PagedLayout, max_query_len: int, num_listed: int = 0) -> int:
    """Bytes of workspace :func:`attend_paged` needs (``num_listed`` = entries per row of a ``block_list``)."""
    return int(_native.load().triattn_attend_workspace_bytes(ctypes.byref(layout), int(max_query_len), int(num_listed)))


def _check_view(view: PagedCacheView, layout: PagedLayout) -> None:
    """The layout handed to the library has to be the view's own: its counts and strides address the cache."""
    for name in ("num_layers", "num_blocks", "block_size", "num_kv_heads", "head_dim", "block_stride", "token_stride", "head_stride"):
        if getattr(layout, name) != getattr(view, name):
            raise ValueError(f"layout has {name} {getattr(layout, name)}, the cache view {getattr(view, name)}")


def evict_paged(view: PagedCacheView, layout: PagedLayout, weight_sums: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor, keep_counts: torch.Tensor, keep_pitch: int, window: int,
                prefill_lens: Optional[torch.Tensor] = None, keep_out: Optional[torch.Tensor] = None,
                status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keep, per layer, request and KV head, the tokens with the largest attention weight sums (``triattn_evict_paged``).

    ``weight_sums`` ``[L, num_blocks, Hkv, block_size]`` fp32, as :func:`attend_paged` fills it layer by layer.  The last
    ``window`` tokens and the first ``prefill_lens[b]`` rank above all others.  K, V and the sums are compacted in place;
    returns keep ``[L, B, Hkv, keep_pitch]`` int32 (ascending, -1 behind ``keep_counts[b]``).
    """
    lib = _native.load()
    _require_cuda(weight_sums, "weight_sums")
    index = weight_sums.get_device()
    _check_view(view, layout)
    L, B, H = view.num_layers, layout.num_reqs, view.num_kv_heads
    if view.k_ptrs.get_device() != index:
        raise ValueError(f"weight_sums is on {weight_sums.device}, the cache on {view.device}")
    p_sums = _expect(weight_sums, "weight_sums", torch.float32, index, (L, view.num_blocks, H, view.block_size))
    p_table = _expect(block_table, "block_table", torch.int32, index, (B, layout.max_blocks_per_req))
    p_lens = _expect(seq_lens, "seq_lens", torch.int32, index, (B,))
    p_counts = _expect(keep_counts, "keep_counts", torch.int32, index, (B,))
    p_prefill = None if prefill_lens is None else _expect(prefill_lens, "prefill_lens", torch.int32, index, (B,))
    p_status = _status_ptr(status, index)
    with _on_device(index):
        if keep_out is None:
            keep_out = weight_sums.new_empty((L, B, H, keep_pitch), dtype=torch.int32)
        p_keep = _expect(keep_out, "keep_out", torch.int32, index, (L, B, H, keep_pitch))
        _native.check(lib.triattn_evict_paged(
            ctypes.byref(layout), view.k_ptrs.data_ptr(), view.v_ptrs.data_ptr(), p_sums, p_table, p_lens, p_counts,
            p_prefill, int(window), p_keep, int(keep_pitch), p_status, _raw_stream(index)), "evict_paged")
    return keep_out


def update_block_bounds(view: PagedCacheView, layout: PagedLayout, bounds: torch.Tensor, block_table: torch.Tensor,
                        first_tokens: torch.Tensor, seq_lens: torch.Tensor, status: Optional[torch.Tensor] = None) -> None:
    """Rebuild the key bounds of every block holding tokens ``first_tokens[b] .. seq_lens[b] - 1``
    (``triattn_update_block_bounds``); ``bounds`` ``[L, num_blocks, Hkv, 2, D]`` bf16 (smallest, largest)."""
    lib = _native.load()
    _require_cuda(bounds, "bounds")
    index, B = bounds.get_device(), layout.num_reqs
    _check_view(view, layout)
    if view.k_ptrs.get_device() != index:
        raise ValueError(f"bounds is on {bounds.device}, the cache on {view.device}")
    p_bounds = _expect(bounds, "bounds", torch.bfloat16, index,
                       (view.num_layers, view.num_blocks, view.num_kv_heads, 2, view.head_dim))
    p_table = _expect(block_table, "block_table", torch.int32, index, (B, layout.max_blocks_per_req))
    p_first = _expect(first_tokens, "first_tokens", torch.int32, index, (B,))
    p_lens = _expect(seq_lens, "seq_lens", torch.int32, index, (B,))
    p_status = _status_ptr(status, index)
    with _on_device(index):
        _native.check(lib.triattn_update_block_bounds(
            ctypes.byref(layout), view.k_ptrs.data_ptr(), p_table, p_first, p_lens, p_bounds, p_status,
            _raw_stream(index)), "update_block_bounds")


def select_blocks(q: torch.Tensor, bounds: torch.Tensor, seq_lens: torch.Tensor, query_start_loc: torch.Tensor,
                  block_table: torch.Tensor, max_query_len: int, block_size: int, num_selected: int, *,
                  sink_blocks: int = 1, recent_blocks: int = 2, block_list: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The ``num_selected`` blocks per request and KV head with the largest bound of the attention logits, summed over
    the request's query tokens and the group's heads (``triattn_select_blocks``).

    ``bounds`` ``[num_blocks, Hkv, 2, D]``: one layer of :func:`update_block_bounds`.  The first ``sink_blocks``, the last
    ``recent_blocks`` and the blocks of the query's own tokens are always among them, so these must fit.  Returns
    ``[B, Hkv, num_selected]`` int32, ascending, -1 behind the request's last block.
    """
    lib = _native.load()
    _require_cuda(q, "q")
    index = q.get_device()
    if bounds.dim() != 4:
        raise ValueError("bounds must be a [num_blocks, Hkv, 2, D] tensor")
    nb, H, _, D = bounds.shape
    g = _check_queries(q, H, D)
    B, width = seq_lens.numel(), block_table.shape[1] if block_table.dim() == 2 else -1
    if B == 0 or width == 0:
        raise ValueError("seq_lens and block_table must not be empty")
    p_bounds = _expect(bounds, "bounds", torch.bfloat16, index, (nb, H, 2, D))
    p_lens = _expect(seq_lens, "seq_lens", torch.int32, index, (B,))
    p_table = _expect(block_table, "block_table", torch.int32, index, (B, width))
    p_start = _expect(query_start_loc, "query_start_loc", torch.int32, index, (B + 1,))
    if block_size <= 0:
        raise ValueError(f"block_size must be positive, got {block_size}")
    own = (max_query_len + block_size - 2) // block_size + 1
    if num_selected < sink_blocks + max(recent_blocks, own):
        raise ValueError(f"num_selected={num_selected} cannot hold {sink_blocks} sink and {max(recent_blocks, own)} recent blocks")
    p_status = _status_ptr(status, index)
    # strides play no part in the choice: any that pass the layout check
    ref, _ = _layer_layout(B, H, g, D, block_size, nb, width, block_size * H * D, H * D, D)
    with _on_device(index):
        if block_list is None:
            block_list = q.new_empty((B, H, num_selected), dtype=torch.int32)
        p_list = _expect(block_list, "block_list", torch.int32, index, (B, H, num_selected))
        workspace, p_ws, ws_bytes = _workspace(workspace, (B * H * width * 4 + 255) // 256 * 256, q)
        _native.check(lib.triattn_select_blocks(
            ref, q.data_ptr(), q.stride(0), q.stride(1), q.shape[0], max_query_len, p_start, p_bounds, p_table, p_lens,
            num_selected, sink_blocks, recent_blocks, p_list, p_ws, ws_bytes, p_status, _raw_stream(index)), "select_blocks")
    return block_list


def select_blocks_workspace_bytes(layout: PagedLayout) -> int:
    """Bytes of workspace :func:`select_blocks` needs."""
    return int(_native.load().triattn_select_blocks_workspace_bytes(ctypes.byref(layout)))
