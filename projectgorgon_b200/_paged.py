"""Argument checks and parameter packing shared by the paged-cache operators.

These operators run once per layer and step, where a call's host time can
exceed its GPU time, so their checks read each tensor attribute once, and a
call's parameters are packed in one ``struct.pack`` (the layouts of
``_abi.PagedKV`` and the structures around it) rather than field by field.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from . import _abi
from ._util import gorgon_dtype

KV_FORMAT = "@ii4q" + "Pqqq" * 4 + "PqqPq"
_STORAGE = {torch.int8: _abi.KV_INT8, torch.float8_e4m3fn: _abi.KV_E4M3}
_COMPUTE = {torch.bfloat16: _abi.BF16, torch.float16: _abi.F16, torch.float32: _abi.F32}
_NO_SCALES = (0, 0, 0, 0, 0, 0, 0, 0)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def packer(tail: str) -> struct.Struct:
    return struct.Struct(KV_FORMAT + tail)


def device_index(what: str, *tensors: Optional[torch.Tensor]) -> int:
    """The CUDA device that every given tensor is on (None is skipped):
    ValueError for host tensors, RuntimeError for mixed devices."""
    dev = -1
    for t in tensors:
        if t is None:
            continue
        d = t.get_device() if isinstance(t, torch.Tensor) else -1
        if d != dev or d < 0:
            if d < 0:
                raise ValueError(f"{what} must be CUDA tensors.")
            if dev >= 0:
                raise RuntimeError(f"{what} must be on one device")
            dev = d
    return dev


def call(dev: int, fn, params: bytes, *more) -> int:
    """``fn(params, *more, stream)`` on torch's current stream of device ``dev``."""
    if torch._C._cuda_getDevice() == dev:
        return fn(params, *more, _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream)
    with torch.cuda.device(dev):
        return fn(params, *more, torch.cuda.current_stream(dev).cuda_stream)


def int32(t: torch.Tensor, name: str, dims: int) -> torch.Tensor:
    """`t` as int32 with its last dimension contiguous."""
    if t.dim() != dims:
        raise RuntimeError(f"{name} must have {dims} dimension(s), got {tuple(t.shape)}")
    if t.dtype is not torch.int32:
        if t.dtype is not torch.int64:
            raise RuntimeError(f"{name} must be int32 or int64, got {t.dtype}")
        t = t.to(torch.int32)
    return t if t.is_contiguous() or t.stride(-1) == 1 else t.contiguous()


def pool_fields(dtype: torch.dtype, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                lens: Optional[torch.Tensor], batch: int, k_scale: Optional[torch.Tensor],
                v_scale: Optional[torch.Tensor], lead: int = 0) -> Tuple:
    """The values of a ``_abi.PagedKV``, in order.  ``lead`` counts leading
    (layer) dimensions of the pages and scales; ``table`` is int32 already."""
    shape, ks, vs, held = k_pages.shape, k_pages.stride(), v_pages.stride(), k_pages.dtype
    if len(shape) != 4 + lead or v_pages.shape != shape:
        raise RuntimeError(f"k_pages and v_pages must both be [pages, heads_kv, page_size, head_dim], got "
                           f"{tuple(shape)} and {tuple(v_pages.shape)}")
    if v_pages.dtype is not held:
        raise RuntimeError(f"k_pages and v_pages must have one dtype, got {held} and {v_pages.dtype}")
    pages, heads, size, d = shape[lead:] if lead else shape
    if (ks[-1] != 1 or vs[-1] != 1) and d > 1:
        raise RuntimeError("the pages' head_dim must be contiguous")
    if heads < 1 or size < 1:
        raise RuntimeError(f"pages need at least one head and one row, got {tuple(shape)}")
    rows, cols = table.shape
    if rows != batch:
        raise RuntimeError(f"block_table has {rows} rows for {batch} sequences")
    if lens is not None and len(lens) != batch:
        raise RuntimeError(f"seq_lens has {len(lens)} entries for {batch} sequences")
    storage = _STORAGE.get(held)
    if storage is None:
        storage, scales = 0, _NO_SCALES
        if k_scale is not None or v_scale is not None:
            raise RuntimeError("scales belong to 8-bit pages only")
        if held is not dtype:
            raise RuntimeError(f"pages of {held} with rows of {dtype}")
    else:
        if k_scale is None or v_scale is None:
            raise RuntimeError("8-bit pages need k_scale and v_scale")
        want = shape[:-1]
        if k_scale.shape != want or v_scale.shape != want or k_scale.dtype is not torch.float32 \
                or v_scale.dtype is not torch.float32:
            raise RuntimeError(f"k_scale and v_scale must be float32 {tuple(want)}")
        a, b = k_scale.stride(), v_scale.stride()
        scales = (k_scale.data_ptr(), a[lead], a[lead + 1], a[lead + 2],
                  v_scale.data_ptr(), b[lead], b[lead + 1], b[lead + 2])
    return (gorgon_dtype(dtype), storage, pages, size, heads, d,
            k_pages.data_ptr(), ks[lead], ks[lead + 1], ks[lead + 2],
            v_pages.data_ptr(), vs[lead], vs[lead + 1], vs[lead + 2], *scales,
            table.data_ptr(), table.stride(0), cols, 0 if lens is None else lens.data_ptr(), batch)


def compute_dtype(dtype: torch.dtype, name: str) -> torch.dtype:
    if dtype not in _COMPUTE:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {dtype}")
    return dtype
