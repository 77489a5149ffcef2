"""A key/value cache in pages: append, read back, trim-on-reject.

The paged counterparts of ``GorgonKVCache``'s operators
(``src/gorgon/inference/kv_cache.py:21-108`` keeps one contiguous tensor per
layer).  Pages hold the rows' own dtype, or 8 bits per value (int8 or
float8_e4m3fn) with one float32 scale per row and kv head; quantisation happens
as rows are written, in the same launch.

``paged_cache_append``, ``paged_cache_read`` and ``paged_cache_trim`` take the
tensors; ``PagedKVCache`` holds them for all layers of a model.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _abi
from .._paged import call, compute_dtype, device_index, int32, packer, pool_fields
from .._util import gorgon_dtype
from ..kernels.paged_attention import paged_attention

_APPEND = packer("PqqqPqqqqqP")
_READ = packer("iPqqPqqqPP")
_TRIM = packer("qqqqqPqqPP")


def paged_cache_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                       block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                       k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                       cu_q: Optional[torch.Tensor] = None) -> None:
    """Writes new rows of K and V as the last rows of each sequence.

    ``k``, ``v`` are ``[B, Hkv, n, D]``, or with ``cu_q`` (int ``[B + 1]``) packed
    ``[total, Hkv, D]``; ``seq_lens[b]`` counts sequence ``b``'s rows with the new
    ones, 0 for an unused slot.  Pages, scales and the block table are
    ``paged_attention``'s.  8-bit pages get, per row and head, the bytes
    ``round(x * inv)`` and the scale ``1 / inv``, with ``inv = largest / amax`` cut to
    12 significant bits (``largest`` 127 for int8, 448 for e4m3); a row with an
    infinity or a NaN reads back as NaN.  Two sequences of one call, or
    two kv heads (by a stride of 0), must not share the page row that they write."""
    dev = device_index("k, v, pages, block_table and seq_lens", k, v, k_pages, v_pages, block_table, seq_lens, k_scale,
                       v_scale, cu_q)
    dtype = compute_dtype(k.dtype, "k")
    if v.dtype is not dtype or v.shape != k.shape:
        raise RuntimeError(f"k and v must have one shape and dtype, got {tuple(k.shape)} {k.dtype} and "
                           f"{tuple(v.shape)} {v.dtype}")
    table = int32(block_table, "block_table", 2)
    lens = int32(seq_lens, "seq_lens", 1)
    if k.stride(-1) != 1:
        k = k.contiguous()
    if v.stride(-1) != 1:
        v = v.contiguous()
    batch = table.shape[0]
    shape = k.shape
    cu = None
    if cu_q is not None:
        cu = int32(cu_q, "cu_q", 1)
        if len(shape) != 3 or cu.shape[0] != batch + 1:
            raise RuntimeError(f"with cu_q [batch + 1], k must be [total, heads_kv, head_dim], got {tuple(shape)} and "
                               f"{cu.shape[0]} entries for {batch} sequences")
        rows, heads, d = shape
        n = 0
        (k_sn, k_sh, _), (v_sn, v_sh, _), k_sb, v_sb = k.stride(), v.stride(), 0, 0
    else:
        if len(shape) != 4 or shape[0] != batch:
            raise RuntimeError(f"k must be [batch, heads_kv, n, head_dim] with block_table's {batch} sequences, got "
                               f"{tuple(shape)}")
        _, heads, n, d = shape
        rows = 0
        (k_sb, k_sh, k_sn, _), (v_sb, v_sh, v_sn, _) = k.stride(), v.stride()
    pool = pool_fields(dtype, k_pages, v_pages, table, lens, batch, k_scale, v_scale)
    if pool[4] != heads or pool[5] != d:
        raise RuntimeError(f"k has {heads} heads of {d}, the pages {pool[4]} of {pool[5]}")
    params = _APPEND.pack(*pool, k.data_ptr(), k_sb, k_sh, k_sn, v.data_ptr(), v_sb, v_sh, v_sn, n, rows,
                          0 if cu is None else cu.data_ptr())
    rc = call(dev, _abi.lib().gorgon_paged_append, params)
    if rc:
        _abi.check(rc, "gorgon_paged_append")


def paged_cache_read(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, cu_rows: torch.Tensor,
                     rows: int, *, starts: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
                     out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of the cache as ragged ``(k, v)`` ``[rows, Hkv, D]``, the form that
    ``tree_attention`` takes with ``cu_seqlens``: row ``cu_rows[b] + i`` is position
    ``starts[b] + i`` (default 0) of sequence ``b``.  ``rows`` sizes the result; rows
    from ``cu_rows[B]`` on are not written (a given ``out`` pair, any strides with
    ``D`` contiguous, keeps them).  ``dtype`` is the result's: default the pages'
    own, or bfloat16 for 8-bit pages.  8-bit values are multiplied by their scale
    in fp32 and rounded once, to the type's largest finite value at most."""
    dev = device_index("pages, block_table and cu_rows", k_pages, v_pages, block_table, cu_rows, starts, k_scale,
                       v_scale, *(out or ()))
    native = k_pages.dtype not in (torch.int8, torch.float8_e4m3fn)
    if out is not None:
        dtype = out[0].dtype if dtype is None else dtype
    elif dtype is None:
        dtype = k_pages.dtype if native else torch.bfloat16
    compute_dtype(dtype, "dtype")
    held = compute_dtype(k_pages.dtype, "k_pages") if native else dtype
    table = int32(block_table, "block_table", 2)
    cu = int32(cu_rows, "cu_rows", 1)
    batch = table.shape[0]
    if cu.shape[0] != batch + 1:
        raise RuntimeError(f"cu_rows has {cu.shape[0]} entries for {batch} sequences")
    if starts is not None:
        starts = int32(starts, "starts", 1)
        if starts.shape[0] != batch:
            raise RuntimeError(f"starts has {starts.shape[0]} entries for {batch} sequences")
    if rows < 0:
        raise RuntimeError("rows must not be negative")
    pool = pool_fields(held, k_pages, v_pages, table, None, batch, k_scale, v_scale)
    shape = (rows, pool[4], pool[5])
    if out is None:
        on = k_pages.device
        k, v = torch.empty(shape, dtype=dtype, device=on), torch.empty(shape, dtype=dtype, device=on)
    else:
        k, v = out
        for x in out:
            if x.shape != shape or x.dtype is not dtype or (x.stride(-1) != 1 and shape[2] > 1):
                raise RuntimeError(f"out must be two tensors {shape} of {dtype} with a contiguous last dimension")
    (k_sn, k_sh, _), (v_sn, v_sh, _) = k.stride(), v.stride()
    params = _READ.pack(*pool, gorgon_dtype(dtype), k.data_ptr(), k_sn, k_sh, v.data_ptr(), v_sn, v_sh, rows,
                        cu.data_ptr(), 0 if starts is None else starts.data_ptr())
    rc = call(dev, _abi.lib().gorgon_paged_read, params)
    if rc:
        _abi.check(rc, "gorgon_paged_read")
    return k, v


def paged_cache_trim(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, src_idx: torch.Tensor,
                     lens: torch.Tensor, dst_start: Union[torch.Tensor, int, None] = None, *,
                     k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> None:
    """Trim-on-reject in place, every layer in one launch: position
    ``dst_start[b] + r`` of sequence ``b`` takes position ``src_idx[b, r]`` for
    ``r < lens[b]``, in every layer and head, as stored (bytes and scales).
    ``GorgonKVCache.trim``'s arguments, over ``[layers, pages, Hkv, page_size, D]``
    (or one layer's ``[pages, Hkv, page_size, D]``); ``dst_start`` ``[B]``, an int, or
    None for 0.  At most 256 columns; few are faster, whatever ``lens`` (of a
    verifier's path pass the first ``max_depth + 1``).  A bad index sets the device
    error bits and leaves its sequence as it is.  A call must not name a sequence
    twice, nor move rows into pages that another of its sequences reads; pages
    expanded over layers or kv heads (strides of 0) are refused."""
    dev = device_index("pages, block_table, src_idx and lens", k_pages, v_pages, block_table, src_idx, lens, k_scale,
                       v_scale, dst_start if isinstance(dst_start, torch.Tensor) else None)
    lead = 1 if k_pages.dim() == 5 else 0
    native = k_pages.dtype not in (torch.int8, torch.float8_e4m3fn)
    held = compute_dtype(k_pages.dtype, "k_pages") if native else torch.bfloat16
    table = int32(block_table, "block_table", 2)
    idx = int32(src_idx.unsqueeze(0) if src_idx.dim() == 1 else src_idx, "src_idx", 2)
    ln = int32(lens if lens.dim() == 1 else lens.reshape(-1), "lens", 1)
    batch = table.shape[0]
    if idx.shape[0] != batch or ln.shape[0] != batch:
        raise RuntimeError("src_idx and lens need one row per sequence")
    if dst_start is None:
        ds = None
    elif isinstance(dst_start, int):
        ds = torch.full((batch,), dst_start, dtype=torch.int32, device=k_pages.device)
    else:
        ds = int32(dst_start if dst_start.dim() == 1 else dst_start.reshape(-1), "dst_start", 1)
        if ds.shape[0] != batch:
            raise RuntimeError("dst_start needs one entry per sequence")
    pool = pool_fields(held, k_pages, v_pages, table, None, batch, k_scale, v_scale, lead)
    if lead:
        layers, k_sl, v_sl = k_pages.shape[0], k_pages.stride(0), v_pages.stride(0)
        ks_sl, vs_sl = (0, 0) if native else (k_scale.stride(0), v_scale.stride(0))
    else:
        layers, k_sl, v_sl, ks_sl, vs_sl = 1, 0, 0, 0, 0
    params = _TRIM.pack(*pool, layers, k_sl, v_sl, ks_sl, vs_sl, idx.data_ptr(), idx.stride(0), idx.shape[1],
                        ln.data_ptr(), 0 if ds is None else ds.data_ptr())
    rc = call(dev, _abi.lib().gorgon_paged_trim, params)
    if rc:
        _abi.check(rc, "gorgon_paged_trim")


class PagedKVCache:
    """The pages of every layer of a model, and the operators on them.

    ``k_pages``, ``v_pages`` ``[layers, pages, Hkv, page_size, D]`` and, for
    ``storage`` "int8" or "fp8", ``k_scale``, ``v_scale``
    ``[layers, pages, Hkv, page_size]``.  Which page belongs to which sequence is the
    caller's block table, passed to every call (it changes from step to step; the
    pages do not move, so calls captured in a CUDA graph stay valid)."""

    _STORAGE = {"native": None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}

    def __init__(self, layers: int, num_pages: int, page_size: int, heads_kv: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, storage: str = "native",
                 device: Union[torch.device, str, None] = None) -> None:
        if storage not in self._STORAGE:
            raise RuntimeError(f"storage must be one of {sorted(self._STORAGE)}")
        self.dtype = compute_dtype(dtype, "dtype")
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise ValueError("PagedKVCache lives on a CUDA device.")
        held = self._STORAGE[storage]
        shape = (layers, num_pages, heads_kv, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=held or dtype, device=dev)
        self.v_pages = torch.zeros(shape, dtype=held or dtype, device=dev)
        self.k_scale = None if held is None else torch.zeros(shape[:-1], dtype=torch.float32, device=dev)
        self.v_scale = None if held is None else torch.zeros(shape[:-1], dtype=torch.float32, device=dev)

    def layer(self, i: int) -> dict:
        """Layer ``i``'s tensors under ``paged_attention``'s argument names."""
        return dict(k_pages=self.k_pages[i], v_pages=self.v_pages[i],
                    k_scale=None if self.k_scale is None else self.k_scale[i],
                    v_scale=None if self.v_scale is None else self.v_scale[i])

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               cu_q: Optional[torch.Tensor] = None) -> None:
        paged_cache_append(k, v, block_table=block_table, seq_lens=seq_lens, cu_q=cu_q, **self.layer(layer))

    def attend(self, layer: int, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, **options):
        """``paged_attention`` over layer ``layer`` (its keyword arguments pass through)."""
        return paged_attention(q, block_table=block_table, seq_lens=seq_lens, **self.layer(layer), **options)

    def read(self, layer: int, block_table: torch.Tensor, cu_rows: torch.Tensor, rows: int,
             starts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        return paged_cache_read(block_table=block_table, cu_rows=cu_rows, rows=rows, starts=starts, dtype=self.dtype,
                                **self.layer(layer))

    def trim(self, block_table: torch.Tensor, src_idx: torch.Tensor, lens: torch.Tensor,
             dst_start: Union[torch.Tensor, int, None] = None) -> None:
        paged_cache_trim(self.k_pages, self.v_pages, block_table, src_idx, lens, dst_start, k_scale=self.k_scale,
                         v_scale=self.v_scale)
