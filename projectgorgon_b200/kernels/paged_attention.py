"""Attention of new tokens over a key/value cache in pages.

``paged_attention`` is ``tree_attention`` for a server's cache: K and V lie in
fixed-size pages (in 16 bits, or in 8 with a scale per row and head), a block
table names each sequence's pages, and the new rows -- one token, a chunk of a
prompt, or a draft tree -- attend to the cached rows and to each other, all of
them or a sliding window and the first few.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch

from .. import _abi
from .._paged import call, compute_dtype, device_index, int32, packer, pool_fields
from .._util import parents_tensor

_ATTN = packer("qqq" + "Pqqq" * 3 + "PPqiqqfi")
_BACKENDS = {"auto": _abi.PAGED_AUTO, "simt": _abi.PAGED_SIMT, "mma": _abi.PAGED_MMA,
             "tcgen05": _abi.PAGED_TCGEN05}
_MANY = 2 ** 31 - 1  # more than any sequence has: options above it mean the same


def _workspace_size_on(dev: int, params: bytes) -> int:
    with torch.cuda.device(dev):  # the schedule counts the current device's SMs
        return _abi.lib().gorgon_paged_attn_workspace_size(params)


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    cu_q: Optional[torch.Tensor] = None,
    max_q: Optional[int] = None,
    parents: Union[Sequence[int], torch.Tensor, None] = None,
    max_depth: Optional[int] = None,
    window: Optional[int] = None,
    sinks: int = 0,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    backend: str = "auto",
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Softmax attention of each sequence's new rows over its pages.

    q            ``[B, Hq, n, D]``, ``n`` new rows per sequence, or with ``cu_q``
                 (int ``[B + 1]``) packed ``[total, Hq, D]``: sequence ``b``'s are
                 rows ``cu_q[b] .. cu_q[b + 1] - 1``, at most ``max_q`` of them
                 (default: ``total``, for which single tokens run on the
                 kernel for chunks: give the bound)
    k_pages, v_pages  ``[pages, Hkv, page_size, D]`` of q's dtype, or int8 /
                 float8_e4m3fn with ``k_scale``, ``v_scale`` float32
                 ``[pages, Hkv, page_size]``; any strides, ``D`` contiguous.  The
                 new rows' K and V are in them already (``paged_cache_append``).
    block_table  int ``[B, columns]``: position ``p`` of a sequence lies in page
                 ``block_table[b, p // page_size]``; unused entries may hold anything
    seq_lens     int ``[B]``: rows of each sequence, its new ones last; 0 marks an
                 unused slot, whose output rows are 0 (log-sum-exp ``-inf``)
    Integer tensors are int32, or int64 with values that fit 32 bits.

    Query head ``h`` reads kv head ``h // (Hq // Hkv)``.  A new row sees the
    cached rows and the new rows up to itself; with ``parents`` (``[n]`` or
    ``[B, n]``, -1 for a root; with ``cu_q`` ``n`` is ``max_q``, and a sequence's tree
    the first of them) the cached rows, itself and its ancestors within
    ``max_depth`` hops.  ``window`` hides rows ``window`` or more positions before
    a row's own (a tree row's position is the cached length plus its depth),
    except the first ``sinks`` rows.  Hidden rows contribute nothing, even when
    they hold infinities or NaN (an 8-bit row holds NaN in its scale, as
    ``paged_cache_append`` writes it; a page filled otherwise must have no e4m3 NaN
    among its bytes).  ``scale`` (default ``D ** -0.5``) is positive.

    Returns ``out`` shaped like ``q``, and with ``return_lse`` also the
    natural-log sum of exponentials, float32 ``[B, Hq, n]`` (packed:
    ``[total, Hq]``).  Packed rows from ``cu_q[B]`` on are not written: a given
    ``out`` keeps them.  16-bit rows of head_dim 64 or 128 in whole 16-byte pieces,
    and 8-bit pages of such, run on the tensor cores; trees of more than 256 nodes
    there pass the cache once per 16 (row, head) pairs.  Everything else, and calls
    whose table's columns times rows of ``max_q`` pass 2^31 units of work, runs on
    the CUDA cores, far slower.  All lengths stay on the device, so a call can be captured
    in a CUDA graph and replayed with other lengths (within the block table).
    """
    dev = device_index("q, pages, block_table and seq_lens", q, k_pages, v_pages, block_table, seq_lens, k_scale,
                       v_scale, cu_q, out)
    dtype = compute_dtype(q.dtype, "q")
    be = _BACKENDS.get(backend)
    if be is None:
        raise RuntimeError(f"backend must be one of {sorted(_BACKENDS)}")
    table = int32(block_table, "block_table", 2)
    lens = int32(seq_lens, "seq_lens", 1)
    if q.stride(-1) != 1:
        q = q.contiguous()
    shape = q.shape
    batch = table.shape[0]
    if cu_q is not None:
        cu = int32(cu_q, "cu_q", 1)
        if len(shape) != 3 or cu.shape[0] != batch + 1:
            raise RuntimeError(f"with cu_q [batch + 1], q must be [total, heads_q, head_dim], got {tuple(shape)} and "
                               f"{cu.shape[0]} entries for {batch} sequences")
        total, hq, d = shape
        n = total if max_q is None else min(int(max_q), total)
        if n < 0:
            raise RuntimeError("max_q must not be negative")
        q_sn, q_sh, _ = q.stride()
        q_sb = 0
    else:
        cu = None
        if len(shape) != 4 or shape[0] != batch:
            raise RuntimeError(f"q must be [batch, heads_q, n, head_dim] with block_table's {batch} sequences, got "
                               f"{tuple(shape)}")
        _, hq, n, d = shape
        q_sb, q_sh, q_sn, _ = q.stride()
    pool = pool_fields(dtype, k_pages, v_pages, table, lens, batch, k_scale, v_scale)
    if pool[5] != d:
        raise RuntimeError(f"q has head_dim {d}, the pages {pool[5]}")
    if hq % pool[4] != 0:
        raise RuntimeError(f"heads_q ({hq}) must be a multiple of heads_kv ({pool[4]})")
    if out is None:
        out = torch.empty_like(q)
        if out.stride(-1) != 1:
            out = torch.empty(shape, dtype=dtype, device=q.device)
    elif out.shape != shape or out.dtype is not dtype or (out.stride(-1) != 1 and d > 1):
        raise RuntimeError(f"out must be {tuple(shape)} of {dtype} with a contiguous last dimension")
    if cu is not None:
        o_sn, o_sh, _ = out.stride()
        o_sb = 0
    else:
        o_sb, o_sh, o_sn, _ = out.stride()
    lse, l_ptr, l_sb, l_sh, l_sn = None, 0, 0, 0, 0
    if return_lse:
        lse = torch.empty(shape[:-1], dtype=torch.float32, device=q.device)
        l_ptr = lse.data_ptr()
        l_sb, l_sh, l_sn = (0, 1, hq) if cu is not None else lse.stride()
    par, p_ptr, p_sb = None, 0, 0
    if parents is not None:
        par = parents_tensor(parents, q.device)
        if cu is not None:
            n = 0 if total == 0 else par.shape[-1] if max_q is None else int(max_q)  # (may pass the packed rows' count)
        if par.dim() == 1 and (par.shape[0] == n or n == 0):
            p_sb = 0
        elif par.dim() == 2 and par.shape[0] == batch and (par.shape[1] == n or n == 0):
            p_sb = par.stride(0)
        else:
            raise RuntimeError(f"parents must be [{n}] or [{batch}, {n}], got {tuple(par.shape)}")
        p_ptr = par.data_ptr()
    if window is not None and window < 1:
        raise RuntimeError(f"window must be at least 1, got {window}")
    if scale is not None and not 0.0 < scale < math.inf:
        raise RuntimeError(f"scale must be positive and finite, got {scale}")
    if sinks < 0:
        raise RuntimeError(f"sinks must not be negative, got {sinks}")
    params = _ATTN.pack(*pool, hq, n, 0 if cu is None else total, q.data_ptr(), q_sb, q_sh, q_sn, out.data_ptr(), o_sb, o_sh, o_sn,
                        l_ptr, l_sb, l_sh, l_sn, 0 if cu is None else cu.data_ptr(), p_ptr, p_sb,
                        -1 if max_depth is None else min(int(max_depth), _MANY), 0 if window is None else min(int(window), _MANY),
                        min(int(sinks), _MANY),
                        0.0 if scale is None else float(scale), be)
    lib = _abi.lib()
    nbytes = lib.gorgon_paged_attn_workspace_size(params) if dev == torch._C._cuda_getDevice() else \
        _workspace_size_on(dev, params)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    rc = call(dev, lib.gorgon_paged_attn, params, ws.data_ptr() if nbytes else 0, nbytes)
    if rc:
        _abi.check(rc, "gorgon_paged_attn")
    return (out, lse) if return_lse else out
