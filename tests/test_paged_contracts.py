"""What the paged operators' documentation promises at its edges (no GPU needed)."""
from __future__ import annotations

import ctypes

from projectgorgon_b200 import _abi
from test_paged import _err, _kv


def test_attention_that_has_something_to_write_needs_its_pointers():
    """Packed rows with n = 0 are written (as too many), so a null out is refused; rows of no values have a log-sum-exp."""
    lib = _abi.lib()
    n = _abi.PagedAttnParams()
    _kv(n.kv)
    n.heads_q, n.n, n.cu_q, n.rows = 2, 0, 4096, 5
    rc, msg = _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))
    assert rc == _abi.GORGON_ERR_INVALID and "null" in msg
    n.rows = 0
    assert lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None) == 0
    n.cu_q = None
    assert lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None) == 0
    n = _abi.PagedAttnParams()
    _kv(n.kv, head_dim=0, seq_lens=None)
    n.heads_q, n.n = 2, 1
    assert lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None) == 0
    n.lse = 4096
    rc, msg = _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))
    assert rc == _abi.GORGON_ERR_INVALID and "null" in msg
    n.kv.seq_lens, n.kv.block_table = 4096, None
    rc, msg = _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))
    assert rc == _abi.GORGON_ERR_INVALID and "null" in msg
