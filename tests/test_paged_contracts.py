"""What the paged operators' documentation promises at its edges (no GPU needed)."""
from __future__ import annotations

import ctypes

import pytest

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


def _trim(storage=_abi.KV_NATIVE, **kw):
    t = _abi.PagedTrimParams()
    _kv(t.kv, storage=storage, head_dim=64)
    t.layers, t.max_len, t.src_idx, t.lens = 3, 8, 4096, 4096
    strides = dict(l=10 ** 6, p=2048, h=1024, s=64)
    for kind, unit in (("k", 64), ("v", 64), ("ks", 1), ("vs", 1)):
        for d, x in strides.items():
            setattr(t if d == "l" else t.kv, f"{kind}_stride_{d}", x // 64 * unit)
    t.kv.k_scale = t.kv.v_scale = 4096
    for name, x in kw.items():
        setattr(t if hasattr(t, name) else t.kv, name, x)
    return t


@pytest.mark.parametrize("kind", ["k", "v", "ks", "vs"])
@pytest.mark.parametrize("dim", ["l", "p", "h", "s"])
def test_trim_refuses_rows_that_are_one_in_memory(kind, dim):
    lib = _abi.lib()
    t = _trim(_abi.KV_INT8, **{f"{kind}_stride_{dim}": 0})
    rc, msg = _err(lib.gorgon_paged_trim(ctypes.byref(t), None))
    assert rc == _abi.GORGON_ERR_UNSUPPORTED and "stride of 0" in msg
