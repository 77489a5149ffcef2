"""The paged operators' refusals and parameter layouts (no GPU needed)."""
from __future__ import annotations

import ctypes
import importlib
import shutil
import subprocess

import pytest
import torch

import projectgorgon_b200 as G
from conftest import ROOT
from projectgorgon_b200 import _abi
from projectgorgon_b200.inference import paged_cache as pc

pa = importlib.import_module("projectgorgon_b200.kernels.paged_attention")

STRUCTS = {"gorgon_paged_kv": _abi.PagedKV, "gorgon_paged_append_params": _abi.PagedAppendParams,
           "gorgon_paged_read_params": _abi.PagedReadParams, "gorgon_paged_trim_params": _abi.PagedTrimParams,
           "gorgon_paged_attn_params": _abi.PagedAttnParams}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_ctypes_layout_matches_c_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "gorgon_b200.h"', "int main(void){"]
    for cname, cls in STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        for fname, _ in cls._fields_:
            lines.append(f'printf("{cname}.{fname} %zu\\n", offsetof({cname}, {fname}));')
    lines.append("return 0;}")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    got = dict(l.split() for l in out if l)
    for cname, cls in STRUCTS.items():
        assert int(got[cname]) == ctypes.sizeof(cls), cname
        for fname, _ in cls._fields_:
            assert int(got[f"{cname}.{fname}"]) == getattr(cls, fname).offset, (cname, fname)


@pytest.mark.parametrize("pack,cls", [(pa._ATTN, _abi.PagedAttnParams), (pc._APPEND, _abi.PagedAppendParams),
                                      (pc._READ, _abi.PagedReadParams), (pc._TRIM, _abi.PagedTrimParams)])
def test_packed_parameters_are_the_structure(pack, cls):
    """Every field's own value comes out of the packed bytes."""
    def leaves(c, at=0):
        for name, t in c._fields_:
            off = at + getattr(c, name).offset
            if issubclass(t, ctypes.Structure):
                yield from leaves(t, off)
            else:
                yield off, t
    fields = list(leaves(cls))
    data = pack.pack(*[float(i + 1) if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(fields)])
    assert len(data) == ctypes.sizeof(cls)
    for i, (off, t) in enumerate(fields):
        assert t.from_buffer_copy(data, off).value == i + 1


def test_host_tensors_are_refused():
    kp = torch.zeros(2, 1, 16, 64)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        G.paged_attention(torch.zeros(1, 1, 1, 64), kp, kp, table, lens)
    with pytest.raises(ValueError):
        G.paged_cache_append(torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, 1, 64), kp, kp, table, lens)
    with pytest.raises(ValueError):
        G.paged_cache_read(kp, kp, table, torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(ValueError):
        G.paged_cache_trim(kp, kp, table, table, lens)
    with pytest.raises(ValueError):
        G.PagedKVCache(1, 2, 16, 1, 64, device="cpu")
    with pytest.raises(RuntimeError, match="storage"):
        G.PagedKVCache(1, 2, 16, 1, 64, storage="int4")


def _err(rc):
    return rc, _abi.lib().gorgon_last_error().decode()


def _kv(kv, **kw):
    base = dict(dtype=_abi.BF16, storage=_abi.KV_NATIVE, num_pages=4, page_size=16, heads_kv=2, head_dim=64, k_pages=4096,
                v_pages=4096, block_table=4096, table_stride_b=2, table_cols=2, seq_lens=4096, batch=1)
    base.update(kw)
    for k, v in base.items():
        setattr(kv, k, v)


@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=9), _abi.GORGON_ERR_INVALID, "dtype"), (dict(storage=3), _abi.GORGON_ERR_INVALID, "storage"),
    (dict(page_size=0), _abi.GORGON_ERR_INVALID, "size"), (dict(heads_kv=0), _abi.GORGON_ERR_INVALID, "size"),
    (dict(num_pages=-1), _abi.GORGON_ERR_INVALID, "size"), (dict(batch=-1), _abi.GORGON_ERR_INVALID, "size"),
    (dict(head_dim=257), _abi.GORGON_ERR_UNSUPPORTED, "head_dim"), (dict(batch=65536), _abi.GORGON_ERR_UNSUPPORTED, "batch"),
    (dict(table_cols=1 << 27), _abi.GORGON_ERR_UNSUPPORTED, "2^30"), (dict(k_pages=None), _abi.GORGON_ERR_INVALID, "null"),
    (dict(block_table=None), _abi.GORGON_ERR_INVALID, "null"), (dict(storage=_abi.KV_INT8), _abi.GORGON_ERR_INVALID, "scale"),
])
def test_bad_pools_are_status_codes(kw, code, word):
    lib = _abi.lib()
    a, r, t, n = _abi.PagedAppendParams(), _abi.PagedReadParams(), _abi.PagedTrimParams(), _abi.PagedAttnParams()
    for p in (a, r, t, n):
        _kv(p.kv, **kw)
    a.n, r.rows, t.layers, t.max_len, n.n, n.heads_q = 1, 1, 1, 1, 1, 2
    for rc in (lib.gorgon_paged_append(ctypes.byref(a), None), lib.gorgon_paged_read(ctypes.byref(r), None),
               lib.gorgon_paged_trim(ctypes.byref(t), None), lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None)):
        got, msg = _err(rc)
        assert got == code and word in msg, msg
    assert lib.gorgon_paged_attn_workspace_size(ctypes.byref(n)) == 0


def test_other_refusals_and_empty_calls():
    lib = _abi.lib()
    for f in (lib.gorgon_paged_append, lib.gorgon_paged_read, lib.gorgon_paged_trim):
        assert _err(f(None, None)) == (_abi.GORGON_ERR_INVALID, f"{f.__name__}: params is null")
    assert _err(lib.gorgon_paged_attn(None, None, 0, None))[0] == _abi.GORGON_ERR_INVALID
    n = _abi.PagedAttnParams()
    _kv(n.kv)
    n.n, n.heads_q, n.q, n.out = 1, 3, 4096, 4096
    assert "multiple" in _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))[1]
    n.heads_q, n.window = 4, -1
    assert "negative" in _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))[1]
    n.window, n.parents, n.n = 0, 4096, 1025
    assert "1024" in _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))[1]
    for bad in (-0.1, float("nan"), float("inf")):
        n.n, n.scale = 1, bad
        assert "scale" in _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))[1]
    n.scale = 0.0
    n.n, n.backend = 1, 99
    assert "backend" in _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))[1]
    n.backend, n.q = 0, None
    assert "null" in _err(lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None))[1]
    n.n = 0
    assert lib.gorgon_paged_attn(ctypes.byref(n), None, 0, None) == 0
    t = _abi.PagedTrimParams()
    _kv(t.kv)
    t.layers, t.max_len = 1, 257
    assert _err(lib.gorgon_paged_trim(ctypes.byref(t), None))[0] == _abi.GORGON_ERR_UNSUPPORTED
    t.max_len = 4
    assert "null" in _err(lib.gorgon_paged_trim(ctypes.byref(t), None))[1]
    t.layers = 0
    assert lib.gorgon_paged_trim(ctypes.byref(t), None) == 0
    a = _abi.PagedAppendParams()
    _kv(a.kv)
    a.n = 1
    assert "null" in _err(lib.gorgon_paged_append(ctypes.byref(a), None))[1]
    a.n = 0
    assert lib.gorgon_paged_append(ctypes.byref(a), None) == 0
    r = _abi.PagedReadParams()
    _kv(r.kv)
    r.rows = 1
    assert "null" in _err(lib.gorgon_paged_read(ctypes.byref(r), None))[1]
    r.rows = 0
    assert lib.gorgon_paged_read(ctypes.byref(r), None) == 0
