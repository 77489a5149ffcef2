"""Paged cache append, read and trim against 64-bit host code: bytes and scales
exactly, for every storage, type, layout and page size."""
from __future__ import annotations

import math
import random

import pytest
import torch

import projectgorgon_b200 as G
from paged_reference import EIGHT, Paged, quantise

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    G.device_error(clear=True)
    yield
    assert G.device_error(clear=True) == 0


def rows_of(p: Paged, pages, b, lo, hi):
    return torch.stack([pages[int(p.table[b, x // p.ps]), :, x % p.ps] for x in range(lo, hi)]) if hi > lo else None


@pytest.mark.parametrize("storage", ["native", "int8", "fp8"])
@pytest.mark.parametrize("dtype,D,ps,layout", [
    (torch.bfloat16, 128, 16, "HSD"), (torch.float16, 64, 12, "SHD"), (torch.bfloat16, 256, 1, "HSD"),
    (torch.float16, 8, 7, "HSD"), (torch.float16, 40, 16, "HSD"), (torch.float32, 128, 16, "HSD"),
    (torch.bfloat16, 128, 8, "pad"), (torch.float32, 33, 5, "SHD"),
])
def test_append_packed(storage, dtype, D, ps, layout):
    H, lens, new = 3, [5, 37, 16, 0, 1, 50], [5, 2, 16, 0, 1, 33]
    p = Paged(lens, H, D, ps, dtype, storage, seed=D, layout=layout, poison=False)
    before = [x.clone() for x in (p.k_pages, p.v_pages)]
    g = torch.Generator().manual_seed(1)
    total = sum(new)
    k, v = ((torch.randn(total + 4, H, D, generator=g) * 3).to(dtype) for _ in range(2))  # 4 rows of padding behind
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
    G.paged_cache_append(k.cuda(), v.cuda(), *p.args, cu_q=cu.cuda(), **p.held)
    for x, pages, scale, old in ((k, p.k_pages, p.k_scale, before[0]), (v, p.v_pages, p.v_scale, before[1])):
        pages, old = pages.cpu(), old.cpu()
        touched = torch.zeros(pages.shape[0], ps, dtype=torch.bool)
        for b, (L, c) in enumerate(zip(lens, new)):
            for i in range(c):
                pos = L - c + i
                pg, r = int(p.table[b, pos // ps]), pos % ps
                touched[pg, r] = True
                row = x[int(cu[b]) + i]
                if storage == "native":
                    assert torch.equal(pages[pg, :, r], row)
                else:
                    # 16-bit rows times a 12-bit factor are exact in 32 bits; a 32-bit row's product is rounded to 24
                    # bits first, which may move a stored byte next to a tie by one step
                    q, s = quantise(row, storage)
                    assert torch.equal(scale.cpu()[pg, :, r], s)
                    off = (pages[pg, :, r].double() - q).abs()
                    if dtype == torch.float32:
                        assert float(off.max()) <= (1 if storage == "int8" else 32) and float((off > 0).float().mean()) < 0.02
                    else:
                        assert float(off.max()) == 0
        keep = ~touched[:, None, :, None].expand_as(pages)
        as_bytes = lambda t: t.contiguous().view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t  # noqa: E731
        assert torch.equal(as_bytes(pages)[keep], as_bytes(old)[keep])


@pytest.mark.parametrize("storage", ["native", "int8", "fp8"])
def test_append_batch_form_equals_packed(storage):
    B, H, n, D, ps = 4, 2, 3, 128, 16
    lens = [3, 40, 0, 17]  # the third slot is unused
    a, b = (Paged(lens, H, D, ps, torch.float16, storage, seed=3, poison=False) for _ in range(2))
    x = torch.randn(2, B, n, H, D, generator=torch.Generator().manual_seed(5)).half().cuda()
    k, v = x[0].transpose(1, 2), x[1].transpose(1, 2)  # [B, H, n, D] views
    G.paged_cache_append(k, v, *a.args, **a.held)
    live = [0, 1, 3]
    packed = x[:, live].reshape(2, -1, H, D)
    cu = torch.tensor([0, 3, 6, 6, 9], dtype=torch.int64).cuda()
    G.paged_cache_append(packed[0], packed[1], *b.args, cu_q=cu, **b.held)
    for p, q in ((a.k_pages, b.k_pages), (a.v_pages, b.v_pages), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)):
        if p is not None:
            assert torch.equal(p.view(torch.uint8) if p.dtype == torch.float8_e4m3fn else p,
                               q.view(torch.uint8) if q.dtype == torch.float8_e4m3fn else q)


@pytest.mark.parametrize("storage", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_special_rows(storage, dtype):
    """Zeros, the smallest and largest values, and rows with infinities or NaN."""
    D, top = 128, torch.finfo(dtype).max
    rows = torch.zeros(7, 1, D, dtype=dtype)
    rows[1, 0, 3] = torch.finfo(dtype).tiny
    rows[2, 0, :] = top
    rows[2, 0, 1::2] = -top
    rows[3, 0, 0] = 1.0
    rows[4, 0, 5], rows[4, 0, 6] = math.inf, 1.0
    rows[5, 0, 5] = math.nan
    rows[6, 0, 0], rows[6, 0, 1] = -1.0, 2.0 ** -9
    p = Paged([7], 1, D, 4, dtype, storage, poison=False)
    G.paged_cache_append(rows.cuda(), rows.cuda(), *p.args, cu_q=torch.tensor([0, 7]).cuda(), **p.held)
    k, v = G.paged_cache_read(p.k_pages, p.v_pages, p.table_d, torch.tensor([0, 7]).cuda(), 7, dtype=torch.float32, **p.held)
    assert torch.equal(torch.nan_to_num(k, nan=9.0), torch.nan_to_num(v, nan=9.0))
    k = k.cpu()[:, 0].double()
    assert torch.isnan(k[4]).all() and torch.isnan(k[5]).all() and float(k[0].abs().max()) == 0
    for i in (1, 2, 3, 6):
        q, s = quantise(rows[i], storage)
        # read as float32: values stop at its largest finite one (the factor's cut may put them 2^-11 above)
        want = (q[0] * s.double()).clamp(-torch.finfo(torch.float32).max, torch.finfo(torch.float32).max)
        # stored values are exact; their product with the scale is rounded to 32 bits once
        assert torch.allclose(k[i], want, rtol=2.0 ** -23, atol=0), i
        step = s.double() if storage == "int8" else want.abs() / 8 + s.double() * 2.0 ** -9
        assert bool(((k[i] - rows[i, 0].double()).abs() <= step / 2 * 1.01 + 1e-37).all())
    same = G.paged_cache_read(p.k_pages, p.v_pages, p.table_d, torch.tensor([0, 7]).cuda(), 7, dtype=dtype, **p.held)[0].cpu()
    assert bool(torch.isfinite(same[:4]).all()) and bool((same[2].abs() == top).all())


@pytest.mark.parametrize("storage", ["native", "int8", "fp8"])
@pytest.mark.parametrize("dtype,D,ps,layout", [
    (torch.bfloat16, 128, 16, "HSD"), (torch.float16, 64, 12, "SHD"), (torch.bfloat16, 256, 1, "HSD"),
    (torch.float16, 8, 7, "HSD"), (torch.float16, 40, 16, "HSD"), (torch.float32, 128, 16, "HSD"),
    (torch.bfloat16, 16, 8, "pad"),
])
def test_read(storage, dtype, D, ps, layout):
    H, lens = 3, [5, 0, 37, 16, 1]
    p = Paged(lens, H, D, ps, dtype, storage, seed=D + 1, layout=layout)
    starts, count = [2, 0, 11, 0, 1], [3, 0, 20, 16, 0]
    cu = torch.tensor([sum(count[:b]) for b in range(6)], dtype=torch.int32).cuda()
    total = sum(count)
    out = tuple(torch.full((total + 3, H, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    got = G.paged_cache_read(p.k_pages, p.v_pages, p.table_d, cu, total + 3, starts=torch.tensor(starts).cuda(), out=out, **p.held)
    assert got[0] is out[0] and got[1] is out[1]
    for x, held in zip(out, (p.k64, p.v64)):
        x = x.cpu()
        assert bool((x[total:] == 7.0).all())
        for b in range(5):
            want = held[b][starts[b]:starts[b] + count[b]]
            have = x[int(cu[b]):int(cu[b + 1])].double()
            if storage == "native":
                assert torch.equal(have, want)
            else:  # the product in 32 bits, then one rounding to the result's type
                half = torch.finfo(dtype).eps / 2
                assert bool(((have - want).abs() <= want.abs() * (half + 2.0 ** -23) + torch.finfo(dtype).tiny * half * 2).all())


def test_read_other_types_and_defaults():
    p = Paged([9, 4], 2, 64, 4, torch.bfloat16, "native", seed=2)
    cu = torch.tensor([0, 9, 13]).cuda()
    k, _ = G.paged_cache_read(p.k_pages, p.v_pages, p.table_d, cu, 13)
    assert k.dtype == torch.bfloat16 and torch.equal(k.cpu().double(), torch.cat(p.k64))
    q = Paged([9, 4], 2, 64, 4, torch.bfloat16, "int8", seed=2)
    k, v = G.paged_cache_read(q.k_pages, q.v_pages, q.table_d, cu, 13, **q.held)
    assert k.dtype == torch.bfloat16
    strided = tuple(torch.zeros(2, 13, 64, dtype=torch.float16, device="cuda").transpose(0, 1) for _ in range(2))
    G.paged_cache_read(q.k_pages, q.v_pages, q.table_d, cu, 13, out=strided, **q.held)
    assert float((strided[0].float() - k.float()).abs().max()) < 0.05
    none = G.paged_cache_read(q.k_pages, q.v_pages, q.table_d, torch.zeros(3, dtype=torch.int32).cuda(), 0, **q.held)
    assert none[0].shape == (0, 2, 64)


@pytest.mark.parametrize("storage", ["native", "int8", "fp8"])
@pytest.mark.parametrize("dtype,D,ps,layout,m", [
    (torch.bfloat16, 128, 16, "HSD", 6), (torch.float16, 64, 12, "SHD", 8), (torch.bfloat16, 128, 16, "HSD", 20),
    (torch.float16, 40, 16, "HSD", 5), (torch.bfloat16, 16, 3, "pad", 5), (torch.bfloat16, 128, 8, "HSD", 100),
    (torch.float32, 128, 16, "HSD", 7),
])
def test_trim_all_layers(storage, dtype, D, ps, layout, m):
    layers, H, B, n = 3, 5, 4, max(20, m + 4)
    rng = random.Random(m)
    lens = [n + x for x in (0, 13, 40, 1)]
    ps_ = [Paged(lens, H, D, ps, dtype, storage, seed=s, layout=layout, poison=False) for s in range(layers)]
    for x in ps_[1:]:
        x.table, x.table_d = ps_[0].table, ps_[0].table_d
    k, v = (torch.stack([getattr(x, a) for x in ps_]) for a in ("k_pages", "v_pages"))
    if layout == "pad":
        k, v = (torch.nn.functional.pad(t.view(torch.uint8) if t.element_size() == 1 else t, (0, 3))[..., :D] for t in (k, v))
        k, v = (t.view(ps_[0].k_pages.dtype) if t.dtype == torch.uint8 else t for t in (k, v))
    ks, vs = (None if storage == "native" else torch.stack([getattr(x, a) for x in ps_]) for a in ("k_scale", "v_scale"))
    count = [m, 0, min(3, m), 1]
    src = torch.zeros(B, m, dtype=torch.int32)
    dst = torch.tensor([L - n for L in lens], dtype=torch.int32)
    for b in range(B):
        path = sorted(rng.sample(range(n), count[b]))
        if b == 2:
            path = [0, 2, 1][: count[b]]  # rows that swap: every row is read before any is written
        for r, t in enumerate(path):
            src[b, r] = lens[b] - n + t
    def as_bytes(t):
        return t.contiguous().view(torch.uint8).clone() if t.dtype == torch.float8_e4m3fn else t.clone()
    want = [as_bytes(t) if t is not None else None for t in (k, v, ks, vs)]
    for t in want:
        if t is None:
            continue
        old = t.clone()
        for b in range(B):
            for r in range(count[b]):
                i, o = int(src[b, r]), int(dst[b]) + r
                t[:, ps_[0].table[b, o // ps], :, o % ps] = old[:, ps_[0].table[b, i // ps], :, i % ps]
    G.paged_cache_trim(k, v, ps_[0].table_d, src.cuda(), torch.tensor(count).cuda(), dst.cuda(), k_scale=ks, v_scale=vs)
    for t, w in zip((k, v, ks, vs), want):
        if w is not None:
            assert torch.equal(as_bytes(t), w)


def test_bad_indices_are_skipped_and_reported():
    """A page outside the pool, a length past the table, a sequence shorter than
    its new rows, a trim index out of range: the error bits, nothing else."""
    ps, H, D = 4, 2, 64
    p = Paged([6, 6, 6], H, D, ps, torch.bfloat16, poison=False, table_cols=2)
    p.table_d[1, 1] = 99
    before = p.k_pages.clone(), p.v_pages.clone()
    k = torch.randn(3, H, 1, D, device="cuda").bfloat16()
    G.paged_cache_append(k, k, *p.args)  # sequence 1's row lies in page 99
    assert G.device_error() == 1 << 6
    assert torch.equal(p.k_pages[int(p.table[0, 1]), :, 1], k[0, :, 0]) and torch.equal(p.k_pages[int(p.table[2, 1]), :, 1], k[2, :, 0])
    p.k_pages.copy_(before[0]), p.v_pages.copy_(before[1])
    G.paged_cache_append(k[:1], k[:1], p.k_pages, p.v_pages, p.table_d[:1], torch.tensor([9]).cuda())  # past the table
    assert G.device_error() == 1 << 6
    k4 = torch.randn(1, H, 4, D, device="cuda").bfloat16()
    G.paged_cache_append(k4, k4, p.k_pages, p.v_pages, p.table_d[:1], torch.tensor([3]).cuda())
    assert G.device_error() == 1 << 3
    for bad in (-1, 8, 10 ** 6):
        G.paged_cache_trim(p.k_pages, p.v_pages, p.table_d[:1], torch.tensor([[0, bad]]).cuda(), torch.tensor([2]).cuda(), 1)
        assert G.device_error() == 1 << 1
    G.paged_cache_trim(p.k_pages, p.v_pages, p.table_d[:1], torch.tensor([[0, 1]]).cuda(), torch.tensor([3]).cuda(), 1)
    assert G.device_error() == 1 << 1
    G.paged_cache_trim(p.k_pages, p.v_pages, p.table_d[1:2], torch.tensor([[0, 5]]).cuda(), torch.tensor([2]).cuda(), 1)
    assert G.device_error() == 1 << 6
    out = torch.full((8, H, D), 3.0, dtype=torch.bfloat16, device="cuda")
    G.paged_cache_read(p.k_pages, p.v_pages, p.table_d[1:2], torch.tensor([0, 6]).cuda(), 8, out=(out, out.clone()))
    assert G.device_error() == 1 << 6 and bool((out[4:] == 3.0).all())
    assert torch.equal(p.k_pages, before[0]) and torch.equal(p.v_pages, before[1])


def test_far_pages():
    """A pool past 2^32 bytes, and past 2^31 elements: offsets are 64 bits."""
    H, ps, D = 8, 16, 128
    pages = (1 << 32) // (H * ps * D) + 40  # int8: a little over 4 GiB each of K and V
    kp, vp = (torch.zeros(pages, H, ps, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, H, ps, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32).cuda()
    k, v = (torch.randn(1, H, 40, D, device="cuda").bfloat16() for _ in range(2))
    G.paged_cache_append(k, v, kp, vp, table, torch.tensor([40]).cuda(), k_scale=ks, v_scale=vs)
    got = G.paged_cache_read(kp, vp, table, torch.tensor([0, 40]).cuda(), 40, k_scale=ks, v_scale=vs)
    for x, y in zip((k, v), got):
        q, s = quantise(x[0].transpose(0, 1).cpu(), "int8")
        want = q * s.double()[..., None]
        assert bool(((y.cpu().double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -23)).all())
    assert int((kp[pages - 1] != 0).sum()) > 0 and int((kp[: 3] != 0).sum()) == 0
