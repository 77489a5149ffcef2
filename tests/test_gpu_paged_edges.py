"""The paged operators at their edges: bad block tables, ragged trees, large
batches and pools, captured calls, waits that run out, refused arguments."""
from __future__ import annotations

import math
import random

import pytest
import torch

import projectgorgon_b200 as G
from paged_reference import Paged, attend, tolerance, visible
from projectgorgon_b200 import _abi
from projectgorgon_b200.trees import random_tree
from test_gpu_paged_attention import check

pytestmark = pytest.mark.gpu

STORES = ["native", "int8", "fp8"]
BAD_PAGE, BAD_LENGTH = 1 << 6, 1 << 3


@pytest.fixture(autouse=True)
def no_device_error():
    G.device_error(clear=True)
    yield
    assert G.device_error(clear=True) == 0


def near(out, q, p, b, see, scale=None):
    """Sequence b's rows [Hq, c, D] against the reference."""
    want, weight, slip, _ = attend(q.cpu(), p.k64[b], p.v64[b], see, p.D ** -0.5 if scale is None else scale)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= tolerance(want, weight, slip, p.dtype)).all()), float(off.max())


@pytest.mark.parametrize("entry", [-1, -2, -7, -2 ** 31, "pages", 2 ** 31 - 1])
@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("ps", [16, 12])
@pytest.mark.parametrize("n", [1, 70])
def test_bad_entries_hide_their_rows(entry, storage, ps, n):
    L = n + 300
    p = Paged([L, L], 2, 128, ps, torch.bfloat16, storage, seed=n)
    q = torch.randn(2, 8, n, 128, device="cuda").bfloat16()
    good = G.paged_attention(q, *p.args, **p.held)
    table = p.table_d.clone()
    table[1, 5] = p.k_pages.shape[0] if entry == "pages" else entry
    for backend in ("auto", "mma", "tcgen05", "simt"):
        out = G.paged_attention(q, p.k_pages, p.v_pages, table, p.lens_d, backend=backend, **p.held)
        assert G.device_error(clear=True) == BAD_PAGE
        if backend == "auto":
            assert torch.equal(out[0], good[0])
        see = visible(L, n)
        see[:, 5 * ps:6 * ps] = False
        near(out[1], q[1], p, 1, see)


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("n,P", [(1, 40), (1, 9000), (70, 100), (70, 5000)])
def test_rows_with_nothing_to_see_are_zero(storage, n, P):
    """Every page of a sequence is bad (one CTA's unit, or one cut between CTAs)."""
    p = Paged([n + P, n + P], 2, 128, 16, torch.bfloat16, storage, seed=n)
    q = torch.randn(2, 8, n, 128, device="cuda").bfloat16()
    table = p.table_d.clone()
    table[1] = -1
    for backend in ("auto", "mma", "tcgen05", "simt"):
        out, lse = G.paged_attention(q, p.k_pages, p.v_pages, table, p.lens_d, backend=backend, return_lse=True, **p.held)
        assert G.device_error(clear=True) == BAD_PAGE
        assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())
        near(out[0], q[0], p, 0, visible(n + P, n))


@pytest.mark.parametrize("new", [[64, 1, 33, 0, 7], [3, 5], [9, 300, 1]])
@pytest.mark.parametrize("storage", STORES)
def test_ragged_trees(new, storage):
    """Packed rows, trees of different sizes: the first nodes of max_q."""
    Hq, D, rng = 4, 128, random.Random(len(new))
    before = [100, 0, 333, 12, 64]
    most = max(new) + 2
    parents = [random_tree(most, rng, 9) for _ in new]
    p = Paged([c + before[b] if c else 0 for b, c in enumerate(new)], 2, D, 16, torch.bfloat16, storage, seed=len(new))
    q = torch.randn(sum(new) + 2, Hq, D, device="cuda").bfloat16()
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    par = torch.tensor(parents, dtype=torch.int32, device="cuda")
    for kw in ({}, {"max_q": most}):
        for backend in ("auto", "simt"):
            out = torch.full_like(q, 3.0)
            G.paged_attention(q, *p.args, cu_q=cu, parents=par, max_depth=4, window=200, out=out, backend=backend, **kw, **p.held)
            assert bool((out[sum(new):] == 3.0).all())
            for b, c in enumerate(new):
                if c:
                    r = slice(int(cu[b]), int(cu[b]) + c)
                    near(out[r].transpose(0, 1), q[r].transpose(0, 1), p, b, visible(p.lens[b], c, parents[b][:c], 4, 200))


@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05", "simt"])
def test_more_rows_than_max_q(backend):
    """A sequence that brings more rows than max_q is left out and reported."""
    new, D = [2, 9, 1], 128
    p = Paged([50, 60, 70], 2, D, 16, torch.float16, seed=1)
    q = torch.randn(sum(new), 20, D, device="cuda").half()
    cu = torch.tensor([0, 2, 11, 12], dtype=torch.int32, device="cuda")
    out, lse = G.paged_attention(q, *p.args, cu_q=cu, max_q=2, return_lse=True, backend=backend)
    assert G.device_error(clear=True) == BAD_LENGTH
    assert bool((out[2:11] == 0).all()) and bool((lse[2:11] == -math.inf).all())
    near(out[:2].transpose(0, 1), q[:2].transpose(0, 1), p, 0, visible(50, 2))
    near(out[11:].transpose(0, 1), q[11:].transpose(0, 1), p, 2, visible(70, 1))


@pytest.mark.parametrize("cu", [[0, -3, 4, 6], [2, 1, 3, 6], [0, 2, 9, 6], [0, 2 ** 31 - 1, 3, 6], [-2 ** 31, 2, 3, 6], [0, 6, 0, 6]])
@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05", "simt"])
def test_counts_out_of_order_are_reported(cu, backend):
    p = Paged([50, 60, 70], 2, 128, 16, torch.float16, seed=1)
    q = torch.randn(6, 16, 128, device="cuda").half()
    G.paged_attention(q, *p.args, cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=4, backend=backend)
    torch.cuda.synchronize()
    assert G.device_error(clear=True) == BAD_LENGTH


@pytest.mark.parametrize("cu", [[0, -3, 4, 6], [2, 5, 3, 6], [0, 5, 2, 6], [0, 2 ** 31 - 1, 3, 6], [-2 ** 31, 2, 3, 6], [0, 6, 0, 6]])
def test_counts_out_of_order_leave_the_pages_alone(cu):
    """Append and read: rows outside their sequence are skipped and reported; pages
    that no row may go to keep their bytes."""
    p = Paged([3, 60, 70], 2, 128, 16, torch.float16, seed=1, poison=False)
    rows = torch.randn(6, 2, 128, device="cuda").half()
    own = torch.unique(p.table[(p.table >= 0) & (p.table < p.k_pages.shape[0])]).cuda()
    other = torch.ones(p.k_pages.shape[0], dtype=torch.bool, device="cuda")
    other[own.long()] = False
    before = p.k_pages.clone()
    cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    G.paged_cache_append(rows, rows, p.k_pages, p.v_pages, p.table_d, p.lens_d, cu_q=cu)
    torch.cuda.synchronize()
    assert torch.equal(p.k_pages[other], before[other])
    G.device_error(clear=True)
    out = torch.full((2, 6, 2, 128), 4.0, device="cuda", dtype=torch.float16)
    for starts in (None, [0, 0, 0], [2 ** 31 - 1] * 3, [-2 ** 31] * 3):
        G.paged_cache_read(p.k_pages, p.v_pages, p.table_d, cu, 6, out=(out[0], out[1]),
                           starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert G.device_error(clear=True) in (0, BAD_LENGTH, BAD_PAGE, BAD_LENGTH | BAD_PAGE)


@pytest.mark.parametrize("batch", [129, 700, 1500])
@pytest.mark.parametrize("packed", [False, True])
def test_many_sequences(batch, packed):
    rng = random.Random(batch)
    new = [rng.choice([0, 1, 1, 2, 19]) for _ in range(batch)] if packed else [1] * batch
    lens = [c + rng.choice([0, 3, 40, 130]) if c else 0 for c in new]
    if not packed:
        lens[::7] = [0] * len(lens[::7])
    p = Paged(lens, 1, 64, 16, torch.bfloat16, "int8", seed=batch)
    check(p, new, 4, packed=packed)


@pytest.mark.parametrize("n", [300, 1000, 1024])
def test_large_trees(n):
    rng = random.Random(n)
    p = Paged([n + 65], 1, 64, 16, torch.bfloat16, seed=n)
    check(p, [n], 2, parents=[random_tree(n, rng, 12)], max_depth=7)


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("ps", [8, 32, 128, 192])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [None, 150])
def test_page_sizes(storage, ps, D, window):
    """Pages of every size that a copy takes in one box, of tiles that begin inside a page."""
    p = Paged([100 + 40, 700 + 40, 40], 2, D, ps, torch.bfloat16, storage, seed=ps)
    check(p, [40] * 3, 8, window=window, sinks=3)


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("n", [1, 40])
def test_pages_repeated_by_strides(storage, n):
    """Kv heads that are one head in memory (stride 0)."""
    p = Paged([n + 90, n + 300], 1, 128, 16, torch.bfloat16, storage, seed=n)
    q = torch.randn(2, 8, n, 128, device="cuda").bfloat16()
    wide = lambda t: None if t is None else t.expand(-1, 4, *t.shape[2:])  # noqa: E731
    out = G.paged_attention(q, wide(p.k_pages), wide(p.v_pages), p.table_d, p.lens_d, k_scale=wide(p.k_scale), v_scale=wide(p.v_scale))
    for b in range(2):
        near(out[b], q[b], p, b, visible(p.lens[b], n))


@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05", "simt"])
@pytest.mark.parametrize("bad", [-2, -2 ** 31, 3, 2 ** 31 - 1])
def test_bad_parents_are_reported(backend, bad):
    """A parent outside the tree ends the walk there, as a root's does."""
    p = Paged([43, 63], 2, 128, 16, torch.bfloat16, seed=1)
    q = torch.randn(2, 16, 3, 128, device="cuda").bfloat16()
    out = G.paged_attention(q, *p.args, parents=torch.tensor([[-1, 0, 1], [-1, bad, 1]]), backend=backend)
    assert G.device_error(clear=True) == 1
    near(out[0], q[0], p, 0, visible(43, 3, [-1, 0, 1]))
    near(out[1], q[1], p, 1, visible(63, 3, [-1, -1, 1]))


@pytest.mark.parametrize("what", [math.inf, -math.inf])
@pytest.mark.parametrize("n", [1, 5, 80])
def test_infinite_keys(what, n):
    """A score of +inf makes its row NaN, one of -inf leaves its key out; hidden ones do nothing."""
    L, D = n + 200, 64
    p = Paged([L], 1, D, 16, torch.bfloat16, seed=n)
    q = torch.randn(1, 2, n, D, device="cuda").bfloat16()
    q[q == 0] = 1
    pos = 150
    p.k_pages[int(p.table[0, pos // 16]), :, pos % 16, 7] = what
    for window in (None, 80):
        out, lse = G.paged_attention(q, *p.args, window=window, return_lse=True)
        see = visible(L, n, window=window)
        up = (q[0, :, :, 7].cpu() * what > 0) & see[:, pos]
        assert torch.equal(torch.isnan(out[0].cpu()).all(-1), up) and torch.equal(torch.isnan(out[0].cpu()).any(-1), up)
        see[:, pos] = False
        p.k64[0][pos] = 0.0
        want, weight, slip, wl = attend(q[0].cpu(), p.k64[0], p.v64[0], see, D ** -0.5)
        tol = tolerance(want, weight, slip, p.dtype)
        assert bool(((out[0].cpu().double() - want).abs() <= tol)[~up].all())
        assert bool(((lse[0].cpu().double() - wl).abs() <= 2 * slip[..., 0] + 64 * 2.0 ** -22 + wl.abs() * 2.0 ** -22)[~up].all())


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("n", [1, 40])
def test_shared_pages(storage, n):
    """Sequences with the same first pages, and one sequence twice."""
    p = Paged([320 + n, 400 + n], 2, 128, 16, torch.bfloat16, storage, seed=n)
    table = torch.cat([p.table_d, p.table_d[:1], p.table_d[1:]])
    table[1, :20] = table[0, :20]
    lens = torch.tensor([320 + n, 400 + n, 320 + n, 400 + n], dtype=torch.int32, device="cuda")
    q = torch.randn(4, 8, n, 128, device="cuda").bfloat16()
    out = G.paged_attention(q, p.k_pages, p.v_pages, table, lens, **p.held)
    k64, v64 = list(p.k64), list(p.v64)
    mixed = [torch.cat([x[0][:320], x[1][320:]]) for x in (k64, v64)]
    p.k64, p.v64 = [k64[0], mixed[0], k64[0], k64[1]], [v64[0], mixed[1], v64[0], v64[1]]
    for b in range(4):
        near(out[b], q[b], p, b, visible(int(lens[b]), n))


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("ps", [16, 12])
def test_pools_past_32_bits(storage, ps):
    """Pages beyond 2^32 bytes (16-bit: 2^33) of a pool, through every operator."""
    Hkv, D, dtype = 2, 128, torch.bfloat16
    small = Paged([333, 90], Hkv, D, ps, dtype, storage, seed=ps)
    used = small.k_pages.shape[0]
    pages = (1 << 32) // (Hkv * ps * D) + used + 10
    first = pages - used
    shape = (pages, Hkv, ps, D)
    big = {}
    for name in ("k_pages", "v_pages"):
        t = getattr(small, name)
        big[name] = torch.empty(shape, dtype=t.dtype, device="cuda")
        big[name][first:].view(torch.uint8).copy_(t.view(torch.uint8))
    for name in ("k_scale", "v_scale"):
        t = getattr(small, name)
        big[name] = None
        if t is not None:
            big[name] = torch.empty(shape[:-1], device="cuda")
            big[name][first:] = t
    table = torch.where(small.table_d < used, small.table_d + first, small.table_d)
    kp, vp, scales = big["k_pages"], big["v_pages"], dict(k_scale=big["k_scale"], v_scale=big["v_scale"])
    for n in (1, 40):
        q = torch.randn(2, 8, n, D, device="cuda").to(dtype)
        for backend in ("auto", "simt"):
            out = G.paged_attention(q, kp, vp, table, small.lens_d, backend=backend, **scales)
            for b in range(2):
                near(out[b], q[b], small, b, visible(small.lens[b], n))
    cu = torch.tensor([0, 333, 423], dtype=torch.int32, device="cuda")
    rows = G.paged_cache_read(kp, vp, table, cu, 423, **scales)
    want = G.paged_cache_read(small.k_pages, small.v_pages, small.table_d, cu, 423, **small.held)
    assert all(torch.equal(a, b) for a, b in zip(rows, want))
    k, v = (torch.randn(2, Hkv, 3, D, device="cuda").to(dtype) for _ in range(2))
    idx = torch.tensor([[2, 7], [5, 80]], dtype=torch.int32, device="cuda")
    two = torch.tensor([2, 2], dtype=torch.int32, device="cuda")
    for pool, tab, held in (((kp, vp), table, scales), ((small.k_pages, small.v_pages), small.table_d, small.held)):
        G.paged_cache_append(k, v, *pool, tab, small.lens_d, **held)
        G.paged_cache_trim(*pool, tab, idx, two, **held)
    rows = G.paged_cache_read(kp, vp, table, cu, 423, **scales)
    want = G.paged_cache_read(small.k_pages, small.v_pages, small.table_d, cu, 423, **small.held)
    assert all(torch.equal(a, b) for a, b in zip(rows, want))


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("n,tree", [(1, False), (64, True), (200, False)])
def test_two_graphs_at_once(storage, n, tree):
    """Two captured calls replayed together on two streams, and again."""
    rng = random.Random(n)
    par = torch.tensor(random_tree(n, rng, 5), dtype=torch.int32, device="cuda") if tree else None
    both = [Paged([n + 900, n, n + 5000], 2, 128, 16, torch.bfloat16, storage, seed=s) for s in (1, 2)]
    q = torch.randn(3, 8, n, 128, device="cuda").bfloat16()
    call = lambda p: G.paged_attention(q, *p.args, parents=par, return_lse=True, **p.held)  # noqa: E731
    want = [call(p) for p in both]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for p in both:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(p))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in both]
    for _ in range(10):
        for o in outs:
            for t in o:
                t.fill_(7.0)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, w in zip(outs, want) for a, b in zip(o, w))
    del graphs


def test_any_strides_of_out_and_table():
    for n in (1, 70):
        p = Paged([n + 200, n + 64], 2, 128, 16, torch.bfloat16, seed=n)
        q = torch.randn(2, 8, n, 128, device="cuda").bfloat16()
        want = G.paged_attention(q, *p.args)
        wide = torch.full((2, n, 8, 131), 9.0, device="cuda", dtype=torch.bfloat16)
        out = wide[..., 1:129].transpose(1, 2)
        assert G.paged_attention(q, *p.args, out=out) is out and torch.equal(out, want)
        assert bool((wide[..., 0] == 9).all()) and bool((wide[..., 129:] == 9).all())
        table = torch.stack([p.table_d, p.table_d], -1).flatten(1).long()[:, ::2]
        assert torch.equal(G.paged_attention(q, p.k_pages, p.v_pages, table, p.lens_d.long()), want)


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("ps", [16, 12])
@pytest.mark.parametrize("n", [64, 20])
def test_waits_that_run_out(storage, ps, n):
    """With the bound of every wait cut to 1 ns the tcgen05 kernel gives up where a
    wait lasts (the bound is looked at every 64 probes), frees what it holds and
    reports it, and the next call is right.  Two short sequences may get through;
    where CTAs have several units, the products of the next wait for the end of one."""
    def pages(like):
        x = torch.randn(400, 2, ps, 128, device="cuda")
        return x.clamp(-3, 3).to(like) if like != torch.int8 else (x * 40).clamp(-127, 127).to(like)

    held = {"native": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}[storage]
    kp, vp = pages(held), pages(held)
    scales = {} if storage == "native" else {s: torch.rand(400, 2, ps, device="cuda") * 0.1 for s in ("k_scale", "v_scale")}
    for batch, P, must in ((2, 3000, False), (200, 100, True)):
        table = torch.randint(0, 400, (batch, -(-(P + n) // ps)), dtype=torch.int32, device="cuda")
        lens = torch.full((batch,), P + n, dtype=torch.int32, device="cuda")
        q = torch.randn(batch, 8, n, 128, device="cuda").bfloat16()
        call = lambda: G.paged_attention(q, kp, vp, table, lens, backend="tcgen05", **scales)  # noqa: E731
        want = call()
        assert G.device_error() == 0 and bool(torch.isfinite(want).all())
        prev = _abi.set_wait_limit_ns(1)
        try:
            call()
            torch.cuda.synchronize()
        finally:
            _abi.set_wait_limit_ns(prev)
        error = G.device_error(clear=True)
        assert error == _abi.ERR_TIMEOUT or (error == 0 and not must)
        assert torch.equal(call(), want)


def test_refused_arguments():
    p = Paged([40, 20], 2, 128, 16, torch.bfloat16, seed=1)
    e = Paged([40, 20], 2, 128, 16, torch.bfloat16, "int8", seed=1)
    q = torch.randn(2, 8, 2, 128, device="cuda").bfloat16()
    kp, vp, table, lens = p.args
    cu = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")

    def refused(word, *args, **kw):
        with pytest.raises(RuntimeError, match=word):
            G.paged_attention(*args, **kw)

    refused("backend", q, *p.args, backend="cpu")
    refused("window", q, *p.args, window=0)
    refused("sinks", q, *p.args, sinks=-1)
    for scale in (0.0, -1.0, math.nan, math.inf):
        refused("scale", q, *p.args, scale=scale)
    refused("head_dim", q[..., :64], *p.args)
    refused("multiple", q[:, :7], *p.args)
    refused("batch", q[:1], *p.args)
    refused("float32, bfloat16 or float16", q.double(), *p.args)
    refused("pages of", q.half(), *p.args)
    refused("scales belong", q, *p.args, k_scale=e.k_scale, v_scale=e.v_scale)
    refused("need k_scale", q, *e.args)
    refused("float32", q, *e.args, k_scale=e.k_scale.half(), v_scale=e.v_scale)
    refused("one dtype", q, kp, e.v_pages, table, lens)
    refused("both be", q, kp, vp[:, :, :8], table, lens)
    refused("int32 or int64", q, kp, vp, table.float(), lens)
    refused("entries", q, kp, vp, table, lens[:1])
    refused("dimension", q, kp, vp, table[0], lens)
    refused("contiguous last", q, *p.args, out=torch.empty(2, 8, 128, 2, device="cuda", dtype=q.dtype).transpose(2, 3))
    refused("out must be", q, *p.args, out=torch.empty_like(q, dtype=torch.float32))
    refused("parents must be", q, *p.args, parents=[-1, 0, 1])
    refused("1024", torch.empty(2, 8, 1025, 128, device="cuda", dtype=q.dtype), *p.args, parents=[-1] * 1025)
    refused("with cu_q", q, *p.args, cu_q=cu)
    refused("with cu_q", q[:, :, 0], *p.args, cu_q=cu[:2])
    refused("max_q", q[:, :, 0], *p.args, cu_q=cu, max_q=-1)
    refused("requested kernel", q.float(), kp.float(), vp.float(), table, lens, backend="mma")
    refused("requested kernel", torch.empty(2, 8, 257, 128, device="cuda", dtype=q.dtype), *p.args, parents=[-1] * 257,
            backend="tcgen05")
    with pytest.raises(ValueError):
        G.paged_attention(q, kp, vp, table.cpu(), lens)
    with pytest.raises(RuntimeError, match="heads of"):
        G.paged_cache_append(q, q, kp, vp, table, lens)
    with pytest.raises(RuntimeError, match="one shape"):
        G.paged_cache_append(q[:, :2], q[:, :2, :1], kp, vp, table, lens)
    with pytest.raises(RuntimeError, match="cu_rows"):
        G.paged_cache_read(kp, vp, table, cu[:2], 3)
    with pytest.raises(RuntimeError, match="starts"):
        G.paged_cache_read(kp, vp, table, cu, 3, starts=cu)
    with pytest.raises(RuntimeError, match="rows"):
        G.paged_cache_read(kp, vp, table, cu, -1)
    with pytest.raises(RuntimeError, match="one row per sequence"):
        G.paged_cache_trim(kp, vp, table, table[:1], lens)
    with pytest.raises(RuntimeError, match="dst_start"):
        G.paged_cache_trim(kp, vp, table, table, lens, lens[:1])


def test_empty_calls():
    p = Paged([40, 20], 2, 128, 16, torch.bfloat16, seed=1)
    kp, vp, table, lens = p.args
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    for q, kw in ((torch.empty(2, 8, 0, 128), {}), (torch.empty(0, 8, 128), {"cu_q": none}),
                  (torch.empty(0, 8, 128), {"cu_q": none, "parents": [-1, 0]})):
        q = q.cuda().bfloat16()
        out, lse = G.paged_attention(q, *p.args, return_lse=True, **kw)
        assert out.shape == q.shape and lse.shape == q.shape[:-1]
    q = torch.empty(0, 8, 1, 128, device="cuda", dtype=torch.bfloat16)
    assert G.paged_attention(q, kp, vp, table[:0], lens[:0]).shape == q.shape
    q = torch.randn(2, 8, 1, 128, device="cuda").bfloat16()
    out, lse = G.paged_attention(q, kp, vp, table, torch.zeros_like(lens), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    out = G.paged_attention(q, kp, vp, table[:, :0], torch.zeros_like(lens))
    assert bool((out == 0).all())
