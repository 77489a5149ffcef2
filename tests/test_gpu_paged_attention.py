"""paged_attention against 64-bit host code, at the sizes, types, layouts and
masks where it can go wrong."""
from __future__ import annotations

import math
import random

import pytest
import torch

import projectgorgon_b200 as G
from paged_reference import Paged, attend, tolerance, visible
from projectgorgon_b200.trees import random_tree

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    G.device_error(clear=True)
    yield
    assert G.device_error(clear=True) == 0


def check(p: Paged, new, Hq, *, packed=False, parents=None, max_depth=None, window=None, sinks=0, scale=None, seed=1,
          backend="auto", q_layout="plain", max_q=None):
    """One call with an `out` that has rows to keep, against the reference."""
    B, D, dtype = len(p.lens), p.D, p.dtype
    n = max(new + [1]) if packed else new[0]
    g = torch.Generator().manual_seed(seed)
    kw = dict(window=window, sinks=sinks, scale=scale, backend=backend, return_lse=True, **p.held)
    if parents is not None:
        kw.update(parents=torch.tensor(parents), max_depth=max_depth)
    if packed:
        total = sum(new)
        q = torch.randn(total + 3, Hq, D, generator=g).to(dtype)
        cu = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32)
        out = torch.full_like(q, 5.0).cuda()
        got, lse = G.paged_attention(q.cuda(), *p.args, cu_q=cu.cuda(), max_q=max_q or n, out=out, **kw)
        got = got.cpu()
        assert bool((got[total:] == 5.0).all())
        rows = lambda b: (q[int(cu[b]):int(cu[b + 1])].transpose(0, 1), got[int(cu[b]):int(cu[b + 1])].transpose(0, 1),  # noqa: E731
                          lse.cpu()[int(cu[b]):int(cu[b + 1])].transpose(0, 1))
    else:
        q = torch.randn(B, Hq, n, D, generator=g).to(dtype)
        qd = q.cuda()
        if q_layout == "BNHD":
            qd = qd.transpose(1, 2).contiguous().transpose(1, 2)
        elif q_layout == "pad":
            qd = torch.nn.functional.pad(qd, (0, 3))[..., :D]
        got, lse = G.paged_attention(qd, *p.args, **kw)
        got, lse = got.cpu(), lse.cpu()
        rows = lambda b: (q[b], got[b], lse[b])  # noqa: E731
    for b, (L, c) in enumerate(zip(p.lens, new)):
        qb, ob, lb = rows(b)
        if L == 0 or c == 0:
            assert bool((ob == 0).all()) and bool((lb == -math.inf).all())
            continue
        par = None if parents is None else (parents[b] if isinstance(parents[0], list) else parents)
        see = visible(L, c, par, max_depth, window, sinks)
        want, weight, slip, wl = attend(qb, p.k64[b], p.v64[b], see, D ** -0.5 if scale is None else scale)
        off = (ob.double() - want).abs()
        tol = tolerance(want, weight, slip, dtype)
        assert torch.equal(torch.isnan(ob), torch.isnan(want))
        bad = (off > tol) & ~torch.isnan(want) & ~torch.isinf(want)
        assert not bool(bad.any()), (b, float((off / tol)[~torch.isnan(off)].max()), torch.nonzero(bad)[:4].tolist())
        assert torch.equal(ob.double()[torch.isinf(want)], want[torch.isinf(want)])
        fin = torch.isfinite(wl)
        # the log of a sum whose terms are off by slip and a few 2^-22, rounded to 32 bits
        assert bool(((lb.double() - wl).abs()[fin] <= (2 * slip[..., 0] + 64 * 2.0 ** -22 + wl.abs() * 2.0 ** -22)[fin]).all())


STORES = ["native", "int8", "fp8"]


@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05", "simt"])
@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,ps", [(8, 2, 128, 16), (5, 1, 64, 12), (4, 4, 128, 1), (14, 2, 128, 7), (16, 1, 64, 64), (20, 1, 128, 16)])
def test_single_tokens(backend, storage, dtype, Hq, Hkv, D, ps):
    p = Paged([1, 17, 0, 300, 129, 64], Hkv, D, ps, dtype, storage, seed=Hq)
    check(p, [1] * 6, Hq, backend=backend)


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (7, 0), (64, 4), (100, 200), (10 ** 6, 5), (129, 1)])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_window_and_sinks(storage, window, sinks, n):
    p = Paged([n, n + 30, n + 257, n + 600], 2, 128, 16, torch.bfloat16, storage, seed=window + n)
    check(p, [n] * 4, 8, window=window, sinks=sinks)


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,ps,n", [(8, 2, 128, 16, 2), (8, 2, 128, 12, 5), (6, 2, 64, 16, 33), (4, 1, 128, 64, 64),
                                           (10, 2, 128, 16, 130), (3, 3, 128, 8, 200), (8, 1, 64, 48, 90)])
def test_chunks(storage, dtype, Hq, Hkv, D, ps, n):
    p = Paged([n, n + 1, n + 150, 0, n + 64], Hkv, D, ps, dtype, storage, seed=n)
    check(p, [n] * 5, Hq, q_layout="BNHD" if n % 2 else "plain")


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("new", [[1, 1, 40, 0, 7, 1], [0, 0, 1], [130, 1, 1, 64], [3, 2, 1, 0]])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3)])
def test_packed_rows(storage, new, window, sinks):
    before = [0, 200, 77, 9, 30, 500]
    p = Paged([c + before[b] if c else 0 for b, c in enumerate(new)], 2, 128, 16, torch.float16, storage, seed=len(new))
    check(p, new, 10, packed=True, window=window, sinks=sinks)
    check(p, new, 10, packed=True, window=window, sinks=sinks, max_q=sum(new))


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("n,max_depth", [(1, None), (2, 5), (7, 5), (31, 5), (31, 1), (64, 5), (64, 0), (100, None), (257, 5)])
@pytest.mark.parametrize("shared", [False, True])
def test_trees(storage, n, max_depth, shared):
    rng = random.Random(n)
    lens = [n, n + 100, n + 333]
    parents = [random_tree(n, rng, 9) for _ in lens]
    p = Paged(lens, 2, 128, 16, torch.bfloat16, storage, seed=n)
    check(p, [n] * 3, 8, parents=parents[0] if shared else parents, max_depth=max_depth)


@pytest.mark.parametrize("n,window,sinks,P", [(31, 4, 2, 50), (64, 100, 4, 300), (64, 3, 0, 0), (20, 2, 30, 5), (100, 1, 0, 64), (9, 40, 1, 30)])
def test_trees_in_a_window(n, window, sinks, P):
    rng = random.Random(n + window)
    p = Paged([n + P, n + 2 * P + 1], 2, 128, 16, torch.float16, seed=n)
    for depth in (None, 2):
        check(p, [n] * 2, 6, parents=[random_tree(n, rng, 12) for _ in range(2)], max_depth=depth, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,D,layout,q_layout", [(torch.float32, 128, "HSD", "plain"), (torch.bfloat16, 40, "HSD", "plain"),
                                                     (torch.float16, 256, "SHD", "BNHD"), (torch.bfloat16, 128, "pad", "plain"),
                                                     (torch.bfloat16, 128, "HSD", "pad"), (torch.float32, 33, "pad", "pad"),
                                                     (torch.bfloat16, 128, "SHD", "BNHD")])
@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("n", [1, 37])
def test_layouts_and_other_sizes(dtype, D, layout, q_layout, storage, n):
    p = Paged([n + 70, n, n + 200], 2, D, 16, dtype, storage, seed=D, layout=layout)
    check(p, [n] * 3, 6, q_layout=q_layout, scale=0.3)


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("n,Hq", [(1, 8), (4, 8), (70, 8)])
def test_long_sequences(storage, n, Hq):
    """Sequences that many CTAs share, beside short ones."""
    p = Paged([n + 9000, n + 3, n + 2500], 1, 128, 16, torch.bfloat16, storage, seed=n)
    check(p, [n] * 3, Hq)
    check(p, [n] * 3, Hq, window=4000, sinks=2)


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n", [1, 4, 70])
def test_infinities_and_nan(where, what, n):
    """A bad value reaches the rows that see it and no others: a new row's
    successors, a cached row's window."""
    lens = [n + 200, n + 90]
    p = Paged(lens, 2, 128, 16, torch.bfloat16, seed=n)
    pages, held = (p.k_pages, p.k64) if where == "k" else (p.v_pages, p.v64)
    for b, pos in ((0, lens[0] - 1), (0, 150), (1, lens[1] - max(1, n // 2))):
        if where == "k":  # a score of +-inf or NaN: whole rows of NaN, where it is seen (an infinite q.k needs one sign)
            held[b][pos, :, 7] = math.nan
            pages[int(p.table[b, pos // 16]), :, pos % 16, 7] = math.nan
        else:
            held[b][pos, :, 7] = what
            pages[int(p.table[b, pos // 16]), :, pos % 16, 7] = what
    check(p, [n] * 2, 8, window=30)
    if n > 1:
        rng = random.Random(n)
        check(p, [n] * 2, 8, parents=[random_tree(n, rng, 5) for _ in range(2)])


@pytest.mark.parametrize("storage", ["int8", "fp8"])
@pytest.mark.parametrize("n", [1, 70])
def test_rows_stored_as_nan(storage, n):
    """8-bit rows with scale NaN poison the rows that see them only."""
    lens = [n + 200]
    p = Paged(lens, 1, 128, 16, torch.float16, storage, seed=n)
    for pos in (20, n + 199):
        pg, r = int(p.table[0, pos // 16]), pos % 16
        p.v_scale[pg, :, r] = math.nan
        p.v64[0][pos] = math.nan
    check(p, [n], 4, window=60 + n)


@pytest.mark.parametrize("storage", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e-4, 100.0, 60000.0])
@pytest.mark.parametrize("n", [1, 70])
def test_rows_of_any_size(storage, dtype, size, n):
    """V far from 1 in size: weights times scales keep their precision."""
    p = Paged([n + 300], 2, 128, 16, dtype, storage, seed=3, scale_of=lambda b, name: size / 4 if name == "v" else 1.0)
    check(p, [n], 4)


@pytest.mark.parametrize("n", [1, 5, 80])
def test_large_scores(n):
    """Scores of hundreds: the running maximum moves by more than exp can span."""
    p = Paged([n + 700], 2, 128, 16, torch.bfloat16, seed=n, scale_of=lambda b, name: 20.0 if name == "k" else 1.0)
    check(p, [n], 8)


def test_streams_and_graph_replay():
    """Two calls on two streams at once, and a captured step replayed with other
    lengths, tables and rows."""
    B, Hq, Hkv, D, ps = 3, 8, 2, 128, 16
    p = Paged([40, 700, 1], Hkv, D, ps, torch.bfloat16, "int8", seed=1, table_cols=60)
    r = Paged([900, 33, 5], Hkv, D, ps, torch.bfloat16, "int8", seed=1, table_cols=60, spare=1)
    q = torch.randn(B, Hq, 1, D, device="cuda").bfloat16()
    want = [G.paged_attention(q, *x.args, **x.held) for x in (p, r)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(20):
        for i, (st, x) in enumerate(zip(streams, (p, r))):
            with torch.cuda.stream(st):
                got[i] = G.paged_attention(q, *x.args, **x.held)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pages = max(p.k_pages.shape[0], r.k_pages.shape[0])
    grow = lambda t: torch.cat([t.view(torch.uint8) if t.element_size() == 1 else t, torch.zeros((pages - t.shape[0],) + t.shape[1:],  # noqa: E731
                               dtype=torch.uint8 if t.element_size() == 1 else t.dtype, device="cuda")]).view(t.dtype)
    bufs = [grow(t) for t in (p.k_pages, p.v_pages, p.k_scale, p.v_scale)]
    table, lens = p.table_d.clone(), p.lens_d.clone()
    call = lambda: G.paged_attention(q, bufs[0], bufs[1], table, lens, k_scale=bufs[2], v_scale=bufs[3])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0])
    for buf, t in zip(bufs, (r.k_pages, r.v_pages, r.k_scale, r.v_scale)):
        buf.copy_(grow(t))
    table.copy_(r.table_d), lens.copy_(r.lens_d)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[1])
    del graph


def test_bad_tables_and_lengths():
    """Bad pages hide their rows, bad lengths make a slot unused; both are reported."""
    D = 128
    p = Paged([40, 40, 40, 40], 2, D, 16, torch.bfloat16, table_cols=3)
    q = torch.randn(4, 8, 2, D, device="cuda").bfloat16()
    good = G.paged_attention(q, *p.args)
    table, lens = p.table_d.clone(), p.lens_d.clone()
    table[1, 1] = -7
    lens[2], lens[3] = 1, 49
    out, lse = G.paged_attention(q, p.k_pages, p.v_pages, table, lens, return_lse=True)
    assert G.device_error() == (1 << 6) | (1 << 3)
    assert torch.equal(out[0], good[0]) and bool(torch.isfinite(out).all())
    assert bool((out[2:] == 0).all()) and bool((lse[2:] == -math.inf).all())
    see = visible(40, 2)
    see[:, 16:32] = False
    want, weight, slip, _ = attend(q[1].cpu(), p.k64[1], p.v64[1], see, D ** -0.5)
    assert bool(((out[1].cpu().double() - want).abs() <= tolerance(want, weight, slip, torch.bfloat16)).all())
    par = torch.tensor([-1, 9], dtype=torch.int32)
    G.paged_attention(q, *p.args, parents=par)
    assert G.device_error() == 1


def test_step_of_a_server():
    """Append, attend, verify-like trim and read together, on an 8-bit cache of
    two layers: each step's attention equals one over the rows read back."""
    layers, Hq, Hkv, D, ps, B = 2, 8, 2, 128, 16, 3
    for storage in STORES:
        cache = G.PagedKVCache(layers, 64, ps, Hkv, D, torch.bfloat16, storage)
        order = torch.randperm(60, generator=torch.Generator().manual_seed(0)).to(torch.int32)
        table = order.reshape(B, 20).cuda()
        lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(1)
        rng = random.Random(5)

        def rows(h, n):
            return torch.randn(B, h, n, D, device="cuda", generator=g).bfloat16()

        for n, tree in ((100, False), (1, False), (40, True), (1, False), (17, True), (30, False)):
            lens += n
            parents = torch.tensor([random_tree(n, rng, 5) for _ in range(B)], dtype=torch.int32, device="cuda") if tree else None
            for layer in range(layers):
                k, v, q = rows(Hkv, n), rows(Hkv, n), rows(Hq, n)
                cache.append(layer, k, v, table, lens)
                out = cache.attend(layer, q, table, lens, parents=parents, max_depth=5 if tree else None)
                cu = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), lens.cumsum(0).to(torch.int32)])
                total = int(cu[-1])
                kk, vv = cache.read(layer, table, cu, total)
                par = parents if tree else torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")
                if n <= 256:
                    ref = G.tree_attention(q.float(), kk.float(), vv.float(), parents=par, max_depth=None if not tree else 5,
                                           cu_seqlens=cu, max_seqlen=int(lens.max()))
                    # rows read back are rounded to bf16 once more when stored in 8 bits (2^-8 of each value, and of
                    # the scores through K: |q . dk| <= 2^-8 * sum |q k| ~ 2^-8 * 128 * 0.6 * 0.09 in ordinary rows)
                    tol = 0.02 if storage == "native" else 0.06
                    assert float((out.float() - ref).abs().max()) < tol
            if tree:
                acc = torch.tensor([rng.randrange(1, 5) for _ in range(B)], dtype=torch.int32, device="cuda")
                path = torch.zeros(B, 5, dtype=torch.int32)
                for b in range(B):
                    at = [0]
                    par_b = parents[b].tolist()
                    while len(at) < int(acc[b]):
                        kids = [j for j in range(n) if par_b[j] == at[-1]]
                        if not kids:
                            break
                        at.append(rng.choice(kids))
                    acc[b] = len(at)
                    path[b, :len(at)] = torch.tensor(at)
                start = lens - n
                before = [cache.read(layer, table, torch.tensor([0, n, 2 * n, 3 * n]).cuda(), B * n, starts=start) for layer in range(layers)]
                cache.trim(table, path.cuda() + start[:, None], acc, start)
                for layer in range(layers):
                    now = cache.read(layer, table, torch.tensor([0, n, 2 * n, 3 * n]).cuda(), B * n, starts=start)
                    for b in range(B):
                        for r in range(int(acc[b])):
                            for i in range(2):
                                assert torch.equal(now[i][b * n + r], before[layer][i][b * n + int(path[b, r])])
                lens = (start + acc).to(torch.int32)
