"""What the paged operators' documentation promises at its edges."""
from __future__ import annotations

import math
import random
import threading

import pytest
import torch

import projectgorgon_b200 as G
from paged_reference import Paged, quantise, visible
from projectgorgon_b200 import _abi
from projectgorgon_b200.trees import random_tree
from test_gpu_paged_attention import check

pytestmark = pytest.mark.gpu

STORES = ["native", "int8", "fp8"]


@pytest.fixture(autouse=True)
def no_device_error():
    G.device_error(clear=True)
    yield
    assert G.device_error(clear=True) == 0


@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05", "simt"])
@pytest.mark.parametrize("tree", [False, True])
def test_rows_where_max_q_is_zero(backend, tree):
    """max_q = 0 is a bound that every sequence with rows passes: zeros, and reported, as for any other."""
    p = Paged([50, 0, 70], 2, 128, 16, torch.bfloat16, seed=1)
    q = torch.randn(9, 8, 128, device="cuda").bfloat16()
    cu = torch.tensor([0, 3, 5, 7], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 3.0)
    parents = torch.tensor([-1, 0, 1]) if tree else None
    _, lse = G.paged_attention(q, *p.args, cu_q=cu, max_q=0, parents=parents, out=out, return_lse=True, backend=backend)
    assert G.device_error(clear=True) == _abi.ERR_BAD_SEQLEN
    assert bool((out[:7] == 0).all()) and bool((lse[:7] == -math.inf).all()) and bool((out[7:] == 3.0).all())
    # nothing but unused slots: zeros, and nothing to report
    out.fill_(3.0)
    _, lse = G.paged_attention(q, p.k_pages, p.v_pages, p.table_d, torch.zeros_like(p.lens_d), cu_q=cu, max_q=0, parents=parents,
                               out=out, return_lse=True, backend=backend)
    assert bool((out[:7] == 0).all()) and bool((lse[:7] == -math.inf).all()) and bool((out[7:] == 3.0).all())


@pytest.mark.parametrize("storage", STORES)
@pytest.mark.parametrize("backend", ["auto", "simt"])
def test_log_sum_exp_of_rows_of_no_values(storage, backend):
    """head_dim 0: every score is 0, so the log-sum-exp is the log of how many keys a row sees."""
    p = Paged([5, 40], 2, 8, 16, torch.bfloat16, storage, seed=1)
    q = torch.empty(2, 4, 3, 0, device="cuda", dtype=torch.bfloat16)
    out, lse = G.paged_attention(q, p.k_pages[..., :0], p.v_pages[..., :0], p.table_d, p.lens_d, window=20, return_lse=True,
                                 backend=backend, **p.held)
    assert out.shape == q.shape
    for b, L in enumerate(p.lens):
        want = visible(L, 3, window=20).sum(-1).double().log()
        assert bool(((lse[b].cpu().double() - want).abs() <= want * 4 * 2.0 ** -23 + 2.0 ** -22).all())


@pytest.mark.parametrize("storage", STORES)
def test_trim_refuses_expanded_pages(storage):
    """Kv heads or layers that are one in memory; a single one may have any stride."""
    p = Paged([40], 1, 64, 16, torch.bfloat16, storage, seed=1, poison=False)
    idx, ln = torch.tensor([[3, 1]], device="cuda"), torch.tensor([2], device="cuda")
    before = [x.clone() for x in (p.k_pages, p.v_pages)]
    for wide in (lambda t: None if t is None else t.expand(-1, 4, *t.shape[2:]), lambda t: None if t is None else t.expand(2, *t.shape)):
        with pytest.raises(RuntimeError, match="stride of 0"):
            G.paged_cache_trim(wide(p.k_pages), wide(p.v_pages), p.table_d, idx, ln, 0, k_scale=wide(p.k_scale), v_scale=wide(p.v_scale))
    as_bytes = lambda t: t.view(torch.uint8)  # noqa: E731
    assert all(torch.equal(as_bytes(a), as_bytes(b)) for a, b in zip(before, (p.k_pages, p.v_pages)))
    one = lambda t: None if t is None else t.as_strided((1,) + t.shape, (0,) + t.stride())  # noqa: E731
    G.paged_cache_trim(one(p.k_pages), one(p.v_pages), p.table_d, idx, ln, 0, k_scale=one(p.k_scale), v_scale=one(p.v_scale))
    first = int(p.table[0, 0])
    assert torch.equal(as_bytes(p.k_pages)[first, :, :2], as_bytes(before[0])[first][:, [3, 1]])


@pytest.mark.parametrize("dtype,D,storage,layout,m", [
    (torch.float32, 256, "native", "HSD", 256), (torch.float32, 256, "native", "pad", 201), (torch.bfloat16, 256, "native", "HSD", 256),
    (torch.float32, 33, "native", "HSD", 256), (torch.bfloat16, 250, "fp8", "HSD", 256), (torch.float16, 128, "int8", "HSD", 255)])
def test_trim_of_as_many_rows_as_documented(dtype, D, storage, layout, m):
    """256 rows of any size, overlapping: a reversal and a shift."""
    H, ps, L = 2, 16, 600
    p = Paged([L, L], H, D, ps, dtype, storage, seed=D, layout=layout, poison=False)
    src = torch.stack([torch.arange(m - 1, -1, -1), torch.arange(m) + 7]).to(torch.int32)
    dst = torch.tensor([0, 3], dtype=torch.int32)
    ln = torch.tensor([m, m - 1], dtype=torch.int32)
    as_bytes = lambda t: t.contiguous().view(torch.uint8) if t.element_size() == 1 else t.contiguous()  # noqa: E731
    want = [as_bytes(t).clone() if t is not None else None for t in (p.k_pages, p.v_pages, p.k_scale, p.v_scale)]
    for t in want:
        if t is not None:
            old = t.clone()
            for b in range(2):
                for r in range(int(ln[b])):
                    i, o = int(src[b, r]), int(dst[b]) + r
                    t[int(p.table[b, o // ps]), :, o % ps] = old[int(p.table[b, i // ps]), :, i % ps]
    G.paged_cache_trim(p.k_pages, p.v_pages, p.table_d, src.cuda(), ln.cuda(), dst.cuda(), **p.held)
    for t, w in zip((p.k_pages, p.v_pages, p.k_scale, p.v_scale), want):
        if w is not None:
            assert torch.equal(as_bytes(t), w)


def test_trims_of_several_host_threads():
    """Trims of different widths, launched by four threads at once, each on its own pages."""
    errors = []

    def work(m):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                p = Paged([300], 2, 128, 16, torch.float32, seed=m, poison=False)
                want = p.k_pages.clone()
                first, second = int(p.table[0, 0]), int(p.table[0, m // 16])
                want[first, :, 0] = p.k_pages[second, :, m % 16]
                idx = torch.full((1, m), m, dtype=torch.int32, device="cuda")
                ln = torch.ones(1, dtype=torch.int32, device="cuda")
                for _ in range(300):
                    G.paged_cache_trim(p.k_pages, p.v_pages, p.table_d, idx, ln)
                st.synchronize()
                assert torch.equal(p.k_pages, want)
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(m,)) for m in (100, 256, 130, 200)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def found(cu, batch, r):
    """The (sequence, number in it) that a search for row r among the counts ends at, or None."""
    if r < cu[0] or r >= cu[batch]:
        return None
    lo, hi = 0, batch - 1
    while lo < hi:
        mid = (lo + hi + 1) // 2
        if cu[mid] <= r:
            lo = mid
        else:
            hi = mid - 1
    if cu[lo] < 0 or not 0 <= r - cu[lo] < cu[lo + 1] - cu[lo]:
        return None
    return lo, r - cu[lo]


COUNTS = [[0, -3, 4, 6], [2, 5, 3, 6], [0, 5, 2, 6], [0, 2 ** 31 - 1, 3, 6], [-2 ** 31, 2, 3, 6], [0, 6, 0, 6], [0, 2, 4, 1], [0, 2, 0, 0],
          [-1, 2, 3, 6], [0, 0, 0, -1], [1, 1, 0, 6]]
IN_ORDER = [[0, 2, 4, 6], [1, 1, 3, 4], [0, 0, 6, 6], [2, 5, 5, 5], [6, 6, 6, 6]]


@pytest.mark.parametrize("cu", COUNTS + IN_ORDER)
@pytest.mark.parametrize("storage", ["native", "int8"])
@pytest.mark.parametrize("D", [128, 40])
@pytest.mark.parametrize("batch", [3, 1500])
def test_counts_are_checked_row_by_row(cu, storage, D, batch):
    """Append and read: every row lands where a search for it says and nowhere else; counts out of order are reported."""
    lens = [60, 50, 70]
    p = Paged(lens, 2, D, 16, torch.float16, storage, seed=1, poison=False)
    rows = torch.randn(2, 6, 2, D, device="cuda").half()
    many = cu + [cu[-1]] * (batch - 3)  # (more sequences than are kept in shared memory, all unused)
    counts = torch.tensor(many, dtype=torch.int32, device="cuda")
    pad = lambda t: torch.cat([t, t.new_zeros((batch - 3,) + t.shape[1:])])  # noqa: E731
    table, seq_lens = pad(p.table_d), pad(p.lens_d)
    word = _abi.ERR_BAD_SEQLEN if cu in COUNTS else 0
    where = [found(many, batch, r) for r in range(6)]
    where = [w if w is None or w[0] < 3 else None for w in where]
    # read first, from the pages as they are
    out = torch.full((2, 6, 2, D), 4.0, device="cuda", dtype=torch.float16)
    every = G.paged_cache_read(p.k_pages, p.v_pages, p.table_d, torch.tensor([0, 60, 110, 180], dtype=torch.int32, device="cuda"), 180,
                               dtype=torch.float16, **p.held)
    G.paged_cache_read(p.k_pages, p.v_pages, table, counts, 6, out=(out[0], out[1]), **p.held)
    assert G.device_error(clear=True) == word
    first = [0, 60, 110]
    for x, whole in zip(out, every):
        for r, w in enumerate(where):
            want = torch.full_like(x[r], 4.0) if w is None else whole[first[w[0]] + w[1]]
            assert torch.equal(x[r], want), (r, w)
    # append: what the rows say, and every other byte as it was
    want = [t.clone() if t is not None else None for t in (p.k_pages, p.v_pages, p.k_scale, p.v_scale)]
    for r, w in enumerate(where):
        if w is not None:
            b, i = w
            pos = lens[b] - (cu[b + 1] - cu[b]) + i
            if pos < 0 or lens[b] < cu[b + 1] - cu[b]:
                continue
            pg, at = int(p.table[b, pos // 16]), pos % 16
            for k in range(2):
                if storage == "native":
                    want[k][pg, :, at] = rows[k, r]
                else:
                    q, s = quantise(rows[k, r].cpu(), storage)
                    want[k][pg, :, at] = q.to(torch.int8).cuda()
                    want[2 + k][pg, :, at] = s.cuda()
    G.paged_cache_append(rows[0], rows[1], p.k_pages, p.v_pages, table, seq_lens, cu_q=counts, **p.held)
    assert G.device_error(clear=True) == word
    for t, w in zip((p.k_pages, p.v_pages, p.k_scale, p.v_scale), want):
        assert t is None or torch.equal(t, w)


@pytest.mark.parametrize("backend", ["mma", "tcgen05", "simt"])
@pytest.mark.parametrize("n,window,sinks,P", [(2, 1, 0, 20), (31, 4, 2, 50), (64, 3, 0, 0), (64, 9, 30, 5), (100, 1, 0, 64), (40, 200, 0, 400)])
def test_trees_in_any_order(backend, n, window, sinks, P):
    """Parents may stand behind their children."""
    rng = random.Random(n + window)
    trees = []
    for _ in range(2):
        tree, at = random_tree(n, rng, 12), list(range(n))
        rng.shuffle(at)
        moved = [-1] * n
        for i, up in enumerate(tree):
            moved[at[i]] = -1 if up < 0 else at[up]
        trees.append(moved)
    trees[0][:2] = [1, -1]  # (whatever hangs below them stays a tree: they are one root and its child)
    trees[0] = [up if i < 2 or up != i else -1 for i, up in enumerate(trees[0])]
    p = Paged([n + P, n + 2 * P + 1], 2, 128, 16, torch.float16, seed=n)
    for depth in (None, 2):
        check(p, [n] * 2, 6, parents=trees, max_depth=depth, window=window, sinks=sinks, backend=backend)
        check(p, [n] * 2, 6, parents=trees, max_depth=depth, backend=backend)


@pytest.mark.parametrize("n,window", [(9, 2), (37, 5)])
def test_float32_trees_in_any_order(n, window):
    """The same in a type that the CUDA cores alone take."""
    parents = [i + 1 for i in range(n - 1)] + [-1]  # a chain from the last row to the first
    p = Paged([n + 30], 2, 64, 16, torch.float32, seed=n)
    check(p, [n], 4, parents=parents, window=window, sinks=1)


@pytest.mark.parametrize("backend", ["mma", "tcgen05", "simt"])
@pytest.mark.parametrize("many", [2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1, 10 ** 30])
def test_options_larger_than_any_sequence(backend, many):
    p = Paged([40, 90], 2, 128, 16, torch.bfloat16, seed=1)
    q = torch.randn(2, 8, 3, 128, device="cuda").bfloat16()
    want = G.paged_attention(q, *p.args, parents=[-1, 0, 1], backend=backend)
    got = G.paged_attention(q, *p.args, parents=[-1, 0, 1], max_depth=many, window=many, sinks=many, backend=backend)
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("storage", STORES)
def test_captured_behind_copies_and_other_streams(n, storage):
    """Lengths and tables that a copy, or a kernel on a joined stream, writes just before a captured call: each replay sees its own."""
    lens = [n + 300, n + 20]
    p = Paged(lens, 2, 128, 16, torch.bfloat16, storage, seed=n)
    q = torch.randn(2, 8, n, 128, device="cuda").bfloat16()
    fresh_lens, seq_lens, table = p.lens_d.clone(), torch.zeros_like(p.lens_d), torch.zeros_like(p.table_d)
    fresh_table = p.table_d.clone()
    call = lambda: G.paged_attention(q, p.k_pages, p.v_pages, table, seq_lens, return_lse=True, **p.held)  # noqa: E731
    cases = [p.lens_d.clone(), torch.tensor([n + 17, n + 5], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda")]
    want = [G.paged_attention(q, p.k_pages, p.v_pages, p.table_d, x, return_lse=True, **p.held) for x in cases]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()

    def by_copy():
        table.copy_(fresh_table)
        seq_lens.copy_(fresh_lens)
        first = call()
        seq_lens.copy_(fresh_lens)
        return first, call()

    def by_join():
        table.copy_(fresh_table)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.add(fresh_lens, 0, out=seq_lens)
        torch.cuda.current_stream().wait_stream(side)
        first = call()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = call()
        torch.cuda.current_stream().wait_stream(side)
        return first, second

    for step in (by_copy, by_join):
        fresh_lens.copy_(cases[0])
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for x, w in list(zip(cases, want)) * 3:
            fresh_lens.copy_(x)
            seq_lens.zero_()
            table.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for got in outs:
                assert all(torch.equal(a, b) for a, b in zip(got, w))
        del graph


def test_calls_of_several_host_threads():
    """Attention of both tensor-core kernels, each thread on its own stream."""
    errors = []

    def work(n, storage):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                p = Paged([n + 200, n + 900], 2, 128, 16, torch.bfloat16, storage, seed=n)
                q = torch.randn(2, 8, n, 128, device="cuda").bfloat16()
                want = G.paged_attention(q, *p.args, **p.held)
                for _ in range(50):
                    assert torch.equal(G.paged_attention(q, *p.args, **p.held), want)
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=a) for a in ((1, "native"), (2, "int8"), (70, "native"), (64, "fp8"))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
