"""paged_attention over 8-bit pages whose V rows differ in size by many powers of
two, hidden from a query or seen by it: what a row sees keeps its precision."""
from __future__ import annotations

import random

import pytest
import torch

import projectgorgon_b200 as G
from paged_reference import Paged, attend, tolerance, visible
from projectgorgon_b200.trees import random_tree
from test_gpu_paged_attention import check

pytestmark = pytest.mark.gpu

EIGHT = ["int8", "fp8"]
KERNELS = ["mma", "tcgen05", "simt"]


@pytest.fixture(autouse=True)
def no_device_error():
    G.device_error(clear=True)
    yield
    assert G.device_error(clear=True) == 0


def sized(lens, rows, storage, dtype, ratio, seed=1, ps=16, small=1.0):
    """Pages whose V rows are of size `small`, those at `rows(L)` `ratio` times as large."""
    def scale_of(b, name):
        s = torch.ones(lens[b], 1, 1)
        if name == "v":
            s *= small
            s[rows(lens[b])] *= ratio
        return s
    return Paged(lens, 2, 128, ps, dtype, storage, seed=seed, scale_of=scale_of)


# (fp16 holds values of 2^-13 and of 2^15 with all their bits: a ratio of 2^28)
SIZES = [(torch.bfloat16, 1.0, 2.0 ** 10), (torch.bfloat16, 1.0, 2.0 ** 20), (torch.bfloat16, 1.0, 2.0 ** 31),
         (torch.bfloat16, 2.0 ** -30, 2.0 ** 60), (torch.bfloat16, 2.0 ** -60, 2.0 ** 120), (torch.bfloat16, 2.0 ** 40, 2.0 ** -70),
         (torch.float16, 2.0 ** -13, 2.0 ** 14), (torch.float16, 2.0 ** -13, 2.0 ** 27)]


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("dtype,small,ratio", SIZES)
@pytest.mark.parametrize("n", [2, 70])
def test_later_rows_of_a_chunk(backend, storage, dtype, small, ratio, n):
    """The chunk's second half is of another size: its first half does not see it."""
    p = sized([n + 200, n], lambda L: slice(L - n // 2, L), storage, dtype, ratio, small=small)
    check(p, [n] * 2, 8, backend=backend)


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("dtype,small,ratio", SIZES)
@pytest.mark.parametrize("n", [7, 64])
def test_other_branches_of_a_tree(backend, storage, dtype, small, ratio, n):
    rng = random.Random(n)
    p = sized([n + 190, n + 3], lambda L: [L - n + i for i in range(1, n) if i % 5 == 2], storage, dtype, ratio, small=small, ps=12)
    check(p, [n] * 2, 8, parents=[random_tree(n, rng, 6) for _ in range(2)], backend=backend)


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("dtype,small,ratio", SIZES)
@pytest.mark.parametrize("n,window,sinks", [(1, 40, 0), (3, 40, 2), (70, 50, 1)])
def test_rows_before_a_window(backend, storage, dtype, small, ratio, n, window, sinks):
    """Rows just before the first new row's window, and one inside the last one's."""
    p = sized([n + 300, n + 100], lambda L: [L - n - window - 1, L - n - window, L - window, L - n - 60], storage, dtype, ratio, small=small)
    check(p, [n] * 2, 8, window=window, sinks=sinks, backend=backend)


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("dtype,small,ratio", SIZES)
@pytest.mark.parametrize("n", [1, 20, 70])
def test_cached_rows_that_all_see(backend, storage, dtype, small, ratio, n):
    """A few large rows early, in the middle and late: also the columns where they hold zeros are right."""
    p = sized([n + 700, n + 90], lambda L: [3, L // 2, L - n - 1], storage, dtype, ratio, small=small)
    check(p, [n] * 2, 8, backend=backend)


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("spread", [4, 30, 100])
@pytest.mark.parametrize("n", [1, 24])
def test_every_row_of_its_own_size(backend, storage, spread, n):
    g = torch.Generator().manual_seed(spread)

    def scale_of(b, name):
        L = (n + 500, n + 70)[b]
        return torch.exp2((torch.rand(L, 1, 1, generator=g) - 0.5) * spread).round(decimals=12) + 2.0 ** -60 if name == "v" else 1.0
    p = Paged([n + 500, n + 70], 2, 128, 16, torch.bfloat16, storage, seed=n, scale_of=scale_of)
    check(p, [n] * 2, 8, backend=backend)


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("n", [1, 24])
def test_sizes_that_drift(backend, storage, up, n):
    """Sizes that rise or fall by 2^120 along the sequence, a little from row to row."""
    def scale_of(b, name):
        L = n + 900
        x = torch.arange(L).view(L, 1, 1) / L * 120 - 60
        return torch.exp2(x if up else -x) if name == "v" else 1.0
    p = Paged([n + 900], 2, 128, 16, torch.bfloat16, storage, seed=n, scale_of=scale_of)
    check(p, [n], 8, backend=backend)


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("n", [1, 40])
def test_a_large_row_of_negligible_weight(backend, storage, n):
    """A row 2^44 times the others whose score is 30 below theirs (a weight of 2^-43): both sides of the sum count."""
    L, D, Hq, pos = n + 300, 128, 8, 120
    p = sized([L], lambda _: [pos], storage, torch.bfloat16, 2.0 ** 44)
    q = torch.randn(1, Hq, n, D).bfloat16()
    q[..., 0] = 16.0
    # the row's K: -21.25 in the first column, zeros elsewhere; as stored bytes times a scale of 1
    pg, r = int(p.table[0, pos // 16]), pos % 16
    byte = -21.0 if storage == "int8" else -22.0
    row = torch.zeros(2, D)
    row[:, 0] = byte
    if storage == "int8":
        p.k_pages[pg, :, r] = row.to(torch.int8).cuda()
    else:
        p.k_pages.view(torch.uint8)[pg, :, r] = row.to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    p.k_scale[pg, :, r] = 1.0
    p.k64[0][pos] = row.double()
    out = G.paged_attention(q.cuda(), *p.args, backend=backend, **p.held)
    want, weight, slip, _ = attend(q[0], p.k64[0], p.v64[0], visible(L, n), D ** -0.5)
    off = (out[0].cpu().double() - want).abs()
    assert bool((off <= tolerance(want, weight, slip, torch.bfloat16)).all()), float((off / tolerance(want, weight, slip, torch.bfloat16)).max())


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("n", [1, 40])
def test_rows_of_zeros(backend, storage, n):
    """Rows of zeros (their scale is 2^-100 / largest) beside ordinary ones and alone."""
    p = sized([n + 200, n + 64], lambda L: slice(0, L, 3) if L > n + 64 else slice(0, L), storage, torch.bfloat16, 0.0)
    check(p, [n] * 2, 8, backend=backend)


@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("n,Hq", [(1, 8), (4, 8), (70, 8)])
def test_pieces_of_other_sizes(storage, n, Hq):
    """A sequence that many CTAs share, its thirds of other sizes: the pieces are joined in one unit."""
    L = n + 9000

    def scale_of(b, name):
        s = torch.ones(L, 1, 1)
        s[3000:6000] = 2.0 ** -40
        s[6000:] = 2.0 ** 30
        s[100] = 2.0 ** 50
        return s if name == "v" else 1.0
    p = Paged([L], 1, 128, 16, torch.bfloat16, storage, seed=n, scale_of=scale_of)
    check(p, [n], Hq)
    check(p, [n], Hq, window=5000, sinks=200)


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("n", [1, 40])
def test_queries_with_one_large_channel(backend, storage, n):
    """A channel 2^28 times the others, where K is 0: the others make the scores."""
    p = sized([n + 200, n + 40], lambda L: slice(0, 0), storage, torch.bfloat16, 1.0)
    p.k_pages.view(torch.uint8)[..., 5] = 0  # (zero bytes are 0 in both formats)
    for k in p.k64:
        k[..., 5] = 0
    q = torch.randn(2, 8, n, 128, generator=torch.Generator().manual_seed(9)).bfloat16()
    q[..., 5] = 2.0 ** 28
    out, lse = G.paged_attention(q.cuda(), *p.args, backend=backend, return_lse=True, **p.held)
    for b in range(2):
        # (the channel adds exact zeros: it takes no part in what the scores lose)
        small = q[b].clone()
        small[..., 5] = 0
        want, weight, slip, wl = attend(small, p.k64[b], p.v64[b], visible(p.lens[b], n), 128 ** -0.5)
        assert bool(((out[b].cpu().double() - want).abs() <= tolerance(want, weight, slip, torch.bfloat16)).all())
        assert bool(((lse[b].cpu().double() - wl).abs() <= 2 * slip[..., 0] + 64 * 2.0 ** -22 + wl.abs() * 2.0 ** -22).all())


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", EIGHT)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ps,Hq,new", [(12, 10, [1, 40, 0, 3]), (64, 2, [130, 1, 7, 1]), (16, 14, [5, 5, 60, 1])])
def test_narrow_heads_and_ragged_batches(backend, storage, dtype, ps, Hq, new):
    """head_dim 64, packed rows, a window: rows of three sizes in turn; and the same bits from call to call."""
    before = [200, 77, 9, 500]
    lens = [c + before[b] if c else 0 for b, c in enumerate(new)]

    def scale_of(b, name):
        i = torch.arange(lens[b]).view(-1, 1, 1)
        return torch.exp2((i % 7 == 3) * 13.0 - (i % 11 == 5) * 12.0) if name == "v" else 1.0
    p = Paged(lens, 2, 64, ps, dtype, storage, seed=ps, scale_of=scale_of)
    check(p, new, Hq, packed=True, window=60, sinks=3, backend=backend)
    check(p, new, Hq, packed=True, backend=backend)
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    q = torch.randn(sum(new), Hq, 64, device="cuda").to(dtype)
    first = G.paged_attention(q, *p.args, cu_q=cu, max_q=max(new), backend=backend, **p.held)
    assert all(torch.equal(first, G.paged_attention(q, *p.args, cu_q=cu, max_q=max(new), backend=backend, **p.held)) for _ in range(3))


@pytest.mark.parametrize("backend", KERNELS)
@pytest.mark.parametrize("storage", ["native", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("gap", [8.0, 14.0, 17.0])
def test_a_sink_that_holds_nothing(backend, storage, dtype, n, gap):
    """The first key takes nearly all weight and its V row is zeros: what the others weigh, e^-gap and less of it, is the output."""
    L, D, Hq = n + 600, 128, 8
    p = sized([L], lambda _: [0], storage, dtype, 0.0)
    q = torch.randn(1, Hq, n, D, generator=torch.Generator().manual_seed(4)).to(dtype)
    q[..., 0] = 16.0
    pg = int(p.table[0, 0])
    row = torch.zeros(2, D)
    row[:, 0] = 8.0  # as stored, and as a value: a score of `gap` with the scale below, 0 from the other columns
    if storage == "fp8":
        p.k_pages.view(torch.uint8)[pg, :, 0] = row.to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    else:
        p.k_pages[pg, :, 0] = row.to(p.k_pages.dtype).cuda()
    if storage != "native":
        p.k_scale[pg, :, 0] = 1.0
    p.k64[0][0] = row.double()
    # the others' scores: about 0, of a standard deviation of at most 1.5
    p.k_pages.view(torch.uint8 if storage != "native" else dtype)[:, :, :, 0] = 0
    p.k_pages.view(torch.uint8 if storage != "native" else dtype)[pg, :, 0, 0] = \
        row[0, 0].to(torch.float8_e4m3fn).view(torch.uint8).item() if storage == "fp8" else 8
    p.k64[0][1:, :, 0] = 0
    scale = gap / 128.0
    out = G.paged_attention(q.cuda(), *p.args, backend=backend, scale=scale, **p.held)
    want, weight, slip, _ = attend(q[0], p.k64[0], p.v64[0], visible(L, n), scale)
    tol = tolerance(want, weight, slip, dtype)
    off = (out[0].cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
