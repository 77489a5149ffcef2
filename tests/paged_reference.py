"""The paged operators in 64 bits on the host, and inputs for their tests."""
from __future__ import annotations

import math
import random

import torch

LARGEST = {"int8": 127.0, "fp8": 448.0}
EIGHT = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def quantise(x: torch.Tensor, storage: str):
    """(values as stored, scale) of rows [..., D], in 64 bits but for the
    rounding that the format itself defines."""
    x = x.double()
    amax = x.abs().amax(-1).clamp(min=2.0 ** -100)
    frac, power = torch.frexp(LARGEST[storage] / amax)
    inv = torch.ldexp(torch.floor(frac * 4096) / 4096, power)
    y = x * inv[..., None]
    if storage == "int8":
        y = torch.round(y)
    else:
        step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 4).clamp(min=-9))
        y = torch.round(y / step) * step
    return y, (1.0 / inv).float()


class Paged:
    """Random pages of one layer with a block table per sequence.  What no
    sequence holds (rows past an end, spare pages) is poison: NaN rows, NaN
    scales; unused table entries are far outside the pool."""

    def __init__(self, lens, Hkv, D, ps, dtype, storage="native", seed=0, layout="HSD", table_cols=None, spare=2,
                 poison=True, scale_of=lambda b, p: 1.0):
        self.lens, self.Hkv, self.D, self.ps, self.dtype, self.storage = list(lens), Hkv, D, ps, dtype, storage
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        need = [-(-x // ps) for x in lens]
        pages = sum(need) + spare
        order = list(range(pages))
        rng.shuffle(order)
        cols = table_cols or max(need + [1])
        self.table = torch.full((len(lens), cols), 10 ** 6, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
            at += k
        self.k64, self.v64 = [], []  # what each sequence's rows stand for, [L, Hkv, D]
        raw = {}
        for name, keep in (("k", self.k64), ("v", self.v64)):
            x = torch.full((pages, Hkv, ps, D), math.nan if poison else 0.0, dtype=torch.float64)
            sc = torch.full((pages, Hkv, ps), math.nan if poison else 0.0, dtype=torch.float32)
            for b, L in enumerate(lens):
                top = torch.finfo(dtype).max  # rows of finite values: what an append of others stores is tested apart
                rows = (torch.randn(L, Hkv, D, generator=g) * scale_of(b, name)).clamp(-top, top).to(dtype).double()
                if storage == "native":
                    vals = rows
                else:
                    q, s = quantise(rows, storage)
                    vals = q * s.double()[..., None]
                keep.append(vals)
                for p in range(L):
                    pg, r = int(self.table[b, p // ps]), p % ps
                    x[pg, :, r] = rows[p] if storage == "native" else q[p]
                    if storage != "native":
                        sc[pg, :, r] = s[p]
            if storage == "native":
                x = x.to(dtype)
            elif storage == "int8":
                x = torch.nan_to_num(x, nan=77.0).to(torch.int8)
            else:
                x = torch.nan_to_num(x, nan=77.0).float().to(torch.float8_e4m3fn)
            raw[name], raw[name + "s"] = x, (None if storage == "native" else sc)
        self.k_pages, self.v_pages = self._laid(raw["k"], layout), self._laid(raw["v"], layout)
        self.k_scale = None if raw["ks"] is None else raw["ks"].cuda()
        self.v_scale = None if raw["vs"] is None else raw["vs"].cuda()
        self.table_d, self.lens_d = self.table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()

    @staticmethod
    def _laid(x, layout):
        if layout == "HSD":
            return x.cuda()
        if layout == "SHD":  # rows of all heads together, as a strided view
            b = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
            b = b.transpose(1, 2).contiguous().cuda()
            return (b.view(x.dtype) if x.dtype == torch.float8_e4m3fn else b).transpose(1, 2)
        if layout == "pad":  # rows 3 elements further apart than they are long: no 16-byte alignment
            y = torch.empty(x.shape[:-1] + (x.shape[-1] + 3,), dtype=x.dtype, device="cuda")
            b = y.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else y
            b[..., : x.shape[-1]] = (x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x).cuda()
            return y[..., : x.shape[-1]]
        raise ValueError(layout)

    @property
    def held(self):
        return dict(k_scale=self.k_scale, v_scale=self.v_scale)

    @property
    def args(self):
        return self.k_pages, self.v_pages, self.table_d, self.lens_d


def visible(L, c, parents=None, max_depth=None, window=None, sinks=0):
    """Boolean [c, L]: what each new row sees."""
    P = L - c
    see = torch.zeros(c, L, dtype=torch.bool)
    pos = list(range(L))
    above = []
    for i in range(c):
        chain = [i]
        if parents is not None:
            while parents[chain[-1]] >= 0:
                chain.append(parents[chain[-1]])
            pos[P + i] = P + len(chain) - 1
        above.append(chain)
    for i in range(c):
        see[i, :P] = True
        if parents is None:
            see[i, P:P + i + 1] = True
        else:
            for hop, j in enumerate(above[i]):
                if max_depth is None or hop <= max_depth:
                    see[i, P + j] = True
        if window is not None:
            for j in range(L):
                if j >= sinks and pos[P + i] - pos[j] >= window:
                    see[i, j] = False
    return see


def attend(q, k, v, see, scale):
    """q [Hq, c, D], k / v [L, Hkv, D], see [c, L], in 64 bits: (out, weight, slip,
    lse): `weight` is sum p |v| / sum p, `slip` bounds what 32-bit scores lose,
    relative to a weight."""
    Hq, c, D = q.shape
    group = Hq // k.shape[1]
    q = q.double()
    kk, vv = k.repeat_interleave(group, 1).transpose(0, 1), v.repeat_interleave(group, 1).transpose(0, 1)
    ok = see[None]
    s = torch.where(ok, q @ torch.nan_to_num(kk).transpose(1, 2) * scale, -math.inf)
    s = torch.where(ok & ~torch.isfinite(kk).all(-1)[:, None], math.nan, s)
    p = torch.softmax(s, -1)
    p0 = torch.where(ok, p, 0.0)
    clean = torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
    out = p0 @ clean
    bad = ~torch.isfinite(vv)
    if bool(bad.any()):  # visible infinities and NaN, one key at a time
        for j in torch.nonzero(bad.any(0).any(-1)).flatten().tolist():
            add = p0[:, :, j, None] * torch.where(bad[:, j], vv[:, j], 0.0)[:, None]
            out = torch.where(see[None, :, j, None], out + add, out)
    weight = p0 @ clean.abs()
    slip = (q.abs() @ torch.nan_to_num(kk).abs().transpose(1, 2) * scale).amax(-1, keepdim=True) * (D + 4) * 2.0 ** -24
    return out, weight, slip, torch.logsumexp(s, -1)


def tolerance(out, weight, slip, dtype, weights_rounded=True):
    """What a kernel may be off by.  Scores are summed in 32 bits (slip: relative
    to every weight, twice: in the sum of weights too); exponentials, sums and
    the division cost a few 2^-22; the weights are rounded to the type of V
    before their product (half a step each, relative to sum p |v|); the result
    is rounded once (half a step), and a 16-bit float's steps end at its
    smallest subnormal."""
    half = torch.finfo(dtype).eps / 2
    rounded = half if weights_rounded and dtype != torch.float32 else 0.0
    return half * out.abs() * 1.01 + weight * (rounded * 1.01 + 2 * slip + 16 * 2.0 ** -22) + torch.finfo(dtype).tiny * half + 1e-30
