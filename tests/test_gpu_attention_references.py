"""Attention on the tensor cores when rows of one warp move their softmax reference in the same key tile for different
reasons: a tile is rescaled once because a row's reference has been outgrown, and again because another row of the warp has
no reference yet or asks for the tile to be redone.  Against 64 bits, in the tolerances of the paged cache's tests."""
from types import SimpleNamespace

import pytest
import torch

import torch_paras  # noqa: F401
from torch_paras import abi

from paged_cases import E4M3, Cache, attend64, attend_tolerance, cu_of, quantise64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
LN2 = 0.6931471805599453
COPIES = 150      # of the same sequence (or head), so that a block walks whole ones, tile after tile

# exponents of 2 that the keys of tile 0, 1, 2, ... get against a query of ones: steps that outgrow a reference by 2^8 (the
# tile is rescaled before the next one) while all older tiles keep a part of the row; one that outgrows it by 2^15 at once
# (the tile is redone) right behind such a step; falling ones
RISING = [0, 3, 6, 9, 12, 15, 18, 20, 24, 26, 28, 30]
JUMPS = [0, 3, 26, 28, 24, 48, 49, 50, 44, 52, 56, 56]


def keys(levels, D, dtype, n):
    level = torch.tensor(levels, dtype=torch.float64).repeat_interleave(128)[:n]
    return level[:, None, None].expand(n, 1, D).to(dtype)


def queries(T, D, dtype, nan_rows):
    # rows that meet the levels in full, in half and not at all, side by side in every warp
    q = torch.ones(T, 1, D)
    q[1::4] *= 0.5
    q[2::4] *= 0.0
    for r in nan_rows:
        q[r, 0, 3] = float("nan")
    return q.to(dtype).to(DEV)


def compare(o, q, c, n, scale, causal, dtype, D, nan_rows):
    # o [copies, rows, 1, D]
    want, _, A, S = attend64(q, c, [q.shape[0]], [n], scale, causal)
    tol = attend_tolerance(want, A, S, dtype, D, n)
    fine = torch.ones(q.shape[0], dtype=torch.bool)
    fine[list(nan_rows)] = False
    err = (o.cpu().double() - want).abs()[:, fine]
    bad = ~(err <= tol[fine])
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol[fine]).max()):.2f} of the tolerance"
    assert torch.isnan(o.cpu()[:, ~fine]).all()


@pytest.mark.parametrize("levels", [RISING, JUMPS], ids=["rising", "jumps"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("nan_rows", [(), (5, 77, 150)], ids=["plain", "nan"])
def test_paged_chunks(nan_rows, cache8, D, levels):
    # a query of NaN has no reference in any tile, and asks for every tile to be redone
    n, T, dtype = 1500, 200, HF if D == 64 else BF
    for causal in (False, True):
        c = Cache([n], 1, D, 64, dtype, cache8, seed=3)
        x = keys(levels, D, dtype, n)
        pos = torch.arange(n)
        where, off = c.table[0].long().cpu()[pos // 64], pos % 64
        if cache8:
            val, e = quantise64(x)
            raw, ex = c.cache[0].view(torch.uint8), c.exps[0]
            raw[where, :, off] = val.float().to(E4M3).view(torch.uint8).to(DEV)
            ex[where, :, off] = (e + 127).to(torch.uint8).to(DEV)
            c.dense[0][0] = val * torch.pow(2.0, e).unsqueeze(-1)
        else:
            c.cache[0][where, :, off] = x.to(DEV)
            c.dense[0][0] = x.double()
        q = queries(T, D, dtype, nan_rows)
        o = abi.paged_attention(q.repeat(COPIES, 1, 1), *c.cache, c.table.repeat(COPIES, 1), c.kv_lens.repeat(COPIES),
                                cu_of([T] * COPIES), T, causal=causal, scale=LN2 / D, **c.kw)
        assert abi.paged_attn_last_kernel() == "paged_tcgen05"
        compare(o.view(COPIES, T, 1, D), q, c, n, LN2 / D, causal, dtype, D, nan_rows)


@pytest.mark.parametrize("levels", [RISING, JUMPS], ids=["rising", "jumps"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nan_rows", [(), (5, 77, 150)], ids=["plain", "nan"])
def test_dense(nan_rows, D, levels):
    n, T, dtype = 1500, 256, HF if D == 64 else BF
    g = torch.Generator().manual_seed(4)
    k, v = keys(levels, D, dtype, n), torch.randn(n, 1, D, generator=g).to(dtype)
    q = queries(T, D, dtype, nan_rows)
    view = lambda t: t.to(DEV).transpose(0, 1).unsqueeze(0).repeat(1, COPIES, 1, 1)     # noqa: E731  [rows, 1, D] -> [1, copies, rows, D]
    o = abi.sdpa_fwd(view(q), view(k), view(v), scale=LN2 / D)
    assert abi.sdpa_last_kernel().startswith("tcgen05")
    c = SimpleNamespace(Hkv=1, page=1, dense=[[k.double()], [v.double()]])
    compare(o[0].unsqueeze(2), q, c, n, LN2 / D, False, dtype, D, nan_rows)
