"""The paged cache on the GPU: its writer and reader bit for bit against the definition in 64 bits, attention over it
within tolerances that count its roundings, at the lengths, masks, pages and layouts where it can go wrong.  Everything a
call must not use is NaN."""
import pytest
import torch

import torch_paras  # noqa: F401
from torch_paras import abi

from paged_cases import E4M3, Cache, attend64, attend_tolerance, cu_of, lse_tolerance, quantise64, values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, dtype, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def widen(c):
    """A page table with the reach that long sequences need, most of it absent: a call that mixes a chunk with single tokens
    is then split (by the positions there may be)."""
    P = -(-4_000_000 // (c.Hkv * (len(c.table) - 1) * c.page))
    c.table = torch.cat([c.table, torch.full((len(c.table), P), -1, dtype=torch.int32, device=c.table.device)], 1)


def check_attention(q_lens, kv_lens, Hq, Hkv, D, page, dtype, cache8, causal=True, order="phd", seed=1, q=None, qscale=1.0,
                    absent=(), route=None, first=0, behind=0, scale=None, max_q=None, wide=False):
    c = Cache(kv_lens, Hkv, D, page, dtype, cache8, seed=seed, order=order)
    if wide:
        widen(c)
    for b, p in absent:
        c.table[b, p] = [-1, c.pages, 2 ** 31 - 1, -2 ** 31][p % 4]
    T = first + sum(q_lens) + behind
    if q is None:
        q = rand(T, Hq, D, dtype=dtype, seed=seed + 1, scale=qscale)
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, Hq, D), 77.0, dtype=dtype, device=DEV)
    o, lse = abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu_of(q_lens, first), max(q_lens + [0]) if max_q is None else max_q,
                                 causal=causal, scale=scale, out=out, return_lse=True, **c.kw)
    torch.cuda.synchronize()
    if route:
        assert abi.paged_attn_last_kernel() == route
    want, wlse, A, S = attend64(q, c, q_lens, kv_lens, scale, causal, first, absent)
    rows = slice(first, first + sum(q_lens))
    tol = attend_tolerance(want, A, S, dtype, D, max(kv_lens + [1]))
    err = (o.cpu().double() - want).abs()[rows]
    bad = ~(err <= tol[rows])
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol[rows]).max()):.2f} of the tolerance"
    l, w = lse.cpu().double()[rows], wlse[rows]
    assert torch.equal(torch.isinf(l), torch.isinf(w))
    fin = torch.isfinite(w)
    assert ((l - w).abs()[fin] <= lse_tolerance(w, S[rows], D, max(kv_lens + [1]))[fin]).all()
    # rows of no sequence keep what they held
    assert bool((o[:first] == 77).all()) and bool((o[first + sum(q_lens):] == 77).all())
    return o


TOKEN = ([1] * 7, [1, 2, 17, 128, 129, 640, 1000])
DRAFT = ([4, 2, 1, 3, 4], [4, 2, 300, 700, 129])
CHUNK = ([200, 1, 0, 77, 130], [200, 900, 50, 333, 131])


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("lens", [TOKEN, DRAFT, CHUNK], ids=["token", "draft", "chunk"])
def test_types(lens, dtype, cache8):
    check_attention(*lens, 8, 2, 128, 16, dtype, cache8)


@pytest.mark.parametrize("D", [1, 8, 40, 64, 80, 96, 128, 200, 256])
@pytest.mark.parametrize("cache8", [False, True])
def test_head_dims(D, cache8):
    check_attention([1, 3, 40], [100, 3, 75], 4, 2, D, 16, BF, cache8)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 64, 100, 128, 256, 512])
@pytest.mark.parametrize("cache8", [False, True])
def test_page_sizes(page, cache8):
    check_attention([1, 2, 30], [515, 129, 300], 4, 2, 64, page, HF, cache8)
    check_attention([1, 1, 1], [515, 129, 1], 4, 2, 128, page, BF, cache8)


@pytest.mark.parametrize("heads", [(1, 1), (2, 1), (3, 1), (6, 2), (5, 1), (7, 1), (16, 2), (12, 1), (16, 1), (17, 1), (64, 1), (130, 1), (8, 8)])
@pytest.mark.parametrize("lens", [([1, 1, 1], [3, 200, 513]), ([90, 3, 1], [200, 3, 513])], ids=["token", "chunk"])
def test_head_groups(heads, lens):
    check_attention(*lens, *heads, 64, 32, BF, False)
    check_attention(*lens, *heads, 128, 16, BF, True)


@pytest.mark.parametrize("lens", [TOKEN, DRAFT, CHUNK], ids=["token", "draft", "chunk"])
@pytest.mark.parametrize("cache8", [False, True])
def test_all_positions_attended(lens, cache8):
    check_attention(*lens, 8, 2, 64, 32, BF, cache8, causal=False)


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [40, 2, 64]], ids=["token", "chunk"])
def test_absent_pages_and_rows_that_attend_nothing(q_lens, dtype, cache8):
    # pages in the first tile, whole tiles, the last page; sequence 1 has none left; sequence 2 keeps only its last
    kv = [400, 48, 272]
    absent = [(0, 0), (0, 3)] + [(0, p) for p in range(8, 17)] + [(0, 24)] + [(1, p) for p in range(3)] + [(2, p) for p in range(16)]
    check_attention(q_lens, kv, 4, 2, 128, 16, dtype, cache8, absent=absent)


def test_more_new_tokens_than_positions_and_empty_sequences():
    # kv < q: the first rows stand before position 0 and attend nothing
    for dtype in (BF, FP):
        for cache8 in (False, True):
            check_attention([5, 1, 0, 3, 40], [2, 0, 0, 3, 9], 4, 2, 64, 16, dtype, cache8)
            check_attention([1, 1, 1], [0, 1, 0], 4, 2, 128, 16, dtype, cache8)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [33, 2, 1]], ids=["token", "chunk"])
def test_layouts_and_rows_of_no_sequence(q_lens):
    for cache8 in (False, True):
        check_attention(q_lens, [70, 300, 1], 8, 4, 128, 16, BF, cache8, order="pdh", first=3, behind=5)
    # q as the middle heads of a wider projection, the odd tokens only
    T = sum(q_lens)
    wide = rand(2 * T, 3 * 8, 64, dtype=HF, seed=5)
    check_attention(q_lens, [70, 300, 1], 8, 4, 64, 32, HF, False, q=wide[1::2, 8:16])
    # rows that are not 16-byte aligned
    odd = rand(T * 8 * 65 + 1, dtype=BF, seed=6)[1:].view(T, 8, 65)[..., :64]
    check_attention(q_lens, [70, 300, 1], 8, 4, 64, 32, BF, False, q=odd)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_lens", [[1, 4], [1, 300]], ids=["token", "chunk"])
@pytest.mark.parametrize("cache8", [False, True])
def test_scores_that_grow_large_and_scales(dtype, q_lens, cache8):
    check_attention(q_lens, [600, 700], 4, 1, 128, 16, dtype, cache8, qscale=30.0)
    check_attention(q_lens, [600, 700], 4, 1, 128, 16, dtype, cache8, scale=0.0)
    check_attention(q_lens, [600, 700], 4, 1, 128, 16, dtype, cache8, scale=-0.1)


def test_rising_scores_move_the_reference():
    # keys that grow along the sequence: every tile outdoes all tiles before it
    c = Cache([1500, 1500], 1, 128, 64, BF, False, seed=3)
    for b in range(2):
        x = torch.ones(1500, 1, 128) * (torch.arange(1500) / 150.0)[:, None, None]
        x = x.to(BF)
        pos = torch.arange(1500)
        c.cache[0][c.table[b].long().cpu()[pos // 64], :, pos % 64] = x.to(DEV)
        c.dense[0][b] = x.double()
    for q_lens in ([1, 2], [1, 130]):
        T = sum(q_lens)
        q = torch.ones(T, 4, 128, dtype=BF, device=DEV)
        q[:, 1] *= -1.0     # ... and every tile falls behind the first
        q[:, 2] *= 8.0
        o = abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu_of(q_lens), max(q_lens))
        want, _, A, S = attend64(q, c, q_lens, [1500, 1500], 128 ** -0.5)
        tol = attend_tolerance(want, A, S, BF, 128, 1500)
        assert ((o.cpu().double() - want).abs() <= tol).all()


def test_small_and_huge_queries_against_an_8_bit_cache():
    # rows of q far outside fp16's range, both ways, next to ordinary ones
    for q_lens in ([1, 2], [1, 60]):
        T = sum(q_lens)
        q = rand(T, 4, 128, dtype=BF, seed=4)
        q[:, 1] *= 1e-30
        q[:, 2] *= 2.0 ** 20
        q[:, 3, ::2] *= 1e-9
        check_attention(q_lens, [200, 300], 4, 1, 128, 16, BF, True, q=q, scale=1e-3)


@pytest.mark.parametrize("q_lens", [[1, 2], [1, 60]], ids=["token", "chunk"])
@pytest.mark.parametrize("cache8", [False, True])
def test_queries_of_zero_and_scales_down_to_nothing(q_lens, cache8):
    T = sum(q_lens)
    q = rand(T, 4, 128, dtype=BF, seed=4)
    q[:, 1] = 0
    q[:, 2] *= 2.0 ** -120
    q[:, 3] *= 2.0 ** -133       # subnormal
    for scale in (0.1, 1e-3, 1e-8, 2.0 ** -99, 1e-31, 1e-38, 1e-45, 1e-60):
        check_attention(q_lens, [200, 300], 4, 1, 128, 16, BF, cache8, q=q, scale=scale)
    with pytest.raises(RuntimeError, match="scale is not finite"):
        check_attention(q_lens, [200, 300], 4, 1, 128, 16, BF, cache8, q=q, scale=1e39)


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("q_lens,kv", [([1, 1], [40, 30000]), ([3, 4], [40, 30000]), ([30, 25], [40, 30000])], ids=["token", "draft", "chunk"])
def test_a_query_of_nan_stays_in_its_row(q_lens, kv, dtype, cache8):
    # in an item that one block finishes, and in one that is cut between many
    c = Cache(kv, 1, 64, 16, dtype, cache8)
    T = sum(q_lens)
    q = rand(T, 4, 64, dtype=dtype, seed=1)
    args = (*c.cache, c.table, c.kv_lens, cu_of(q_lens), max(q_lens))
    want, wlse = abi.paged_attention(q, *args, return_lse=True, **c.kw)
    gone = torch.zeros(T, 4, dtype=torch.bool, device=DEV)
    for row, head in ((0, 1), (T - 1, 2)):
        q[row, head, 5] = float("nan")
        gone[row, head] = True
    out, lse = abi.paged_attention(q, *args, return_lse=True, **c.kw)
    assert torch.isnan(out[gone]).all() and torch.isnan(lse[gone]).all()
    tol = 4 * torch.finfo(dtype).eps      # (a row's neighbours may be summed against another reference: half a step of P and of the result, twice)
    assert torch.allclose(out[~gone].float(), want[~gone].float(), rtol=tol, atol=tol) and torch.allclose(lse[~gone], wlse[~gone], atol=1e-4)


def test_max_q_bounds_what_is_computed():
    c = Cache([50, 60], 1, 64, 16, BF, False)
    q = rand(30, 2, 64, dtype=BF, seed=2)
    full = abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu_of([10, 20]), 20)
    for m in (0, 1, 4, 12):
        out = torch.full_like(q, 5.0)
        abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu_of([10, 20]), m, out=out)
        for b, (f, n) in enumerate([(0, 10), (10, 20)]):
            k = min(m, n)
            assert torch.allclose(out[f:f + k].float(), full[f:f + k].float(), atol=2e-2) and bool((out[f + k:f + n] == 5).all())


def test_lengths_that_point_outside_are_held_back():
    # kv_lens past the table's reach and cu_q past the tokens: what exists is attended, nothing else is touched
    c = Cache([64, 64], 1, 64, 16, BF, False)
    q = rand(8, 2, 64, dtype=BF, seed=2)
    for m in (4, 8):
        for kv, cu in (([2 ** 31 - 1, -5], [0, 4, 8]), ([64, 1 << 20], [0, 4, 1 << 30]), ([64, 64], [-7, 4, 8]), ([64, 64], [8, 4, 2])):
            out = torch.full_like(q, 5.0)
            abi.paged_attention(q, *c.cache, c.table, torch.tensor(kv, dtype=torch.int32, device=DEV),
                                torch.tensor(cu, dtype=torch.int32, device=DEV), m, out=out)
            torch.cuda.synchronize()
            assert not torch.isnan(out).any()


@pytest.mark.parametrize("lens", [TOKEN, CHUNK], ids=["token", "chunk"])
@pytest.mark.parametrize("cache8", [False, True])
def test_the_same_call_gives_the_same_bits_on_any_stream(lens, cache8):
    q_lens, kv_lens = lens
    c = Cache(kv_lens, 2, 128, 16, BF, cache8)
    q = rand(sum(q_lens), 8, 128, dtype=BF, seed=9)
    args = (q, *c.cache, c.table, c.kv_lens, cu_of(q_lens), max(q_lens))
    ref = abi.paged_attention(*args, **c.kw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(abi.paged_attention(*args, **c.kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


@pytest.mark.parametrize("lens", [([1, 1, 1], [100, 700, 300]), ([90, 1, 5], [100, 700, 300])], ids=["token", "chunk"])
@pytest.mark.parametrize("cache8", [False, True])
def test_captured_steps_follow_the_lengths_on_the_device(lens, cache8):
    q_lens, kv_lens = lens
    H, Hkv, D = 8, 2, 128
    c = Cache(kv_lens, Hkv, D, 16, BF, cache8)
    cu, T = cu_of(q_lens), sum(q_lens)
    q, k, v = rand(T, H, D, dtype=BF, seed=1), rand(T, Hkv, D, dtype=BF, seed=2), rand(T, Hkv, D, dtype=BF, seed=3)
    out = torch.empty_like(q)
    ws = torch.empty(max(16, abi.paged_attn_workspace_bytes(q, *c.cache, c.table, c.kv_lens, cu, max(q_lens), **c.kw)),
                     dtype=torch.uint8, device=DEV)

    def step(o, **kw):
        abi.paged_kv_write(k, v, *c.cache, c.table, c.kv_lens, cu, **c.kw)
        abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu, max(q_lens), out=o, **c.kw, **kw)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(out)
    torch.cuda.synchronize()
    graphs = []
    for kw in ({}, {"workspace": ws}):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            step(out, **kw)
        graphs.append(g)
    for lens_now in ([100, 700, 300], [95, 650, 299], [90, 699, 5]):
        c.kv_lens.copy_(torch.tensor(lens_now, dtype=torch.int32))
        want = torch.empty_like(q)
        step(want)
        for g in graphs:
            out.fill_(3.0)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_a_cache_past_2_31_elements():
    page, Hkv, D = 16, 8, 128
    pages = (1 << 31) // (page * Hkv * D) + 40
    for dtype, q_lens in ((BF, [1, 2]), (BF, [1, 40]), (E4M3, [2, 1]), (E4M3, [40, 1])):
        small = Cache([100, 200], Hkv, D, page, BF, dtype == E4M3, seed=8)
        big = [torch.empty((pages, Hkv, page, D), dtype=torch.uint8 if dtype == E4M3 else BF, device=DEV) for _ in range(2)]
        off = pages - small.pages
        for i in range(2):
            src = small.cache[i]
            big[i][off:] = src.view(torch.uint8) if dtype == E4M3 else src
        kw = {}
        if dtype == E4M3:
            big = [x.view(E4M3) for x in big]
            ex = [torch.zeros((pages, Hkv, page), dtype=torch.uint8, device=DEV) for _ in range(2)]
            for i in range(2):
                ex[i][off:] = small.exps[i]
            kw = {"k_exp": ex[0], "v_exp": ex[1]}
        table = torch.where(small.table >= 0, small.table + off, small.table)
        q = rand(sum(q_lens), 16, D, dtype=BF, seed=9)
        a = abi.paged_attention(q, *small.cache, small.table, small.kv_lens, cu_of(q_lens), max(q_lens), **small.kw)
        b = abi.paged_attention(q, *big, table, small.kv_lens, cu_of(q_lens), max(q_lens), **kw)
        assert torch.equal(a, b)
        cu_kv = cu_of([100, 200])
        ka, va = abi.paged_kv_read(*small.cache, small.table, cu_kv, 300, dtype=BF, **small.kw)
        kb, vb = abi.paged_kv_read(*big, table, cu_kv, 300, dtype=BF, **kw)
        assert torch.equal(ka, kb) and torch.equal(va, vb)
        for x in big:
            (x.view(torch.uint8) if dtype == E4M3 else x)[off:].zero_()
        if kw:
            kw["k_exp"][off:] = 0
            kw["v_exp"][off:] = 0
        abi.paged_kv_write(ka, va, *big, table, small.kv_lens, cu_kv, **kw)
        kc, vc = abi.paged_kv_read(*big, table, cu_kv, 300, dtype=BF, **kw)
        assert torch.equal(ka, kc) and torch.equal(va, vc)      # (8-bit rows that are read and written again stay as they are)
        del big, kw, table, a, b


def test_routes():
    def route(q_lens, Hq, Hkv, D, page, dtype, cache8=False, kv=300, **kw):
        check_attention(q_lens, [kv] * len(q_lens), Hq, Hkv, D, page, dtype, cache8, **kw)
        return abi.paged_attn_last_kernel()

    for cache8 in (False, True):
        for dtype in (BF, HF):
            assert route([1, 1], 8, 2, 128, 16, dtype, cache8) == "paged_decode"
            assert route([4, 1], 8, 2, 64, 256, dtype, cache8) == "paged_decode"
            assert route([9, 9], 8, 2, 128, 16, dtype, cache8) == "paged_tcgen05"
            assert route([1, 1], 34, 2, 64, 8, dtype, cache8) == "paged_tcgen05"
            assert route([60, 1, 1, 1], 8, 2, 128, 16, dtype, cache8) == "paged_tcgen05"
            assert route([60, 1, 1, 1], 8, 2, 128, 16, dtype, cache8, wide=True) == "paged_tcgen05+paged_decode"
            assert route([60, 30, 1, 1], 8, 2, 128, 16, dtype, cache8, wide=True) == "paged_tcgen05"
        assert route([3], 8, 2, 128, 16, FP, cache8) == "paged_simt"
        assert route([3], 8, 2, 96, 16, BF, cache8) == "paged_simt"
        assert route([3], 8, 2, 128, 24, BF, cache8) == "paged_simt"
        assert route([3], 130, 1, 64, 16, BF, cache8) == "paged_simt"
        assert route([30], 8, 2, 128, 16, BF, cache8, scale=0.0) == "paged_simt"


MIXED = ([1, 300, 2, 1, 0, 3, 1], [513, 900, 129, 1, 70, 260, 640])


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 128)])
def test_chunks_and_single_tokens_in_one_call(D, page, dtype, cache8):
    route = "paged_tcgen05+paged_decode"
    check_attention(*MIXED, 8, 2, D, page, dtype, cache8, route="paged_tcgen05")
    check_attention(*MIXED, 8, 2, D, page, dtype, cache8, route=route, wide=True)
    check_attention(*MIXED, 8, 2, D, page, dtype, cache8, route=route, wide=True, causal=False, first=2, behind=4, order="pdh")
    absent = [(0, 0), (1, 0), (1, 2), (3, 0), (6, 0), (6, 1)]
    check_attention(*MIXED, 8, 2, D, page, dtype, cache8, route=route, wide=True, absent=absent)


@pytest.mark.parametrize("cache8", [False, True])
def test_a_captured_mixed_call_follows_tokens_that_change_places(cache8):
    c = Cache([600, 400, 500, 300], 2, 128, 16, BF, cache8)
    widen(c)
    T = 70
    q = rand(T, 8, 128, dtype=BF, seed=1)
    cu = cu_of([67, 1, 1, 1])
    args = (q, *c.cache, c.table, c.kv_lens, cu, 67)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        abi.paged_attention(*args, out=out, **c.kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        abi.paged_attention(*args, out=out, **c.kw)
    assert abi.paged_attn_last_kernel() == "paged_tcgen05+paged_decode"
    for q_lens in ([67, 1, 1, 1], [1, 4, 64, 1], [0, 5, 60, 5], [17, 18, 17, 18], [4, 4, 4, 4], [0, 0, 0, 0]):
        cu.copy_(cu_of(q_lens))
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        want, _, A, S = attend64(q[:sum(q_lens)], c, q_lens, [600, 400, 500, 300], 128 ** -0.5)
        tol = attend_tolerance(want, A, S, BF, 128, 600)
        assert ((out[:sum(q_lens)].cpu().double() - want).abs() <= tol).all()
        assert bool((out[sum(q_lens):] == 5).all())


@pytest.mark.parametrize("q_lens", [[1], [16], [40]], ids=["token", "draft", "chunk"])
@pytest.mark.parametrize("cache8", [False, True])
def test_one_item_cut_between_all_multiprocessors(q_lens, cache8):
    # one kv head, more tiles than multiprocessors: every CTA leaves a part of the same rows
    check_attention(q_lens, [40000], 1, 1, 64, 128, BF, cache8)


def test_more_sequences_than_threads():
    for cache8 in (False, True):
        B = 700
        kv = [1 + (37 * b) % 300 for b in range(B)]
        check_attention([1] * B, kv, 2, 1, 64, 32, BF, cache8, route="paged_decode")
        check_attention([(b * 7) % 3 for b in range(B - 1)] + [50], kv, 2, 1, 64, 32, BF, cache8, route="paged_tcgen05+paged_decode", wide=True)
        check_attention([24 if b % 50 == 0 else 18 for b in range(B)], [n + 24 for n in kv], 2, 1, 64, 32, BF, cache8, route="paged_tcgen05", wide=True)


@pytest.mark.parametrize("q_lens", [[1, 1], [50, 40], [50, 1, 1]], ids=["token", "chunk", "mixed"])
def test_workspaces(q_lens):
    kv = [400 + 100 * i for i in range(len(q_lens))]
    c = Cache(kv, 2, 128, 16, BF, False)
    widen(c)
    T = sum(q_lens)
    q = rand(T, 8, 128, dtype=BF, seed=1)
    cu = cu_of(q_lens)
    args = lambda q: (q, *c.cache, c.table, c.kv_lens, cu, max(q_lens))      # noqa: E731
    n = abi.paged_attn_workspace_bytes(*args(q))
    want = abi.paged_attention(*args(q))
    ws = torch.zeros(n + 16, dtype=torch.uint8, device=DEV)
    with pytest.raises(RuntimeError, match="too small"):
        abi.paged_attention(*args(q), workspace=ws[:n - 1])
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        abi.paged_attention(*args(q), workspace=ws[8:8 + n])
    # exactly as much as is asked for, nothing written behind it; rows with a stride on D are copied first
    ws.fill_(7)
    strided = torch.empty(T, 8, 128, 2, dtype=BF, device=DEV)[..., 0].copy_(q)
    assert abi.paged_attn_workspace_bytes(*args(strided)) == n
    for x in (q, strided):
        assert torch.equal(abi.paged_attention(*args(x), workspace=ws[:n]), want)
    assert bool((ws[n:] == 7).all())
    # two captured graphs with one workspace, replayed in turn
    q2 = -q
    outs = [torch.empty_like(q) for _ in range(2)]
    side = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for x, o in zip((q, q2), outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            abi.paged_attention(*args(x), workspace=ws[:n], out=o)
        graphs.append(g)
    want2 = abi.paged_attention(*args(q2))
    for _ in range(3):
        for g, o, w in zip(graphs, outs, (want, want2)):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, w)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [90, 1, 5]], ids=["token", "chunk"])
def test_captured_calls_that_run_at_the_same_time(q_lens):
    # scratch from the pool: each graph has its own, on whatever stream it is replayed
    kv = [3000, 700, 2000]
    c = Cache(kv, 2, 128, 16, BF, False)
    cu = cu_of(q_lens)
    qs = [rand(sum(q_lens), 8, 128, dtype=BF, seed=i) for i in range(3)]
    want = [abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu, max(q_lens)) for q in qs]
    outs = [torch.empty_like(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    graphs = []
    for q, o, s in zip(qs, outs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for _ in range(4):
                abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu, max(q_lens), out=o)
        graphs.append(g)
    for turn in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(3):
            with torch.cuda.stream(streams[(i + turn) % 3]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_a_given_stream():
    q_lens, kv = [1, 40], [300, 500]
    c = Cache(kv, 2, 128, 16, BF, False)
    q = rand(41, 8, 128, dtype=BF, seed=1)
    args = (*c.cache, c.table, c.kv_lens, cu_of(q_lens), 40)
    want = abi.paged_attention(q, *args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    out = torch.empty_like(q)
    got = abi.paged_attention(q, *args, out=out, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want)
    strided = torch.empty(41, 8, 128, 2, dtype=BF, device=DEV)[..., 0].copy_(q)
    assert torch.equal(abi.paged_attention(strided, *args), want)
    with pytest.raises(RuntimeError, match="contiguous rows"):
        abi.paged_attention(strided, *args, stream=s.cuda_stream)
    with pytest.raises(RuntimeError, match="contiguous rows"):
        abi.paged_kv_write(strided[:, :2], strided[:, :2], *c.cache, c.table, c.kv_lens, cu_of(q_lens), stream=s.cuda_stream)


def test_rows_of_nothing_but_nan():
    for dtype in (BF, HF, FP):
        for T in (3, 4000):      # a warp per row, several heads a warp
            c = Cache([T], 6, 64, 16, dtype, True)
            k = rand(T, 6, 64, dtype=dtype, seed=1)
            k[1, 2], k[2] = float("nan"), float("inf")
            k[0, 1] = -0.0
            abi.paged_kv_write(k, -k, *c.cache, c.table, c.kv_lens, cu_of([T]), **c.kw)
            for got, x in zip(abi.paged_kv_read(*c.cache, c.table, cu_of([T]), T, dtype=FP, **c.kw), (k, -k)):
                q, e = quantise64(x)
                want = (q * torch.pow(2.0, e).unsqueeze(-1)).float()
                assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
                assert torch.equal(got.cpu().nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("q_lens", [[2], [40]], ids=["token", "chunk"])
def test_positions_past_2_30(q_lens):
    # one page of zeros again and again, then one whose keys outweigh them all: it has to be found at its place
    page, n, D = 32768, q_lens[0], 64
    k = torch.zeros(2, 1, page, D, dtype=torch.uint8, device=DEV).view(E4M3)
    v = torch.zeros_like(k)
    exps = [torch.full((2, 1, page), 127, dtype=torch.uint8, device=DEV) for _ in range(2)]
    last = 100
    k[1, 0, :last] = torch.full((D,), 8.0, device=DEV).to(E4M3)
    v[1, 0, :last] = torch.arange(1, last + 1, device=DEV).float()[:, None].expand(last, D).to(E4M3)
    whole = (1 << 30) // page
    table = torch.zeros(1, whole + 1, dtype=torch.int32, device=DEV)
    table[0, whole] = 1
    kv = torch.tensor([whole * page + last], dtype=torch.int32, device=DEV)
    q = torch.ones(n, 1, D, dtype=BF, device=DEV)
    out, lse = abi.paged_attention(q, k, v, table, kv, cu_of([n]), n, scale=1 / 8.0, k_exp=exps[0], v_exp=exps[1], return_lse=True)
    seen = last - n + 1 + torch.arange(n)
    vals = v[1, 0, :last, 0].cpu().double()
    want = torch.stack([vals[:m].mean() for m in seen])          # (the zeros weigh 2^30 e^-64 of a key)
    u = torch.finfo(BF).eps / 2
    assert ((out[:, 0].cpu().double() - want[:, None]).abs() <= 2.0 * u * want[:, None]).all()
    assert ((lse[:, 0].cpu().double() - (64 + seen.double().log())).abs() <= 1e-4).all()


# ---------------------------------------------------------------- writing and reading

def rows_for(T, H, D, dtype, seed):
    x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed))
    mag = torch.tensor([1.0, 1e-3, 300.0, 1e-6, 448.0, 20000.0, 0.0, 2.0 ** -17])
    x = x * mag[torch.arange(T) % len(mag)][:, None, None]
    x[::5, :, :1] = 448.0 * 2.0 ** -3       # a largest value on the border between two exponents
    x[::5, :, 1:] = x[::5, :, 1:].clamp(-40, 40)
    return x.to(dtype)


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D,page,Hkv", [(128, 16, 8), (64, 32, 2), (1, 1, 1), (40, 3, 3), (100, 16, 2), (256, 64, 1), (200, 16, 1), (133, 7, 2)])
def test_rows_written_and_read_back(D, page, Hkv, dtype, cache8):
    q_lens, kv_lens = [1, 0, 30, 7, 3], [5, 4, 30, 100, 2]     # the last: one row stands before position 0
    first, behind = 2, 3
    T = first + sum(q_lens) + behind
    for order in ("phd", "pdh"):
        c = Cache(kv_lens, Hkv, D, page, dtype, cache8, order=order)
        before = [x.view(torch.uint8).cpu().clone() if cache8 else x.cpu().clone() for x in c.cache]
        k, v = rows_for(T, Hkv, D, dtype, 1), rows_for(T, Hkv, D, dtype, 2)
        if dtype != FP and D > 2:
            k[4, :, 1], v[5, :, 2], v[6, :, 0] = float("nan"), float("inf"), float("-inf")
        abi.paged_kv_write(k.to(DEV), v.to(DEV), *c.cache, c.table, c.kv_lens, cu_of(q_lens, first), **c.kw)
        torch.cuda.synchronize()
        table = c.table.cpu().long()
        for i, x in enumerate((k, v)):
            raw = c.cache[i].view(torch.uint8).cpu() if cache8 else c.cache[i].cpu()
            want = before[i].clone()
            exps = c.exps[i].cpu() if cache8 else None
            t = first
            for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
                for j in range(n):
                    pos = L - n + j
                    if pos >= 0:
                        at = (int(table[b, pos // page]), slice(None), pos % page)
                        row = x[t + j]
                        if cache8:
                            qv, e = quantise64(torch.where(torch.isinf(row), torch.sign(row) * 57344.0, row) if torch.isinf(row).any() else row)
                            if torch.isinf(row).any():      # an infinite row takes the largest exponent
                                e = torch.where(torch.isinf(row).any(-1), torch.full_like(e, 7.0), e)
                            want[at] = qv.to(E4M3).view(torch.uint8) if not torch.isnan(qv).any() else raw[at]
                            if torch.isnan(qv).any():
                                got = raw[at].view(E4M3).double()
                                assert torch.equal(torch.isnan(got), torch.isnan(qv))
                                fin = ~torch.isnan(qv)
                                assert torch.equal(got[fin], qv[fin])
                            assert torch.equal(exps[at].double(), e + 127)
                        else:
                            want[at] = row
                t += n
            # every other place keeps what it held
            if cache8:
                assert torch.equal(raw & 0x7f, want & 0x7f) and torch.equal((raw[(raw & 0x7f) != 0]), want[(raw & 0x7f) != 0])
            else:
                assert torch.equal(raw.nan_to_num(nan=1e4), want.nan_to_num(nan=1e4))
        # read back: dense rows, rows of no sequence as they were
        cu_kv, total = cu_of(kv_lens, first), first + sum(kv_lens) + behind
        for to in ([dtype] if not cache8 else [BF, HF, FP]):
            ro = [torch.full((total, Hkv, D), 9.0, dtype=to, device=DEV) for _ in range(2)]
            abi.paged_kv_read(*c.cache, c.table, cu_kv, total, out=ro, **c.kw)
            torch.cuda.synchronize()
            for i in range(2):
                dense = values(c.cache[i], c.exps[i])
                got = ro[i].cpu().double()
                assert bool((got[:first] == 9).all()) and bool((got[first + sum(kv_lens):] == 9).all())
                t = first
                for b, L in enumerate(kv_lens):
                    for pos in range(L):
                        w = dense[int(table[b, pos // page]), :, pos % page]
                        assert torch.equal(torch.isnan(got[t + pos]), torch.isnan(w))
                        assert torch.equal(got[t + pos].nan_to_num(), w.nan_to_num())
                    t += L


def test_absent_pages_take_nothing_and_read_as_zeros():
    for cache8 in (False, True):
        c = Cache([40, 40], 2, 64, 16, BF, cache8)
        c.table[0, 1], c.table[1, 0], c.table[1, 2] = -1, c.pages, 2 ** 31 - 1
        before = [x.view(torch.uint8).clone() for x in c.cache]
        k = rand(80, 2, 64, dtype=BF, seed=1)
        abi.paged_kv_write(k, k, *c.cache, c.table, c.kv_lens, cu_of([40, 40]), **c.kw)
        a, b = abi.paged_kv_read(*c.cache, c.table, cu_of([40, 40]), 80, dtype=BF, **c.kw)
        torch.cuda.synchronize()
        for x in (a, b):
            assert bool((x[16:32] == 0).all()) and bool((x[40:56] == 0).all()) and bool((x[72:80] == 0).all())
            assert not torch.isnan(x).any()
        used = {int(c.table[0, 0]), int(c.table[0, 2]), int(c.table[1, 1])}
        for i in range(2):
            now = c.cache[i].view(torch.uint8)
            for p in range(c.pages):
                if p not in used:
                    assert torch.equal(now[p], before[i][p])
        # lengths beyond the table's reach: dropped
        abi.paged_kv_write(k[:4], k[:4], *c.cache, c.table, torch.tensor([2 ** 31 - 1, -3], dtype=torch.int32, device=DEV),
                           cu_of([2, 2]), **c.kw)
        torch.cuda.synchronize()


def test_many_sequences_find_their_rows():
    # more sequences than one probe of the search covers, some of them empty
    for B in (31, 33, 1000, 1100):
        q_lens = [(7 * b) % 3 for b in range(B)]
        kv_lens = [n + (b % 5) for b, n in enumerate(q_lens)]
        c = Cache(kv_lens, 1, 64, 16, BF, False)
        T = sum(q_lens)
        k = rand(T, 1, 64, dtype=BF, seed=3)
        abi.paged_kv_write(k, -k, *c.cache, c.table, c.kv_lens, cu_of(q_lens), **c.kw)
        a, b_ = abi.paged_kv_read(*c.cache, c.table, cu_of(kv_lens), sum(kv_lens))
        t = at = 0
        idx = []
        for n, L in zip(q_lens, kv_lens):
            idx += list(range(at + L - n, at + L))
            at += L
        assert torch.equal(a[idx], k) and torch.equal(b_[idx], -k)
        check_attention([min(1, n) for n in q_lens], kv_lens, 2, 1, 64, 16, BF, False)


# ---------------------------------------------------------------- on the paras device

def test_a_layer_step_on_the_device():
    """Residual norm, projections, cache write, attention, read back: as a decoder layer runs them, on `paras` tensors,
    against 64 bits with each operator's own inputs."""
    from torch_paras import nn
    import torch.nn.functional as F
    H, Hkv, D, page, hid = 8, 2, 64, 16, 256
    g = torch.Generator().manual_seed(0)
    q_lens, kv_before = [1, 20, 1], [33, 0, 90]
    kv_lens = [a + b for a, b in zip(q_lens, kv_before)]
    T = sum(q_lens)
    for cache8 in (False, True):
        c = Cache(kv_lens, Hkv, D, page, BF, cache8, dev="cpu")
        dev = "paras:1"
        x, res = (torch.randn(T, hid, generator=g).to(BF) for _ in range(2))
        w = (1 + 0.1 * torch.randn(hid, generator=g)).to(BF)
        wq, wk, wv = (torch.randn(n * D, hid, generator=g).mul(hid ** -0.5).to(BF) for n in (H, Hkv, Hkv))
        caches = [t.to(dev) for t in c.cache]
        exps = {} if not cache8 else {"k_exp": c.exps[0].to(dev), "v_exp": c.exps[1].to(dev)}
        table, lens, cu = c.table.to(dev), c.kv_lens.to(dev), cu_of(q_lens, dev="cpu").to(dev)
        y, h = nn.add_rms_norm(x.to(dev), res.to(dev), w.to(dev))
        q, k, v = (F.linear(y, m.to(dev)).view(T, -1, D) for m in (wq, wk, wv))
        nn.paged_kv_write(k, v, *caches, table, lens, cu, **exps)
        out, lse = nn.paged_attention(q, *caches, table, lens, cu, max(q_lens), return_lse=True, **exps)
        q8, scales, h2 = nn.add_rms_norm_quant(F.linear(out.view(T, -1), torch.randn(hid, H * D, generator=g).to(BF).to(dev)), h, w.to(dev), group=64)
        kr, vr = nn.paged_kv_read(*caches, table, cu_of(kv_lens, dev="cpu").to(dev), sum(kv_lens), dtype=BF, **exps)
        assert q8.shape == (T, hid) and scales.shape == (T, 4) and h2.shape == h.shape
        assert torch.equal(h.cpu(), (x.float() + res.float()).to(BF))
        # what the cache holds now
        at = 0
        for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
            rows = slice(sum(q_lens[:b]), sum(q_lens[:b]) + n)
            for i, (new, read) in enumerate(((k, kr), (v, vr))):
                r = read.cpu()[at:at + L].double()
                qv, e = quantise64(new.cpu()[rows])
                want = qv * torch.pow(2.0, e).unsqueeze(-1) if cache8 else new.cpu()[rows].double()
                assert torch.equal(r[L - n:], want)
                assert torch.equal(r[:L - n], c.dense[i][b][:L - n])
                c.dense[i][b] = r
            at += L
        want, wlse, A, S = attend64(q.cpu(), c, q_lens, kv_lens, D ** -0.5)
        assert ((out.cpu().double() - want).abs() <= attend_tolerance(want, A, S, BF, D, max(kv_lens))).all()
        assert ((lse.cpu().double() - wlse).abs() <= lse_tolerance(wlse, S, D, max(kv_lens))).all()


def test_refusals_on_the_device():
    c = Cache([20], 2, 64, 16, BF, False)
    q = rand(1, 4, 64, dtype=BF, seed=1)
    cu = cu_of([1])
    with pytest.raises(RuntimeError, match="multiple of key/value heads"):
        abi.paged_attention(q[:, :3], *c.cache, c.table, c.kv_lens, cu, 1)
    with pytest.raises(RuntimeError, match="k_exp"):
        abi.paged_attention(q, *[x.to(E4M3) for x in c.cache], c.table, c.kv_lens, cu, 1)
    with pytest.raises(RuntimeError, match="8-bit cache"):
        abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu, 1, k_exp=torch.zeros(1), v_exp=torch.zeros(1))
    with pytest.raises(RuntimeError, match="rows' type"):
        abi.paged_attention(q.half(), *c.cache, c.table, c.kv_lens, cu, 1)
    with pytest.raises(RuntimeError, match="int32"):
        abi.paged_attention(q, *c.cache, c.table, c.kv_lens.long(), cu, 1)
    with pytest.raises(RuntimeError, match="2 entries"):
        abi.paged_attention(q, *c.cache, c.table, c.kv_lens, torch.zeros(3, dtype=torch.int32, device=DEV), 1)
    with pytest.raises(RuntimeError, match="scale is not finite"):
        abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu, 1, scale=float("nan"))
    with pytest.raises(RuntimeError, match="head dim"):
        abi.paged_attention(rand(1, 4, 257, dtype=BF, seed=1), *[torch.zeros(2, 2, 16, 257, dtype=BF, device=DEV)] * 2, c.table,
                            c.kv_lens, cu, 1)
    with pytest.raises(RuntimeError, match="different devices"):
        abi.paged_kv_write(q[:, :2], q[:, :2], *c.cache, c.table.cpu(), c.kv_lens, cu)
    # nothing to do
    abi.paged_attention(q[:0], *c.cache, c.table, c.kv_lens, cu_of([0]), 0)
    abi.paged_attention(q, *c.cache, c.table[:0], c.kv_lens[:0], cu[:1], 1)
    abi.paged_kv_write(q[:0, :2], q[:0, :2], *c.cache, c.table, c.kv_lens, cu_of([0]))
    # a cache without pages: nothing is attended
    none = [torch.empty(0, 2, 16, 64, dtype=BF, device=DEV)] * 2
    assert bool((abi.paged_attention(q, *none, c.table, c.kv_lens, cu, 1) == 0).all())
    assert bool((abi.paged_attention(q, *c.cache, c.table[:, :0], c.kv_lens, cu, 1) == 0).all())
