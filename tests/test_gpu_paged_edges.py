"""Edges of the paged cache's calls on the GPU."""
import pytest
import torch

import torch_paras  # noqa: F401
from torch_paras import abi

from paged_cases import Cache, attend64, attend_tolerance, cu_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def rand(*shape, dtype, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [4, 1, 3, 2], [60, 1, 40, 2]], ids=["token", "draft", "chunk"])
def test_exponent_bytes_wherever_they_lie(q_lens, dtype, D):
    # word by word where they are aligned and there, byte by byte else: the same bits either way, over many turns of a block's
    # ring of tiles, beside pages that are absent (which take the second way alone)
    kv = [30000, 700, 9000, 4100]
    c = Cache(kv, 2, D, 16, dtype, True, seed=2)
    absent = [(0, p) for p in range(1, 1800, 3)] + [(2, 0), (2, 5), (3, 200)]
    for b, p in absent:
        c.table[b, p] = -1
    q = rand(sum(q_lens), 8, D, dtype=dtype, seed=3)
    args = (q, *c.cache, c.table, c.kv_lens, cu_of(q_lens), max(q_lens))
    ref, lse = abi.paged_attention(*args, return_lse=True, **c.kw)
    want, _, A, S = attend64(q, c, q_lens, kv, D ** -0.5, absent=absent)
    assert ((ref.cpu().double() - want).abs() <= attend_tolerance(want, A, S, dtype, D, max(kv))).all()
    shape = c.exps[0].shape
    for turn in range(5):
        ways = []
        for e in c.exps:
            spaced = torch.full((*shape, 2), 255, dtype=torch.uint8, device=DEV)
            spaced[..., 0] = e
            shifted = torch.full((e.numel() + 1,), 255, dtype=torch.uint8, device=DEV)[1:].view(shape)
            shifted.copy_(e)
            across = e.transpose(1, 2).contiguous().transpose(1, 2)
            ways.append((spaced[..., 0], shifted, across))
        for k_exp, v_exp in zip(*ways):
            out, l2 = abi.paged_attention(*args, return_lse=True, k_exp=k_exp, v_exp=v_exp)
            assert torch.equal(out, ref) and torch.equal(l2, lse)


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
def test_bits_do_not_depend_on_what_ran_before(dtype, D, cache8):
    # a call for single tokens after one whose query rows fill whole tiles with other values: what its own tiles of query rows
    # do not cover in shared memory must not show, and neither must a neighbour's row
    kv = [30000, 700, 9000, 4100]
    c = Cache(kv, 2, D, 16, dtype, cache8, seed=2)
    q = rand(4, 8, D, dtype=dtype, seed=3)
    args = (*c.cache, c.table, c.kv_lens)
    before = [torch.zeros(16, 8, D, dtype=dtype, device=DEV)] + [rand(16, 8, D, dtype=dtype, seed=5 + i, scale=s)
                                                                 for i, s in enumerate((1.0, 30.0, 300.0))]
    ref = None
    for turn in range(3):
        for other in before:
            abi.paged_attention(other, *args, cu_of([4] * 4), 4, **c.kw)
            out, lse = abi.paged_attention(q, *args, cu_of([1] * 4), 1, return_lse=True, **c.kw)
            assert abi.paged_attn_last_kernel() == "paged_decode"
            ref = ref or (out, lse)
            assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1])
    # one head's query changes: the others keep their bits
    for scale in (0.0, 30.0):
        q2 = q.clone()
        q2[:, 1] *= scale
        q2[:, 6] = float("nan")
        out, lse = abi.paged_attention(q2, *args, cu_of([1] * 4), 1, return_lse=True, **c.kw)
        for h in (0, 2, 3, 4, 5, 7):
            assert torch.equal(out[:, h], ref[0][:, h]) and torch.equal(lse[:, h], ref[1][:, h])


@pytest.mark.parametrize("cache8", [False, True])
def test_an_item_that_lasts_longer_than_any_wait(cache8):
    # a sequence of 2^26 positions for every multiprocessor (all of one page of zeros, then one whose keys outweigh them): a
    # block's item takes more than half a second, for all of which its idle warps wait for the next one
    page, D, H, last = 32768, 64, 128, 100
    B = torch.cuda.get_device_properties(0).multi_processor_count
    whole = (1 << 26) // page
    k, v = torch.zeros(2, 1, page, D, device=DEV), torch.zeros(2, 1, page, D, device=DEV)
    k[1, 0, :last] = 8.0
    v[1, 0, :last] = torch.arange(1, last + 1, device=DEV).float()[:, None]
    kind = torch.float8_e4m3fn if cache8 else BF
    k, v = k.to(kind), v.to(kind)
    exps = {n: torch.full((2, 1, page), 127, dtype=torch.uint8, device=DEV) for n in ("k_exp", "v_exp")} if cache8 else {}
    table = torch.zeros(1, whole + 1, dtype=torch.int32, device=DEV)
    table[0, whole] = 1
    kv = torch.full((B,), whole * page + last, dtype=torch.int32, device=DEV)
    q = torch.ones(B, H, D, dtype=BF, device=DEV)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    out, lse = abi.paged_attention(q, k, v, table.expand(B, -1), kv, cu_of([1] * B), 1, scale=1 / 8.0, return_lse=True, **exps)
    end.record()
    torch.cuda.synchronize()
    assert abi.paged_attn_last_kernel() == "paged_tcgen05"
    abi.paged_attention(q, k, v, table.expand(B, -1), torch.ones_like(kv), cu_of([1] * B), 1, scale=1 / 8.0, **exps)      # (would report a wait that ran out)
    want = v[1, 0, :last, 0].cpu().double().mean()          # (the zeros weigh 2^26 e^-64 of a key)
    u = torch.finfo(BF).eps / 2
    assert ((out.cpu().double() - want).abs() <= 2 * u * want).all()
    assert ((lse.cpu().double() - (64 + torch.tensor(float(last)).double().log())).abs() <= 1e-4).all()
    assert start.elapsed_time(end) > 400      # (twice the limit of a wait: the case is what it claims to be)


def test_a_block_that_gives_up_leaves_its_copies_time_to_land():
    # the exit of the chunk and streaming kernels and of the self-test kernel, whose wait runs out after 0.2 ms
    import time
    abi.selftest_bounded_wait(0, 200)
    t0 = time.perf_counter()
    status, word = abi.selftest_bounded_wait(0, 200)
    assert status == -6 and word & (1 << 27)
    assert time.perf_counter() - t0 >= 1.2e-3
    check = torch.ones(4, device=DEV).sum()
    assert check.item() == 4


def test_outputs_that_are_given_to_the_reader():
    c = Cache([40, 20], 2, 64, 16, BF, True)
    k, v = (torch.full((60, 2, 64), 5.0, dtype=HF, device=DEV) for _ in range(2))
    args = (*c.cache, c.table, cu_of([40, 20]), 60)
    with pytest.raises(RuntimeError, match="not the dtype asked for"):
        abi.paged_kv_read(*args, dtype=BF, out=(k, v), **c.kw)
    for out in ((k, None), (None, v)):
        with pytest.raises(RuntimeError, match="both or not at all"):
            abi.paged_kv_read(*args, out=out, **c.kw)
    assert bool((k == 5).all()) and bool((v == 5).all())
    want = abi.paged_kv_read(*args, dtype=HF, **c.kw)
    for dtype in (None, HF):
        got = abi.paged_kv_read(*args, dtype=dtype, out=(k, v), **c.kw)
        assert got[0].data_ptr() == k.data_ptr() and torch.equal(k, want[0]) and torch.equal(v, want[1])
        k.zero_()


def test_the_last_kernel_is_that_of_the_library_that_ran(tmp_path):
    # with the ctypes bindings pointed at another build, the paged calls still run, and report on, the one `_C` is linked to
    import os
    import shutil
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    package = os.path.dirname(os.path.dirname(abi.__file__))
    other = shutil.copy(os.path.join(package, "torch_paras", "libparas_b200.so"), tmp_path / "libother.so")
    code = ("import torch, torch_paras\nfrom torch_paras import abi\nfrom paged_cases import Cache, cu_of\n"
            "c = Cache([300], 2, 64, 16, torch.bfloat16, False)\nq = torch.ones(1, 4, 64, dtype=torch.bfloat16, device='cuda:0')\n"
            "abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu_of([1]), 1)\ntorch.cuda.synchronize()\n"
            "print(abi._LIB_PATH, abi.paged_attn_last_kernel())\n")
    env = dict(os.environ, PARAS_B200_LIB=str(other), PYTHONPATH=os.pathsep.join([package, here]))
    out = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert out.stdout.split() == [str(other), "paged_decode"]


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("dtype,q_lens,max_q", [(BF, [4, 4], 4), (BF, [40, 60], 60), (torch.float32, [4, 7], 7)], ids=["token", "chunk", "simt"])
def test_a_sequence_that_goes_on_past_the_rows_there_are(dtype, q_lens, max_q, cache8):
    # the rows of a longer batch that are there stand where they stood
    kv = [n + 1 for n in q_lens]
    c = Cache(kv, 2, 64, 16, dtype, cache8)
    T = sum(q_lens)
    q = rand(T, 4, 64, dtype=dtype, seed=1)
    args = (*c.cache, c.table, c.kv_lens, cu_of(q_lens), max_q)
    full = abi.paged_attention(q, *args, **c.kw)
    for there in (T - 1, T - 3):
        out = abi.paged_attention(q[:there], *args, **c.kw)
        tol = 2 * torch.finfo(dtype).eps      # (shared out between other blocks: half a step of P and of the result, twice)
        assert torch.allclose(out.float(), full[:there].float(), rtol=tol, atol=tol)


@pytest.mark.parametrize("q_lens", [[1, 2], [1, 60]], ids=["token", "chunk"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_what_the_heaviest_key_adds_nothing_to(dtype, q_lens):
    # scores so far apart that a row is nearly one key's, whose value is zero in every fourth column: what is left there are weights
    # down to nothing, which fp16 holds to 2^-25 of the reference, each times its value
    kv = [300, 200]
    c = Cache(kv, 1, 128, 16, dtype, True, seed=4)
    for b in range(2):
        c.dense[1][b][:, :, ::4] *= (torch.arange(kv[b]) % 2)[:, None, None]
        pos = torch.arange(kv[b])
        where, off = c.table[b].long().cpu()[pos // 16], pos % 16
        raw = c.cache[1].view(torch.uint8)
        row = raw[where, :, off]
        row[::2, :, ::4] = 0
        raw[where, :, off] = row
    q = rand(sum(q_lens), 4, 128, dtype=dtype, seed=5, scale=20.0)
    out = abi.paged_attention(q, *c.cache, c.table, c.kv_lens, cu_of(q_lens), max(q_lens), **c.kw)
    want, _, A, S = attend64(q, c, q_lens, kv, 128 ** -0.5)
    small = torch.cat([c.dense[1][b].abs().sum(0).expand(n, 4, 128) for b, n in enumerate(q_lens)])
    tol = attend_tolerance(want, A, S, dtype, 128, max(kv)) + 2.0 ** -25 * small
    assert ((out.cpu().double() - want).abs() <= tol).all()
