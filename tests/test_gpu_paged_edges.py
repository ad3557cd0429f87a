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
