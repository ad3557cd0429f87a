"""Limits of the paged cache's calls that need no GPU."""
import ctypes

import pytest

import torch_paras  # noqa: F401
from torch_paras import abi


def cache_args(args):
    buf = (ctypes.c_char * 64)()
    args._keep = buf
    p = ctypes.addressof(buf)
    c = args.cache
    c.k = c.v = c.page_table = args.kv_lens = args.cu = p
    c.cache_dtype, c.pages, c.page, c.Hkv, c.D, c.B, c.max_pages = abi.BF16, 4, 16, 2, 64, 1, 4
    args.T, args.dtype = 1, abi.BF16
    return args


def calls():
    lib = abi.lib()
    kv = cache_args(abi.PagedKvArgs())
    kv.k = kv.v = kv.cache.k
    at = cache_args(abi.PagedAttnArgs())
    at.q = at.out = at.cache.k
    at.Hq, at.max_q, at.scale = 4, 1, 0.125
    n = ctypes.c_size_t(0)
    yield kv, lambda: lib.paras_b200_paged_kv_write(ctypes.byref(kv))
    yield kv, lambda: lib.paras_b200_paged_kv_read(ctypes.byref(kv))
    yield at, lambda: lib.paras_b200_paged_attn(ctypes.byref(at))
    yield at, lambda: lib.paras_b200_paged_attn_workspace_bytes(ctypes.byref(at), ctypes.byref(n))


@pytest.mark.parametrize("page,max_pages", [(1, 2 ** 31 - 1), (1, 2 ** 31 - 255), (49981, 42966), (64, 2 ** 25 - 1), (128, 2 ** 24 - 1),
                                            (8, 2 ** 28 - 31), (65536, 2 ** 15)])
def test_a_table_that_reaches_past_the_positions_is_refused(page, max_pages):
    # positions are counted in 32 bits, in steps and tiles of up to 128: the last 255 below 2^31 have no room for the next step
    for args, call in calls():
        args.cache.page, args.cache.max_pages = page, max_pages
        assert call() == -1
        assert "max_pages * page exceeds 2^31 - 256" in abi.lib().paras_b200_last_error().decode()


@pytest.mark.parametrize("page,max_pages", [(1, 2 ** 31 - 256), (64, 2 ** 25 - 4), (128, 2 ** 24 - 2), (65536, 2 ** 15 - 1)])
def test_the_widest_table_is_taken(page, max_pages):
    # (the next check that fails is another one)
    for args, call in calls():
        args.cache.page, args.cache.max_pages, args.cache.k = page, max_pages, None
        assert call() == -1
        assert "null cache" in abi.lib().paras_b200_last_error().decode()


@pytest.mark.parametrize("dtype", ["bfloat16", 15, float, object()])
def test_a_dtype_that_is_none_is_refused(dtype):
    import torch
    pool, table = torch.zeros(2, 1, 16, 64), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(TypeError, match="torch.dtype"):
        abi.paged_kv_read(pool, pool, table, torch.zeros(2, dtype=torch.int32), 4, dtype=dtype)
