"""Refusals of the paged cache and of the residual norm that need no GPU, and the definition the GPU tests compare with."""
import ctypes

import pytest
import torch

import torch_paras
from torch_paras import abi

from paged_cases import E4M3, quantise64


def kv_args():
    a = abi.PagedKvArgs()
    c = a.cache
    buf = (ctypes.c_char * 64)()
    a._keep = buf
    p = ctypes.addressof(buf)
    c.k = c.v = c.k_exp = c.v_exp = c.page_table = a.k = a.v = a.kv_lens = a.cu = p
    c.cache_dtype, c.pages, c.page, c.Hkv, c.D, c.B, c.max_pages = abi.BF16, 4, 16, 2, 64, 1, 4
    a.T, a.dtype = 1, abi.BF16
    return a


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=7), -2, "unsupported dtype"), (dict(dtype=abi.E4M3), -2, "unsupported dtype"),
    (dict(dtype=abi.F16), -1, "rows' type"), (dict(D=0), -2, "head dim"), (dict(D=257), -2, "head dim"),
    (dict(page=0), -1, "a page holds"), (dict(page=65537), -1, "a page holds"), (dict(pages=-1), -1, "negative size"),
    (dict(B=-1), -1, "negative size"), (dict(Hkv=0), -1, "no kv heads"), (dict(max_pages=1 << 30), -1, "exceeds 2"),
    (dict(page_table=None), -1, "null page table"), (dict(k=None), -1, "null cache"), (dict(T=-1), -1, "negative"),
    (dict(cache_dtype=abi.E4M3, k_exp=None), -1, "exponent bytes"),
])
def test_bad_arguments_are_refused_before_the_gpu_is_used(change, status, text):
    for entry in ("write", "read"):
        a = kv_args()
        for name, value in change.items():
            setattr(a if name in ("T", "dtype") else a.cache, name, value)
        f = getattr(abi.lib(), "paras_b200_paged_kv_" + entry)
        assert f(ctypes.byref(a)) == status
        assert text in abi.lib().paras_b200_last_error().decode()
    assert abi.lib().paras_b200_paged_kv_write(None) == -1 and abi.lib().paras_b200_paged_kv_read(None) == -1


def test_attention_refusals():
    lib = abi.lib()
    a = abi.PagedAttnArgs()
    k = kv_args()
    a.cache = k.cache
    a.T, a.Hq, a.max_q, a.dtype, a.scale = 1, 4, 1, abi.BF16, 0.125
    n = ctypes.c_size_t(0)
    for name, value, text in (("Hq", 3, "multiple of key/value heads"), ("Hq", 0, "multiple of"), ("max_q", -1, "negative"),
                              ("scale", float("inf"), "scale"), ("T", -1, "negative"), ("dtype", 9, "unsupported")):
        old = getattr(a, name)
        setattr(a, name, value)
        assert lib.paras_b200_paged_attn(ctypes.byref(a)) < 0
        assert text in lib.paras_b200_last_error().decode()
        assert lib.paras_b200_paged_attn_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) < 0
        setattr(a, name, old)
    assert lib.paras_b200_paged_attn(None) == -1


def test_norm_refusals():
    lib = abi.lib()
    buf = (ctypes.c_char * 64)()
    assert lib.paras_b200_add_rmsnorm_fwd(0, buf, buf, buf, buf, buf, None, -1, 8, 1e-6, abi.BF16, None) == -1
    assert lib.paras_b200_add_rmsnorm_fwd(0, buf, buf, buf, buf, buf, None, 1, 8, 1e-6, abi.E4M3, None) == -2
    assert lib.paras_b200_add_rmsnorm_quant_fwd(0, buf, buf, buf, buf, buf, buf, 1, 8, 1e-6, 48, abi.BF16, None) == -1
    assert b"group" in lib.paras_b200_last_error()
    assert lib.paras_b200_add_rmsnorm_bwd(0, buf, None, buf, buf, buf, buf, buf, 1, 1 << 40, abi.BF16, None) == -2


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU error path")
def test_no_gpu_is_said_so():
    a = kv_args()
    assert abi.lib().paras_b200_paged_kv_write(ctypes.byref(a)) == -4
    buf = (ctypes.c_char * 64)()
    assert abi.lib().paras_b200_add_rmsnorm_fwd(0, buf, buf, buf, buf, buf, None, 1, 8, 1e-6, abi.BF16, None) == -4
    with pytest.raises(RuntimeError):
        torch_paras.nn.add_rms_norm(torch.zeros(2, 8, device="paras:0"), torch.zeros(2, 8, device="paras:0"), torch.zeros(8, device="paras:0"))


def test_struct_sizes_match_the_header():
    assert ctypes.sizeof(abi.PagedCache) == 4 * 8 + 4 * 24 + 16 + 8 * 4
    assert ctypes.sizeof(abi.PagedKvArgs) == ctypes.sizeof(abi.PagedCache) + 16 + 32 + 16 + 16 + 8
    assert ctypes.sizeof(abi.PagedAttnArgs) == ctypes.sizeof(abi.PagedCache) + 24 + 32 + 16 + 24 + 8 + 16 + 8


def test_the_definition_rounds_to_values_that_e4m3_holds():
    x = torch.randn(200, 64, dtype=torch.float64) * torch.logspace(-8, 5, 200, dtype=torch.float64)[:, None]
    q, e = quantise64(x)
    assert torch.equal(q.to(E4M3).double(), q)                              # every value is an e4m3 value
    assert torch.equal((q * torch.pow(2.0, e)[:, None]).to(torch.float16).double(), q * torch.pow(2.0, e)[:, None])
    ordinary = (e > -15) & (e < 7)
    assert (q.abs().amax(-1)[ordinary] > 223).all() and (q.abs() <= 448).all()
    # torch's own rounding to e4m3 agrees
    assert torch.equal((x / torch.pow(2.0, e)[:, None]).clamp(-448, 448).float().to(E4M3).double()[ordinary], q[ordinary])
