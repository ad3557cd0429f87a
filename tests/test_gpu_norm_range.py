"""The residual norm over the whole range of its types: rows whose squares do not fit fp32, beside ordinary ones, at widths of
every kernel.  Against 64 bits, with tolerances that count the roundings as for ordinary rows."""
import pytest
import torch

import torch_paras  # noqa: F401
from torch_paras import abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
F32 = 2.0 ** -24     # half a step of fp32
WIDTHS = [1, 7, 64, 200, 577, 1000, 2048, 4096, 5001, 8192, 16384, 32768, 40961]
# magnitude of a row's elements; with eps = 0 for those that eps would cover
ROWS = [(1.0, 1e-6), (1e20, 1e-6), (1e30, 1e-6), (1e37, 1e-6), (1e-25, 0.0), (1e-35, 0.0), (1e-12, 0.0), (1e12, 0.0)]


def rand(rows, width, dtype, seed, scale=1.0):
    return (torch.randn(rows, width, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def close(got, want, tol):
    err = (got.cpu().double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.2f} of the tolerance"


def rows_of(width, dtype, scale):
    # ordinary rows around the ones in question; in one of these a single element is large
    x, r = rand(5, width, dtype, 1), rand(5, width, dtype, 2)
    x[1] = (x[1].double() * scale).to(dtype)
    r[1] = (r[1].double() * scale).to(dtype)
    x[3] = (x[3].double() * scale).to(dtype)
    r[3] = 0
    if scale > 1e18:
        x[4, width // 2] = scale
    return x, r, rand(1, width, dtype, 3)[0]


def norm64(h, w, eps):
    h = h.cpu().double()
    s = 1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return h * s * w.cpu().double(), s


@pytest.mark.parametrize("scale,eps", ROWS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("width", WIDTHS)
def test_forward_and_8_bits(width, dtype, scale, eps):
    u = torch.finfo(dtype).eps / 2
    x, r, w = rows_of(width, dtype, scale)
    y, h, rstd = abi.add_rmsnorm_fwd(x, r, w, eps, return_rstd=True)
    want, rs = norm64(h, w, eps)
    close(y, want, (u + 40 * F32) * want.abs() + torch.finfo(dtype).smallest_normal * u * 2)
    close(rstd, rs[:, 0], 40 * F32 * rs[:, 0])
    for group in (0, 128):
        q, s, _ = abi.add_rmsnorm_quant(x, r, w, eps, group=group)
        g = group or width
        n = -(-width // g)
        top = (torch.nn.functional.pad(want.abs(), (0, n * g - width)).view(5, n, g).amax(-1) / 448.0).clamp_min(2.0 ** -126)
        close(s, top, 44 * F32 * top)
        se = torch.repeat_interleave(s.cpu().double(), g, 1)[:, :width]
        close(q.cpu().float().double() * se, want, (2.0 ** -4 + 48 * F32) * want.abs() + 2.0 ** -10 * se * (1 + 1e-5))


@pytest.mark.parametrize("scale,eps", ROWS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("width", WIDTHS)
def test_gradients(width, dtype, scale, eps):
    u = torch.finfo(dtype).eps / 2
    x, r, w = rows_of(width, dtype, scale)
    h = (x.double() + r.double()).to(dtype)
    gy, gh = rand(5, width, dtype, 4), rand(5, width, dtype, 5)
    rs = 1.0 / torch.sqrt(h.cpu().double().square().mean(-1, keepdim=True) + eps)
    rstd = rs[:, 0].float().to(DEV)
    for g2 in (gh, None):
        gx, gw = abi.add_rmsnorm_bwd(gy, g2, h, w, rstd)
        n, a = h.cpu().double() * rs, gy.cpu().double() * w.cpu().double()
        add = 0 if g2 is None else g2.cpu().double()
        wx = rs * (a - n * (a * n).mean(-1, keepdim=True)) + add
        size = rs * (a.abs() + n.abs() * (a * n).abs().mean(-1, keepdim=True)) + (0 if g2 is None else add.abs())
        close(gx, wx, u * wx.abs() + 96 * F32 * size + torch.finfo(dtype).tiny)
        gn = gy.cpu().double() * n
        close(gw, gn.sum(0), u * gn.sum(0).abs() + 64 * F32 * gn.abs().sum(0) + torch.finfo(dtype).tiny)


def test_the_ends_of_fp16():
    for width in (577, 4096, 40961):
        x = rand(4, width, HF, 1)
        x[0], x[1] = 60000.0, 6e-8
        x[2] *= 1e-7
        r, w = torch.zeros_like(x), rand(1, width, HF, 3)[0]
        for eps in (0.0, 1e-6):
            y, h = abi.add_rmsnorm_fwd(x, r, w, eps)
            want, _ = norm64(h, w, eps)
            close(y, want, (2.0 ** -11 + 40 * F32) * want.abs() + 2.0 ** -25)
