"""Residual addition with RMSNorm: forward, 8-bit forward and gradients against 64 bits, with tolerances that count the
roundings: half a step of the result, and a few dozen half steps of fp32 for the sums."""
import pytest
import torch

import torch_paras  # noqa: F401
from torch_paras import abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
F32 = 2.0 ** -24     # half a step of fp32
# one warp's rows, several warps', the longest in registers, longer ones, and rows of no whole 16 bytes
WIDTHS = [1, 7, 8, 64, 100, 256, 264, 511, 512, 1000, 1024, 1032, 2048, 4096, 5000, 6144, 8192, 8200, 16384, 30000, 32768, 33000, 40961]


def data(rows, width, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, width, generator=g) * scale).to(dtype).to(DEV)


def norm64(h, w, eps):
    h = h.cpu().double()
    r = 1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return h * r * (1.0 if w is None else w.cpu().double()), r


def close(got, want, tol):
    err = (got.cpu().double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("width", WIDTHS)
def test_forward(width, dtype):
    u = torch.finfo(dtype).eps / 2
    for rows in (1, 5):
        x, r, w = data(rows, width, dtype, 1), data(rows, width, dtype, 2, 3.0), data(1, width, dtype, 3)[0]
        for res in (r, None):
            for wt in (w, None):
                y, h, rstd = abi.add_rmsnorm_fwd(x, res, wt, 1e-6, return_rstd=True)
                assert torch.equal(h, x if res is None else (x.float() + r.float()).to(dtype))
                want, rs = norm64(h, wt, 1e-6)
                # sum of squares: at most 64 terms one after the other; three fp32 roundings on the way to y
                close(y, want, (u + 40 * F32) * want.abs() + torch.finfo(dtype).smallest_normal * u * 2)
                close(rstd, rs[:, 0], 40 * F32 * rs[:, 0])


@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("width", WIDTHS)
def test_forward_in_8_bits(width, dtype, group):
    rows = 3
    x, r, w = data(rows, width, dtype, 1), data(rows, width, dtype, 2, 3.0), data(1, width, dtype, 3)[0]
    x[1], r[1] = 0, 0                                # a row of zeros
    for res in (r, None):
        q, s, h = abi.add_rmsnorm_quant(x, res, w, 1e-6, group=group)
        assert torch.equal(h, x if res is None else (x.float() + r.float()).to(dtype))
        want, _ = norm64(h, w, 1e-6)
        g = group or width
        n = -(-width // g)
        assert s.shape == (rows, n) and q.dtype == torch.float8_e4m3fn
        top = torch.nn.functional.pad(want.abs(), (0, n * g - width)).view(rows, n, g).amax(-1) / 448.0
        top = top.clamp_min(2.0 ** -126)
        close(s, top, 44 * F32 * top)
        se = torch.repeat_interleave(s.cpu().double(), g, 1)[:, :width]
        got = q.cpu().float().double() * se
        # half a step of e4m3, subnormal steps being 2^-9 of the scale; the fp32 arithmetic before it
        close(got, want, (2.0 ** -4 + 48 * F32) * want.abs() + 2.0 ** -10 * se * (1 + 1e-5))


def grads64(gy, gh, h, w, rstd_eps):
    gy, h = gy.cpu().double(), h.cpu().double()
    w = torch.ones(h.shape[-1], dtype=torch.float64) if w is None else w.cpu().double()
    r = 1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + rstd_eps)
    n, a = h * r, gy * w
    m = (a * n).mean(-1, keepdim=True)
    gx = r * (a - n * m) + (0 if gh is None else gh.cpu().double())
    size = r * (a.abs() + n.abs() * (a * n).abs().mean(-1, keepdim=True)) + (0 if gh is None else gh.cpu().double().abs())
    return gx, (gy * n).sum(0), size, (gy * n).abs().sum(0)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("width", [1, 7, 64, 100, 256, 520, 1024, 2048, 3001, 4096, 5000, 8192, 8200, 16384, 16392])
def test_backward(width, dtype):
    u = torch.finfo(dtype).eps / 2
    for rows in (1, 3, 700):
        if rows * width > 4_000_000:
            continue
        h, w = data(rows, width, dtype, 1, 2.0), data(1, width, dtype, 3)[0]
        gy, gh = data(rows, width, dtype, 4), data(rows, width, dtype, 5)
        _, rs = norm64(h, None, 1e-6)
        rstd = rs[:, 0].float().to(DEV)
        for g2 in (gh, None):
            for wt in (w, None):
                gx, gw = abi.add_rmsnorm_bwd(gy, g2, h, wt, rstd)
                wx, ww, sx, sw = grads64(gy, g2, h, wt, 1e-6)
                close(gx, wx, u * wx.abs() + 96 * F32 * sx + torch.finfo(dtype).tiny)
                if wt is None:
                    assert gw is None
                else:
                    close(gw, ww, u * ww.abs() + 64 * F32 * sw + torch.finfo(dtype).tiny)


def test_differences_and_autograd_on_the_device():
    from torch_paras import nn
    torch.manual_seed(0)
    x, r, w = (torch.randn(3, 40, dtype=torch.float32) for _ in range(3))
    w = w[0].contiguous()
    a, b = torch.randn(3, 40), torch.randn(3, 40)

    def f(x, r, w):      # in 64 bits
        h = x + r
        return ((h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w) * a.double()).sum() + (h * b.double()).sum()

    leaves = [t.to("paras:1").requires_grad_() for t in (x, r, w)]
    y, h = nn.add_rms_norm(*leaves)
    torch.autograd.backward([y, h], [a.to("paras:1"), b.to("paras:1")])
    for i, t in enumerate((x, r, w)):
        base = [v.double() for v in (x, r, w)]
        num = torch.zeros_like(base[i])
        for j in range(t.numel()):
            p = [v.clone() for v in base]
            m = [v.clone() for v in base]
            p[i].view(-1)[j] += 1e-5
            m[i].view(-1)[j] -= 1e-5
            num.view(-1)[j] = (f(*p) - f(*m)) / 2e-5
        assert (leaves[i].grad.cpu().double() - num).abs().max() <= 1e-4 * num.abs().max()
    # one of the two results unused; the same tensor twice
    for which in (0, 1):
        leaves = [t.to("paras:1").requires_grad_() for t in (x, r, w)]
        out = nn.add_rms_norm(*leaves)[which]
        out.backward(a.to("paras:1"))
        assert torch.equal(leaves[0].grad.cpu(), leaves[1].grad.cpu())
        assert (leaves[2].grad is None) == (which == 1)
    leaf, wd = x.to("paras:1").requires_grad_(), w.to("paras:1")
    y, h = nn.add_rms_norm(leaf, leaf, wd)
    h.backward(a.to("paras:1"))
    assert torch.allclose(leaf.grad.cpu(), 2 * a)


def test_infinities_and_nan_stay_in_their_row():
    x, r, w = data(4, 1000, BF, 1), data(4, 1000, BF, 2), data(1, 1000, BF, 3)[0]
    clean = abi.add_rmsnorm_fwd(x, r, w), abi.add_rmsnorm_quant(x, r, w, group=128)
    x[1, 5], r[2, 7] = float("nan"), float("inf")
    y, h = abi.add_rmsnorm_fwd(x, r, w)
    q, s, _ = abi.add_rmsnorm_quant(x, r, w, group=128)
    for row in (0, 3):
        assert torch.equal(y[row], clean[0][0][row]) and torch.equal(s[row], clean[1][1][row])
        assert torch.equal(q[row].view(torch.uint8), clean[1][0][row].view(torch.uint8))
    assert torch.isnan(y[1]).all() and torch.isnan(q[1].float()).all()
    assert torch.isnan(y[2, 7]) and bool((y[2, :7] == 0).all())


def test_in_place_streams_capture_and_refusals():
    x, r, w = data(64, 4096, BF, 1), data(64, 4096, BF, 2), data(1, 4096, BF, 3)[0]
    ref = abi.add_rmsnorm_fwd(x, r, w)
    torch.cuda.synchronize()
    # h over residual, through the C entry
    h = r.clone()
    y = torch.empty_like(x)
    abi.check(abi.lib().paras_b200_add_rmsnorm_fwd(0, x.data_ptr(), h.data_ptr(), w.data_ptr(), h.data_ptr(), y.data_ptr(), None,
                                                   64, 4096, 1e-6, abi.BF16, torch.cuda.current_stream().cuda_stream or 1))
    torch.cuda.synchronize()
    assert torch.equal(h, ref[1]) and torch.equal(y, ref[0])
    side = torch.cuda.Stream()
    gy = data(64, 4096, BF, 5)
    rstd = abi.add_rmsnorm_fwd(x, r, w, return_rstd=True)[2]
    gref = abi.add_rmsnorm_bwd(gy, None, ref[1], w, rstd)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = abi.add_rmsnorm_fwd(x, r, w)
        gout = abi.add_rmsnorm_bwd(gy, None, out[1], w, rstd)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], ref[0]) and torch.equal(gout[0], gref[0]) and torch.equal(gout[1], gref[1])
    with pytest.raises(RuntimeError, match="group"):
        abi.add_rmsnorm_quant(x, r, w, group=48)
    with pytest.raises(RuntimeError, match="one shape"):
        abi.add_rmsnorm_fwd(x, r[:1], w)
    with pytest.raises(RuntimeError, match="one type"):
        abi.add_rmsnorm_fwd(x, r, w.float())
    y, h = abi.add_rmsnorm_fwd(x[:0], r[:0], w)
    assert y.shape == (0, 4096)
    gx, gw = abi.add_rmsnorm_bwd(x[:0], None, x[:0], w, torch.empty(0, device=DEV))
    assert bool((gw == 0).all())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("width", [7, 577, 4096, 5001, 16384, 33000, 40961])
def test_the_sum_over_either_of_its_terms(width, dtype):
    # through the C entries: h is the memory of x or of residual, on every kernel
    code = abi.BF16 if dtype == BF else abi.F32
    x, r, w = data(9, width, dtype, 1), data(9, width, dtype, 2), data(1, width, dtype, 3)[0]
    ref, quant = abi.add_rmsnorm_fwd(x, r, w), abi.add_rmsnorm_quant(x, r, w, group=64)
    stream = torch.cuda.current_stream().cuda_stream or 1
    for over in (0, 1):
        a, b, y = x.clone(), r.clone(), torch.empty_like(x)
        h = b if over else a
        abi.check(abi.lib().paras_b200_add_rmsnorm_fwd(0, a.data_ptr(), b.data_ptr(), w.data_ptr(), h.data_ptr(), y.data_ptr(), None,
                                                       9, width, 1e-6, code, stream))
        assert torch.equal(h, ref[1]) and torch.equal(y, ref[0])
        a, b = x.clone(), r.clone()
        h, q, s = b if over else a, torch.empty_like(quant[0]), torch.empty_like(quant[1])
        abi.check(abi.lib().paras_b200_add_rmsnorm_quant_fwd(0, a.data_ptr(), b.data_ptr(), w.data_ptr(), h.data_ptr(), q.data_ptr(),
                                                             s.data_ptr(), 9, width, 1e-6, 64, code, stream))
        assert torch.equal(h, ref[1]) and torch.equal(s, quant[1]) and torch.equal(q.view(torch.uint8), quant[0].view(torch.uint8))


def test_a_given_stream_takes_no_copies():
    x, w = data(8, 512, BF, 1), data(1, 512, BF, 3)[0]
    wide = data(8, 1024, BF, 2)[:, ::2]
    want = abi.add_rmsnorm_fwd(x, wide, w)
    assert torch.equal(want[1], (x.float() + wide.float()).to(BF))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = abi.add_rmsnorm_fwd(x, wide.contiguous(), w, stream=torch.cuda.current_stream().cuda_stream or 1)
    assert torch.equal(got[0], want[0])
    for call in (lambda: abi.add_rmsnorm_fwd(x, wide, w, stream=s.cuda_stream),
                 lambda: abi.add_rmsnorm_quant(wide, x, w, stream=s.cuda_stream),
                 lambda: abi.add_rmsnorm_bwd(wide, None, x, w, torch.ones(8, device=DEV), stream=s.cuda_stream)):
        with pytest.raises(RuntimeError, match="contiguous rows"):
            call()


def test_a_second_derivative_is_refused():
    from torch_paras import nn
    x, r, w = (torch.randn(n, 16, dtype=torch.float32).squeeze(0).to("paras:1").requires_grad_() for n in (3, 3, 1))
    ones = torch.ones(3, 16).to("paras:1")
    for grad_y, text in ((ones, "does not require grad"), (ones.clone().requires_grad_(), "once_differentiable")):
        y, h = nn.add_rms_norm(x, r, w)
        g = torch.autograd.grad(y, x, grad_y, create_graph=True)[0]
        with pytest.raises(RuntimeError, match=text):
            g.backward(ones)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("width", [64, 256, 512, 1000, 2048])
def test_backward_of_many_rows(width, dtype):
    # every block walks several rows, and its ring of rows goes round
    rows, u = 10_001, torch.finfo(dtype).eps / 2
    h, w = data(rows, width, dtype, 1, 2.0), data(1, width, dtype, 3)[0]
    gy, gh = data(rows, width, dtype, 4), data(rows, width, dtype, 5)
    rstd = norm64(h, None, 1e-6)[1][:, 0].float().to(DEV)
    gx, gw = abi.add_rmsnorm_bwd(gy, gh, h, w, rstd)
    wx, ww, sx, sw = grads64(gy, gh, h, w, 1e-6)
    close(gx, wx, u * wx.abs() + 96 * F32 * sx + torch.finfo(dtype).tiny)
    # a column's products go through fp32 in runs of at most 32 rows (10001 / 592 and fewer), in 64 bits between the runs
    close(gw, ww, u * ww.abs() + 64 * F32 * sw + torch.finfo(dtype).tiny)
    again = abi.add_rmsnorm_bwd(gy, gh, h, w, rstd)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)
