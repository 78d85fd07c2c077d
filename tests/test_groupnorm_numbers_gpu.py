"""Group norm where its numbers are hard.

Statistics are sums in fp64 of values that fp64 holds exactly (squares too), so mean and 1 / sqrt(variance + eps) are their definitions rounded to
fp32: off by u = 2^-24 of the mean, and of rstd by u plus what E[x^2] - mean^2 loses: additions of some hundred values a thread, each off by at most 2^-53 of a partial sum and in either direction, 2^-50
(1 + mean^2 / variance).  y = (x - mean) rstd w + b then adds the
difference's and two products' roundings and that of the mean over the deviation: 4 u |xh w| + u |mean| rstd |w| + u |y|."""
import math

import pytest
import torch

from unet_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def check_forward(x, groups, w, b, stored=0.0):
    n, c = x.shape[0], x.shape[-1]
    y, stats = ops.groupnorm_act_fwd(x, groups, w, b, act="none")
    xd = x.double().cpu().reshape(n, -1, groups, c // groups)
    mean = xd.mean((1, 3), keepdim=True)
    var = (xd - mean).square().mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + float(torch.tensor(1e-5, dtype=torch.float32)))
    lost = 2.0 ** -50 * (1 + mean ** 2 / (var + 1e-5))
    s = stats.double().cpu()
    assert ((s[..., 0] - mean[:, 0, :, 0]).abs() <= 1.01 * U * mean[:, 0, :, 0].abs() + 1e-37).all()
    rel = (s[..., 1] / rstd[:, 0, :, 0] - 1).abs()
    assert (rel <= 1.01 * U + lost[:, 0, :, 0]).all(), float(rel.max() / U)
    xh = (xd - mean) * rstd
    wd, bd = w.double().cpu().reshape(groups, -1), b.double().cpu().reshape(groups, -1)
    want = xh * wd + bd
    tol = (4 * U + lost) * (xh * wd).abs() + 1.01 * U * mean.abs() * rstd * wd.abs() + (U + stored) * want.abs() + 1e-37
    err = (y.double().cpu().reshape(want.shape) - want).abs()
    assert (err <= 1.01 * tol).all(), float((err / tol).max())


@pytest.mark.parametrize("n,sp,c,groups", [(2, (256, 256), 32, 8), (1, (64, 64, 64), 16, 4), (1, (200, 210), 30, 5), (3, (16, 16), 256, 32), (2, (5, 7), 8, 2), (1, (300, 300), 8, 8)])
@pytest.mark.parametrize("level", [0.0, 100.0])
def test_a_pixel_unlike_all_others(dev, n, sp, c, groups, level):
    """A bright pixel on an even background, at the first place of what a thread adds up or anywhere else: the variance is its doing alone."""
    g = torch.Generator().manual_seed(c)
    x = torch.full((n, math.prod(sp), c), level)
    w, b = (1 + 0.2 * torch.randn(c, generator=g)).to(dev), (0.2 * torch.randn(c, generator=g)).to(dev)
    for at in (0, 1, math.prod(sp) // 2, math.prod(sp) - 1):
        y = x.clone()
        y[:, at] += 0.5 + 2.5 * torch.rand(n, c, generator=g)
        check_forward(y.reshape(n, *sp, c).to(dev), groups, w, b)


@pytest.mark.parametrize("n,sp,c,groups", [(2, (256, 256), 32, 8), (1, (130, 170), 30, 5), (2, (12, 20), 64, 8), (1, (700, 700), 4, 1)])
@pytest.mark.parametrize("mean,std", [(0.0, 1.0), (50.0, 1.0), (1000.0, 0.25), (3.0, 1e-2)])
def test_statistics_are_their_definitions_rounded(dev, n, sp, c, groups, mean, std):
    g = torch.Generator().manual_seed(c + int(mean))
    x = (torch.randn(n, *sp, c, generator=g) * std + mean).to(dev)
    w, b = (1 + 0.2 * torch.randn(c, generator=g)).to(dev), (0.2 * torch.randn(c, generator=g)).to(dev)
    check_forward(x, groups, w, b)
    check_forward(x.bfloat16(), groups, w, b, stored=2.0 ** -8)


def test_gelu_is_good_relatively_in_its_tail(dev):
    """weight = 0: the activation sees the biases, exactly.  Phi(-|u|) is off by the fit, 4.8e-7, the exponential's 2^-23 and three roundings of its
    exponent, 1.5 u^2 2^-24; the product with u adds 2^-24, and 1 - Phi another."""
    u = torch.cat([torch.linspace(-12.5, 8.0, 4000), torch.tensor([0.0, -1e-30, 1e-30, -1e-3, 1e-3]), torch.linspace(-0.5, 0.5, 91)])
    c = u.numel()
    x = torch.randn(1, 3, 3, c, generator=torch.Generator().manual_seed(1)).to(dev)
    y, _ = ops.groupnorm_act_fwd(x, 1, torch.zeros(c, device=dev), u.to(dev), act="gelu")
    ud = u.double()
    want = 0.5 * ud * torch.erfc(-ud * 0.5 ** 0.5)
    rel = (y.double().cpu()[0].reshape(9, c) / want - 1).abs()
    rel = torch.where(want == 0, torch.zeros_like(rel), rel)
    bound = 4.8e-7 + (2 + 1.5 * ud ** 2 + 2) * U
    assert (rel <= bound).all(), float((rel / bound).max())
    assert not y[..., u.to(dev) == 0].any()


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_gradient_beyond_2_31_elements(dev, mode):
    """One image whose upstream gradient is 0 except at its last pixels, 2^31 elements behind the first: the sums, and the gradient at both
    ends, follow from those pixels alone.  Means of few values over all: u of each product."""
    c, groups, last = 32, 4, 1000
    npix = (1 << 31) // c + 5000
    dt = torch.float32 if mode == "fp32" else torch.bfloat16
    x = torch.empty(1, npix, 1, c, dtype=dt, device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(1))
    dy = torch.zeros(1, npix, 1, c, dtype=dt, device=dev)
    g = torch.Generator().manual_seed(2)
    dy[0, -last:, 0] = torch.randn(last, c, generator=g).to(dt).to(dev) * 1e3
    w, b = (1 + 0.2 * torch.randn(c, generator=g)).to(dev), (0.2 * torch.randn(c, generator=g)).to(dev)
    stats = torch.stack([0.01 * torch.randn(1, groups, generator=g), 1 + 0.1 * torch.rand(1, groups, generator=g)], -1).to(dev)
    dx, dw, db, _ = ops.groupnorm_act_bwd(dy, x, stats, groups, w, b, act="relu")
    mean, rstd = (stats[0, :, k].double().cpu().repeat_interleave(c // groups) for k in (0, 1))
    wd, bd = w.double().cpu(), b.double().cpu()

    def parts(rows):
        xh = (x[0, rows, 0].double().cpu() - mean) * rstd
        return xh, dy[0, rows, 0].double().cpu() * (xh * wd + bd > 0)

    xh, gr = parts(slice(npix - last, npix))
    for got, want, size in ((db, gr.sum(0), gr.abs().sum(0)), (dw, (gr * xh).sum(0), (gr * xh).abs().sum(0))):
        assert ((got.double().cpu() - want).abs() <= 260 * U * size).all()                 # up to 256 values of a thread in fp32
    count = npix * (c // groups)
    m0 = ((gr * wd).sum(0).reshape(groups, -1).sum(1) / count).repeat_interleave(c // groups)
    m1 = ((gr * wd * xh).sum(0).reshape(groups, -1).sum(1) / count).repeat_interleave(c // groups)
    size = ((gr * wd).abs() * (1 + xh.abs())).sum() / count
    assert float(size) > 1e-4
    for rows in (slice(0, 50), slice(npix - last, npix)):
        xh, gr = parts(rows)
        want = rstd * (wd * gr - m0 - xh * m1)
        tol = rstd * (8 * U * (wd * gr).abs() + 300 * U * size * (1 + xh.abs())) + (2.0 ** -8 if mode == "bf16" else U) * want.abs()
        err = (dx[0, rows, 0].double().cpu() - want).abs()
        assert (err <= 1.01 * tol).all(), float((err / tol).max())
