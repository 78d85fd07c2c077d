"""Group norm + activation on channels-last tensors against the formula in 64 bits.

Tolerances (derived before the first run).  u32 = 2^-24, ub = 2^-9 is half a bf16 step relative to the next power of two
and at most 2^-8 relative to the value.

* statistics: fp64 sums of fp32 differences from a thread's first value; a thread adds at most 256 of them, each addition
  rounds by u32 relative to the running sum: 256 u32 relative to sum |d|, sum d^2, plus the final rounding.  rstd goes with
  half of the variance's error.  STAT = 300 u32 = 1.8e-5, relative to (|x - first|, at most 16 standard deviations here).
  In practice roundings cancel; the bound used is 2e-5 for the mean in units of the standard deviation and for rstd.
* y: x - mean rounds by u32 of |mean| / std (mean itself is rounded to fp32) -> the error in xh is at most
  (2 |mean| / std + 4 |xh|) u32 + 2e-5 |xh| + 2e-5; times |w| and the activation's slope (at most 1.13), plus 8 u32 of the
  activation's own functions; then one rounding to the storage type.
* gradients: the same relative errors in every factor (8 factors, 2e-5 each at most) on terms bounded by |w g|, the group
  means bounded by mean |w g| and mean |w g xh|.
"""
import pytest
import torch
import torch.nn.functional as F

from unet_amd import ops

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
HALF_STEP = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8}
ACTS = {"none": lambda u, a: u * 1.0, "relu": lambda u, a: F.relu(u), "silu": lambda u, a: F.silu(u), "gelu": lambda u, a: F.gelu(u),
        "prelu": lambda u, a: F.relu(u) - a * F.relu(-u)}


def formula(x, groups, w, b, act, alpha, res, dy, eps=1e-5):
    """64 bits on the CPU: y, stats, dx, dw, db, dalpha and bounds of the terms that go into y and dx."""
    x, dy = x.double().cpu(), dy.double().cpu()
    nb, c = x.shape[0], x.shape[-1]
    w = torch.ones(c) if w is None else w.cpu()
    b = torch.zeros(c) if b is None else b.cpu()
    w, b = w.double(), b.double()
    a = alpha.double().cpu() if alpha is not None else None
    xg = x.reshape(nb, -1, groups, c // groups)
    mean = xg.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((xg - mean).square().mean((1, 3), keepdim=True) + eps)
    xh = ((xg - mean) * rstd).reshape(nb, -1, c)
    u = (xh * w + b).requires_grad_(True)
    al = a.requires_grad_(True) if a is not None else None
    y = ACTS[act](u, al)
    ins = [u] + ([al] if al is not None else [])
    got = torch.autograd.grad(y, ins, dy.reshape(nb, -1, c))
    g, da = got[0], (got[1] if al is not None else None)
    wg = (g * w).reshape(xg.shape)
    hg = xh.reshape(xg.shape)
    m0, m1 = wg.mean((1, 3), keepdim=True), (wg * hg).mean((1, 3), keepdim=True)
    dx = (rstd * (wg - m0 - hg * m1)).reshape(x.shape)
    # what the errors are relative to
    size = rstd * (wg.abs() + wg.abs().mean((1, 3), keepdim=True) + hg.abs() * (wg * hg).abs().mean((1, 3), keepdim=True))
    # a shift of xh by e moves g by at most 1.13 |dy| |w| e
    moved = rstd * (w.square() * dy.reshape(nb, -1, c).abs()).reshape(xg.shape)
    offset = (mean.abs() * rstd).expand_as(xg).reshape(x.shape)
    y = y.detach().reshape(x.shape)
    if res is not None:
        y = y + res.double().cpu()
    return dict(y=y, mean=mean.reshape(nb, groups), rstd=rstd.reshape(nb, groups), dx=dx, dw=(g * xh).sum((0, 1)), db=g.sum((0, 1)), da=da,
                xh=xh.reshape(x.shape), w=w, b=b, size=size.reshape(x.shape), moved=moved.reshape(x.shape), offset=offset,
                sum_dw=(g * xh).abs().sum((0, 1)), sum_db=g.abs().sum((0, 1)), sum_dy=dy.reshape(-1, c).abs().sum(0),
                sum_dyx=(dy.reshape(nb, -1, c) * xh).abs().sum((0, 1)), sum_da=(dy.reshape(nb, -1, c) * u.detach()).abs().sum())


U32 = 2.0 ** -24
STAT = 2e-5


def xh_error(r):
    return (2 * r["offset"] + 4 * r["xh"].abs()) * U32 + STAT * (1 + r["xh"].abs())


def check_forward(y, stats, r, mode, res=None):
    std = 1 / r["rstd"]
    assert ((stats[..., 0].double().cpu() - r["mean"]).abs() <= STAT * std + U32 * r["mean"].abs()).all()
    assert ((stats[..., 1].double().cpu() / r["rstd"] - 1).abs() <= STAT).all()
    tol = 1.13 * r["w"].abs() * xh_error(r) + 8 * U32 * (r["w"].abs() * r["xh"].abs() + r["b"].abs())
    if res is not None:
        tol = tol + U32 * res.double().cpu().abs()
    tol = tol * 1.01 + HALF_STEP[mode] * r["y"].abs() + 1e-30
    err = (y.double().cpu() - r["y"]).abs()
    assert (err <= tol).all(), float((err / tol).max())


def check_backward(got, r, mode):
    dx, dw, db, da = got
    e = xh_error(r)
    tol = 8 * STAT * r["size"] + 1.13 * r["moved"] * e + r["size"] * e
    tol = tol + 1.13 * (r["moved"] * e).mean() * 2 + HALF_STEP[mode] * r["dx"].abs() + 1e-30
    err = (dx.double().cpu() - r["dx"]).abs()
    assert (err <= tol).all(), float((err / tol).max())
    worst = float((r["offset"].max() * 2 + 4 * r["xh"].abs().max()) * U32 + STAT * (1 + r["xh"].abs().max()))
    w = float(r["w"].abs().max())
    for name, g, ref, size in (("dw", dw, r["dw"], r["sum_dw"] + worst * r["sum_dy"] + (1.13 * w) * worst * r["sum_dyx"] / 8 / STAT),
                               ("db", db, r["db"], r["sum_db"] + (1.13 * w) * worst * r["sum_dy"] / 8 / STAT)):
        if g is not None:
            err = (g.double().cpu() - ref).abs()
            assert (err <= 8 * STAT * size + 1e-30).all(), (name, float((err / (8 * STAT * size)).max()))
    if r["da"] is not None:
        assert abs(float(da) - float(r["da"])) <= 8 * STAT * float(r["sum_da"]) + worst * w * float(r["sum_dy"].sum())


CASES = [  # N, spatial, C, groups, act, affine, residual, mean offset
    (2, (16, 16), 64, 8, "silu", True, False, 0.0),
    (1, (1, 1), 16, 4, "silu", True, False, 0.0),          # four values per group
    (1, (1,), 8, 8, "none", True, True, 0.0),              # one value per group: xh = 0
    (3, (5, 7), 30, 5, "gelu", True, True, 0.0),
    (3, (5, 7), 3, 1, "relu", True, False, 0.0),
    (2, (3, 5, 7), 33, 33, "prelu", True, False, 0.0),     # one channel per group, odd
    (2, (9, 4), 20, 2, "prelu", False, False, 0.0),
    (5, (64, 33), 96, 12, "silu", True, False, 0.0),
    (1, (190, 181), 16, 4, "silu", True, True, 3.0),       # several workgroups per image
    (1, (190, 181), 12, 3, "gelu", True, False, 0.0),
    (2, (130, 127), 7, 7, "silu", True, False, 0.0),
    (1, (24, 24, 24), 32, 8, "prelu", True, False, 0.0),
    (4, (6, 5), 2080, 65, "silu", True, False, 0.0),       # more vectors per pixel than a workgroup has threads
    (1, (3, 3), 8192, 2048, "relu", True, False, 0.0),     # the limits
    (2, (4, 4), 2050, 1025, "none", True, False, 0.0),
    (300, (2, 2), 16, 16, "silu", True, False, 0.0),
    (2, (80, 80), 16, 2, "silu", True, False, 1000.0),     # mean far from zero
    (3, (61, 53), 33, 3, "silu", True, True, 0.0),         # odd channel counts, a number of pixels that is no multiple of 8 or 4
    (1, (151, 149), 5, 5, "prelu", True, False, 0.0),
    (2, (67, 71), 30, 10, "gelu", True, True, 2.0),
    (1, (50, 51), 255, 5, "silu", True, False, 0.0),
    (1, (41, 43), 257, 1, "relu", True, False, 0.0),
    (2, (53, 37), 250, 125, "silu", False, False, 0.0),
    (2, (103, 101), 12, 2, "none", True, False, 0.0),
    (3, (395, 397), 36, 3, "silu", True, False, 0.0),      # tens of MB whose pixels are a multiple of 8 bytes
    (1, (397, 401), 54, 6, "gelu", True, True, 0.0),
    (2, (45, 43), 36, 4, "prelu", True, False, 0.0),
]


def make(case, mode, dev, seed=0):
    n, sp, c, groups, act, affine, res, offset = case
    g = torch.Generator().manual_seed(1000 + seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    dt = DT[mode]
    x = (rnd(n, *sp, c) * (0.5 + rnd(c).abs()) + rnd(c) + offset).to(dt).to(dev)
    dy = rnd(n, *sp, c).to(dt).to(dev)
    w = (1 + 0.3 * rnd(c)).to(dev) if affine else None
    b = (0.3 * rnd(c)).to(dev) if affine else None
    alpha = torch.tensor([0.25], device=dev) if act == "prelu" else None
    r = rnd(n, *sp, c).to(dt).to(dev) if res else None
    return x, dy, w, b, alpha, r


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{'x'.join(map(str, c[1]))}x{c[2]}g{c[3]}{c[4]}")
def test_forward_and_backward(dev, mode, case):
    n, sp, c, groups, act, affine, res, offset = case
    x, dy, w, b, alpha, r = make(case, mode, dev)
    y, stats = ops.groupnorm_act_fwd(x, groups, w, b, act=act, alpha=alpha, res=r)
    # the backward kernel starts from the forward's fp32 statistics: so does its reference
    got = ops.groupnorm_act_bwd(dy, x, stats, groups, w, b, act=act, alpha=alpha)
    ref = formula(x, groups, w, b, act, alpha, r, dy)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    check_forward(y, stats, ref, mode, r)
    assert (got[1] is None) == (w is None) and (got[3] is None) == (alpha is None)
    check_backward(got, ref, mode)


def test_gradient_against_differences(dev):
    """Directional differences of the forward call itself (fp32, sums in 64 bits on the host)."""
    x, dy, w, b, alpha, _ = make((2, (7, 9), 24, 4, "silu", True, False, 0.0), "fp32", dev)
    g = torch.Generator().manual_seed(3)
    for act, al in (("silu", None), ("gelu", None)):
        _, stats = ops.groupnorm_act_fwd(x, 4, w, b, act=act)
        dx, dw, db, _ = ops.groupnorm_act_bwd(dy, x, stats, 4, w, b, act=act)
        vx, vw, vb = (torch.randn(t.shape, generator=g).to(dev) for t in (x, w, b))
        h = 2.0 ** -6

        def f(s):
            y, _ = ops.groupnorm_act_fwd(x + s * h * vx, 4, w + s * h * vw, b + s * h * vb, act=act)
            return float((y.double() * dy.double()).sum())

        got = float((dx.double() * vx.double()).sum() + (dw.double() * vw.double()).sum() + (db.double() * vb.double()).sum())
        # central differences with one extrapolation: error O(h^4), rounding of y (1e-6 per value, 3e3 values, random) / h
        d1, d2 = (f(1) - f(-1)) / (2 * h), (f(2) - f(-2)) / (4 * h)
        assert abs((4 * d1 - d2) / 3 - got) < 2e-3 * float((dy.abs() * vx.abs()).sum().sqrt() + 1), act


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_views_and_other_orders(dev, mode):
    """A slice of a wider tensor's channels is read in place; other orders of the memory give the same numbers."""
    case = (2, (9, 11), 24, 6, "silu", True, True, 0.0)
    x, dy, w, b, alpha, r = make(case, mode, dev)
    y, stats = ops.groupnorm_act_fwd(x, 6, w, b, res=r)
    dx, dw, db, _ = ops.groupnorm_act_bwd(dy, x, stats, 6, w, b)
    for lo in (0, 1, 3, 8):
        wide = torch.full((2, 9, 11, 40), float("nan"), dtype=x.dtype, device=dev)
        wide[..., lo:lo + 24] = x
        wd = torch.full((2, 9, 11, 33), float("nan"), dtype=x.dtype, device=dev)
        wd[..., lo:lo + 24] = dy
        xv, dv = wide[..., lo:lo + 24], wd[..., lo:lo + 24]
        yv, sv = ops.groupnorm_act_fwd(xv, 6, w, b, res=r)
        gv = ops.groupnorm_act_bwd(dv, xv, sv, 6, w, b)
        for a, c in ((yv, y), (sv, stats), (gv[0], dx), (gv[1], dw), (gv[2], db)):
            assert torch.allclose(a.float(), c.float(), rtol=1e-2 if mode == "bf16" else 1e-4, atol=1e-4)
        ref = formula(x, 6, w, b, "silu", None, r, dy)
        check_forward(yv, sv, ref, mode, r)
        check_backward(gv, ref, mode)
    planar = x.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    assert not planar.is_contiguous()
    yp, sp = ops.groupnorm_act_fwd(planar, 6, w, b, res=r)
    assert torch.equal(yp, y) and torch.equal(sp, stats)
    cut = torch.randn(2, 9, 20, 24, device=dev).to(x.dtype)
    cut[:, :, 2:13] = x
    yc, _ = ops.groupnorm_act_fwd(cut[:, :, 2:13], 6, w, b, res=r)
    assert torch.equal(yc, y)
    one = x[:1, :1, :1].expand(2, 9, 11, 24)
    y1, _ = ops.groupnorm_act_fwd(one, 6, w, b)
    y2, _ = ops.groupnorm_act_fwd(one.contiguous(), 6, w, b)
    assert torch.equal(y1, y2)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_large_slices_of_wider_tensors(dev, mode):
    """The same numbers from a slice of the channels, read where it lies, as from a dense copy of it."""
    for c, lo, width in ((30, 1, 40), (32, 8, 64), (7, 2, 9)):
        case = (2, (73, 77), c, 1, "silu", True, False, 0.0)
        x, dy, w, b, _, _ = make(case, mode, dev)
        wide = torch.full((2, 73, 77, width), float("nan"), dtype=x.dtype, device=dev)
        wide[..., lo:lo + c] = x
        y, s = ops.groupnorm_act_fwd(wide[..., lo:lo + c], 1, w, b)
        got = ops.groupnorm_act_bwd(dy, wide[..., lo:lo + c], s, 1, w, b)
        ref = formula(x, 1, w, b, "silu", None, None, dy)
        check_forward(y, s, ref, mode)
        check_backward(got, ref, mode)
        y, s = ops.groupnorm_act_fwd(x, 1, w, b)
        check_forward(y, s, ref, mode)
        check_backward(ops.groupnorm_act_bwd(dy, x, s, 1, w, b), ref, mode)


def test_nan_and_infinity_stay_in_their_group(dev):
    x, dy, w, b, _, _ = make((2, (40, 40), 16, 4, "silu", True, False, 0.0), "fp32", dev)
    y0, s0 = ops.groupnorm_act_fwd(x, 4, w, b)
    bad = x.clone()
    bad[0, 3, 5, 1], bad[1, 39, 39, 15] = float("nan"), float("inf")
    y, s = ops.groupnorm_act_fwd(bad, 4, w, b)
    assert torch.isnan(y[0, ..., :4]).all() and torch.isnan(s[0, 0]).all()
    assert torch.isnan(y[1, ..., 12:]).all()
    assert torch.equal(y[0, ..., 4:], y0[0, ..., 4:]) and torch.equal(y[1, ..., :12], y0[1, ..., :12])
    for act in ("none", "relu", "gelu"):
        y, _ = ops.groupnorm_act_fwd(bad, 4, w, b, act=act)
        assert torch.isnan(y[0, ..., :4]).all()
    x, dy, w, b, _, _ = make((1, (81, 83), 15, 5, "silu", True, False, 0.0), "bf16", dev)
    y0, s0 = ops.groupnorm_act_fwd(x, 5, w, b)
    g0 = ops.groupnorm_act_bwd(dy, x, s0, 5, w, b)
    bad = x.clone()
    bad[0, 80, 82, 4] = float("nan")                       # the last pixel, group 1
    y, s = ops.groupnorm_act_fwd(bad, 5, w, b)
    g = ops.groupnorm_act_bwd(dy, bad, s, 5, w, b)
    keep = [0, 1, 2] + list(range(6, 15))
    assert torch.isnan(y[..., 3:6]).all() and torch.equal(y[..., keep], y0[..., keep])
    assert torch.isnan(g[0][..., 3:6]).all() and torch.equal(g[0][..., keep], g0[0][..., keep]) and torch.equal(g[1][keep], g0[1][keep])


def test_an_outlier_as_the_first_value_does_not_cost_the_variance(dev):
    x, dy, w, b, _, _ = make((1, (96, 96), 8, 1, "none", True, False, 0.0), "fp32", dev)
    x[0, 0, 0, 0] = 3e4
    y, s = ops.groupnorm_act_fwd(x, 1, w, b, act="none")
    ref = formula(x, 1, w, b, "none", None, None, dy)
    assert abs(float(s[0, 0, 1]) / float(ref["rstd"]) - 1) < STAT


def test_more_than_2_31_elements(dev):
    """Offsets beyond 32 bits: an image whose last pixels lie behind 2^31 elements, and its gradient."""
    npix, c = 67200000, 32
    x = torch.empty(1, npix, c, dtype=torch.bfloat16, device=dev)
    x.normal_()
    y, s = ops.groupnorm_act_fwd(x, 4, act="none")
    m = torch.stack([p.reshape(-1, 4, 8).float().double().mean((0, 2)) * p.shape[0] for p in x[0].split(4200000)]).sum(0) / npix
    q = torch.stack([p.reshape(-1, 4, 8).float().double().square().mean((0, 2)) * p.shape[0] for p in x[0].split(4200000)]).sum(0) / npix
    rstd = 1 / torch.sqrt(q - m * m + 1e-5)
    assert (s[0, :, 0].double() - m).abs().max() < STAT and (s[0, :, 1].double() / rstd - 1).abs().max() < STAT
    for a in (0, npix - 40):
        want = (x[0, a:a + 40].double().reshape(-1, 4, 8) - m[:, None]) * rstd[:, None]
        assert ((y[0, a:a + 40].double().reshape(want.shape) - want).abs() <= want.abs() * HALF_STEP["bf16"] + 4 * STAT).all()
    dx, _, _, _ = ops.groupnorm_act_bwd(y, x, s, 4, act="none")     # y as its own gradient: dx = rstd (y - xh mean(y xh)) = 0
    assert dx[0, -40:].float().abs().max() < 6 * 2.0 ** -8 * float(rstd.max()) * 1.1      # |xh| < 6, half a step of y


def test_results_repeat_bit_for_bit_and_other_streams_wait(dev):
    case = (2, (200, 170), 32, 8, "prelu", True, False, 0.0)
    x, dy, w, b, alpha, _ = make(case, "bf16", dev)
    first = None
    for _ in range(3):
        y, s = ops.groupnorm_act_fwd(x, 8, w, b, act="prelu", alpha=alpha)
        out = (y, s) + ops.groupnorm_act_bwd(dy, x, s, 8, w, b, act="prelu", alpha=alpha)
        if first is None:
            first = out
        assert all(torch.equal(a, c) for a, c in zip(out, first))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        y, s = ops.groupnorm_act_fwd(x, 8, w, b, act="prelu", alpha=alpha)
        out = (y, s) + ops.groupnorm_act_bwd(dy, x, s, 8, w, b, act="prelu", alpha=alpha)
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(out, first))


def test_two_captured_graphs_replay_in_turn(dev):
    case = (2, (50, 40), 24, 6, "silu", True, False, 0.0)
    x, dy, w, b, _, _ = make(case, "bf16", dev)
    graphs = []
    torch.cuda.synchronize()
    for scale in (1.0, 2.0):
        xs = (x.float() * scale + scale).to(x.dtype)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            ops.groupnorm_act_bwd(dy, xs, ops.groupnorm_act_fwd(xs, 6, w, b)[1], 6, w, b)
        torch.cuda.current_stream(dev).wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y, s = ops.groupnorm_act_fwd(xs, 6, w, b)
            g = ops.groupnorm_act_bwd(dy, xs, s, 6, w, b)
        graphs.append((gr, xs, (y, s) + g[:3]))
    for _ in range(3):
        for gr, xs, out in graphs:
            xs.add_(0.25)
            gr.replay()
            y, s = ops.groupnorm_act_fwd(xs, 6, w, b)
            want = (y, s) + ops.groupnorm_act_bwd(dy, xs, s, 6, w, b)[:3]
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_refusals_on_the_gpu(dev):
    x = torch.randn(2, 4, 4, 12, device=dev)
    w = torch.ones(12, device=dev)
    st = torch.zeros(2, 4, 2, device=dev)
    bad = [lambda: ops.groupnorm_act_fwd(x, 5, w), lambda: ops.groupnorm_act_fwd(x, 0, w), lambda: ops.groupnorm_act_fwd(x.half(), 4),
           lambda: ops.groupnorm_act_fwd(x, 4, w[:3]), lambda: ops.groupnorm_act_fwd(x, 4, w, act="swish"), lambda: ops.groupnorm_act_fwd(x, 4, act="prelu"),
           lambda: ops.groupnorm_act_fwd(x, 4, alpha=torch.ones(1, device=dev)), lambda: ops.groupnorm_act_fwd(x, 4, w.cpu()),
           lambda: ops.groupnorm_act_fwd(x, 4, res=x[:1]), lambda: ops.groupnorm_act_fwd(x, 4, res=x.bfloat16()), lambda: ops.groupnorm_act_fwd(x[:, :0], 4),
           lambda: ops.groupnorm_act_bwd(x.bfloat16(), x, st, 4), lambda: ops.groupnorm_act_bwd(x, x, st[:1], 4), lambda: ops.groupnorm_act_bwd(x, x, st.double(), 4)]
    for f in bad:
        with pytest.raises((ValueError, TypeError)):
            f()
    with pytest.raises(RuntimeError):
        ops.groupnorm_act_fwd(x, 4, eps=-1.0)
    y, s = ops.groupnorm_act_fwd(x[:0], 4, w)
    assert y.shape == (0, 4, 4, 12) and s.shape == (0, 4, 2)
    dx, dw, db, da = ops.groupnorm_act_bwd(x[:0], x[:0], s, 4, w)
    assert dx.shape == (0, 4, 4, 12) and not dw.any() and db is None and da is None
