"""The distillation loss where it is easily wrong without a word: NaN and infinities in the teacher's lists, tangents, what is kept
between forward and backward, temperatures at which its terms cancel."""
import math
import threading

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import unet_amd
from unet_amd import ops

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---- NaN and +inf in the teacher --------------------------------------------------------------------------------------
@pytest.mark.parametrize("t_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("v,k", [(2, 1), (16, 4), (16, 2), (40, 40), (133, 5), (64, 16), (1000, 60), (600, 200), (4000, 6), (4000, 100), (4000, 256), (140000, 8)])
def test_nan_and_inf_of_the_teacher_reach_the_loss(dev, mode, v, k, t_dtype):
    """softmax over a list with a NaN or a +inf is NaN in every slot: so are the row's loss and its gradient at the listed classes,
    wherever in the list the value stands, and no other row's."""
    g = torch.Generator().manual_seed(v + k)
    bad = [(n, value) for n in sorted({0, k // 2, k - 1}) for value in (math.nan, math.inf)]
    rows = 2 * len(bad) + 3
    z = torch.randn(rows, v, generator=g).to(DT[mode]).to(dev)
    t = torch.randn(rows, k, generator=g)
    i = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(rows)])
    if k > 2:
        i[:, 1] = torch.where(torch.arange(rows) % 2 == 0, i[:, 1], torch.tensor(-1))        # an unused slot in every second row
    where = []
    for n, (slot, value) in enumerate(bad):
        row = 2 * n + 1
        t[row, slot] = value
        if int(i[row, slot]) >= 0:
            where.append(row)
    t[rows - 1] = math.nan                                 # and a list of nothing else
    where.append(rows - 1)
    spoilt = torch.zeros(rows, dtype=torch.bool)
    spoilt[where] = True
    t, i = t.to(t_dtype).to(dev), i.to(dev)
    z.requires_grad_(True)
    each = unet_amd.TopLogitDistillationLoss(2.0, "none")
    with torch.no_grad():
        assert torch.equal(torch.isnan(each(z, t, i)).cpu(), spoilt)
    out = each(z, t, i)
    assert torch.equal(torch.isnan(out).cpu(), spoilt) and torch.isfinite(out[~spoilt.to(dev)]).all()
    (dz,) = torch.autograd.grad(out, z, torch.ones_like(out))
    listed = torch.zeros(rows, v + 1, dtype=torch.bool, device=dev).scatter_(1, torch.where(i < 0, v, i), True)[:, :v]
    assert torch.equal(torch.isnan(dz), listed & spoilt.to(dev)[:, None])
    for reduction in ("mean", "sum"):
        fn = unet_amd.TopLogitDistillationLoss(2.0, reduction)
        out = fn(z, t, i)
        assert torch.isnan(out)
        (dz,) = torch.autograd.grad(out, z)
        assert torch.equal(torch.isnan(dz), listed & spoilt.to(dev)[:, None])
        keep = torch.where(spoilt.to(dev)[:, None], torch.full_like(i, -1), i)               # the rows left out
        assert torch.isfinite(fn(z, t, keep))


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("v,k", [(16, 4), (300, 16), (5000, 8)])
def test_a_teacher_pixel_of_nan_reaches_the_loss_through_its_top_logits(dev, mode, v, k):
    g = torch.Generator().manual_seed(v)
    teacher = torch.randn(6, v, generator=g).to(DT[mode]).to(dev)
    z = torch.randn(6, v, generator=g).to(DT[mode]).to(dev)
    teacher[2, v // 3] = math.nan
    t, i = ops.top_logits(teacher, k)
    assert torch.isnan(t[2, 0])
    out = unet_amd.TopLogitDistillationLoss(2.0, "none")(z, t, i)
    assert torch.isnan(out).tolist() == [False, False, True, False, False, False]


@pytest.mark.parametrize("rows,v", [(5, 16), (5, 5000)])
def test_forward_mode_tangents_are_refused(dev, rows, v):
    """A tangent that the loss cannot carry on must not vanish without a word."""
    z = torch.randn(rows, v, device=dev)
    t, i = torch.randn(rows, 3, device=dev), torch.zeros(rows, 3, dtype=torch.int32, device=dev)
    fn = unet_amd.TopLogitDistillationLoss()
    with forward_ad.dual_level():
        plain = fn(z, t, i)                                # no tangent: nothing to refuse
        dual = forward_ad.make_dual(z, torch.ones_like(z))
        with pytest.raises(RuntimeError):
            fn(dual, t, i)
        with torch.no_grad(), pytest.raises(RuntimeError):
            fn(dual, t, i)
    assert torch.equal(plain, fn(z, t, i))


# ---- the gradient that the forward call of long rows leaves behind -----------------------------------------------------
# Written by the forward call or computed again, a gradient scale (p - q) is off by (V / 256 + 64 + 8 |x|) u of scale p, at a listed class also by
# (2 k + 32 + 8 |y|) u of scale q, u = 2^-24 (sums, exponents, weights); with V <= 9000, k = 5 and |x|, |y| <= 8: 163 u and 106 u.  Twice that between two.
def close(a, b, scale):
    return ((a - b).abs() <= 2 * 163 * 2.0 ** -24 * b.abs() + 2 * (163 + 106) * 2.0 ** -24 * scale).all()


def test_saved_tensor_hooks_see_all_that_a_training_step_keeps(dev):
    rows, v = 300, 9000
    g = torch.Generator().manual_seed(1)
    z = torch.randn(rows, v, generator=g).to(dev).requires_grad_(True)
    t, i = torch.randn(rows, 5, generator=g).to(dev), torch.randint(0, v, (rows, 5), generator=g).to(dev)
    fn = unet_amd.TopLogitDistillationLoss(2.0)
    (want,) = torch.autograd.grad(fn(z, t, i), z)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(dev)
    with torch.autograd.graph.save_on_cpu():
        out = fn(z, t, i)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated(dev) - before < z.numel()              # bytes: a quarter of the gradient
    (dz,) = torch.autograd.grad(out, z, retain_graph=True)
    (again,) = torch.autograd.grad(out, z, torch.full((), 3.0, device=dev))
    assert torch.equal(dz, want)
    assert close(again, 3.0 * want, 3.0 * 2.0 / rows)


def test_threads_share_a_retained_graph(dev):
    """Every backward call gets a tensor of its own, also when several threads run them at once and change what they get."""
    rows, v = 64, 5000
    g = torch.Generator().manual_seed(2)
    z = torch.randn(rows, v, generator=g).to(dev).requires_grad_(True)
    t, i = torch.randn(rows, 5, generator=g).to(dev), torch.randint(0, v, (rows, 5), generator=g).to(dev)
    fn = unet_amd.TopLogitDistillationLoss(2.0)
    for _ in range(10):
        out = fn(z, t, i)
        got, start = [], threading.Barrier(4)

        def run():
            start.wait()
            (dz,) = torch.autograd.grad(out, z, retain_graph=True)
            got.append(dz)

        threads = [threading.Thread(target=run) for _ in range(4)]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
        torch.cuda.synchronize()
        assert len(got) == 4 and len({d.data_ptr() for d in got}) == 4
        assert all(close(d, got[0], 2.0 / rows) for d in got)
    (first,) = torch.autograd.grad(out, z, retain_graph=True)
    kept = first.clone()
    first.zero_()                                          # the caller's own
    (second,) = torch.autograd.grad(out, z)
    assert torch.equal(second, kept)


def test_gradients_accumulate_over_a_retained_graph(dev):
    z = torch.randn(40, 5000, device=dev, requires_grad=True)
    t, i = torch.randn(40, 5, device=dev), torch.randint(0, 5000, (40, 5), device=dev)
    out = unet_amd.TopLogitDistillationLoss(2.0)(z, t, i)
    out.backward(retain_graph=True)
    once = z.grad.clone()
    out.backward(retain_graph=True)
    out.backward()
    assert close(z.grad, 3.0 * once, 3.0 * 2.0 / 40)


# ---- temperatures -----------------------------------------------------------------------------------------------------
# The definition in numpy's long double (2^-64: T^2 times the 64-bit one's own error passes the loss at T = 1e6), and a row's tolerance, u = 2^-24.
# x_j = log q_j - log p_j.  Short rows add q_j phi(x_j), phi(x) = x - 1 + exp(-x), and R = 1 - sum p_j.  An x is off by dx = (3 |a| + 3 |b| + 3 |a - b|) u / T
# + 2 |x| u (a, b: gaps of t and z to their maxima; differences, 1 / T, products) and, all alike, by d = (V / 64 + k + 16 + 2 ln V + mean |a| / T) u (sums, two
# logarithms), which enters as R d and d^2 / 2.  A weight q is off by eq = (k + 8 + 4 |a| / T) u relatively, a probability by ep = (V / 64 + 12 + 4 |b| / T) u.
# For |x| < 1/2 (up to dx) phi is a series: q (|x| dx + phi (eq + 16 u)); beyond, q dx + (q (|x| + 1) + p) (eq + ep + 16 u).
# R: fp64 sums above T = 4, R (16 + 4 max |b| / T) u; below, sums of fp32 are off by at most 32 u (and so is what they set to zero).
# Long rows: T^2 u (V / 256 + 2 k + 64 + 8 (1 + M)^2), M the largest |a| or |b| over T of a listed class.
U = 2.0 ** -24


def rows_in_long_double(z, t, i, temperature, short):
    L = np.longdouble
    T = L(np.float32(temperature))
    z, t, i = z.float().cpu().numpy().astype(L), t.float().cpu().numpy().astype(L), i.cpu().numpy()
    loss, tol = [], []
    v, k = z.shape[1], t.shape[1]
    for zr, tr, ir in zip(z, t, i):
        used = (ir >= 0) & (ir < v) & (tr > -np.inf)
        tr, ir = tr[used], ir[used]
        b, a = zr - zr.max(), tr - tr.max()
        with np.errstate(all="ignore"):
            lp, lq = b / T - np.log(np.exp(b / T).sum()), a / T - np.log(np.exp(a / T).sum())
            p, q, bl = np.exp(lp), np.exp(lq), b[ir]
            x = np.where(q > 0, lq - lp[ir], 0)
            pj = p[ir]
            loss.append(T * T * np.where(q > 0, q * x, 0).sum())
            A, B = np.abs(a) / T, np.where(np.isfinite(bl), np.abs(bl), 0) / T
            if not short:
                M = max(np.where(q > 1e-30, np.maximum(A, B), 0).max(), 0)
                tol.append(T * T * U * (v / 256 + 2 * k + 64 + 8 * (1 + M) ** 2))
                continue
            dx = (3 * A + 3 * B + 3 * np.where(np.isfinite(bl), np.abs(a - bl), 0) / T) * U + 2 * np.abs(x) * U
            d = (v / 64 + k + 16 + 2 * np.log(L(v)) + (q * A).sum()) * U
            eq, ep = (k + 8 + 4 * A) * U, (v / 64 + 12 + 4 * B) * U
            phi = x - 1 + np.exp(-x)
            near = q * (np.abs(x) * dx + dx * dx + np.abs(phi) * (eq + 16 * U))
            far = q * dx + (q * (np.abs(x) + 1) + pj) * (eq + ep + 16 * U)
            e = np.where(np.abs(x) < 0.5 - dx, near, np.where(np.abs(x) > 0.5 + dx, far, np.maximum(near, far))).sum()
            R = abs(1 - pj.sum())
            most = np.where(p > 0, np.abs(np.where(p > 0, b, 0)), 0).max() / T
            e += R * d + (R * (16 + 4 * most) * U if temperature > 4 else 32 * U) + (64 * U * d if temperature > 4 else d * d)
            tol.append(T * T * e + 8 * U * abs(loss[-1]))
    return np.array(loss, dtype=np.float64), np.array(tol, dtype=np.float64)


def check_rows(z, t, i, temperature, short):
    want, tol = rows_in_long_double(z, t, i, temperature, short)
    got = unet_amd.TopLogitDistillationLoss(temperature, "none")(z, t, i).double().cpu().numpy()
    err = np.abs(got - want)
    assert (err <= tol + 1e-37).all(), (temperature, float((err / (tol + 1e-37)).max()), float(got[(err / (tol + 1e-37)).argmax()]), float(want[(err / (tol + 1e-37)).argmax()]))
    return got, want, tol


@pytest.mark.parametrize("temperature", [0.5, 1.0, 4.0, 4.5, 20.0, 100.0, 1e3, 1e4, 1e6])
@pytest.mark.parametrize("v,k", [(1, 1), (2, 2), (5, 2), (16, 16), (16, 4), (40, 40), (133, 100), (256, 256), (300, 256), (600, 20), (1000, 200)])
def test_short_rows_keep_their_digits_at_any_temperature(dev, v, k, temperature):
    g = torch.Generator().manual_seed(v + k)
    for spread in (2.0, 20.0):
        z = torch.randn(24, v, generator=g) * spread
        i = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(24)])
        t = z.gather(1, i) + 0.5 * torch.randn(24, k, generator=g)
        t[::6] = z.gather(1, i)[::6]                       # a student that agrees
        for zt in (torch.float32, torch.bfloat16):
            got, want, tol = check_rows(z.to(zt).to(dev), t.to(dev), i.to(dev), temperature, True)
            assert (got >= -tol).all()                     # no class twice: a divergence


@pytest.mark.parametrize("temperature", [1.0, 20.0, 1e3])
@pytest.mark.parametrize("v,k", [(16, 16), (64, 64), (900, 10)])
def test_what_a_short_list_cancels(dev, v, k, temperature):
    """The figure in words: the loss of lists that hold all the mass, 0.02 to 0.3 here, is good to 2^-14 of itself."""
    g = torch.Generator().manual_seed(v)
    i = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(64)])
    z = torch.randn(64, v, generator=g)
    z = torch.full_like(z, -math.inf).scatter_(1, i, z.gather(1, i))                       # classes that are not listed are masked
    t = z.gather(1, i) + 0.5 * torch.randn(64, k, generator=g)
    got, want, tol = check_rows(z.to(dev), t.to(dev), i.to(dev), temperature, True)
    big = want > 0.02
    assert big.sum() > 32 and (np.abs(got - want)[big] <= 2.0 ** -14 * want[big]).all()


@pytest.mark.parametrize("temperature", [0.5, 2.0, 50.0])
@pytest.mark.parametrize("v,k", [(16, 20), (3, 200), (400, 64)])
def test_short_lists_with_repeats_and_unused_slots(dev, v, k, temperature):
    g = torch.Generator().manual_seed(v)
    z = torch.randn(30, v, generator=g) * 3
    i = torch.randint(-1, v + 1, (30, k), generator=g)
    i[:, 0] = 0
    t = torch.randn(30, k, generator=g) * 3
    check_rows(z.to(dev), t.to(dev), i.to(dev), temperature, True)


@pytest.mark.parametrize("temperature", [0.5, 20.0, 1e3])
@pytest.mark.parametrize("v,k", [(3000, 5), (5000, 256), (40000, 40)])
def test_long_rows_at_high_temperatures(dev, v, k, temperature):
    g = torch.Generator().manual_seed(v)
    z = torch.randn(7, v, generator=g) * 3
    i = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(7)])
    t = z.gather(1, i) + 0.5 * torch.randn(7, k, generator=g)
    for zt in (torch.float32, torch.bfloat16):
        check_rows(z.to(zt).to(dev), t.to(dev), i.to(dev), temperature, False)


@pytest.mark.parametrize("temperature", [0.01, 0.5, 1.0])
@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("v,k", [(16, 4), (300, 70), (5000, 4), (5000, 100)])
def test_listed_classes_masked_with_the_lowest_value(dev, mode, v, k, temperature):
    """Temperatures below 1 make the gap to such a class larger than fp32 holds; the loss, T times q times the gap, is not."""
    g = torch.Generator().manual_seed(v + k)
    z = torch.randn(6, v, generator=g) * 2
    i = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(6)])
    t = torch.randn(6, k, generator=g) * temperature
    for row, slot in ((0, 0), (1, k // 2), (2, k - 1)):
        z[row, i[row, slot]] = torch.finfo(DT[mode]).min
    z = z.to(DT[mode]).to(dev)
    for reduction in ("none", "sum"):
        fn = unet_amd.TopLogitDistillationLoss(temperature, reduction)
        leaf = z.clone().requires_grad_(True)
        out = fn(leaf, t.to(dev), i.to(dev))
        assert torch.isfinite(out).all()
        (dz,) = torch.autograd.grad(out.sum(), leaf)
        assert torch.isfinite(dz).all()
    got, want, tol = check_rows(z, t.to(dev), i.to(dev), temperature, v <= 1024)
    assert (want[:3] > 1e33).all()


def test_checkpointed_step_gives_the_gradient_of_the_plain_one(dev):
    from torch.utils.checkpoint import checkpoint

    g = torch.Generator().manual_seed(3)
    fn = unet_amd.TopLogitDistillationLoss(2.0)
    for v in (40, 5000):
        x = torch.randn(30, v, generator=g).to(dev).requires_grad_(True)
        t, i = torch.randn(30, 5, generator=g).to(dev), torch.randint(0, v, (30, 5), generator=g).to(dev)
        (want,) = torch.autograd.grad(fn(x * 1.5, t, i), x)
        (got,) = torch.autograd.grad(checkpoint(lambda a: fn(a * 1.5, t, i), x, use_reentrant=False), x)
        assert torch.equal(got, want)
