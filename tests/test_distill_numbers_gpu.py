"""The distillation loss where it is easily wrong without a word: NaN and infinities in the teacher's lists, tangents, and what is kept
between forward and backward."""
import math
import threading

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
