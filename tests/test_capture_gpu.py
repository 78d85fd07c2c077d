"""Operators replayed from captured graphs: several times, with eager work and new inputs in between, every replay against the
eager result.  Sums that atomics add in fp64 may differ in the order of addition: by less than 2^-45, which the rounding of such a sum to
fp32 makes one step, 2^-23 of it; it then enters a result at most at the size of the largest one, with a factor of at most 2."""
import pytest
import torch

import unet_amd
from unet_amd import _lib, ops
from unet_amd.metrics import confusion_counts

pytestmark = pytest.mark.gpu


def replay(dev, inputs, step):
    """``inputs`` change in place; ``step`` returns tensors."""
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        with torch.no_grad():
            for t in inputs:
                t.copy_(t.roll(1, 0) if n % 2 else t.flip(0))
                if t.is_floating_point():
                    t.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.isfinite(a.double()).all()
            assert ((a.double() - b.double()).abs() <= 2.0 ** -22 * b.double().abs().max()).all()


@pytest.mark.parametrize("ce", [0.0, 1.0])
def test_segmentation_loss_replays(dev, ce):
    g = torch.Generator().manual_seed(1)
    z = torch.randn(3, 1, 37, 41, generator=g).to(dev).requires_grad_(True)
    t = (torch.rand(3, 1, 37, 41, generator=g) > 0.6).to(torch.uint8).to(dev)
    fn = unet_amd.DiceCELoss(sigmoid=True, lambda_ce=ce)

    def step():
        out = fn(z, t)
        return out.detach(), torch.autograd.grad(out, z)[0]

    replay(dev, [z], step)


def test_loss_without_allocation_replays(dev):
    g = torch.Generator().manual_seed(2)
    z = torch.randn(5, 1, 33, 20, generator=g).to(dev)
    t = (torch.rand(5, 1, 33, 20, generator=g) > 0.6).float().to(dev)
    lib = _lib.load()

    def step():
        loss = torch.zeros(1, device=dev)
        _lib.check(lib.mi_dice_ce_loss_fwd_noalloc(z.data_ptr(), t.data_ptr(), 0, 0, 5, 660, 1e-5, 1e-5, 1.0, 1.0, loss.data_ptr(), 0,
                                                   _lib.current_stream(dev)), "mi_dice_ce_loss_fwd_noalloc")
        return (loss,)

    replay(dev, [z], step)


def test_confusion_counts_replay(dev):
    g = torch.Generator().manual_seed(3)
    p = torch.randn(4, 1, 50, 30, generator=g).to(dev)
    t = (torch.rand(4, 1, 50, 30, generator=g) > 0.5).to(dev).float()
    replay(dev, [p], lambda: (confusion_counts(p, t, binary=False, threshold=0.0),))


def test_instance_norm_backward_replays(dev):
    g = torch.Generator().manual_seed(4)
    nb, c, side = 2, 16, 200                               # more than the one-launch form takes
    raw = torch.randn(nb, side, side, c, generator=g).to(dev)
    dy = torch.randn(nb, side, side, c, generator=g).to(dev)
    alpha = torch.full((1,), 0.25, device=dev)
    x = raw.double().reshape(nb, -1, c)
    stats = torch.zeros(nb, 8, c, 2, dtype=torch.float64, device=dev)
    stats[:, 0] = torch.stack([x.sum(1), x.square().sum(1)], -1)

    replay(dev, [dy], lambda: ops.instnorm_prelu_bwd(dy, raw, stats, alpha)[:1])


def test_passes_over_the_network_are_refused_under_capture(dev):
    """Nothing of a refused step stays behind: the next eager step leaves the parameters where it leaves them without the attempt."""
    x = torch.rand(2, 1, 32, 32, device=dev)
    t = (torch.rand(2, 1, 32, 32, device=dev) > 0.6).float()

    def make():
        torch.manual_seed(11)
        m = unet_amd.UNet(2, 1, 1, (16, 32), (2,), num_res_units=2, dropout=0.1, compute_dtype=torch.float32).to(dev).train()
        return m, unet_amd.Trainer(m, unet_amd.DiceCELoss(sigmoid=True), unet_amd.AdamW(m.parameters(), lr=1e-3, model=m))

    (m0, tr0), (m1, tr1) = make(), make()
    for tr in (tr0, tr1):
        tr.step(x, t)
    torch.cuda.synchronize()
    plan, flat = m1._plan_for(x, True), m1._ensure_flat(dev)
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=dev)
    y, g = torch.empty_like(x), torch.zeros_like(flat)
    for attempt in (lambda: tr1.step(x, t), lambda: m1(x), lambda: plan.forward(flat, x, y, ws, True, 3), lambda: plan.backward(flat, x, y, g, ws, True, 3)):
        scratch = torch.ones(8, device=dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scratch.zero_()
            with pytest.raises(RuntimeError, match="captured"):
                attempt()
    for m, tr in ((m0, tr0), (m1, tr1)):
        tr.step(x, t)
    torch.cuda.synchronize()
    assert torch.equal(m0.flat_parameters(), m1.flat_parameters())
