"""Top logits of a teacher and the distillation loss on them, against the definitions in 64 bits.

Tolerances (derived before the first run), u = 2^-24.  The sum of exponentials: a thread adds at most V / 256 + 32 terms, the
lanes and waves join in 10 more steps, each rounding by u; an exponent x = (z - max) / T is off by 3 u |x| (difference,
factor, base change), which moves its term by as much relatively; exp2 and log2 are good to one unit.  So, relative to p:
ep = (V / 256 + 64 + 8 |x|) u, and to q: eq = (2 k + 32 + 8 |y|) u with y = (t - max t) / T.  A row's loss is T^2 times sums of
q (|x| + |y|), log Sz and log Sq: T^2 u (V / 256 + 2 k + 64 + 8 (1 + M)^2), M the largest |x| or |y| of a listed class.  Gradients:
|scale| (p ep + q eq) plus half a step of the type.
"""
import math

import pytest
import torch

import unet_amd
from unet_amd import ops

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
HALF_STEP = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8}
U = 2.0 ** -24


# ---- top logits -------------------------------------------------------------------------------------------------------
def sorted_lists(x, k):
    """Largest first, NaN in front, equal values by ascending index: Python's own stable order."""
    x = x.cpu().double()
    if x.numel() > 200000:                                 # torch's stable order on the CPU, NaN largest
        return x.sort(dim=-1, descending=True, stable=True).indices[:, :k].int()
    key = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x)
    nan = torch.isnan(x)
    out = []
    for row, isnan in zip(key.tolist(), nan.tolist()):
        order = sorted(range(len(row)), key=lambda i: (not isnan[i], -row[i], i))
        out.append(order[:k])
    return torch.tensor(out, dtype=torch.int32)


def check_top(x, k):
    values, index = ops.top_logits(x, k)
    want = sorted_lists(x.reshape(-1, x.shape[-1]), k).reshape(index.shape)
    assert index.dtype == torch.int32 and values.dtype == x.dtype and values.shape == x.shape[:-1] + (k,)
    assert torch.equal(index.cpu(), want)
    picked = x.cpu().gather(-1, want.long())
    assert torch.equal(values.cpu().float().nan_to_num(7e30), picked.float().nan_to_num(7e30))


TOP = [(1, 1, 1), (7, 2, 2), (300, 3, 2), (300, 16, 4), (65, 16, 16), (130, 21, 5), (33, 64, 64), (40, 133, 8), (9, 255, 255), (5, 256, 256),
       (17, 257, 17), (6, 512, 16), (6, 513, 40), (5, 1024, 100), (5, 1025, 16), (5, 1025, 200), (4, 2048, 16), (4, 2049, 3), (3, 5000, 256), (2, 50001, 32),
       (1, 128000, 64), (1, 4097, 1), (600, 2100, 20), (520, 4200, 100), (513, 20000, 70), (513, 40000, 200), (3, 70000, 256), (2, 140000, 256), (2, 2049, 256), (300, 176, 17), (40, 700, 130), (5, 2100, 24), (5, 2100, 200), (5, 4200, 60),
       (5, 9000, 42), (9, 1025, 85), (600, 1025, 85), (9, 1030, 86), (7, 1999, 64), (12, 517, 33), (600, 1025, 1), (520, 10241, 9), (520, 20500, 171),
       (520, 100001, 5), (300, 150, 9), (300, 23, 9), (70, 600, 33), (70, 1100, 33), (70, 1100, 20), (66000, 130, 40)]


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("case", TOP, ids=lambda c: "x".join(map(str, c)))
def test_top_logits(dev, mode, case):
    rows, v, k = case
    g = torch.Generator().manual_seed(rows * v + k)
    check_top((torch.randn(rows, v, generator=g) * 2).to(DT[mode]).to(dev), k)
    # few different values: nearly everything is a tie
    check_top(torch.randint(-2, 3, (rows, v), generator=g).to(DT[mode]).to(dev), k)
    check_top(torch.zeros(min(rows, 2), v, dtype=DT[mode], device=dev), k)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("k", range(1, 17))
def test_top_logits_of_every_pattern(dev, mode, k):
    """All rows of 16 zeros and ones: a network of exchanges that orders these orders everything."""
    n = torch.arange(1 << 16)
    bits = ((n[:, None] >> torch.arange(16)) & 1).to(DT[mode]).to(dev)
    check_top(bits, k)
    g = torch.Generator().manual_seed(k)
    for v in (9, 23, 70, 300, 1100):
        x = torch.rand(400, v, generator=g).argsort(-1).to(DT[mode]).to(dev)            # bf16: ties above 256
        check_top(x, min(k, v))


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("v", [17, 31, 32, 33, 64, 65, 100, 128, 129, 200, 255, 256, 300, 511, 512])
def test_top_logits_of_whole_rows(dev, mode, v):
    """Lists up to the whole row: orders, reversed orders, steps at every class, ties and special values."""
    g = torch.Generator().manual_seed(v)
    up = torch.arange(v, dtype=torch.float32)
    steps = (up[:, None] >= up[None, :]).float()
    x = torch.cat([torch.rand(300, v, generator=g).argsort(-1).float() - 100, up[None], -up[None], steps, 1 - steps, torch.randn(100, v, generator=g),
                   torch.randint(0, 3, (100, v), generator=g).float()])
    x[0, v // 2], x[1, 3], x[2, ::2], x[3, 1::2] = math.nan, -math.nan, -math.inf, math.inf
    x[4] = torch.where(torch.arange(v) % 2 == 0, torch.tensor(0.0), torch.tensor(-0.0))
    x = x.to(DT[mode]).to(dev)
    for k in sorted({min(k, v, 256) for k in (5, 9, 12, 33, 100, v // 2, v - 1, v)}):
        check_top(x, k)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("v,k", [(16, 4), (300, 16), (2100, 24), (9000, 5)])
def test_top_logits_of_special_values(dev, mode, v, k):
    g = torch.Generator().manual_seed(v)
    x = torch.randn(6, v, generator=g)
    x[0, ::3] = -math.inf
    x[1] = -math.inf
    x[2, v // 2:] = math.inf
    x[3, 5], x[3, v - 1] = math.nan, -math.nan
    x[4] = torch.where(torch.arange(v) % 2 == 0, torch.tensor(0.0), torch.tensor(-0.0))
    x[5] = torch.finfo(DT[mode]).min
    x = x.to(DT[mode]).to(dev)
    check_top(x, k)
    values, _ = ops.top_logits(x, k)
    assert torch.equal(torch.signbit(values[4]).cpu(), torch.arange(k) % 2 == 1)      # the values themselves are kept


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_top_logits_of_views(dev, mode):
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(2, 5, 7, 40, generator=g).to(DT[mode]).to(dev)
    for lo, hi in ((0, 33), (1, 22), (3, 40)):
        check_top(wide[..., lo:hi], 6)
    check_top(wide.permute(0, 3, 1, 2), 3)
    check_top(wide[:, 1:4], 3)
    check_top(wide[0, 0, 0], 5)
    check_top(wide[0, 0, :1].expand(7, 40), 5)
    v, i = ops.top_logits(wide[:0], 3)
    assert v.shape == (0, 5, 7, 3) and i.shape == (0, 5, 7, 3)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_top_logits_of_long_views(dev, mode):
    """Rows that begin at any element, with the largest classes first and last."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(5, 9007, generator=g)
    for lo, hi in ((0, 9007), (1, 9007), (1, 9001), (2, 9007), (3, 1030), (1, 2050), (5, 8199)):
        x = wide.clone()
        x[:, lo], x[:, hi - 1] = 9.0, 9.0
        check_top(x.to(DT[mode]).to(dev)[:, lo:hi], 20)


def test_top_logits_refusals(dev):
    x = torch.randn(4, 10, device=dev)
    for bad in (lambda: ops.top_logits(x, 0), lambda: ops.top_logits(x, 11), lambda: ops.top_logits(x.half(), 2), lambda: ops.top_logits(x.long(), 2),
                lambda: ops.top_logits(torch.randn(1, 300, device=dev), 257), lambda: ops.top_logits(x[:, :0], 1)):
        with pytest.raises(ValueError):
            bad()


# ---- the loss ---------------------------------------------------------------------------------------------------------
def definition(z, t, i, temperature, reduction, gout):
    """64 bits on the CPU: loss, gradient and their tolerances without the storage type's rounding."""
    z, t, i = z.detach().double().cpu(), t.double().cpu(), i.long().cpu()
    v, k = z.shape[-1], i.shape[-1]
    shape = i.shape[:-1]
    z, t, i = z.reshape(-1, v), t.reshape(-1, k), i.reshape(-1, k)
    used = (i >= 0) & (i < v) & (t > -math.inf)
    some = used.any(-1)
    ts = (t / temperature).masked_fill(~used, -math.inf)
    y = ts - ts.max(-1, keepdim=True).values
    logq = torch.where(some[:, None], ts, torch.zeros_like(ts)).log_softmax(-1).masked_fill(~used, -math.inf)
    q = logq.exp()
    x = z / temperature
    x = x - x.max(-1, keepdim=True).values
    logp = (z / temperature).log_softmax(-1)
    at = i.clamp(0, v - 1)
    part = torch.where(q > 0, q * (logq - logp.gather(1, at)), torch.zeros_like(q))
    row = part.sum(-1) * temperature ** 2
    count = max(1, int(some.sum()))
    scale = gout.double().cpu().reshape(-1, 1) * temperature / (count if reduction == "mean" else 1)
    p = logp.exp()
    target = torch.zeros_like(z).scatter_add_(1, at, q)
    dz = torch.where(some[:, None], (p - target) * scale, torch.zeros_like(z))
    y0 = torch.where(used & some[:, None], y, torch.zeros_like(y)).abs()
    x0 = torch.where(used, x.gather(1, at), torch.zeros_like(y)).abs()
    big = torch.where(q > 1e-30, torch.maximum(x0, y0), torch.zeros_like(y)).amax(-1)
    tol_row = temperature ** 2 * U * (v / 256 + 2 * k + 64 + 8 * (1 + big) ** 2)
    tol_row = torch.where(some, tol_row, torch.zeros_like(tol_row))
    eq = (2 * k + 32 + 8 * y0) * U * q
    tol_q = torch.zeros_like(z).scatter_add_(1, at, eq)
    xa = torch.where(p > 0, x, torch.zeros_like(x)).abs()
    tol_dz = scale.abs() * ((v / 256 + 64 + 8 * xa) * U * p + tol_q) + 4 * U * dz.abs()
    tol_dz = torch.where(some[:, None], tol_dz, torch.zeros_like(tol_dz))
    if reduction == "none":
        loss, tol = row.reshape(shape), tol_row.reshape(shape)
    else:
        n = count if reduction == "mean" else 1
        loss, tol = row.sum() / n, tol_row.sum() / n + 2 * U * row.sum().abs() / n
    full = tuple(shape) + (v,)
    return loss, tol, dz.reshape(full), tol_dz.reshape(full)


def check_loss(z, t, i, temperature, reduction, mode, one=False):
    z = z.detach().requires_grad_(True)
    fn = unet_amd.TopLogitDistillationLoss(temperature, reduction)
    with torch.no_grad():
        alone = fn(z, t, i)                                # without a gradient to come
    out = fn(z, t, i)
    g = torch.Generator().manual_seed(9)
    gout = torch.ones(out.shape) if one else torch.rand(out.shape, generator=g) + 0.5
    gout = gout.to(z.device)
    (dz,) = torch.autograd.grad(out, z, gout, retain_graph=True)
    first = dz.clone()
    (again,) = torch.autograd.grad(out, z, gout)           # a second backward call: the same numbers, another tensor
    assert torch.equal(first, dz) and again.data_ptr() != dz.data_ptr()
    loss, tol, ref, tol_dz = definition(z, t, i, temperature, reduction, gout)
    assert out.dtype == torch.float32 and out.shape == loss.shape and dz.shape == z.shape and dz.dtype == z.dtype
    err = (out.detach().double().cpu() - loss).abs()
    assert (err <= tol + 1e-37).all(), float((err / (tol + 1e-37)).max())
    bound = tol_dz * 1.01 + HALF_STEP[mode] * ref.abs() + 1e-37
    err = (dz.double().cpu() - ref).abs()
    assert (err <= bound).all(), float((err / bound).max())
    for other, limit in ((alone, tol + 1e-37),):
        assert ((other.double().cpu() - loss).abs() <= limit).all()
    assert ((again.double().cpu() - ref).abs() <= bound).all()
    return out.detach(), dz


def lists(rows, v, k, g, dev, t_dtype=torch.float32, i_dtype=torch.int32, ragged=True):
    i = torch.randint(0, v, (rows, k), generator=g)
    if ragged:
        used = torch.arange(k) < torch.randint(0, k + 1, (rows, 1), generator=g)
        used[rows // 2] = False
        if rows > 1:
            used[0] = True
        i = torch.where(used, i, torch.randint(0, 2, (rows, k), generator=g) * (v + 1) - 1)      # -1 or V
    t = (torch.randn(rows, k, generator=g) * 2).to(t_dtype)
    return t.to(dev), i.to(i_dtype).to(dev)


LOSS = [(1, 1, 1), (5, 2, 1), (64, 3, 3), (300, 16, 4), (257, 21, 5), (70, 16, 256), (700, 64, 16), (1000, 133, 8), (33, 512, 64), (17, 1024, 33),
        (17, 2048, 256), (9, 2049, 7), (9, 1023, 256), (5000, 7, 2), (3, 50001, 32), (1, 32001, 64), (4100, 2050, 3), (7, 8200, 12), (5, 16390, 9), (3, 33000, 4),
        (2, 70000, 8), (2, 131072, 5), (2, 131080, 5),
        (520, 9000, 4), (513, 34000, 3), (600, 29, 12), (2, 5, 1), (2050, 16, 1), (90, 2043, 2), (300, 1021, 17),
        (40, 1100, 16), (40, 600, 20), (130, 140, 7), (130, 75, 40), (40000, 140, 40), (140000, 68, 5), (530000, 5, 2)]


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("case", LOSS, ids=lambda c: "x".join(map(str, c)))
def test_loss_and_gradient(dev, mode, case):
    rows, v, k = case
    g = torch.Generator().manual_seed(rows + v + k)
    z = (torch.randn(rows, v, generator=g) * 3).to(DT[mode]).to(dev)
    for n, (reduction, temperature, td, idt) in enumerate((("mean", 1.0, torch.float32, torch.int32), ("sum", 2.0, torch.bfloat16, torch.int64),
                                                           ("none", 0.5, torch.float32, torch.int64))):
        t, i = lists(rows, v, k, g, dev, td, idt, ragged=rows > 1)
        check_loss(z, t, i, temperature, reduction, mode)
        check_loss(z, t, i, temperature, reduction, mode, one=True)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,v", [(513, 2600), (513, 4700), (513, 5900), (513, 7001), (513, 9003), (513, 11111), (513, 13001), (513, 19501), (513, 23502),
                                    (513, 28003), (513, 32775), (513, 39999), (513, 48001), (513, 56003), (514, 66001), (3, 45001), (3, 60007), (2, 90001), (2, 105003)])
def test_step_at_every_number_of_vectors(dev, mode, rows, v):
    """Few rows have a list: theirs is the loss, and the gradient of all others is exactly 0."""
    g = torch.Generator().manual_seed(v)
    gd = torch.Generator(device=dev).manual_seed(v)
    z = (torch.randn(rows, v, generator=gd, device=dev) * 3).to(DT[mode]).requires_grad_(True)
    some = sorted({0, 1, rows // 2, rows - 1})
    t, i = lists(rows, v, 7, g, torch.device("cpu"), ragged=False)
    i[:, 0], i[:, 1] = 0, v - 1                            # the first class and the last
    keep = torch.zeros(rows, 1, dtype=torch.bool)
    keep[some] = True
    i = torch.where(keep, i, torch.full_like(i, -1))
    t, i = t.to(dev), i.to(dev)
    out = unet_amd.TopLogitDistillationLoss(1.5, "mean")(z, t, i)
    (dz,) = torch.autograd.grad(out, z)
    loss, tol, ref, tol_dz = definition(z[some], t[some], i[some], 1.5, "mean", torch.ones(()))
    assert (out.detach().double().cpu() - loss).abs() <= tol
    bound = tol_dz * 1.01 + HALF_STEP[mode] * ref.abs() + 1e-37
    err = (dz[some].double().cpu() - ref).abs()
    assert (err <= bound).all(), float((err / bound).max())
    assert int((dz != 0).any(-1).sum()) == len(some) and not dz.isnan().any()


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_long_rows_at_any_offset(dev, mode):
    g = torch.Generator().manual_seed(8)
    wide = (torch.randn(6, 9001, generator=g) * 2).to(DT[mode]).to(dev)
    for lo, hi in ((0, 9001), (1, 9001), (1, 3000), (2, 2101), (3, 8201), (33, 2090), (63, 8999)):
        z = wide[:, lo:hi]
        t, i = lists(6, hi - lo, 5, g, dev)
        check_loss(z, t, i, 1.0, "mean", mode, one=True)
        check_loss(z, t, i, 2.0, "none", mode)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("v", [16, 300, 4000])
def test_masks_infinities_and_repeats(dev, mode, v):
    g = torch.Generator().manual_seed(v)
    low = torch.finfo(DT[mode]).min
    z = (torch.randn(12, v, generator=g) * 2)
    t, i = lists(12, v, 6, g, torch.device("cpu"), ragged=False)
    i = i.long()
    i[0] = 3                                              # one class in every slot
    i[1, 3:] = i[1, :3]                                   # every class twice
    i[2], i[3] = -1, torch.tensor([v, v + 1, -7, 2 ** 40, -2 ** 40, 2 ** 31])      # nothing used
    z[2, 1], z[3, 0] = math.nan, math.inf                 # and what the row holds does not matter
    t[4] = -math.inf                                      # weights of zero only: nothing used
    t[5, 2:] = -math.inf
    i[6, :] = torch.arange(6) % v
    t[6, 1] = low                                         # a weight that underflows
    keep = torch.zeros(v, dtype=torch.bool)
    keep[i[7].clamp(0, v - 1)] = True
    z[7, ~keep] = -math.inf                               # classes masked out of the student
    z[8, ~keep] = low
    i[8] = i[7]
    t[9, :] = low                                         # equal weights at the type's lowest value
    i[10, 1:] = -1
    z[11] = low
    z = z.to(DT[mode]).to(dev)
    if mode == "bf16":
        t = t.bfloat16()
    t, i = t.to(dev), i.to(dev)
    for reduction in ("mean", "sum", "none"):
        # row 11: equal logits at the type's lowest value are a uniform distribution
        out, dz = check_loss(z, t, i, 1.0, reduction, mode)
        check_loss(z, t, i, 1.0, reduction, mode, one=True)
        assert not dz[2].any() and not dz[3].any() and not dz[4].any()
        assert torch.isfinite(dz).all()
    assert not out[2:5].any()
    # a teacher's class that the student rules out: infinite loss, finite gradient
    z2 = z.clone()
    z2[10, int(i[10, 0])] = -math.inf
    z2.requires_grad_(True)
    out = unet_amd.TopLogitDistillationLoss(reduction="none")(z2, t, i)
    assert out[10] == math.inf and torch.isfinite(out[:10]).all()
    (dz,) = torch.autograd.grad(out.sum(), z2)
    assert torch.isfinite(dz).all() and dz[10, int(i[10, 0])] == -1
    # NaN and +inf in a row that counts reach its loss, and no other row
    z3 = z.clone()
    z3[5, v - 1], z3[6, 0] = math.nan, math.inf
    out3 = unet_amd.TopLogitDistillationLoss(reduction="none")(z3, t, i)
    assert torch.isnan(out3[5:7]).all() and torch.isfinite(out3[:5]).all() and torch.isfinite(out3[7:]).all()
    z3[7] = -math.inf
    assert torch.isnan(unet_amd.TopLogitDistillationLoss(reduction="none")(z3, t, i)[7])
    z3[7] = math.nan
    assert torch.isnan(unet_amd.TopLogitDistillationLoss(reduction="none")(z3, t, i)[7])


@pytest.mark.parametrize("i_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("t_dtype", [torch.float32, torch.bfloat16])
def test_lists_at_any_address(dev, t_dtype, i_dtype):
    """Full and ragged lists whose tensors begin at any element."""
    g = torch.Generator().manual_seed(12)
    for rows, v, k in ((130, 16, 4), (77, 40, 8), (65, 300, 32), (9, 600, 256)):
        z = (torch.randn(rows, v, generator=g) * 2).to(dev)
        t, i = lists(rows, v, k, g, dev, t_dtype, i_dtype)
        for off in (1, 2, 3):
            tt = torch.zeros(rows * k + off, dtype=t_dtype, device=dev)[off:].view(rows, k).copy_(t)
            ii = torch.zeros(rows * k + off, dtype=i_dtype, device=dev)[off:].view(rows, k).copy_(i)
            check_loss(z, tt, ii, 1.0, "mean", "fp32")


def test_nothing_to_learn_from(dev):
    for shape, v in (((6,), 16), ((2, 3, 4), 16), ((3,), 5000)):
        z = torch.randn(*shape, v, device=dev, requires_grad=True)
        t, i = torch.zeros(*shape, 3, device=dev), torch.full((*shape, 3), -1, dtype=torch.int32, device=dev)
        for reduction in ("mean", "sum", "none"):
            out = unet_amd.TopLogitDistillationLoss(2.0, reduction)(z, t, i)
            (dz,) = torch.autograd.grad(out.sum(), z)
            assert not out.any() and not dz.any()
    for reduction in ("mean", "sum", "none"):
        z = torch.randn(0, 4, 16, device=dev, requires_grad=True)
        out = unet_amd.TopLogitDistillationLoss(2.0, reduction)(z, torch.zeros(0, 4, 3, device=dev), torch.zeros(0, 4, 3, dtype=torch.int32, device=dev))
        (dz,) = torch.autograd.grad(out.sum(), z)
        assert dz.shape == z.shape and not out.any()


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_views_and_other_orders(dev, mode):
    g = torch.Generator().manual_seed(4)
    wide = (torch.randn(2, 5, 7, 40, generator=g) * 2).to(DT[mode]).to(dev)
    t, i = lists(70, 21, 4, g, dev)
    t, i = t.reshape(2, 5, 7, 4), i.reshape(2, 5, 7, 4)
    for lo in (0, 1, 2, 8, 19):
        check_loss(wide[..., lo:lo + 21], t, i, 1.5, "mean", mode)
    check_loss(wide[..., :21].permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1), t, i, 1.5, "mean", mode)
    ts, ist = t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0), i.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    check_loss(wide[..., :21], ts, ist, 1.5, "none", mode)
    long = (torch.randn(3, 5000, generator=g) * 2).to(DT[mode]).to(dev)
    t, i = lists(3, 4097, 9, g, dev)
    for lo in (0, 1, 3, 800):
        check_loss(long[:, lo:lo + 4097], t, i, 1.0, "sum", mode)
    check_loss(long[:1, :4097].expand(3, 4097), t, i, 1.0, "sum", mode)


def test_the_gradient_reaches_views_and_other_types(dev):
    g = torch.Generator().manual_seed(5)
    base = torch.randn(6, 30, generator=g).to(dev)
    t, i = lists(6, 21, 3, g, dev)
    fn = unet_amd.TopLogitDistillationLoss(2.0)
    for dt in (torch.float64, torch.float16):
        z = base.to(dt).requires_grad_(True)
        out = fn(z[:, 4:25], t.to(dt), i)
        (dz,) = torch.autograd.grad(out, z)
        zf = base.to(dt).float()[:, 4:25].contiguous().requires_grad_(True)
        (want,) = torch.autograd.grad(fn(zf, t.to(dt).float(), i), zf)
        assert dz.dtype == dt and not dz[:, :4].any() and not dz[:, 25:].any() and torch.equal(dz[:, 4:25], want.to(dt))


def test_gradient_against_differences(dev):
    g = torch.Generator().manual_seed(6)
    for v in (21, 2500):
        z = torch.randn(8, v, generator=g).to(dev)
        t, i = lists(8, v, 5, g, dev)
        fn = unet_amd.TopLogitDistillationLoss(1.5, "none")
        d = torch.randn(8, v, generator=g).to(dev)
        zr = z.clone().requires_grad_(True)
        (dz,) = torch.autograd.grad(fn(zr, t, i).sum(), zr)
        f = lambda s: fn(z + s * d, t, i).double()
        h = 2.0 ** -4
        d1, d2 = (f(h) - f(-h)) / (2 * h), (f(2 * h) - f(-2 * h)) / (4 * h)
        # fourth-order differences of a smooth function: h^4 / 30 of its fifth derivative (a cumulant of d, of order 10), rounding 1e-5 / h
        assert ((4 * d1 - d2) / 3 - (dz.double() * d.double()).sum(-1)).abs().max() < 1e-3


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("v", [48, 5000])
def test_weight_scales_loss_and_gradient(dev, mode, v):
    g = torch.Generator().manual_seed(v)
    z = (torch.randn(9, v, generator=g) * 2).to(DT[mode]).to(dev).requires_grad_(True)
    t, i = lists(9, v, 4, g, dev)
    for reduction in ("mean", "sum", "none"):
        one = unet_amd.TopLogitDistillationLoss(2.0, reduction)(z, t, i)
        half = unet_amd.TopLogitDistillationLoss(2.0, reduction, weight=-0.5)(z, t, i)
        assert torch.equal(half, -0.5 * one)               # a power of two: no rounding
        (d1,) = torch.autograd.grad(one.sum(), z)
        (d2,) = torch.autograd.grad(half.sum(), z)
        assert torch.equal(d2, -0.5 * d1)


def test_refusals(dev):
    z = torch.randn(4, 10, device=dev)
    t, i = torch.randn(4, 3, device=dev), torch.zeros(4, 3, dtype=torch.int32, device=dev)
    fn = unet_amd.TopLogitDistillationLoss()
    for bad in (lambda: fn(z[:3], t, i), lambda: fn(z, t[:, :2], i), lambda: fn(z, t, i.float()), lambda: fn(z, t, i.short()), lambda: fn(z.long(), t, i),
                lambda: fn(z, t.long(), i), lambda: fn(z, t.cpu(), i), lambda: fn(z, t, i.cpu()), lambda: fn(z, t[:, :0], i[:, :0]), lambda: fn(z[:, :0], t, i),
                lambda: fn(z, torch.randn(4, 257, device=dev), torch.zeros(4, 257, dtype=torch.int32, device=dev)), lambda: fn(z[0], t, i)):
        with pytest.raises(ValueError):
            bad()
    z.requires_grad_(True)
    (dz,) = torch.autograd.grad(fn(z, t, i), z, create_graph=True)
    with pytest.raises(RuntimeError):
        dz.sum().backward()


def test_results_repeat_bit_for_bit_also_on_another_stream(dev):
    g = torch.Generator().manual_seed(7)
    for rows, v, k in ((5000, 16, 4), (600, 3001, 20)):
        z = torch.randn(rows, v, generator=g).to(dev).requires_grad_(True)
        t, i = lists(rows, v, k, g, dev)
        i = (i % 5).int()                                  # many repeats
        fn = unet_amd.TopLogitDistillationLoss(2.0)

        def step():
            out = fn(z, t, i)
            return out.detach(), torch.autograd.grad(out, z)[0], *ops.top_logits(z.detach(), min(k, v))

        first = step()
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream(dev).wait_stream(side)
        for out in (step(), other):
            assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_captured_steps_replay(dev):
    g = torch.Generator().manual_seed(8)
    graphs = []
    fn = unet_amd.TopLogitDistillationLoss(2.0)
    for rows, v, k in ((700, 16, 4), (40, 3001, 20)):
        z = torch.randn(rows, v, generator=g).to(dev).requires_grad_(True)
        teacher = torch.randn(rows, v, generator=g).to(dev)

        def step(z=z, teacher=teacher, k=k):
            t, i = ops.top_logits(teacher, k)
            out = fn(z, t, i)
            return out.detach(), torch.autograd.grad(out, z)[0], t, i

        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream(dev).wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, z, teacher, out, step))
    for n in range(3):
        for gr, z, teacher, out, step in graphs:
            with torch.no_grad():
                z.mul_(0.9)
                teacher.copy_(teacher.roll(1, 0))
            gr.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_more_than_2_31_logits(dev):
    """Offsets beyond 32 bits: the last rows of 66000 x 32800 bf16 logits against calls on those rows alone."""
    rows, v, k = 66000, 32800, 3
    x = torch.empty(rows, v, dtype=torch.bfloat16, device=dev)
    x.normal_()
    g = torch.Generator().manual_seed(12)
    t, i = lists(rows, v, k, g, dev)
    i[-5:] = torch.tensor([v - 1, 0, 5], device=dev)
    values, index = ops.top_logits(x, k)
    last = slice(rows - 3, rows)
    v1, i1 = ops.top_logits(x[last].clone(), k)
    assert torch.equal(values[last], v1) and torch.equal(index[last], i1)
    del values, index
    fn = unet_amd.TopLogitDistillationLoss(2.0, "none")
    x.requires_grad_(True)
    out = fn(x, t, i)
    (dz,) = torch.autograd.grad(out, x, torch.ones_like(out))
    x1 = x[last].detach().clone().requires_grad_(True)
    o1 = fn(x1, t[last], i[last])
    (d1,) = torch.autograd.grad(o1, x1, torch.ones_like(o1))
    assert torch.allclose(out[last], o1, rtol=1e-5) and torch.allclose(dz[last].float(), d1.float(), rtol=2.0 ** -7, atol=1e-9)
    del dz, d1
    total = unet_amd.TopLogitDistillationLoss(2.0, "sum")
    (dz,) = torch.autograd.grad(total(x, t, i), x)
    (d1,) = torch.autograd.grad(total(x1, t[last], i[last]), x1)
    assert torch.allclose(dz[last].float(), d1.float(), rtol=2.0 ** -7, atol=1e-9)


# ---- together ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_a_student_step_out_of_the_operators(dev, mode):
    """Convolution -> group norm + SiLU -> 1x1 convolution -> distillation from a teacher's top logits, and back; compared
    with the same network differentiated in 64 bits on the CPU."""
    dt = DT[mode]
    g = torch.Generator().manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g)
    x = rnd(2, 12, 20, 16).to(dt).to(dev)
    w1, w2 = (rnd(32, 16, 3, 3) * 0.1), (rnd(48, 32, 1, 1) * 0.3)
    if mode == "bf16":
        w1, w2 = w1.bfloat16().float(), w2.bfloat16().float()
    gamma, beta = 1 + 0.2 * rnd(32), 0.2 * rnd(32)
    teacher = (rnd(2, 12, 20, 48) * 2).to(dev)
    t, i = ops.top_logits(teacher, 6)
    i[:, :, ::5] = -1                                      # pixels that nobody labelled

    c = ops.conv_forward(x, w1.to(dev))
    h, stats = ops.groupnorm_act_fwd(c, 8, gamma.to(dev), beta.to(dev))
    z = ops.conv_forward(h, w2.to(dev), ksize=1).requires_grad_(True)
    loss = unet_amd.TopLogitDistillationLoss(2.0)(z, t, i)
    (dz,) = torch.autograd.grad(loss, z)
    dw2, _ = ops.conv_wgrad(h, dz, tuple(w2.shape), ksize=1)
    dh = ops.conv_dgrad(dz, w2.to(dev), tuple(h.shape), ksize=1)
    dc, dgamma, dbeta, _ = ops.groupnorm_act_bwd(dh, c, stats, 8, gamma.to(dev), beta.to(dev))
    dw1, _ = ops.conv_wgrad(x, dc, tuple(w1.shape))

    F = torch.nn.functional
    leaf = [p.double().requires_grad_(True) for p in (w1, gamma, beta, w2)]
    a = F.conv2d(x.double().cpu().permute(0, 3, 1, 2), leaf[0], padding=1)
    a = F.silu(F.group_norm(a, 8, leaf[1], leaf[2]))
    zr = F.conv2d(a, leaf[3]).permute(0, 2, 3, 1)
    ir, used = i.long().cpu(), (i >= 0).cpu()
    q = (t.double().cpu() / 2).softmax(-1)
    rows = (q * (q.log() - (zr / 2).log_softmax(-1).gather(-1, ir.clamp(min=0)))).sum(-1) * 4
    ref = rows[used[..., 0]].mean()
    ref.backward()
    # storage rounding of the tensors between the operators: five of them, each half a step, plus fp32 sums
    tol = 2e-5 if mode == "fp32" else 5 * 2.0 ** -8
    assert abs(float(loss.detach()) - float(ref.detach())) < tol * float(ref.detach())
    for got, p in ((dw1, leaf[0]), (dgamma, leaf[1]), (dbeta, leaf[2]), (dw2, leaf[3])):
        err = (got.double().cpu() - p.grad).norm() / p.grad.norm()
        assert err < tol, float(err)
