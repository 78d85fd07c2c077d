"""``DiceLoss`` / ``DiceCELoss`` with MONAI's call surface (reference/train.py:88,116,142), computed by
single-pass HIP reductions: per-sample sums of sigmoid(z)*t, sigmoid(z), t and the BCE-with-logits
terms in one kernel, the gradient w.r.t. the logits in another.  ``TopLogitDistillationLoss`` trains a student on
the top logits of a teacher.
"""
from __future__ import annotations

import functools

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib
from .ops import _DT, _pixels


class _DiceCEFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, smooth_nr, smooth_dr, lambda_dice, lambda_ce, fold2):
        lib = _lib.load()
        nb = logits.shape[0]
        npix = logits[0].numel()
        dev = logits.device
        sums = torch.empty(nb * 4, dtype=torch.float64, device=dev)
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        st = _lib.current_stream(dev)
        _lib.check(lib.mi_dice_ce_loss_fwd(logits.data_ptr(), target.data_ptr(), _lib.label_dtype_code(target),
                                           1 if fold2 else 0, nb, npix, smooth_nr, smooth_dr, lambda_dice, lambda_ce,
                                           sums.data_ptr(), loss.data_ptr(), 0, st), "mi_dice_ce_loss_fwd")
        ctx.save_for_backward(logits, target, sums)
        ctx.cfg = (smooth_nr, smooth_dr, lambda_dice, lambda_ce, fold2)
        return loss.reshape(())

    @staticmethod
    def backward(ctx, gout):
        logits, target, sums = ctx.saved_tensors
        smooth_nr, smooth_dr, lambda_dice, lambda_ce, fold2 = ctx.cfg
        lib = _lib.load()
        nb = logits.shape[0]
        npix = logits[0].numel()
        dz = torch.empty_like(logits)
        g = gout.contiguous().float()
        _lib.check(lib.mi_dice_ce_loss_bwd(logits.data_ptr(), target.data_ptr(), _lib.label_dtype_code(target),
                                           1 if fold2 else 0, nb, npix, smooth_nr, smooth_dr, lambda_dice, lambda_ce,
                                           sums.data_ptr(), g.data_ptr(), 1.0, dz.data_ptr(),
                                           _lib.current_stream(logits.device)), "mi_dice_ce_loss_bwd")
        return dz, None, None, None, None, None, None


def _prepare(input: torch.Tensor, target: torch.Tensor):
    if input.dim() != target.dim():
        raise ValueError("the number of dimensions for input and target should be the same, "
                         f"got shape {input.shape} (nb dims: {len(input.shape)}) and {target.shape} "
                         f"(nb dims: {len(target.shape)}).")
    if target.shape != input.shape:
        raise AssertionError(f"ground truth has different shape ({target.shape}) from input ({input.shape})")
    if input.shape[1] != 1:
        raise NotImplementedError("unet_amd losses implement the one-channel sigmoid case (reference/train.py:88)")
    if not input.is_cuda:
        raise RuntimeError("unet_amd losses run on an AMD GPU only (no CPU or eager fallback)")
    x = input.as_subclass(torch.Tensor) if type(input) is not torch.Tensor else input
    t = target.as_subclass(torch.Tensor) if type(target) is not torch.Tensor else target
    x = x.contiguous()
    if x.dtype != torch.float32:
        x = x.float()
    t = t.contiguous()
    if _lib.label_dtype_code(t) < 0:
        t = t.float()
    return x, t


class DiceCELoss(nn.Module):
    """``monai.losses.DiceCELoss`` for one-channel logits: ``lambda_dice * Dice(sigmoid(x), t) +
    lambda_ce * BCEWithLogits(x, t)`` (MONAI >= 1.3 semantics).  ``lambda_ce=0`` gives the plain Dice loss.

    ``fold_label_two=True`` treats label value 2 as 1 inside the kernels, i.e. fuses
    ``labels[labels == 2] = 1`` (reference/train.py:112-113) into the loss read.
    """

    def __init__(self, include_background=True, to_onehot_y=False, sigmoid=False, softmax=False, other_act=None,
                 squared_pred=False, jaccard=False, reduction="mean", smooth_nr=1e-5, smooth_dr=1e-5, batch=False,
                 weight=None, lambda_dice=1.0, lambda_ce=1.0, fold_label_two=False):
        super().__init__()
        bad = []
        if not sigmoid: bad.append("sigmoid=True is required")
        if softmax or other_act is not None: bad.append("softmax / other_act")
        if to_onehot_y or squared_pred or jaccard or batch or weight is not None: bad.append("to_onehot_y / squared_pred / jaccard / batch / weight")
        if not include_background: bad.append("include_background=False")
        if reduction != "mean": bad.append("reduction must be 'mean'")
        if bad:
            raise NotImplementedError("unet_amd.DiceCELoss: unsupported options: " + "; ".join(bad))
        if lambda_dice < 0.0 or lambda_ce < 0.0:
            raise ValueError("lambda_dice and lambda_ce should be no less than 0.0.")
        self.smooth_nr, self.smooth_dr = float(smooth_nr), float(smooth_dr)
        self.lambda_dice, self.lambda_ce = float(lambda_dice), float(lambda_ce)
        self.fold_label_two = bool(fold_label_two)

    def forward(self, input: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        x, t = _prepare(input, target)
        return _DiceCEFunction.apply(x, t, self.smooth_nr, self.smooth_dr, self.lambda_dice, self.lambda_ce,
                                     self.fold_label_two)


class DiceLoss(DiceCELoss):
    """``monai.losses.DiceLoss(sigmoid=True)``: the Dice term alone."""

    def __init__(self, include_background=True, to_onehot_y=False, sigmoid=False, softmax=False, other_act=None,
                 squared_pred=False, jaccard=False, reduction="mean", smooth_nr=1e-5, smooth_dr=1e-5, batch=False,
                 fold_label_two=False):
        super().__init__(include_background=include_background, to_onehot_y=to_onehot_y, sigmoid=sigmoid,
                         softmax=softmax, other_act=other_act, squared_pred=squared_pred, jaccard=jaccard,
                         reduction=reduction, smooth_nr=smooth_nr, smooth_dr=smooth_dr, batch=batch,
                         lambda_dice=1.0, lambda_ce=0.0, fold_label_two=fold_label_two)


_REDUCTION = {"none": 0, "mean": 1, "sum": 2}
_INDEX = {torch.int64: 2, torch.int32: 3}


@functools.lru_cache(maxsize=256)
def _distill_sizes(dt, rows, v, k, red):
    lib = _lib.load()
    return lib.mi_distill_loss_saved_bytes(dt, rows, v, k), bool(lib.mi_distill_loss_step_ready(dt, rows, v, k, red))


def _distill_call(logits, teacher, index, temperature, weight, red, train):
    """The forward call: (loss, what the backward call reads, the gradient for an upstream gradient of 1 or None)."""
    lib, dev = _lib.load(), logits.device
    z, pitch = _pixels(logits, "input")
    v, k = z.shape[-1], index.shape[-1]
    rows = index.numel() // k
    dt = _DT[z.dtype]
    nbytes, in_one = _distill_sizes(dt, rows, v, k, red)
    loss = teacher.new_empty(index.shape[:-1] if red == 0 else (), dtype=torch.float32)
    saved = index.new_empty(nbytes, dtype=torch.uint8)
    args = (dt, rows, v, pitch, z.data_ptr(), k, _DT[teacher.dtype], teacher.data_ptr(), _INDEX[index.dtype],
            index.data_ptr(), temperature, weight, red, loss.data_ptr(), saved.data_ptr())
    with _lib.on_device(dev):
        if train and in_one:
            dz = z.new_empty(z.shape)
            _lib.check(lib.mi_distill_loss_step(*args, v, dz.data_ptr(), _lib.stream_of(dev)), "mi_distill_loss_step")
            return loss, saved, dz
        _lib.check(lib.mi_distill_loss_fwd(*args, _lib.stream_of(dev)), "mi_distill_loss_fwd")
    return loss, saved, None


def _distill_gradient(ctx, gout):
    logits, teacher, index, saved, dz = ctx.saved_tensors
    temperature, weight, red = ctx.cfg
    lib, dev = _lib.load(), logits.device
    z, pitch = _pixels(logits, "input")
    v, k = z.shape[-1], index.shape[-1]
    try:                                     # the first backward call gives it away (one of several threads: a list pops once)
        done = ctx.first.pop()
    except IndexError:
        done = False
    dz = dz.data if done else z.new_empty(z.shape)       # the receiver may change it in place: not the saved tensor itself
    g = gout if gout.dtype == torch.float32 and gout.is_contiguous() else gout.contiguous().float()
    with _lib.on_device(dev):
        _lib.check(lib.mi_distill_loss_bwd(_DT[z.dtype], index.numel() // k, v, pitch, z.data_ptr(), k, _DT[teacher.dtype], teacher.data_ptr(),
                                           _INDEX[index.dtype], index.data_ptr(), temperature, weight, red, g.data_ptr(), saved.data_ptr(),
                                           1 if done else 0, v, dz.data_ptr(), _lib.stream_of(dev)), "mi_distill_loss_bwd")
    return dz, None, None, None, None, None


_distill_gradient_once = torch.autograd.function.once_differentiable(_distill_gradient)


class _DistillFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, index, temperature, weight, red):
        loss, saved, dz = _distill_call(logits, teacher, index, temperature, weight, red, True)
        ctx.save_for_backward(logits, teacher, index, saved, dz)
        ctx.first = [True] if dz is not None else []
        ctx.cfg = (temperature, weight, red)
        return loss

    @staticmethod
    def backward(ctx, gout):
        # only a graph of the gradient itself (create_graph) needs the refusal of a second derivative
        return _distill_gradient_once(ctx, gout) if torch.is_grad_enabled() else _distill_gradient(ctx, gout)


class TopLogitDistillationLoss(nn.Module):
    """Trains a student on the top logits of a teacher (``ops.top_logits``):
    ``weight * temperature**2 * KL(q || softmax(input / temperature))`` per pixel, where ``q`` is the softmax of the pixel's listed
    teacher logits over ``temperature``.

    ``forward(input, teacher_logits, teacher_index)``: ``input`` [.., V] class logits of the student, channels last, fp32 or
    bf16 (other types are read as fp32); ``teacher_logits`` [.., k] (fp32, bf16; others are read as fp32) and ``teacher_index``
    [.., k] (int32 or int64), k at most 256.  A slot whose index lies outside [0, V), or whose logit is -inf, is unused: -1
    fills up short lists and leaves out pixels.  The weights of a class listed twice add.  ``reduction``: "mean" over the pixels with a used slot (0 if
    there are none), "sum", or "none" (one loss per pixel, 0 where no slot is used).  The gradient flows to ``input`` alone.

    The loss of a pixel is good to a few 2^-24 of its parts, none of which is negative where no class repeats, also where the list holds all that
    the student's distribution does (up to temperature 4: and to 2^-15 ``weight``; beyond 2048 bf16 or 1024 fp32 classes: and to ``(64 + classes / 256 + 2 k) 2^-24 weight
    temperature**2``).  The gradient is good to about 2^-20 of the two probabilities that it is the difference of.

    With more classes than 64 lanes hold (2048 bf16, 1024 fp32) the forward call of a training step writes the gradient along, for
    an upstream gradient of 1: ``backward`` then has nothing left to do, and computes it again for any other (give ``weight``
    instead of multiplying the loss).
    """

    def __init__(self, temperature=1.0, reduction="mean", weight=1.0):
        super().__init__()
        temperature, weight = float(temperature), float(weight)
        if not 1e-6 <= temperature <= 1e6:
            raise ValueError(f"temperature must be in 1e-6 .. 1e6, got {temperature}")
        if not abs(weight) < float("inf"):
            raise ValueError(f"weight must be finite, got {weight}")
        if not abs(weight) * max(1.0, temperature, temperature * temperature) <= 3.4e38:
            raise ValueError(f"weight * temperature**2 must be within fp32, got {weight} and {temperature}")
        if reduction not in _REDUCTION:
            raise ValueError(f"reduction must be one of {sorted(_REDUCTION)}, got {reduction!r}")
        self.temperature, self.reduction, self.weight = temperature, reduction, weight

    def forward(self, input: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor) -> torch.Tensor:
        x = input.as_subclass(torch.Tensor) if type(input) is not torch.Tensor else input
        t, i = teacher_logits, teacher_index
        if x.dim() < 1 or t.shape != i.shape or t.shape[:-1] != x.shape[:-1] or t.dim() != x.dim():
            raise ValueError(f"input [.., V] and the teacher's lists [.., k] must agree in front of the last dimension, got {tuple(x.shape)}, "
                             f"{tuple(t.shape)} and {tuple(i.shape)}")
        if x.shape[-1] < 1 or not 1 <= i.shape[-1] <= 256:
            raise ValueError(f"the lists must have 1 .. 256 slots and the input at least one class, got {i.shape[-1]} and {x.shape[-1]}")
        if i.dtype not in _INDEX:
            raise ValueError(f"teacher_index must be torch.int32 or torch.int64, got {i.dtype}")
        if not x.is_floating_point() or not t.is_floating_point():
            raise ValueError(f"input and teacher_logits must be floating point, got {x.dtype} and {t.dtype}")
        if not x.is_cuda:
            raise RuntimeError("unet_amd losses run on an AMD GPU only (no CPU or eager fallback)")
        if t.device != x.device or i.device != x.device:
            raise ValueError(f"the teacher's lists are on {t.device} and {i.device}, expected {x.device}")
        if x.dtype not in _DT:
            x = x.float()
        if t.requires_grad:
            t = t.detach()
        if t.dtype not in _DT:
            t = t.float()
        red = _REDUCTION[self.reduction]
        if i.numel() == 0:
            total = x.float().sum(-1)                              # nothing to learn from: zeros that know the input
            return total if red == 0 else total.sum()
        t, i = t.contiguous(), i.contiguous()
        # a tangent of forward-mode differentiation is refused by autograd; without a level there is none (asking takes 1 us)
        tangent = forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None
        if tangent or x.requires_grad and torch.is_grad_enabled():
            return _DistillFunction.apply(x, t, i, self.temperature, self.weight, red)
        return _distill_call(x, t, i, self.temperature, self.weight, red, False)[0]
