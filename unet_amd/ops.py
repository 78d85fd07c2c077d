"""Operator-level Python bindings (channels-last tensors) over the C ABI: convolution forward / data
gradient / weight gradient, instance-norm + PReLU, group norm + activation and the top logits of a teacher.  Used by the operator parity tests and by
callers that want to assemble other networks from the same kernels.

Tensors are ``[N, (D,) H, W, C]`` contiguous, dtype ``torch.bfloat16`` or ``torch.float32``.  These are the kernels' calls, without autograd: results do
not require a gradient, and the caller of a forward operator calls the backward one.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import Optional

import torch

from . import _lib

_DT = {torch.float32: 0, torch.bfloat16: 1}


def _desc(x_shape, cin, cout, ksize, stride, transposed, dtype):
    d = _lib.MiConvDesc()
    nd = len(x_shape) - 2
    d.ndim, d.transposed, d.ksize, d.stride = nd, 1 if transposed else 0, ksize, stride
    d.cin, d.cout, d.nb = cin, cout, x_shape[0]
    sp = [1] * (3 - nd) + [int(v) for v in x_shape[1:-1]]
    for i in range(3):
        d.in_dims[i] = sp[i]
    d.dtype = _DT[dtype]
    return d


def _ten(t: Optional[torch.Tensor], coff: int = 0):
    m = _lib.MiTensor()
    if t is not None:
        m.ptr, m.pitch, m.coff = t.data_ptr(), t.shape[-1], coff
    return m


def _out_spatial(sp, ksize, stride, transposed):
    if transposed:
        return [2 * s for s in sp]
    pad = (ksize - 1) // 2
    return [(s + 2 * pad - ksize) // stride + 1 for s in sp]


def pack_weights(w: torch.Tensor, x_shape, ksize, stride, transposed, dtype, dgrad=False) -> torch.Tensor:
    lib = _lib.load()
    cin, cout = (w.shape[0], w.shape[1]) if transposed else (w.shape[1], w.shape[0])
    d = _desc(x_shape, cin, cout, ksize, stride, transposed, dtype)
    nbytes = lib.mi_conv_packed_bytes(C.byref(d))
    out = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
    wf = w.contiguous().float()
    _lib.check(lib.mi_conv_pack(C.byref(d), 1 if dgrad else 0, wf.data_ptr(), out.data_ptr(),
                                _lib.current_stream(w.device)), "mi_conv_pack")
    return out


def conv_forward(x, w, bias=None, ksize=3, stride=1, transposed=False, addend=None, want_stats=False):
    """x: channels-last; w: torch layout fp32.  Returns y (channels-last) [, stats [N,8,Cout,2] fp64]."""
    lib = _lib.load()
    cin, cout = (w.shape[0], w.shape[1]) if transposed else (w.shape[1], w.shape[0])
    d = _desc(x.shape, cin, cout, ksize, stride, transposed, x.dtype)
    packed = pack_weights(w, x.shape, ksize, stride, transposed, x.dtype, False)
    osp = _out_spatial(list(x.shape[1:-1]), ksize, stride, transposed)
    y = torch.empty([x.shape[0]] + osp + [cout], dtype=x.dtype, device=x.device)
    stats = torch.zeros(x.shape[0], 8, cout, 2, dtype=torch.float64, device=x.device) if want_stats else None
    b = bias.contiguous().float() if bias is not None else None
    tx, ty, ta = _ten(x), _ten(y), _ten(addend)
    _lib.check(lib.mi_conv_forward(C.byref(d), C.byref(tx), packed.data_ptr(), _lib.ptr(b), C.byref(ty),
                                   C.byref(ta) if addend is not None else None, _lib.ptr(stats),
                                   _lib.current_stream(x.device)), "mi_conv_forward")
    return (y, stats) if want_stats else y


def conv_dgrad(dy, w, x_shape, ksize=3, stride=1, transposed=False, addend=None):
    lib = _lib.load()
    cin, cout = (w.shape[0], w.shape[1]) if transposed else (w.shape[1], w.shape[0])
    d = _desc(x_shape, cin, cout, ksize, stride, transposed, dy.dtype)
    packed = pack_weights(w, x_shape, ksize, stride, transposed, dy.dtype, True)
    dx = torch.empty(list(x_shape[:-1]) + [cin], dtype=dy.dtype, device=dy.device)
    tdy, tdx, ta = _ten(dy), _ten(dx), _ten(addend)
    _lib.check(lib.mi_conv_dgrad(C.byref(d), C.byref(tdy), packed.data_ptr(), C.byref(tdx),
                                 C.byref(ta) if addend is not None else None, _lib.current_stream(dy.device)),
               "mi_conv_dgrad")
    return dx


def conv_wgrad(x, dy, w_shape, ksize=3, stride=1, transposed=False):
    """Returns (dw in the torch layout, db [cout] or None for transposed convolutions)."""
    lib = _lib.load()
    cin, cout = (w_shape[0], w_shape[1]) if transposed else (w_shape[1], w_shape[0])
    d = _desc(x.shape, cin, cout, ksize, stride, transposed, x.dtype)
    ws = torch.empty(lib.mi_conv_wgrad_workspace_bytes(C.byref(d)), dtype=torch.uint8, device=x.device)
    dw = torch.empty(w_shape, dtype=torch.float32, device=x.device)
    db = None if transposed else torch.empty(cout, dtype=torch.float32, device=x.device)
    tx, tdy = _ten(x), _ten(dy)
    _lib.check(lib.mi_conv_wgrad(C.byref(d), C.byref(tx), C.byref(tdy), dw.data_ptr(), _lib.ptr(db), ws.data_ptr(),
                                 _lib.current_stream(x.device)), "mi_conv_wgrad")
    return dw, db


def _dims3(sp):
    return (C.c_int32 * 3)(*([1] * (3 - len(sp)) + [int(v) for v in sp]))


def conv1_forward(x, w, bias=None, dtype=torch.float32, split=None, want_stats=False):
    """F.conv (k 3, stride 2, padding 1) of a one-channel fp32 tensor ``x`` [N, (D,) H, W] with ``w`` [C, 1, 3, ..]:
    channels-last result of ``dtype``; ``split``: write the channels from ``split`` on to a second tensor (returned as
    a pair).  With ``want_stats`` also the [N, 8, C, 2] fp64 sums of the bias-free result."""
    lib = _lib.load()
    nd, n = x.dim() - 1, w.shape[0]
    osp = [v // 2 for v in x.shape[1:]]
    c1 = n if split is None else split
    y = torch.empty([x.shape[0]] + osp + [c1], dtype=dtype, device=x.device)
    y2 = torch.empty([x.shape[0]] + osp + [n - c1], dtype=dtype, device=x.device) if split is not None else None
    ty = _ten(y)
    if y2 is not None:
        ty.ptr2, ty.pitch2, ty.coff2, ty.c1 = y2.data_ptr(), y2.shape[-1], 0, c1
    stats = torch.zeros(x.shape[0], 8, n, 2, dtype=torch.float64, device=x.device) if want_stats else None
    wf = w.contiguous().float()
    b = bias.contiguous().float() if bias is not None else None
    _lib.check(lib.mi_conv1_forward(_DT[dtype], nd, x.shape[0], _dims3(x.shape[1:]), n, x.data_ptr(), wf.data_ptr(), _lib.ptr(b),
                                    C.byref(ty), _lib.ptr(stats), _lib.current_stream(x.device)), "mi_conv1_forward")
    out = y if y2 is None else (y, y2)
    return (out, stats) if want_stats else out


def conv1_transposed(y, w, bias=None, y2=None, want_stats=False):
    """F.conv_transpose (k 3, stride 2, padding 1, output_padding 1) of channels-last ``y`` (+ ``y2``) with ``w``
    [C, 1, 3, ..] to ONE output channel: fp32 [N, (D,) H, W] on the fine grid."""
    lib = _lib.load()
    nd = y.dim() - 2
    n = y.shape[-1] + (y2.shape[-1] if y2 is not None else 0)
    fsp = [2 * v for v in y.shape[1:-1]]
    out = torch.empty([y.shape[0]] + fsp, dtype=torch.float32, device=y.device)
    ty = _ten(y)
    if y2 is not None:
        ty.ptr2, ty.pitch2, ty.coff2, ty.c1 = y2.data_ptr(), y2.shape[-1], 0, y.shape[-1]
    stats = torch.zeros(y.shape[0], 8, 1, 2, dtype=torch.float64, device=y.device) if want_stats else None
    wf = w.contiguous().float()
    b = bias.contiguous().float() if bias is not None else None
    _lib.check(lib.mi_conv1_transposed(_DT[y.dtype], nd, y.shape[0], _dims3(fsp), n, C.byref(ty), wf.data_ptr(), _lib.ptr(b),
                                       out.data_ptr(), _lib.ptr(stats), _lib.current_stream(y.device)), "mi_conv1_transposed")
    return (out, stats) if want_stats else out


def conv1_wgrad(x, y, y2=None):
    """Weight and bias gradient of the 3^d stride-2 convolution between a one-channel fp32 tensor ``x``
    ([N, (D,) H, W], fine grid) and channels-last ``y`` (coarse grid; ``y2``: a second source whose channels follow
    those of ``y``).  Returns (dw [C, 1, 3, ..] fp32, db [C] fp32)."""
    lib = _lib.load()
    nd = x.dim() - 1
    n = y.shape[-1] + (y2.shape[-1] if y2 is not None else 0)
    dims = _dims3(x.shape[1:])
    ws = torch.empty(lib.mi_conv1_wgrad_workspace_bytes(nd, n, dims), dtype=torch.uint8, device=x.device)
    dw = torch.empty([n, 1] + [3] * nd, dtype=torch.float32, device=x.device)
    db = torch.empty(n, dtype=torch.float32, device=x.device)
    ty = _ten(y)
    if y2 is not None:
        ty.ptr2, ty.pitch2, ty.coff2, ty.c1 = y2.data_ptr(), y2.shape[-1], 0, y.shape[-1]
    _lib.check(lib.mi_conv1_wgrad(_DT[y.dtype], nd, x.shape[0], dims, n, x.data_ptr(), C.byref(ty), dw.data_ptr(),
                                  db.data_ptr(), ws.data_ptr(), _lib.current_stream(x.device)), "mi_conv1_wgrad")
    return dw, db


def instnorm_prelu_fwd(raw, stats, alpha, res=None, dropout=0.0, seed=0, layer=0):
    lib = _lib.load()
    nb, c = raw.shape[0], raw.shape[-1]
    npix = raw[0].numel() // c
    out = torch.empty_like(raw)
    traw, tres, tout = _ten(raw), _ten(res), _ten(out)
    _lib.check(lib.mi_instnorm_prelu_fwd(_DT[raw.dtype], nb, npix, c, C.byref(traw), stats.data_ptr(), alpha.data_ptr(),
                                         C.byref(tres) if res is not None else None, C.byref(tout), float(dropout),
                                         C.c_uint64(seed), layer, _lib.current_stream(raw.device)),
               "mi_instnorm_prelu_fwd")
    return out


def instnorm_prelu_bwd(dy, raw, stats, alpha, dropout=0.0, seed=0, layer=0):
    """Returns (dx, dalpha [1])."""
    lib = _lib.load()
    nb, c = raw.shape[0], raw.shape[-1]
    npix = raw[0].numel() // c
    dx = torch.empty_like(raw)
    bstats = torch.empty(nb * 8 * c * 2, dtype=torch.float64, device=raw.device)
    dalpha = torch.zeros(1, dtype=torch.float32, device=raw.device)
    tdy, traw, tdx = _ten(dy), _ten(raw), _ten(dx)
    _lib.check(lib.mi_instnorm_prelu_bwd(_DT[raw.dtype], nb, npix, c, C.byref(tdy), C.byref(traw), stats.data_ptr(),
                                         alpha.data_ptr(), bstats.data_ptr(), dalpha.data_ptr(), C.byref(tdx),
                                         float(dropout), C.c_uint64(seed), layer, _lib.current_stream(raw.device)),
               "mi_instnorm_prelu_bwd")
    return dx, dalpha


_ACT = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "prelu": 4}


def _pixels(t, name, like=None):
    """``t`` [N, .., C] as (tensor, pitch): pixels at one common distance, channels side by side.  A slice of the channels
    of a wider tensor is taken as it lies; any other order of the memory is copied into a dense tensor."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if like is not None:
        if t.shape != like.shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(like.shape)}")
        if t.dtype != like.dtype or t.device != like.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {like.dtype} on {like.device}")
    if t.is_contiguous():
        return t, t.shape[-1]
    c, pitch, span = t.shape[-1], None, 1
    dense = t.stride(-1) == 1 or c == 1
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if pitch is None:
            pitch = stride
        dense = dense and stride == pitch * span
        span *= size
    if pitch is None:
        pitch = c
    if not dense or pitch < c or pitch > 0x7FFFFFFF:
        return t.contiguous(), c
    return t, pitch


def _view(t, pitch):
    return C.byref(_lib.MiTensor(t.data_ptr(), pitch))


def _channel_param(t, n, x, name):
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must have shape ({n},), got {tuple(t.shape)}")
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, expected {x.device}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.detach().contiguous().float()


@functools.lru_cache(maxsize=256)
def _groupnorm_workspace(dt, nb, npix, c, groups, backward):
    return _lib.load().mi_groupnorm_act_workspace_bytes(dt, nb, npix, c, groups, backward)


def _groupnorm_args(x, groups, weight, bias, act, alpha):
    if not isinstance(x, torch.Tensor) or x.dim() < 2:
        raise ValueError("x must be a channels-last tensor [N, .., C]")
    if not x.is_cuda:
        raise RuntimeError("unet_amd.ops run on an AMD GPU only (no CPU or eager fallback)")
    if x.dtype not in _DT:
        raise ValueError(f"x must be torch.float32 or torch.bfloat16, got {x.dtype}")
    if act not in _ACT:
        raise ValueError(f"act must be one of {sorted(_ACT)}, got {act!r}")
    if (alpha is None) == (act == "prelu"):
        raise ValueError("alpha (one slope) belongs to act='prelu' and to no other")
    nb, c, groups = x.shape[0], x.shape[-1], int(groups)
    if c < 1 or groups < 1 or c % groups:
        raise ValueError(f"{groups} groups do not divide {c} channels")
    npix = math.prod(x.shape[1:-1])
    if npix == 0:
        raise ValueError("an image without pixels has no mean")
    return (nb, npix, c, groups, _channel_param(weight, c, x, "weight"), _channel_param(bias, c, x, "bias"),
            _channel_param(alpha, 1, x, "alpha"))


def groupnorm_act_fwd(x, groups, weight=None, bias=None, act="silu", alpha=None, res=None, eps=1e-5):
    """``act(F.group_norm(x, groups, weight, bias, eps)) (+ res)`` of a channels-last ``x`` [N, .., C]; ``act`` is one of
    "none", "relu", "silu", "gelu" (erf) and "prelu" (with its one slope ``alpha`` [1]).  ``weight`` and ``bias`` [C] and
    ``alpha`` are read as fp32.  Returns (y, stats [N, groups, 2] fp32: mean and 1 / sqrt(variance + eps), for the backward call)."""
    nb, npix, c, groups, weight, bias, alpha = _groupnorm_args(x, groups, weight, bias, act, alpha)
    x, xp = _pixels(x, "x")
    out = x.new_empty(x.shape)
    stats = x.new_empty((nb, groups, 2), dtype=torch.float32)
    if res is not None:
        res, rp = _pixels(res, "res", x)
    if nb == 0:
        return out, stats
    lib, dt = _lib.load(), _DT[x.dtype]
    with _lib.on_device(x.device):
        ws = x.new_empty(_groupnorm_workspace(dt, nb, npix, c, groups, 0), dtype=torch.uint8)
        _lib.check(lib.mi_groupnorm_act_fwd(dt, nb, npix, c, groups, _view(x, xp), _lib.ptr(weight), _lib.ptr(bias), _ACT[act],
                                            _lib.ptr(alpha), _view(res, rp) if res is not None else None, _view(out, c), eps, stats.data_ptr(), ws.data_ptr(), _lib.stream_of(x.device)), "mi_groupnorm_act_fwd")
    return out, stats


def groupnorm_act_bwd(dy, x, stats, groups, weight=None, bias=None, act="silu", alpha=None):
    """Gradients of ``groupnorm_act_fwd`` from its input and its ``stats``: (dx, dweight, dbias, dalpha), fp32 for the
    parameters and None for those that were not given.  The gradient with respect to ``res`` is ``dy`` itself."""
    nb, npix, c, groups, weight, bias, alpha = _groupnorm_args(x, groups, weight, bias, act, alpha)
    dy, dp = _pixels(dy, "dy", x)
    x, xp = _pixels(x, "x")
    if tuple(stats.shape) != (nb, groups, 2) or stats.dtype != torch.float32 or stats.device != x.device:
        raise ValueError(f"stats must be the fp32 tensor [{nb}, {groups}, 2] of the forward call")
    stats = stats.contiguous()
    dx = x.new_empty(x.shape)
    new = x.new_zeros if nb == 0 else x.new_empty
    dw = new(c, dtype=torch.float32) if weight is not None else None
    db = new(c, dtype=torch.float32) if bias is not None else None
    da = new(1, dtype=torch.float32) if alpha is not None else None
    if nb == 0:
        return dx, dw, db, da
    lib, dt = _lib.load(), _DT[x.dtype]
    with _lib.on_device(x.device):
        ws = x.new_empty(_groupnorm_workspace(dt, nb, npix, c, groups, 1), dtype=torch.uint8)
        _lib.check(lib.mi_groupnorm_act_bwd(dt, nb, npix, c, groups, _view(dy, dp), _view(x, xp), stats.data_ptr(), _lib.ptr(weight),
                                            _lib.ptr(bias), _ACT[act], _lib.ptr(alpha), _view(dx, c), _lib.ptr(dw), _lib.ptr(db),
                                            _lib.ptr(da), ws.data_ptr(), _lib.stream_of(x.device)), "mi_groupnorm_act_bwd")
    return dx, dw, db, da


def top_logits(logits, k):
    """The ``k`` (at most 256) largest of the class logits [.., V] of every pixel, largest first, equal ones by ascending class:
    (values [.., k] of the logits' type, index [.., k] int32), the lists that ``TopLogitDistillationLoss`` reads.
    NaN counts as the largest value."""
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1:
        raise ValueError("logits must be a tensor [.., V]")
    if not logits.is_cuda:
        raise RuntimeError("unet_amd.ops run on an AMD GPU only (no CPU or eager fallback)")
    if logits.dtype not in _DT:
        raise ValueError(f"logits must be torch.float32 or torch.bfloat16, got {logits.dtype}")
    v, k = logits.shape[-1], int(k)
    if not 1 <= k <= min(v, 256):
        raise ValueError(f"k must be in 1 .. {min(v, 256)} for {v} classes, got {k}")
    x, pitch = _pixels(logits, "logits")
    shape = logits.shape[:-1] + (k,)
    values = x.new_empty(shape)
    index = x.new_empty(shape, dtype=torch.int32)
    rows = index.numel() // k
    if rows:
        with _lib.on_device(x.device):
            _lib.check(_lib.load().mi_top_logits(_DT[x.dtype], rows, v, pitch, x.data_ptr(), k, values.data_ptr(), index.data_ptr(),
                                                 _lib.stream_of(x.device)), "mi_top_logits")
    return values, index
