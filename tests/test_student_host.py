"""Argument checks of the student-training operators that need no GPU: every call fails before any launch."""
import ctypes

import pytest
import torch

import unet_amd
from unet_amd import _lib, ops


def _tensor(ptr=4096, pitch=32, coff=0):
    t = _lib.MiTensor()
    t.ptr, t.pitch, t.coff = ptr, pitch, coff
    return t


def test_group_norm_arguments_are_checked_on_the_host():
    lib = _lib.load()
    size = lib.mi_groupnorm_act_workspace_bytes
    assert size(1, 2, 100, 32, 8, 0) > 0 and size(1, 2, 100, 32, 8, 1) > size(1, 2, 100, 32, 8, 0)
    for bad in ((2, 2, 100, 32, 8), (1, 0, 100, 32, 8), (1, 2, 0, 32, 8), (1, 2, 100, 0, 1), (1, 2, 100, 32, 7), (1, 2, 100, 32, 0),
                (1, 2, 100, 8200, 8), (1, 2, 100, 4096, 4096), (1, 2, -5, 32, 8)):
        assert size(*bad, 0) == 0 and lib.mi_last_error()
    t = _tensor()
    ref = ctypes.byref

    def fwd(x=t, out=t, act=2, alpha=None, res=None, eps=1e-5, stats=4096, ws=4096, c=32, dtype=1):
        return lib.mi_groupnorm_act_fwd(dtype, 2, 100, c, 8, ref(x) if x else None, None, None, act, alpha, ref(res) if res else None,
                                        ref(out) if out else None, eps, stats, ws, None)

    for kw, text in ((dict(act=5), b"activation"), (dict(act=-1), b"activation"), (dict(act=4), b"alpha"), (dict(act=2, alpha=4096), b"alpha"),
                     (dict(stats=None), b"null"), (dict(ws=None), b"null"), (dict(x=None), b"null"), (dict(out=None), b"null"), (dict(eps=-1.0), b"eps"),
                     (dict(x=_tensor(pitch=31)), b"pitch"), (dict(x=_tensor(coff=1)), b"pitch"), (dict(x=_tensor(coff=-1)), b"pitch"),
                     (dict(x=_tensor(ptr=4097)), b"address"), (dict(res=_tensor(pitch=8)), b"pitch"), (dict(c=36), b"groups"), (dict(dtype=3), b"dtype")):
        assert fwd(**kw) != 0 and text in lib.mi_last_error(), (kw, lib.mi_last_error())
    two = _tensor()
    two.ptr2 = 4096
    assert fwd(x=two) != 0 and b"second source" in lib.mi_last_error()

    def bwd(act=2, alpha=None, dalpha=None, stats=4096, ws=4096, dy=t):
        return lib.mi_groupnorm_act_bwd(1, 2, 100, 32, 8, ref(dy) if dy else None, ref(t), stats, None, None, act, alpha, ref(t), None, None, dalpha, ws, None)

    for kw, text in ((dict(act=4), b"alpha"), (dict(dalpha=4096), b"alpha"), (dict(stats=None), b"null"), (dict(ws=None), b"null"), (dict(dy=None), b"null")):
        assert bwd(**kw) != 0 and text in lib.mi_last_error(), (kw, lib.mi_last_error())


def test_group_norm_has_no_cpu_path():
    x = torch.randn(1, 2, 2, 8)
    with pytest.raises(RuntimeError):
        ops.groupnorm_act_fwd(x, 2)
    with pytest.raises(ValueError):
        ops.groupnorm_act_fwd(torch.randn(8), 2)


def test_top_logits_and_distillation_arguments_are_checked_on_the_host():
    lib = _lib.load()
    ok = dict(dtype=1, rows=4, v=16, pitch=16, x=4096, k=4, values=4096, index=4096)

    def top(**kw):
        a = dict(ok, **kw)
        return lib.mi_top_logits(a["dtype"], a["rows"], a["v"], a["pitch"], a["x"], a["k"], a["values"], a["index"], None)

    for kw, text in ((dict(dtype=2), b"dtype"), (dict(rows=0), b"row"), (dict(v=0), b"classes"), (dict(v=2 ** 28 + 1), b"classes"), (dict(k=0), b"list"),
                     (dict(k=17), b"list"), (dict(v=300, pitch=300, k=257), b"list"), (dict(pitch=15), b"pitch"), (dict(x=None), b"null"),
                     (dict(values=None), b"null"), (dict(index=None), b"null"), (dict(x=4097), b"address"), (dict(index=4098), b"address")):
        assert top(**kw) != 0 and text in lib.mi_last_error(), (kw, lib.mi_last_error())

    size = lib.mi_distill_loss_saved_bytes
    assert size(1, 4, 16, 4) >= 32 and size(1, 4, 50000, 4) >= 64
    for bad in ((2, 4, 16, 4), (1, 0, 16, 4), (1, 4, 0, 4), (1, 4, 16, 0), (1, 4, 16, 257)):
        assert size(*bad) == 0 and lib.mi_last_error()
    ok = dict(dtype=1, rows=4, v=16, pitch=16, z=4096, k=4, td=0, t=4096, idt=3, i=4096, temp=1.0, w=1.0, red=1, loss=4096, saved=4096, dp=16, dz=4096, g=4096, after=0)

    def fwd(a):
        return lib.mi_distill_loss_fwd(a["dtype"], a["rows"], a["v"], a["pitch"], a["z"], a["k"], a["td"], a["t"], a["idt"], a["i"], a["temp"], a["w"], a["red"],
                                       a["loss"], a["saved"], None)

    def bwd(a):
        return lib.mi_distill_loss_bwd(a["dtype"], a["rows"], a["v"], a["pitch"], a["z"], a["k"], a["td"], a["t"], a["idt"], a["i"], a["temp"], a["w"], a["red"],
                                       a["g"], a["saved"], a["after"], a["dp"], a["dz"], None)

    both = ((dict(dtype=-1), b"dtype"), (dict(td=2), b"teacher dtype"), (dict(idt=0), b"index dtype"), (dict(rows=0), b"row"), (dict(v=0), b"classes"),
            (dict(k=0), b"list"), (dict(k=257), b"list"), (dict(pitch=15), b"pitch"), (dict(z=None), b"null"), (dict(t=None), b"null"), (dict(i=None), b"null"),
            (dict(saved=None), b"null"), (dict(temp=0.0), b"temperature"), (dict(temp=-1.0), b"temperature"), (dict(temp=float("inf")), b"temperature"),
            (dict(temp=float("nan")), b"temperature"), (dict(red=3), b"reduction"), (dict(w=float("nan")), b"weight"), (dict(z=4097), b"address"), (dict(t=4098), b"address"), (dict(i=4097), b"address"))
    for kw, text in both:
        for call in (fwd, bwd):
            assert call(dict(ok, **kw)) != 0 and text in lib.mi_last_error(), (kw, lib.mi_last_error())
    def step(a):
        return lib.mi_distill_loss_step(a["dtype"], a["rows"], a["v"], a["pitch"], a["z"], a["k"], a["td"], a["t"], a["idt"], a["i"], a["temp"], a["w"], a["red"],
                                        a["loss"], a["saved"], a["dp"], a["dz"], None)

    wide = dict(ok, v=5000, pitch=5000, dp=5000)
    ready = lib.mi_distill_loss_step_ready
    assert ready(1, 4, 5000, 4, 1) == 1 and ready(0, 4, 5000, 4, 2) == 1
    assert ready(1, 4, 16, 4, 1) == 0 and ready(1, 4, 5000, 4, 0) == 0 and ready(1, 4, 200000, 4, 1) == 0 and ready(2, 4, 5000, 4, 1) == 0
    assert step(ok) != 0 and b"step_ready" in lib.mi_last_error()
    assert step(dict(wide, red=0)) != 0 and b"step_ready" in lib.mi_last_error()
    assert bwd(dict(ok, after=1)) != 0 and b"step" in lib.mi_last_error()
    for kw, text in both[:-3] + ((dict(dp=15), b"pitch"), (dict(dz=None), b"null"), (dict(loss=None), b"null"), (dict(saved=4100), b"aligned")):
        assert step(dict(wide, **kw)) != 0 and text in lib.mi_last_error(), (kw, lib.mi_last_error())
    for kw, text in ((dict(dp=15), b"pitch"), (dict(dz=None), b"null"), (dict(g=None), b"null"), (dict(dz=4097), b"address")):
        assert bwd(dict(ok, **kw)) != 0 and text in lib.mi_last_error(), (kw, lib.mi_last_error())
    assert fwd(dict(ok, loss=None)) != 0 and b"null" in lib.mi_last_error()


def test_distillation_has_no_cpu_path_and_checks_its_options():
    z, t, i = torch.randn(3, 8), torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        unet_amd.TopLogitDistillationLoss()(z, t, i)
    with pytest.raises(RuntimeError):
        ops.top_logits(z, 2)
    for bad in (dict(temperature=0), dict(temperature=-1), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(reduction="batchmean"), dict(weight=float("inf"))):
        with pytest.raises(ValueError):
            unet_amd.TopLogitDistillationLoss(**bad)
