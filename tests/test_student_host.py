"""Argument checks of the student-training operators that need no GPU: every call fails before any launch."""
import ctypes

import pytest
import torch

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
