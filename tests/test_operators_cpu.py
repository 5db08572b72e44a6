"""Refusals of the operators at the end of a token model that need no GPU: tensors off the device through the public
functions, bad arguments through the C ABI (an error code and a text, nothing launched)."""
import ctypes as C

import pytest
import torch


def _addr():
    buf = C.create_string_buffer(256)
    return buf, C.addressof(buf) + (-C.addressof(buf)) % 16


def test_layer_norm_needs_device_tensors():
    from scmomer_amd.norm import layer_norm
    with pytest.raises(ValueError):
        layer_norm(torch.randn(2, 8))
    with pytest.raises(TypeError):
        layer_norm(torch.zeros(2, 8, dtype=torch.int64))


@pytest.mark.parametrize("change", [dict(x=None), dict(y=None), dict(T=0), dict(D=0), dict(D=16385), dict(T=1 << 31),
                                    dict(ldx=-1), dict(xt=3), dict(xt=1, yt=0), dict(xt=2, yt=1), dict(xt=0, yt=2),
                                    dict(rstd=None)])
def test_norm_fwd_rejects(change):
    from scmomer_amd._lib import lib
    keep, a = _addr()
    k = dict(x=a, xt=0, ldx=8, T=1, D=8, y=a, yt=0, mean=a, rstd=a)
    k.update(change)
    rc = lib.scm_norm_fwd(k["x"], k["xt"], k["ldx"], None, None, k["T"], k["D"], 1e-5, k["y"], k["yt"], k["mean"],
                          k["rstd"], None)
    assert rc < 0 and b"scm_norm_fwd" in lib.scm_last_error()


@pytest.mark.parametrize("change", [dict(dy=None), dict(x=None), dict(mean=None), dict(lddy=-1), dict(ws=None),
                                    dict(dx=None, dg=None, db=None, ws=None), dict(dg=None, db=None), dict(D=20000)])
def test_norm_bwd_rejects(change):
    from scmomer_amd._lib import lib
    keep, a = _addr()
    k = dict(dy=a, lddy=8, x=a, D=8, mean=a, dx=a, ws=a, dg=a, db=a)
    k.update(change)
    rc = lib.scm_norm_bwd(k["dy"], 0, k["lddy"], k["x"], 0, 8, k["mean"], a, None, 1, k["D"], k["dx"], k["ws"], k["dg"],
                          k["db"], None)
    assert rc < 0 and b"scm_norm_bwd" in lib.scm_last_error()


def test_norm_workspace_sizes():
    from scmomer_amd._lib import lib
    assert lib.scm_norm_bwd_ws_floats(0, 8) == 0 and lib.scm_norm_bwd_ws_floats(8, 16385) == 0
    assert lib.scm_norm_bwd_ws_floats(1, 7) == 14
    assert lib.scm_norm_bwd_ws_floats(1 << 30, 4096) <= 2 * 4096 * 2048
