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


def test_token_logprobs_needs_device_tensors():
    from scmomer_amd.logits import token_logprobs
    with pytest.raises(ValueError):
        token_logprobs(torch.randn(2, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        token_logprobs(torch.zeros(2, 8, dtype=torch.int64))


@pytest.mark.parametrize("change", [dict(x=None), dict(type=3), dict(ldx=-1), dict(T=0), dict(T=1 << 31), dict(V=0),
                                    dict(V=(1 << 30) + 1), dict(tau=0.0), dict(tau=-1.0), dict(tau=float("inf")),
                                    dict(tau=float("nan")), dict(tau=1e-38), dict(k=-1), dict(k=65), dict(k=9), dict(target=None),
                                    dict(logprob=None), dict(top=None), dict(index=None), dict(V=100000, k=3, ws=None),
                                    dict(ws_off=4)])
def test_score_fwd_rejects(change):
    from scmomer_amd._lib import lib
    keep, a = _addr()
    k = dict(x=a, type=0, ldx=8, T=1, V=8, tau=1.0, target=a, k=2, logprob=a, top=a, index=a, ws=a, ws_off=0)
    k.update(change)
    ws = k["ws"] + k["ws_off"] if k["ws"] else None
    rc = lib.scm_score_fwd(k["x"], k["type"], k["ldx"], k["T"], k["V"], k["tau"], k["target"], -100, k["k"], k["logprob"],
                           a, a, k["top"], k["index"], a, ws, None)
    assert rc < 0 and b"scm_score_fwd" in lib.scm_last_error()


@pytest.mark.parametrize("change", [dict(x=None), dict(tape=None), dict(dx=None), dict(target=None), dict(entropy=None),
                                    dict(index=None), dict(k=0), dict(type=-1), dict(tau=0.0)])
def test_score_bwd_rejects(change):
    from scmomer_amd._lib import lib
    keep, a = _addr()
    k = dict(x=a, type=0, tau=1.0, target=a, k=2, tape=a, entropy=a, index=a, dx=a)
    k.update(change)
    rc = lib.scm_score_bwd(k["x"], k["type"], 8, 1, 8, k["tau"], k["target"], -100, k["k"], k["tape"], k["entropy"],
                           k["index"], a, a, a, a, k["dx"], None)
    assert rc < 0 and b"scm_score_bwd" in lib.scm_last_error()


def test_score_workspace_holds_every_split():
    """a split row's keys and statistics fit the workspace, and the join's limits hold"""
    from scmomer_amd._lib import lib
    for t in (1, 3, 100, 511, 512, 100000):
        for v in (1, 64, 8192, 8193, 131072, 1 << 30):
            for k in (0, 1, 20, 64):
                n = lib.scm_score_ws_floats(t, v, k)
                s = n // (t * (2 * k + 3))
                assert n == s * t * (2 * k + 3) and s <= 64 and s * k <= 2048 and s != 1
    assert lib.scm_score_ws_floats(1, 100, 65) == 0 and lib.scm_score_ws_floats(0, 100, 1) == 0


def test_topk_distillation_needs_device_tensors():
    from scmomer_amd.logits import topk_distillation, topk_distillation_grad
    x, idx, lp = torch.randn(2, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for f in (topk_distillation, topk_distillation_grad):
        with pytest.raises(ValueError):
            f(x, idx, lp)


@pytest.mark.parametrize("entry", ["fwd", "bwd", "step"])
@pytest.mark.parametrize("change", [dict(x=None), dict(type=7), dict(T=0), dict(V=0), dict(ldx=-2), dict(tau=0.0), dict(k=0),
                                    dict(k=65), dict(index=None), dict(lp=None), dict(rows=None), dict(dx=None),
                                    dict(tape=None, V=100), dict(wsum=None), dict(ws=None, V=100000), dict(gloss=None),
                                    dict(T=(1 << 31) - 1, V=1 << 30)])
def test_topk_distill_rejects(entry, change):
    from scmomer_amd._lib import lib
    only = {"rows": ("fwd", "step"), "dx": ("bwd", "step"), "tape": ("bwd", "step"), "wsum": ("bwd", "step"),
            "ws": ("fwd", "step"), "gloss": ("bwd",)}
    if any(entry not in only.get(n, (entry,)) for n in change):
        pytest.skip("not an argument of this entry point, or allowed there")
    keep, a = _addr()
    k = dict(x=a, type=0, ldx=8, T=1, V=8, tau=1.0, index=a, lp=a, k=2, rows=a, dx=a, tape=a, wsum=a, ws=a, gloss=a)
    k.update(change)
    head = (k["x"], k["type"], k["ldx"], k["T"], k["V"], k["tau"], k["index"], k["lp"], k["k"], 1, a, 1)
    if entry == "fwd":
        rc = lib.scm_topk_distill_fwd(*head, k["rows"], a, k["wsum"], k["tape"], k["ws"], None)
    elif entry == "bwd":
        rc = lib.scm_topk_distill_bwd(*head, k["wsum"], k["gloss"], 0, k["tape"], k["dx"], None)
    else:
        rc = lib.scm_topk_distill_step(*head, 1.0, k["rows"], a, k["wsum"], k["tape"], k["ws"], k["dx"], None)
    assert rc < 0 and f"scm_topk_distill_{entry}".encode() in lib.scm_last_error()


def test_topk_distill_workspaces():
    from scmomer_amd._lib import lib
    assert lib.scm_topk_distill_tape_floats(10, 64, 5) == 70 and lib.scm_topk_distill_tape_floats(100000, 64, 5) == 0
    assert lib.scm_topk_distill_ws_floats(1000, 131072) == 0                 # one workgroup per row
    assert lib.scm_topk_distill_ws_floats(1000, 131073) == 4000              # more tokens than a workgroup marks
    assert lib.scm_topk_distill_ws_floats(16384, 7) == 0 and lib.scm_topk_distill_ws_floats(16385, 7) == 1024   # parts of the sums
    assert lib.scm_topk_distill_ws_floats(64, 131072) == 0
    for t in (1, 7, 63):
        n = lib.scm_topk_distill_ws_floats(t, 100000)
        assert n % (2 * t) == 0 and 2 <= n // (2 * t) <= 64
