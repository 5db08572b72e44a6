"""Calls of the operators at a model's end that their documentation allows, or has to refuse, beyond values of their inputs:
forward-mode differentiation through them, and their backward pass."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.fixture(scope="module")
def M():
    from types import SimpleNamespace
    from scmomer_amd import logits, norm
    return SimpleNamespace(layer_norm=norm.layer_norm, token_logprobs=logits.token_logprobs,
                           topk_distillation=logits.topk_distillation, topk_distillation_grad=logits.topk_distillation_grad)


def _calls(M, t=6, v=300, k=4):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(t, v, generator=gen).to(DEV)
    idx = torch.rand(t, v, generator=gen).topk(k, 1).indices.to(DEV)
    lp = torch.full((t, k), -2.0, device=DEV)
    return x, {"norm": lambda z: M.layer_norm(z), "score": lambda z: M.token_logprobs(z).lse,
               "entropy": lambda z: M.token_logprobs(z).entropy,
               "distill": lambda z: M.topk_distillation(z, idx, lp, reduction="none"),
               "step": lambda z: M.topk_distillation_grad(z, idx, lp)[0]}


@pytest.mark.parametrize("name", ["norm", "score", "entropy", "distill", "step"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_raises(M, name, grad):
    x, calls = _calls(M)
    with fwAD.dual_level():
        z = fwAD.make_dual(x.detach().requires_grad_(grad), torch.randn_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            calls[name](z)
    assert torch.isfinite(calls[name](x)).all()          # a call that was refused leaves the next one alone


@pytest.mark.parametrize("name", ["norm", "score", "entropy", "distill"])
def test_forward_mode_of_the_incoming_gradient_raises(M, name):
    x, calls = _calls(M)
    z = x.detach().requires_grad_()
    y = calls[name](z)
    with fwAD.dual_level():
        g = fwAD.make_dual(torch.ones_like(y), torch.randn_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, z, g, retain_graph=True)
    assert torch.isfinite(torch.autograd.grad(y, z, torch.ones_like(y))[0]).all()


@pytest.mark.parametrize("name", ["norm", "score", "distill"])
def test_a_mode_that_only_counts_changes_nothing(M, name):
    from torch.utils.flop_counter import FlopCounterMode
    x, calls = _calls(M)
    z = x.detach().requires_grad_()
    want = calls[name](z)
    dw, = torch.autograd.grad(want.sum(), z)
    with FlopCounterMode(display=False):
        got = calls[name](z)
        dg, = torch.autograd.grad(got.sum(), z)
    assert torch.equal(want, got) and torch.equal(dw, dg)
