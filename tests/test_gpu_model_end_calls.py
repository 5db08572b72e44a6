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


def _negated(shape, seed):
    """f32 of that shape whose memory holds the values with the other sign (a view that notes the change only)"""
    gen = torch.Generator().manual_seed(seed)
    z = torch.complex(torch.zeros(shape), torch.randn(shape, generator=gen)).to(DEV)
    n = z.conj().imag
    assert n.is_neg()
    return n, n.clone().resolve_neg()


def test_views_that_note_a_sign(M):
    """every operand with one element a row or one element at all, where no copy for its stride would write the sign"""
    for t in (1, 5):
        n, x = _negated((t, 1), t)
        assert torch.equal(M.token_logprobs(n).lse, M.token_logprobs(x).lse)
        idx, lp, w = torch.zeros(t, 1, dtype=torch.int64, device=DEV), torch.zeros(t, 1, device=DEV), torch.ones(t, device=DEV)
        y = torch.ones(t, 1, device=DEV)
        assert torch.equal(M.topk_distillation(y, idx, n, reduction="none"), M.topk_distillation(y, idx, x, reduction="none"))
        n1, x1 = _negated((1,), 7)
        for a, b in ((M.layer_norm(n, n1, n1), M.layer_norm(x, x1, x1)), (M.layer_norm(y, None, n1), M.layer_norm(y, None, x1)),
                     (M.topk_distillation(y[:1], idx[:1], lp[:1] - 1, tail=True, weight=n1, reduction="sum"),
                      M.topk_distillation(y[:1], idx[:1], lp[:1] - 1, tail=True, weight=x1, reduction="sum"))):
            assert torch.equal(a, b)
        z = y.clone().requires_grad_()
        b = torch.zeros(1, device=DEV, requires_grad=True)
        for f, v in ((lambda: M.layer_norm(z, None, b), b), (lambda: M.token_logprobs(z).lse[:, None], z)):
            want, = torch.autograd.grad(f(), v, x)
            got, = torch.autograd.grad(f(), v, n)
            assert torch.equal(want, got) and want.abs().max() > 0


@pytest.mark.parametrize("name", ["norm", "score", "entropy", "distill"])
def test_an_incoming_gradient_that_is_only_noted_to_be_zero(M, name):
    x, calls = _calls(M)
    z = x.detach().requires_grad_()
    y = calls[name](z)
    g, = torch.autograd.grad(y, z, torch._efficientzerotensor(tuple(y.shape), device=DEV))
    assert g.shape == x.shape and not g.any()


@pytest.mark.parametrize("name", ["norm", "score", "distill"])
@pytest.mark.parametrize("layers", [1, 3])
def test_capture_beside_an_eager_graph_of_a_leaf_further_up(M, name, layers):
    """The leaf is a weight some products before the operator; its accumulator lives on the default stream for as long as the
    eager graph does.  Refused then, before anything is launched; captured once that graph is gone, and for a weight that no
    graph holds."""
    import gc
    x, calls = _calls(M)
    w = torch.rand(6, 300, generator=torch.Generator().manual_seed(1)).to(DEV).requires_grad_()

    def loss(weight):
        h = x
        for _ in range(layers):
            h = h * weight
        y = calls[name](h)
        return (y * y).sum()
    alive = loss(w)
    want, = torch.autograd.grad(alive, w, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other = w.detach().requires_grad_()
        got, = torch.autograd.grad(loss(other), other)
        h = x.detach().requires_grad_()                    # a leaf of its own: the held weight takes no part
        side, = torch.autograd.grad((calls[name](h * w) ** 2).sum(), h)
        with pytest.raises(RuntimeError, match="default stream"):
            torch.autograd.grad(loss(w), w)
        with pytest.raises(RuntimeError, match="default stream"):
            loss(w).backward()
    del alive
    gc.collect()          # the refusals' tracebacks hold graphs too
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        got2, = torch.autograd.grad(loss(w), w)
    for _ in range(3):
        graph.replay()
        again.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(got2, want) and torch.isfinite(side).all()
        got.zero_()
        got2.zero_()
        torch.cuda.synchronize()
    assert w.grad is None
