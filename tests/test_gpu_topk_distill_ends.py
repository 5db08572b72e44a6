"""topk_distillation at the ends of its ranges: entries whose mass together is next to nothing, what the C entry points write
of the weights' sum, and the sizes at which its kernels change.  Bounds as in test_gpu_topk_distill."""
import pytest
import torch

from test_gpu_topk_distill import _case, _check, _terms, _within, HALF, U

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")


@pytest.fixture(scope="module")
def L():
    from scmomer_amd import logits as m
    return m


@pytest.mark.parametrize("t,v,k", [(9, 40, 5), (21000, 40, 5), (7, 700, 64), (5, 9000, 7), (3, 100000, 20), (300, 20000, 3)])
@pytest.mark.parametrize("top", [-41.0, -50.0, -88.0, -104.0, -200.0, -700.0, -760.0, -5000.0, -3e37])
def test_renormalised_entries_of_hardly_any_mass(L, t, v, k, top):
    """Renormalised, only differences of the entries' log probabilities count: q = softmax over the entries, log q exact in
    64 bits.  f32 rounds lp - max(lp) once (u of at most 8) and the logarithm of a sum in [1, 64] (below 4.2) to a few u: 16 u on
    each log q, next to the rounding of log p that _terms counts; q moves by as much, relative."""
    x, idx, _, w = _case(t, v, k, torch.float32, t + v)
    gen = torch.Generator().manual_seed(k)
    step = 1.0 if abs(top) < 1e6 else abs(top) * 2.0 ** -18      # a step that f32 holds there
    lp = (top - step * torch.randint(0, 9, (t, k), generator=gen).float()).to(DEV)
    lp[0, 1:] = -INF                                              # one entry, and others of no probability
    idx[1, 0] = -1
    used = idx >= 0
    z = torch.log_softmax(x.double(), 1)
    lq = torch.log_softmax(torch.where(used, lp.double(), -INF), 1)
    q = lq.exp()
    logp = z.gather(1, torch.where(used, idx, 0))
    want = torch.where(q > 0, q * (lq - logp), 0.0).sum(1)
    tol = (_terms(v) + 64) * U + 8 * U * torch.where(q > 0, q * (lq.abs() + logp.abs()), 0.0).sum(1) + 16 * U * (1 + want.abs())
    rows = L.topk_distillation(x, idx, lp, tail=False, reduction="none")
    _within(rows, want, tol, "rows")
    p = z.exp()
    share = torch.zeros_like(p).scatter_add_(1, torch.where(used, idx, 0), q)
    wd = w.double()[:, None]
    _, dx = L.topk_distillation_grad(x, idx, lp, tail=False, weight=w, reduction="sum")
    g, gtol = wd * (p - share), wd * (2 * _terms(v) + 160 + 64) * U * (p + share)
    _within(dx, g, gtol + 8 * U * g.abs() + 2.0 ** -126, "dx")
    xg = x.detach().requires_grad_()
    d2, = torch.autograd.grad(L.topk_distillation(xg, idx, lp, tail=False, weight=w, reduction="sum"), xg)
    _within(d2, g, gtol + 8 * U * g.abs() + 2.0 ** -126, "dx")


@pytest.mark.parametrize("t,v", [(5, 40), (21000, 40), (700, 900), (1025, 900), (17000, 100), (3, 100000)])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("mean", [0, 1])
def test_the_sum_of_the_weights_is_written(t, v, weighted, mean):
    """by both entry points whenever there is room for it, with and without a loss; U relative: a 64-bit sum rounded once"""
    from scmomer_amd._lib import check, lib
    k = 3
    x, idx, lp, w = _case(t, v, k, torch.float32, t + v)
    want = w.double().sum() if weighted else torch.tensor(float(t), dtype=torch.float64, device=DEV)
    p = lambda a: a.data_ptr() if a is not None else None
    head = (p(x), 0, v, t, v, 1.0, p(idx), p(lp), k, 1, p(w) if weighted else None, mean)
    rows = torch.empty(t, device=DEV)
    tape = torch.empty(max(1, lib.scm_topk_distill_tape_floats(t, v, k)), device=DEV)
    ws = torch.empty(lib.scm_topk_distill_ws_floats(t, v) + 2, device=DEV)
    loss, dx = torch.empty((), device=DEV), torch.empty_like(x)
    s = torch.cuda.current_stream().cuda_stream
    for out in (None, loss):
        wsum = torch.full((), -7.0, device=DEV)
        check(lib.scm_topk_distill_fwd(*head, p(rows), p(out), p(wsum), p(tape), p(ws), s), "fwd")
        assert abs(wsum.double() - want) <= U * want, out
    wsum = torch.full((), -7.0, device=DEV)
    check(lib.scm_topk_distill_step(*head, 1.0, p(rows), p(loss), p(wsum), p(tape), p(ws), p(dx), s), "step")
    assert abs(wsum.double() - want) <= U * want
