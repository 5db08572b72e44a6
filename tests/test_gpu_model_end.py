"""The operators at a model's end together, as a distillation step uses them, and what autograd is owed by each: a teacher
(norm, head, token_logprobs with alternatives) and a student (norm, head, topk_distillation) against the same step in 64
bits; gradients wanted of any subset of the inputs; a graph kept, used twice, differentiated twice, broken by an in-place
change."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.fixture(scope="module")
def M():
    from types import SimpleNamespace
    from scmomer_amd import logits, norm
    return SimpleNamespace(layer_norm=norm.layer_norm, token_logprobs=logits.token_logprobs,
                           topk_distillation=logits.topk_distillation, topk_distillation_grad=logits.topk_distillation_grad)


def _step64(h_t, h_s, w, b, head_t, head_s, k, tau, weight):
    """teacher entries and the student's loss by torch in 64 bits; -> loss, gradients of h_s, w, b, head_s"""
    ln = torch.nn.functional.layer_norm
    d = h_s.shape[-1]
    h_s, w, b, head_s = (t.double().detach().requires_grad_() for t in (h_s, w, b, head_s))
    top = torch.log_softmax(ln(h_t.double(), (d,), eps=1e-5) @ head_t.double().T / tau, -1).topk(k, -1)
    lp = torch.log_softmax(ln(h_s, (d,), w, b, 1e-5) @ head_s.T / tau, -1)
    q, r = top.values.exp(), 1 - top.values.exp().sum(-1)
    named = torch.zeros_like(lp, dtype=torch.bool).scatter_(-1, top.indices, True)
    rest = torch.logsumexp(lp.masked_fill(named, float("-inf")), -1)
    rows = (q * (top.values - lp.gather(-1, top.indices))).sum(-1) + r * (torch.log(r) - rest)
    loss = (weight.double() * rows).sum() / weight.double().sum()
    return loss.detach(), torch.autograd.grad(loss, (h_s, w, b, head_s)), top


@pytest.mark.parametrize("v", [7, 900, 16906])
@pytest.mark.parametrize("fused", [False, True])
def test_a_distillation_step(M, v, fused):
    """f32 throughout: the products between the operators run in 64 bits and are rounded once to f32 (u relative), so what
    differs from the 64-bit step is the operators' own rounding.  A logit is a sum over d = 200 columns of magnitude
    |h| |head| ~ 1: its error is below (d + 64) u times that, 300 u; the loss and the gradients move with the logits'
    differences, times 1 / tau and the entries' weights below 1: 4 x 300 u of their own scale, and as much again for the
    operators (their own tests); 1e-4 of the largest element is three times that."""
    gen = torch.Generator().manual_seed(v)
    b_, n, d, k, tau = 2, 33, 200, min(3, v - 1), 1.4
    mk = lambda *s, sc=1.0: (torch.randn(*s, generator=gen) * sc).to(DEV)
    h_t, h_s, head_t, head_s = mk(b_, n, d), mk(b_, n, d), mk(v, d, sc=0.15), mk(v, d, sc=0.15)
    w, b = 1 + mk(d, sc=0.2), mk(d, sc=0.1)
    weight = (torch.rand(b_, n, generator=gen) < 0.8).float().to(DEV)
    want, grads, top64 = _step64(h_t, h_s, w, b, head_t, head_s, k, tau, weight)

    class Head(torch.autograd.Function):      # the product in 64 bits, rounded once
        @staticmethod
        def forward(ctx, x, m):
            ctx.save_for_backward(x, m)
            return (x.double() @ m.double().T).float()

        @staticmethod
        def backward(ctx, g):
            x, m = ctx.saved_tensors
            return (g.double() @ m.double()).float(), (g.double().flatten(0, 1).T @ x.double().flatten(0, 1)).float()

    with torch.no_grad():
        t = M.token_logprobs(Head.apply(M.layer_norm(h_t, None, None, 1e-5), head_t), k=k, temperature=tau, entropy=False)
    assert torch.equal(t.top_index, top64.indices)
    leaves = [z.detach().requires_grad_() for z in (h_s, w, b, head_s)]
    logits = Head.apply(M.layer_norm(leaves[0], leaves[1], leaves[2], 1e-5), leaves[3])
    if fused:
        loss, dl = M.topk_distillation_grad(logits, t.top_index, t.top_logprob, temperature=tau, weight=weight)
        got = torch.autograd.grad(logits, leaves, dl)
    else:
        loss = M.topk_distillation(logits, t.top_index, t.top_logprob, temperature=tau, weight=weight)
        got = torch.autograd.grad(loss, leaves)
    assert abs(loss.double() - want) <= 1e-4 * abs(want)
    for g, r in zip(got, grads):
        assert (g.double() - r).abs().max() <= 1e-4 * r.abs().max()


@pytest.mark.parametrize("want", range(1, 8))
def test_layer_norm_gradients_of_any_subset(M, want):
    gen = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, generator=gen).to(DEV) for s in ((9, 70), (70,), (70,)))
    dy = torch.randn(9, 70, generator=gen).to(DEV)
    every = [z.detach().requires_grad_() for z in (x, w, b)]
    full = torch.autograd.grad(M.layer_norm(*every), every, dy)
    some = [z.detach().requires_grad_(bool(want >> i & 1)) for i, z in enumerate((x, w, b))]
    y = M.layer_norm(*some)
    got = torch.autograd.grad(y, [z for z in some if z.requires_grad], dy)
    assert all(torch.equal(g, f) for g, f in zip(got, [f for i, f in enumerate(full) if want >> i & 1]))
    if want >> 2:      # a bias without a weight
        bb = b.detach().requires_grad_()
        db, = torch.autograd.grad(M.layer_norm(x, None, bb), bb, dy)
        assert torch.equal(db, full[2])


def _calls(M):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(6, 300, generator=gen).to(DEV)
    idx = torch.rand(6, 300, generator=gen).topk(4, 1).indices.to(DEV)
    lp = torch.full((6, 4), -2.0, device=DEV)
    tg = torch.randint(0, 300, (6,), generator=gen).to(DEV)
    w = torch.ones(300, device=DEV)
    return x, {"norm": lambda z: M.layer_norm(z, w).pow(2).sum(), "score": lambda z: M.token_logprobs(z, tg, k=2).logprob.sum(),
               "lse": lambda z: M.token_logprobs(z, entropy=False).lse.sum(),
               "top": lambda z: M.token_logprobs(z, k=3, entropy=False).top_logprob[:, 1].sum(),
               "distill": lambda z: M.topk_distillation(z, idx, lp),
               "rows": lambda z: M.topk_distillation(z, idx, lp, reduction="none").sum()}


@pytest.mark.parametrize("name", ["norm", "score", "lse", "top", "distill", "rows"])
def test_graph_used_twice_and_accumulated(M, name):
    x, calls = _calls(M)
    f = calls[name]
    z = x.detach().requires_grad_()
    loss = f(z)
    a, = torch.autograd.grad(loss, z, retain_graph=True)
    b, = torch.autograd.grad(loss, z)
    assert torch.equal(a, b) and a.abs().max() > 0
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, z)          # the graph is gone
    z = x.detach().requires_grad_()
    f(z).backward()
    f(z).backward()
    assert torch.equal(z.grad, a + a)


@pytest.mark.parametrize("name", ["norm", "score", "distill"])
def test_second_derivatives_are_refused(M, name):
    x, calls = _calls(M)
    z = x.detach().requires_grad_()
    first, = torch.autograd.grad(calls[name](z), z, create_graph=True)
    plain, = torch.autograd.grad(calls[name](z), z)
    assert torch.equal(first.detach(), plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), z)


@pytest.mark.parametrize("name", ["norm", "score", "distill"])
def test_an_input_changed_in_place_is_noticed(M, name):
    x, calls = _calls(M)
    z = x.detach().requires_grad_()
    y = z * 1.0
    loss = calls[name](y)
    y.add_(1.0)
    with pytest.raises(RuntimeError):
        loss.backward()


@pytest.mark.parametrize("name", ["norm", "score", "distill"])
def test_saved_tensors_may_move(M, name):
    """under hooks that keep saved tensors on the host (their storage is another one in the backward pass)"""
    x, calls = _calls(M)
    z = x.detach().requires_grad_()
    want, = torch.autograd.grad(calls[name](z), z)
    with torch.autograd.graph.save_on_cpu():
        loss = calls[name](z)
    got, = torch.autograd.grad(loss, z)
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", ["norm", "score", "distill"])
def test_capture_beside_an_eager_graph_of_the_same_leaf(M, name):
    """The eager graph keeps the leaf's accumulator on the default stream, which cannot take part in a capture: the backward
    pass is refused; a gradient of other tensors, and the same call once the eager graph is gone, are captured."""
    x, calls = _calls(M)
    z = x.detach().requires_grad_()
    alive = calls[name](z)
    want, = torch.autograd.grad(alive, z, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other = z.detach().requires_grad_()
        got, = torch.autograd.grad(calls[name](other), other)
        with pytest.raises(RuntimeError, match="default stream"):
            torch.autograd.grad(calls[name](z), z)
    del alive
    gc.collect()          # the refusal's traceback holds a graph too
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        got2, = torch.autograd.grad(calls[name](z), z)
    for _ in range(3):
        graph.replay()
        again.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(got2, want)
        got.zero_()
        got2.zero_()
        torch.cuda.synchronize()


@pytest.mark.parametrize("t,v", [(5, 1), (600, 1), (5, 40), (20600, 40), (5, 700), (300, 9000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_one_token_with_all_the_probability(M, t, v, dtype):
    """its log probability is 0 and nothing has a gradient, exactly"""
    x = torch.full((t, v), float("-inf"), device=DEV, dtype=dtype)
    at = torch.randint(0, v, (t,), device=DEV)
    x.scatter_(1, at[:, None], torch.randn(t, 1, device=DEV).to(dtype))
    z = x.requires_grad_()
    o = M.token_logprobs(z, at, k=1, temperature=0.7)
    g = torch.randn(3, t, device=DEV)
    dx, = torch.autograd.grad((o.logprob, o.entropy), z, (g[0], g[1]))
    assert torch.equal(o.top_index[:, 0], at) and not o.logprob.any() and not o.entropy.any() and not dx.any()
    lp = -torch.rand(t, 1, device=DEV)
    for tail in (True, False):
        rows = M.topk_distillation(z, at[:, None], lp, temperature=0.7, tail=tail, reduction="none")
        dz, = torch.autograd.grad(rows, z, g[2])
        _, dx = M.topk_distillation_grad(z, at[:, None], lp, temperature=0.7, tail=tail, weight=g[2].abs())
        assert torch.isfinite(rows).all() and not dz.any() and not dx.any()


def test_inference_mode_and_no_grad(M):
    x, calls = _calls(M)
    z = x.detach().requires_grad_()
    for name, f in calls.items():
        with torch.no_grad():
            a = f(z)
        with torch.inference_mode():
            b = f(z)
        assert not a.requires_grad and torch.equal(a, b) and torch.equal(a, f(z).detach()), name


def test_two_threads_at_once(M):
    """each on a stream of its own"""
    import threading
    x, calls = _calls(M)
    want = {}
    for name, f in calls.items():
        z = x.detach().requires_grad_()
        want[name] = torch.autograd.grad(f(z), z)[0]
    torch.cuda.synchronize()
    errors = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                for name, f in calls.items():
                    z = x.detach().requires_grad_()
                    g, = torch.autograd.grad(f(z), z)
                    s.synchronize()
                    if not torch.equal(g, want[name]):
                        errors.append(name)
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
