"""topk_distillation and topk_distillation_grad (scm_topk_distill_*) against the definition in 64 bits.

Tolerances, u = 2^-24: lse and lse_R are within n u of the exact values, n as for the scores (V / 64 or V / 256 sequential
additions, + 104 for joins and exponents; + 64 for the named tokens that join afterwards).  A row's loss adds up to 65
terms q (l - logp): each carries q n u and a few roundings of its two parts; r = 1 - sum q is within 2 u, which the
logarithms multiply.  The gradient's terms carry the same relative errors, and the type's half step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
INF = float("inf")


@pytest.fixture(scope="module")
def L():
    from scmomer_amd import logits as m
    return m


def _terms(v):
    return (v / 64 if v <= 2048 else v / 256) + 168


def _exact(x, idx, lp, tau, tail, w=None):
    """-> row loss, gradient of each row's loss in x (f64), and what the tolerances need"""
    z = x.double() / tau
    t, v = z.shape
    used = idx >= 0
    safe = torch.where(used, idx, 0)
    named = torch.zeros(t, v, dtype=torch.int64, device=x.device).scatter_add_(1, safe, used.long()) > 0
    lp = lp.double()
    q = torch.where(used, torch.exp(lp), 0.0)
    tot = q.sum(1, keepdim=True)
    m = z.amax(1, keepdim=True)
    dead = m == -INF
    # from here on relative to the row's maximum: a row near -3.4e38 has a step of 2^75 in 64 bits, which would swallow
    # the logarithm of the sum; the loss and the gradient depend on differences of logits only
    z = torch.where(dead, 0.0, z - m)
    lse = torch.logsumexp(z, 1, keepdim=True)
    rest = z.masked_fill(named, -INF)
    some = (rest > -INF).any(1, keepdim=True)
    lse_r = torch.where(some, torch.logsumexp(torch.where(some, rest, 0.0), 1, keepdim=True), 0.0)
    if tail:
        r = torch.where(some, (1 - tot).clamp(min=0), 0.0)
    else:
        lp = torch.where(tot > 0, lp - torch.log(tot), lp)
        q = torch.where(tot > 0, q / tot, 0.0)
        r = torch.zeros_like(tot)
    logp = z.gather(1, safe) - lse
    terms = torch.where(q > 0, q * (lp - logp), 0.0)
    rl = torch.where(r > 0, torch.log(r) - lse_r + lse, 0.0)
    loss = terms.sum(1) + (r * rl)[:, 0]
    a = q.sum(1, keepdim=True) + r
    p = torch.exp(z - lse)
    share = torch.where(named | ~some, 0.0, torch.exp(rest - lse_r))
    qd = torch.zeros_like(z).scatter_add_(1, safe, q)
    g = (a * p - qd - r * share) / tau
    loss = torch.where(dead[:, 0], 0.0, loss)
    g = torch.where(dead, 0.0, g)
    n = _terms(v)
    # the parts of (lp - logp), each rounded: lp, x / tau and lse; r off by 2 u times its logarithms
    parts = torch.where(q > 0, q * (lp.abs() + logp.abs() + (z.gather(1, safe)).abs()), 0.0).nan_to_num(posinf=0.0, neginf=0.0).sum(1)
    ltol = n * U * a[:, 0] + 8 * U * parts + 4 * U * (1 + rl.abs()[:, 0]) + 8 * U * (r * (lse_r.abs() + lse.abs()))[:, 0]
    gtol = 2 * n * U * (a * p + qd + r * share) / tau + 4 * U * share / tau
    # the exponents: x - m is exact to u |x - m|, and c to u: 80 u of a term above 2^-40
    return loss, g, ltol, gtol + 160 * U * (a * p + r * share) / tau


def _case(t, v, k, dtype, seed, mass=0.9):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(t, v, generator=gen) * 2.5).to(dtype).to(DEV)
    idx = torch.rand(t, v, generator=gen).topk(k, dim=1).indices.to(DEV)
    lp = torch.log(torch.softmax(torch.randn(t, k, generator=gen) * 2, 1) * (mass if k < v else 1.0)).to(DEV)
    w = (torch.rand(t, generator=gen) * 2).to(DEV)
    if t > 2:
        w[1] = 0
    return x, idx, lp, w


def _within(got, want, tol, what):
    off = (got.double() - want).abs()
    ok = (off <= tol) | (got.double() == want)
    assert ok.all(), f"{what}: off by {off[~ok].max()}"


def _check(L, x, idx, lp, w, tau, tail):
    loss, g, ltol, gtol = _exact(x, idx, lp, tau, tail)
    wd = w.double()
    on = wd > 0
    loss, g = torch.where(on, loss, 0.0), torch.where(on[:, None], g, 0.0)
    kw = dict(temperature=tau, tail=tail, weight=w)
    rows = L.topk_distillation(x, idx, lp, reduction="none", **kw)
    _within(rows, wd * loss, wd * ltol + 2 * U * (wd * loss).abs(), "rows")
    small = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126
    for reduction in ("mean", "sum"):
        div = wd.sum() if reduction == "mean" else 1.0
        want, wg = (wd * loss).sum() / div, wd[:, None] * g / div
        tol, wtol = (wd * ltol).sum() / div + 4 * U * (wd * loss).abs().sum() / div, wd[:, None] * gtol / div
        xg = x.detach().requires_grad_()
        out = L.topk_distillation(xg, idx, lp, reduction=reduction, **kw)
        _within(out.detach(), want, tol, reduction)
        dx, = torch.autograd.grad(out, xg, torch.tensor(1.5, device=DEV))
        assert dx.dtype == x.dtype and dx.shape == x.shape
        _within(dx, 1.5 * wg, 1.5 * wtol + (HALF[x.dtype] + 4 * U) * (1.5 * wg).abs() + small, "dx")
        out2, dx2 = L.topk_distillation_grad(x, idx, lp, reduction=reduction, scale=0.25, **kw)
        _within(out2, want, tol, "step " + reduction)
        _within(dx2, 0.25 * wg, 0.25 * wtol + (HALF[x.dtype] + 4 * U) * (0.25 * wg).abs() + small, "step dx")
    gr = torch.linspace(-1, 2, len(w), device=DEV)
    xg = x.detach().requires_grad_()
    dx, = torch.autograd.grad(L.topk_distillation(xg, idx, lp, reduction="none", **kw), xg, gr)
    s = (wd * gr.double())[:, None]
    _within(dx, s * g, s.abs() * gtol + (HALF[x.dtype] + 4 * U) * (s * g).abs() + small, "dx none")


@pytest.mark.parametrize("t,v,k", [(1, 1, 1), (70, 2, 1), (129, 7, 3), (64, 64, 64), (65, 33, 20), (5, 65, 64), (9, 100, 5),
                                   (600, 1000, 16), (3, 2048, 64), (700, 2049, 33), (2, 8192, 64), (2, 8193, 64), (520, 8200, 8),
                                   (3, 50001, 20), (1, 131072, 64), (40, 16906, 5), (2, 300007, 50), (513, 140001, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tail", [True, False])
def test_loss_and_gradient(L, t, v, k, dtype, tail):
    x, idx, lp, w = _case(t, v, k, dtype, 11 * t + v + k)
    _check(L, x, idx, lp, w, 1.0 if t % 2 else 1.7, tail)


# where rows are split, by the elements of a thread in a segment, and from where on they are not
@pytest.mark.parametrize("t,v,k", [(40, 40003, 20), (30, 131072, 64), (63, 16906, 7), (64, 16906, 7), (64, 131072, 20),
                                   (65, 131073, 5), (256, 140001, 3), (257, 50001, 12), (1024, 1500, 9), (1025, 1500, 9),
                                   (1025, 2500, 64), (1024, 5003, 2), (1025, 5003, 2), (256, 16385, 4), (257, 12001, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_few_rows(L, t, v, k, dtype):
    x, idx, lp, w = _case(t, v, k, dtype, t + v)
    _check(L, x, idx, lp, w, 1.0, True)


# short rows in numbers: a thread per row
@pytest.mark.parametrize("t,v,k", [(520, 1, 1), (1100, 2, 2), (3700, 7, 3), (8201, 16, 16), (16900, 33, 20), (32800, 64, 64),
                                   (33001, 64, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_many_short_rows(L, t, v, k, dtype):
    x, idx, lp, w = _case(t, v, k, dtype, t + v)
    _check(L, x, idx, lp, w, 1.3, bool(t % 2))


def _odd_rows(v):
    x, idx, lp, w = _case(14, v, 6, torch.float32, v)
    w[:] = 1
    x[0] = -INF                                   # nothing left
    idx[1, 2:] = -1                               # few entries
    idx[2] = -1                                   # none
    idx[3, 3] = idx[3, 1]                         # named twice, not side by side
    idx[3, 5] = idx[3, 1]
    lp[4, 2] = -INF                               # an entry of probability 0 on a token the student excludes
    x[4, idx[4, 2]] = -INF
    x[5] = torch.finfo(torch.float32).min         # uniform
    x[6] = -INF                                   # the student knows the entries only
    x[6].scatter_(0, idx[6], torch.randn(6, device=DEV))
    x[7].scatter_(0, idx[7], 60.0)                # the student is sure of the entries: p outside near e^-60
    x[8].scatter_(0, idx[8], -80.0)               # or nearly excludes them
    lp[9] = torch.log_softmax(lp[9], 0)           # the entries hold all of the teacher's mass
    x[10, ::2] = -INF                             # some entries excluded: an infinite loss, a finite gradient
    idx[10, 0] = 2
    return x, idx, lp, w


@pytest.mark.parametrize("tail", [True, False])
def test_conventions_of_many_short_rows(L, tail):
    x, idx, lp, w = _odd_rows(40)
    _check(L, x.repeat(1500, 1), idx.repeat(1500, 1), lp.repeat(1500, 1), w.repeat(1500), 1.0, tail)


@pytest.mark.parametrize("v", [40, 700, 9000, 20000])
@pytest.mark.parametrize("tail", [True, False])
def test_conventions(L, v, tail):
    x, idx, lp, w = _odd_rows(v)
    _check(L, x, idx, lp, w, 1.0, tail)
    rows = L.topk_distillation(x, idx, lp, tail=tail, reduction="none")
    assert rows[0] == 0 and abs(rows[2]) <= _terms(v) * U and rows[10] == INF and torch.isfinite(rows[[1, 3, 4, 5, 6, 7, 8, 9]]).all()


@pytest.mark.parametrize("t,v", [(4, 40), (20500, 40), (4, 700), (4, 9000), (600, 9000)])
def test_broken_rows_stay_by_themselves(L, t, v):
    x, idx, lp, w = _case(t, v, 4, torch.float32, v)
    idx[0, 1] = v                                 # outside the vocabulary
    x[2, 3] = float("nan")
    for fused in (False, True):
        if fused:
            loss, dx = L.topk_distillation_grad(x, idx, lp, reduction="sum")
        else:
            xg = x.detach().requires_grad_()
            loss = L.topk_distillation(xg, idx, lp, reduction="sum")
            dx, = torch.autograd.grad(loss, xg)
        assert torch.isnan(loss) and torch.isnan(dx[[0, 2]]).all() and torch.isfinite(dx[[1, 3]]).all()
        # weight 0 keeps them out, unread
        w = torch.ones(t, device=DEV)
        w[[0, 2]] = 0
        if fused:
            loss, dx = L.topk_distillation_grad(x, idx, lp, weight=w)
        else:
            loss = L.topk_distillation(xg, idx, lp, weight=w)
            dx, = torch.autograd.grad(loss, xg)
        assert torch.isfinite(loss) and torch.equal(dx[[0, 2]], torch.zeros_like(dx[[0, 2]])) and torch.isfinite(dx).all()


def test_no_weight_at_all_and_no_rows(L):
    x, idx, lp, _ = _case(5, 90, 3, torch.float32, 1)
    w = torch.zeros(5, device=DEV)
    assert torch.isnan(L.topk_distillation(x, idx, lp, weight=w))
    assert L.topk_distillation(x, idx, lp, weight=w, reduction="sum") == 0
    loss, dx = L.topk_distillation_grad(x, idx, lp, weight=w)
    assert torch.isnan(loss) and torch.equal(dx, torch.zeros_like(dx))
    e = x[:0].detach().requires_grad_()
    loss = L.topk_distillation(e, idx[:0], lp[:0], reduction="sum")
    assert loss == 0 and torch.autograd.grad(loss, e)[0].shape == (0, 90)
    loss, dx = L.topk_distillation_grad(x[:0], idx[:0], lp[:0])
    assert torch.isnan(loss) and dx.shape == (0, 90)


def test_shapes_strides_and_unaligned_rows(L):
    x, idx, lp, w = _case(15, 1003, 9, torch.bfloat16, 5)
    wide = torch.zeros(3, 5, 1010, dtype=torch.bfloat16, device=DEV)
    wide[..., 3:1006] = x.view(3, 5, 1003)
    view = wide[..., 3:1006].detach().requires_grad_()
    shape = lambda a: a.view(3, 5, *a.shape[1:])
    want_x = x.detach().requires_grad_()
    want = L.topk_distillation(want_x, idx, lp, weight=w)
    got = L.topk_distillation(view, shape(idx), shape(lp), weight=shape(w))
    assert torch.equal(want, got)
    g1, = torch.autograd.grad(want, want_x)
    g2, = torch.autograd.grad(got, view)
    assert g2.shape == (3, 5, 1003) and torch.equal(g1, g2.reshape(15, 1003))
    loss, d = L.topk_distillation_grad(view.detach(), shape(idx), shape(lp), weight=shape(w))
    assert torch.equal(loss, want) and d.shape == (3, 5, 1003)
    # entries with a stride of their own
    two = torch.stack([idx, idx], 2)
    assert torch.equal(L.topk_distillation(x, two[..., 0], lp, weight=w), want)


def test_from_a_teacher_to_its_student(L):
    """the entries token_logprobs returns, fed to the loss: the teacher itself has loss 0 and gradient 0 up to rounding"""
    gen = torch.Generator().manual_seed(2)
    for t, v in ((50, 7), (20, 5000)):
        x = (torch.randn(t, v, generator=gen) * 2).to(DEV)
        top = L.token_logprobs(x, k=min(5, v), temperature=1.3)
        for tail in (True, False):
            if tail:
                loss, dx = L.topk_distillation_grad(x, top.top_index, top.top_logprob, temperature=1.3)
                assert abs(loss) <= 8 * _terms(v) * U and dx.abs().max() <= 8 * _terms(v) * U / t
            y = x + 0.5 * torch.randn(t, v, generator=gen).to(DEV)
            assert L.topk_distillation(y, top.top_index, top.top_logprob, temperature=1.3, tail=tail) > 1e-3


def test_gradient_against_differences(L):
    x, idx, lp, w = _case(6, 40, 5, torch.float32, 3)
    v = torch.randn(6, 40, generator=torch.Generator().manual_seed(4)).to(DEV)
    for tail in (True, False):
        f = lambda z: L.topk_distillation(z, idx, lp, weight=w, tail=tail, reduction="none").double().sum()
        _, dx = L.topk_distillation_grad(x, idx, lp, weight=w, tail=tail, reduction="sum")
        h = 2.0 ** -7
        num = (f(x + h * v) - f(x - h * v)) / (2 * h)
        # third derivatives of log-sum-exp along v are below |v|_inf^3 ~ 40 per row, weights below 2
        assert abs(num - (dx.double() * v.double()).sum()) <= 12 * 80 * h * h + 12 * 300 * U / h


def test_repeats_streams_and_graphs(L):
    for t, v, k in ((100, 7, 3), (3, 40000, 20), (600, 3000, 64)):
        x, idx, lp, w = _case(t, v, k, torch.bfloat16, v)

        def all_of(z):
            zg = z.detach().requires_grad_()
            loss = L.topk_distillation(zg, idx, lp, weight=w)
            g, = torch.autograd.grad(loss, zg)
            return [loss.detach(), g, *L.topk_distillation_grad(z, idx, lp, weight=w, temperature=2.0)]
        want = all_of(x)
        xs = x.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())      # after the copy that the other stream reads
        with torch.cuda.stream(side):
            got = all_of(xs)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = all_of(xs)
            graphs.append((g, out))
        for rep in range(3):
            xs.copy_(x.flip(1) if rep % 2 else x)
            want = all_of(xs)
            for g, _ in graphs:
                g.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(want, out)), (t, v, rep)


def test_offsets_past_32_bits(L):
    t, v = 70000, 40000
    row = torch.randn(v, device=DEV).half()
    x = row.expand(t, v).contiguous()
    idx = torch.tensor([5, 39999, 17], device=DEV).expand(t, 3)
    lp = torch.log(torch.tensor([0.5, 0.2, 0.1], device=DEV)).expand(t, 3)
    w = torch.zeros(t, device=DEV)
    w[0] = w[-1] = 1
    loss, dx = L.topk_distillation_grad(x, idx, lp, weight=w)
    assert torch.equal(dx[0], dx[-1]) and not dx[1:-1].any() and dx[0].any()
    xg = x.requires_grad_()
    loss2 = L.topk_distillation(xg, idx, lp, weight=w)
    g, = torch.autograd.grad(loss2, xg)
    assert torch.equal(g, dx) and torch.equal(loss, loss2)


def test_more_rows_than_a_launch(L):
    """the rows behind the first 2^21 against a call of their own"""
    t, v = (1 << 21) + 1001, 65
    x = torch.randn(t, v, device=DEV).half()
    idx = torch.rand(t, v, device=DEV).topk(3, 1).indices
    lp = torch.log_softmax(torch.randn(t, 4, device=DEV), 1)[:, :3].contiguous()
    w = torch.rand(t, device=DEV)
    gr = torch.randn(t, device=DEV)
    def rows(cut):
        z = x[cut].detach().requires_grad_()
        o = L.topk_distillation(z, idx[cut], lp[cut], weight=w[cut], reduction="none")
        g, = torch.autograd.grad(o, z, gr[cut])
        loss, d = L.topk_distillation_grad(x[cut], idx[cut], lp[cut], weight=w[cut], reduction="sum")
        return o.detach(), g, d, loss
    whole = rows(slice(None))
    for cut in (slice(0, 700), slice((1 << 21) - 300, None)):
        part = rows(cut)
        assert all(torch.equal(a[cut], b) for a, b in zip(whole[:3], part[:3])), cut
    assert abs(whole[3].double() - whole[0].double().sum()) <= U * whole[0].double().sum()
    # the mean without weights divides by all rows
    loss, d = L.topk_distillation_grad(x, idx, lp)
    plain, ds = L.topk_distillation_grad(x[-900:], idx[-900:], lp[-900:], reduction="sum")
    want = ds.double() / t
    assert (d[-900:].double() - want).abs().max() <= 2.0 ** -24        # both below the step of a subnormal half


@pytest.mark.parametrize("t", [16384, 16385, 70001, 1_100_000])
def test_sums_over_many_rows(L, t):
    """one workgroup's sum, and parts joined: rows of one known loss each, sums in 64 bits rounded once"""
    gen = torch.Generator().manual_seed(t)
    x = torch.randn(t, 3, generator=gen).to(DEV)
    idx = torch.randint(0, 3, (t, 1), generator=gen).to(DEV)
    lp = torch.full((t, 1), -0.3, device=DEV)
    w = torch.rand(t, generator=gen).to(DEV)
    rows = L.topk_distillation(x, idx, lp, weight=w, reduction="none")
    for reduction, div in (("sum", 1.0), ("mean", w.double().sum())):
        want = rows.double().sum() / div
        for got in (L.topk_distillation(x, idx, lp, weight=w, reduction=reduction),
                    L.topk_distillation_grad(x, idx, lp, weight=w, reduction=reduction)[0]):
            assert abs(got.double() - want) <= 2 * U * abs(want)
    assert abs(L.topk_distillation(x, idx, lp).double() - L.topk_distillation(x, idx, lp, reduction="none").double().mean()) <= 4 * U
    _, dx = L.topk_distillation_grad(x, idx, lp, weight=w)
    _, ds = L.topk_distillation_grad(x, idx, lp, weight=w, reduction="sum")
    # an entry is A p - q - r share with A p, q, r share <= 1, each scaled by the row's weight (and 1 / sum) and rounded
    # before the difference: 2 roundings a part and one of the scale on either side, 3 parts, 2 x 3 x 3 u of the weight
    assert ((dx.double() * w.double().sum() - ds.double()).abs() <= 18 * U * w.double()[:, None]).all()


def test_refusals(L):
    x, idx, lp, w = _case(4, 90, 3, torch.float32, 1)
    f, s = L.topk_distillation, L.topk_distillation_grad
    for bad, err in ((lambda: f(x.double(), idx, lp), TypeError), (lambda: f(x, idx.int(), lp), TypeError),
                     (lambda: f(x, idx, lp.half()), TypeError), (lambda: f(x, idx[:2], lp[:2]), ValueError),
                     (lambda: f(x, idx, lp[:, :2]), ValueError), (lambda: f(x, idx[:, :0], lp[:, :0]), ValueError),
                     (lambda: f(x, idx[0], lp[0]), ValueError), (lambda: f(x, idx.cpu(), lp), ValueError),
                     (lambda: f(x, idx.repeat(1, 22), lp.repeat(1, 22)), ValueError),
                     (lambda: f(x, idx, lp, weight=w[:2]), ValueError), (lambda: f(x, idx, lp, weight=w.double()), TypeError),
                     (lambda: f(x, idx, lp, temperature=-1.0), ValueError), (lambda: f(x, idx, lp, reduction="max"), ValueError),
                     (lambda: s(x, idx, lp, reduction="none"), ValueError),
                     (lambda: f(x, idx, lp.detach().requires_grad_()), ValueError),
                     (lambda: f(x, idx, lp, weight=w.detach().requires_grad_()), ValueError)):
        with pytest.raises(err):
            bad()
