"""token_logprobs (scm_score_fwd / scm_score_bwd) against the definition in 64 bits.

Tolerances, u = 2^-24: a thread adds at most V / 64 (one wave) or V / 256 terms in a row before a tree of 8 + 6 joins,
so s is within n u of the exact sum, n = V / 64 + 64 (V <= 2048) or V / 256 + 64, the exponentials' own two roundings and
the rescalings among the 64.  A term 2^d carries d's rounding: |d| u relative; terms with |d| > 40 weigh nothing, so at
most 40 u more.  lse, logprob: (n + 40) u absolute plus 4 roundings of the result and of x - m.  Entropy: the same error
relative to each of its two parts.  Gradient: the same error relative to every term, and the type's half step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
INF = float("inf")


@pytest.fixture(scope="module")
def token_logprobs():
    from scmomer_amd.logits import token_logprobs as f
    return f


def _terms(v):
    return (v / 64 if v <= 2048 else v / 256) + 104


def _order(x, k):
    """the k largest per row by (value, lowest index), NaN first, in plain sorting"""
    key = torch.where(torch.isnan(x), INF, x.double())
    nan_first = torch.sort(torch.isnan(x).to(torch.int8), dim=-1, descending=True, stable=True).indices
    by_value = torch.sort(key.gather(-1, nan_first), dim=-1, descending=True, stable=True).indices
    return nan_first.gather(-1, by_value)[..., :k]


def _exact(x, target, k, tau, ignore=-100):
    z = x.double() / tau
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -INF, 0.0, m)
    s = torch.exp(z - m).sum(-1, keepdim=True)
    lse = m + torch.log(s)
    logp = torch.where(lse == -INF, -INF, (z - m) - torch.log(s))     # z - lse would lose log s next to 3e38
    p = torch.exp(logp)
    ent = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    r = dict(lse=lse[..., 0], logp=logp, p=p, ent=ent)
    if target is not None:
        safe = target.clamp(0, x.shape[-1] - 1)
        lp = logp.gather(-1, safe[..., None])[..., 0]
        lp = torch.where((target < 0) | (target >= x.shape[-1]), float("nan"), lp)
        r["lp"] = torch.where(target == ignore, 0.0, lp)
    r["idx"] = _order(x, k)
    r["top"] = logp.gather(-1, r["idx"])
    return r


def _close(got, want, tol, what):
    same = (got.double() == want) | (torch.isnan(got) & torch.isnan(want))
    off = (got.double() - want).abs()
    assert (same | (off <= tol)).all(), f"{what}: off by {off[~same].max()} (tolerance {tol if isinstance(tol, float) else tol.max()})"


def _check(out, x, target, k, tau):
    r = _exact(x, target, k, tau)
    n = _terms(x.shape[-1])
    span = 4 * U * (x.double() / tau).masked_fill(~torch.isfinite(x), 0.0).abs().amax(-1)
    _close(out.lse, r["lse"], n * U + span, "lse")
    near = lambda lp: n * U + 8 * U * lp.abs().masked_fill(~torch.isfinite(lp), 0.0)      # x - m and the result rounded
    if target is not None:
        _close(out.logprob, r["lp"], near(r["lp"]), "logprob")
    if out.entropy is not None:
        _close(out.entropy, r["ent"], 2 * n * U * (1 + r["ent"].abs()), "entropy")
    if k:
        assert torch.equal(out.top_index, r["idx"])
        _close(out.top_logprob, r["top"], near(r["top"]), "top")
    return r


def _logits(t, v, dtype, seed, scale=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(t, v, generator=gen) * scale).to(dtype).to(DEV)
    target = torch.randint(0, v, (t,), generator=gen).to(DEV)
    return x, target


SIZES = [(1, 1, 1), (70, 2, 2), (129, 7, 3), (64, 64, 64), (65, 33, 20), (63, 64, 1), (5, 65, 64), (9, 100, 5), (600, 1000, 20),
         (3, 2047, 64), (3, 2048, 7), (700, 2049, 33), (2, 8192, 64), (1, 8193, 64), (520, 8200, 8), (3, 50001, 20),
         (1, 131072, 64), (40, 16906, 5), (513, 20000, 0), (2, 300007, 50), (40, 300, 64), (33, 512, 33), (12, 513, 64),
         (600, 5000, 64), (520, 9000, 64), (515, 30000, 33), (514, 100000, 40)]


@pytest.mark.parametrize("t,v,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scores(token_logprobs, t, v, k, dtype):
    x, target = _logits(t, v, dtype, t * 7 + v)
    if t > 2:
        target[1] = -100
    for tau in (1.0, 0.7):
        _check(token_logprobs(x, target, k=k, temperature=tau), x, target, k, tau)


# short rows in numbers (a thread per row), and as many as not yet
@pytest.mark.parametrize("t,v,k", [(2100, 17, 17), (2200, 17, 3), (4097, 33, 20), (4300, 33, 20), (8192, 64, 5), (8193, 64, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scores_of_many_short_rows(token_logprobs, t, v, k, dtype):
    x, target = _logits(t, v, dtype, t + v)
    _check(token_logprobs(x, target, k=k), x, target, k, 1.0)


# where rows are split, by the elements of a thread in a segment, and from where on they are not
@pytest.mark.parametrize("t,v,k", [(40, 16906, 20), (40, 40003, 20), (40, 40003, 0), (30, 131072, 64), (63, 65537, 64),
                                   (64, 9001, 64), (64, 131072, 20), (127, 131072, 20),
                                   (128, 131072, 20), (128, 131073, 20), (200, 70001, 40), (255, 140001, 8),
                                   (256, 140001, 3), (257, 9000, 64), (512, 2500, 3), (513, 2500, 3), (513, 2500, 0),
                                   (1024, 5003, 20), (1025, 5003, 20), (1025, 1500, 9), (1025, 2500, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_of_few_rows(token_logprobs, t, v, k, dtype):
    x, target = _logits(t, v, dtype, t + v)
    _check(token_logprobs(x, target, k=k), x, target, k, 1.0)


@pytest.mark.parametrize("v", [7, 64, 100, 1500, 9000, 40000])
def test_masks_ties_and_special_values(token_logprobs, v):
    x, target = _logits(12, v, torch.float32, v)
    k = min(v, 17)
    x[0] = -INF                                  # nothing left
    x[1] = torch.finfo(torch.float32).min        # masked by the type's lowest value throughout: uniform
    x[2, 1:] = -INF                              # one token left
    x[3, ::2] = -INF
    x[4] = 0.0                                   # all equal
    x[5] = torch.where(torch.arange(v, device=DEV) % 2 == 0, 0.0, -0.0)
    x[6, v // 2] = float("nan")
    x[7, v - 1] = INF
    x[8, 1:] = torch.finfo(torch.float32).min
    x[9] = torch.arange(v, device=DEV).float() * 0.01          # ascending: every thread's last chunk is its largest
    x[10] = -torch.arange(v, device=DEV).float() * 0.01
    x[11, 0] = 1e30
    out = token_logprobs(x, target, k=k)
    keep = [0, 1, 2, 3, 4, 5, 8, 9, 10, 11]
    part = type(out)(*(None if o is None else o[keep] for o in out))
    _check(part, x[keep], target[keep], k, 1.0)
    assert out.entropy[0] == 0 and out.lse[0] == -INF and torch.equal(out.top_index[0], torch.arange(k, device=DEV))
    for row in (6, 7):
        assert torch.isnan(out.logprob[row]) and torch.isnan(out.entropy[row]) and torch.isnan(out.lse[row])
        assert torch.isnan(out.top_logprob[row]).all()
    assert torch.equal(out.top_index[[6, 7]], _order(x[[6, 7]], k))


@pytest.mark.parametrize("t,v", [(2, 3000), (600, 3000), (2, 70000), (520, 30000)])
def test_large_values_in_few_threads(token_logprobs, t, v):
    """all large logits in the elements of one or two threads: more candidates than the threads' maxima tell apart"""
    x = torch.randn(t, v, generator=torch.Generator().manual_seed(v)).to(DEV)
    i = torch.arange(v, device=DEV)
    x[0] += 50.0 * ((i // 4) % 64 == 3)
    x[1] += 50.0 * ((i // 4) % 256 == 200)
    _check(token_logprobs(x, None, k=64), x, None, 64, 1.0)


def test_bfloat16_ties(token_logprobs):
    """bf16 logits of a wide vocabulary repeat values: equal logits come in index order"""
    x = (torch.randn(6, 120000, generator=torch.Generator().manual_seed(1)) * 0.01).bfloat16().to(DEV)
    x[3, :60000] = -INF
    x[4] = -INF
    x[4, 100::7777] = 1.0
    _check(token_logprobs(x, None, k=64, entropy=False), x, None, 64, 1.0)


def test_targets(token_logprobs):
    x, target = _logits(9, 50, torch.float32, 5)
    target[:4] = torch.tensor([-100, -1, 50, 7], device=DEV)
    x[3, 7] = -INF
    out = token_logprobs(x, target)
    assert out.logprob[0] == 0 and torch.isnan(out.logprob[1:3]).all() and out.logprob[3] == -INF
    assert torch.isfinite(out.logprob[4:]).all() and out.top_index is None and out.top_logprob is None
    out = token_logprobs(x, target, ignore_index=7, entropy=False)
    assert out.logprob[3] == 0 and torch.isnan(out.logprob[0]) and out.entropy is None
    out = token_logprobs(x)
    assert out.logprob is None and out.lse.shape == (9,)


def test_shapes_and_strides(token_logprobs):
    gen = torch.Generator().manual_seed(4)
    wide = torch.randn(3, 5, 311, generator=gen).to(torch.bfloat16).to(DEV)
    target = torch.randint(0, 207, (3, 5), generator=gen).to(DEV)
    a = token_logprobs(wide[..., 3:210], target, k=4)
    b = token_logprobs(wide[..., 3:210].contiguous(), target, k=4)
    assert a.logprob.shape == (3, 5) and a.top_index.shape == (3, 5, 4)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    t = wide[0].t()                                      # classes not contiguous
    assert torch.equal(token_logprobs(t, k=2).top_index, token_logprobs(t.contiguous(), k=2).top_index)
    e = token_logprobs(wide[0, :1].expand(6, 311), k=3)  # one row for all
    assert (e.top_index == e.top_index[0]).all() and (e.lse == e.lse[0]).all()
    one = token_logprobs(wide[0, 0], torch.tensor(5, device=DEV), k=2)
    assert one.logprob.shape == () and one.top_index.shape == (2,)
    none = token_logprobs(wide[:0], target[:0], k=2)
    assert none.logprob.shape == (0, 5) and none.top_index.shape == (0, 5, 2)
    # rows behind the ones that are given stay unread and unwritten
    big = torch.full((4, 100), float("nan"), device=DEV)
    big[:2] = 1.0
    assert torch.isfinite(token_logprobs(big[:2]).lse).all()


def _grad(token_logprobs, x, target, k, tau, gl, gh, gz, gt):
    x = x.detach().requires_grad_()
    o = token_logprobs(x, target, k=k, temperature=tau)
    outs = [(o.logprob, gl), (o.entropy, gh), (o.lse, gz)] + ([(o.top_logprob, gt)] if k else [])
    outs = [(a, b) for a, b in outs if b is not None]
    return torch.autograd.grad([a for a, _ in outs], x, [b for _, b in outs])[0]


def _check_grad(dx, x, target, k, tau, gl, gh, gz, gt):
    r = _exact(x, target, k, tau)
    t, v = x.shape
    g = torch.zeros(t, v, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(g)
    if gl is not None:
        on = (target != -100).double() * gl.double()
        g.scatter_add_(1, target.clamp(min=0)[:, None], on[:, None])
    if gt is not None and k:
        g.scatter_add_(1, r["idx"], gt.double())
    tot = g.sum(1, keepdim=True) - (gz.double()[:, None] if gz is not None else 0)
    mag = g.abs() + r["p"] * (g.abs().sum(1, keepdim=True) + (gz.double().abs()[:, None] if gz is not None else 0))
    dz = g - r["p"] * tot
    if gh is not None:
        lp = torch.where(r["p"] > 0, r["logp"], 0.0)
        dz = dz - gh.double()[:, None] * r["p"] * (lp + r["ent"][:, None])
        mag = mag + gh.double().abs()[:, None] * r["p"] * (lp.abs() + r["ent"][:, None] + 1)
    want = dz / tau
    tol = 4 * _terms(v) * U * mag / tau + HALF[x.dtype] * want.abs() + (2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    _close(dx, want, tol, "dx")


@pytest.mark.parametrize("t,v,k", [(70, 7, 2), (3, 64, 64), (65, 20, 0), (5, 65, 64), (600, 1000, 5), (4, 2049, 20),
                                   (3, 8193, 64), (1021, 5001, 3), (2, 131072, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients(token_logprobs, t, v, k, dtype):
    x, target = _logits(t, v, dtype, t + 3 * v, 2.0)
    x[0, ::3] = -INF
    target[0] = 1
    if k:
        target[1] = _order(x[1:2], 1)[0, 0]          # the target is the most likely token
    if t > 2:
        target[2] = -100
    gen = torch.Generator().manual_seed(v)
    gl, gh, gz = (torch.randn(t, generator=gen).to(DEV) for _ in range(3))
    gt = torch.randn(t, k, generator=gen).to(DEV) if k else None
    for tau, g in ((1.0, (gl, None, None, None)), (0.7, (gl, gh, gz, gt)), (1.0, (None, gh, None, gt))):
        if k or any(a is not None for a in g):
            _check_grad(_grad(token_logprobs, x, target, k, tau, *g), x, target, k, tau, *g)


@pytest.mark.parametrize("v", [20, 300, 9000])
def test_gradients_of_empty_masked_and_broken_rows(token_logprobs, v):
    x, target = _logits(6, v, torch.float32, v)
    x[0] = -INF
    x[1, 3] = float("nan")
    x[2] = torch.finfo(torch.float32).min
    x[3, 1:] = -INF
    target[4] = v
    gl, gh = torch.ones(6, device=DEV), torch.ones(6, device=DEV)
    dx = _grad(token_logprobs, x, target, 3, 1.0, gl, gh, gl, torch.ones(6, 3, device=DEV))
    assert torch.equal(dx[0], torch.zeros_like(dx[0])) and torch.isnan(dx[1]).all() and torch.isnan(dx[4]).all()
    assert torch.isfinite(dx[[2, 3, 5]]).all()


@pytest.mark.parametrize("t,v,k", [(3600, 7, 2), (10300, 20, 20), (10200, 20, 0), (32800, 64, 3)])
def test_gradients_of_many_short_rows(token_logprobs, t, v, k):
    x, target = _logits(t, v, torch.float32, t)
    x[::6] = -INF
    x[2::6] = torch.finfo(torch.float32).min
    x[3::6, 1:] = -INF
    target[5] = -100
    g = torch.randn(3, t, generator=torch.Generator().manual_seed(v)).to(DEV)
    gt = torch.randn(t, k, generator=torch.Generator().manual_seed(v + 1)).to(DEV) if k else None
    dx = _grad(token_logprobs, x, target, k, 1.0, g[0], g[1], g[2], gt)
    assert torch.equal(dx[::6], torch.zeros_like(dx[::6]))
    keep = torch.arange(t, device=DEV) % 6 != 0
    _check_grad(dx[keep], x[keep], target[keep], k, 1.0, g[0][keep], g[1][keep], g[2][keep], gt[keep] if k else None)


def test_gradient_of_an_expanded_row(token_logprobs):
    x, target = _logits(1, 400, torch.float32, 8)
    xe = x.detach().requires_grad_()
    tg = torch.arange(11, device=DEV)
    dx, = torch.autograd.grad(token_logprobs(xe.expand(11, 400), tg).logprob.sum(), xe)
    p = torch.softmax(x.double(), 1)[0]
    want = (torch.arange(400, device=DEV) < 11).double() - 11 * p
    assert ((dx[0].double() - want).abs() <= 11 * 400 * U).all()


def test_gradient_against_differences(token_logprobs):
    x, target = _logits(4, 30, torch.float32, 10, 1.0)
    gen = torch.Generator().manual_seed(3)
    gl, gh = torch.randn(4, generator=gen).to(DEV), torch.randn(4, generator=gen).to(DEV)
    v = torch.randn(4, 30, generator=gen).to(DEV)

    def f(z):
        o = token_logprobs(z, target)
        return ((o.logprob * gl).double() + (o.entropy * gh).double()).sum()
    h = 2.0 ** -7
    num = (f(x + h * v) - f(x - h * v)) / (2 * h)
    ana = (_grad(token_logprobs, x, target, 0, 1.0, gl, gh, None, None).double() * v.double()).sum()
    # third derivatives of a softmax along v are below 10 |v|^3 here; the values are off by 200 u each
    assert abs(num - ana) <= 200 * h * h + 4 * 30 * 200 * U / h


def test_results_repeat_capture_and_streams(token_logprobs):
    for t, v, k in ((100, 7, 2), (3, 40000, 20), (600, 3000, 8)):
        x, target = _logits(t, v, torch.bfloat16, v)
        gl, gh = torch.randn(t, device=DEV), torch.randn(t, device=DEV)

        def both(z):
            z = z.detach().requires_grad_()
            o = token_logprobs(z, target, k=k)
            g, = torch.autograd.grad((o.logprob, o.entropy), z, (gl, gh))
            return [a.detach() for a in o] + [g]
        want = both(x)
        xs = x.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())      # after the copy that the other stream reads
        with torch.cuda.stream(side):
            got = both(xs)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        graphs = []
        for _ in range(2):                                 # two graphs, replayed in turn
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = both(xs)
            graphs.append((g, out))
        for rep in range(3):
            xs.copy_(x.flip(1) if rep % 2 else x)
            want = both(xs)
            for g, out in graphs:
                g.replay()
            torch.cuda.synchronize()
            for g, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(want, out)), (t, v, rep)


def test_offsets_past_32_bits(token_logprobs):
    t, v = 70000, 40000                                     # 2.8e9 elements
    row = torch.randn(v, device=DEV).half()
    x = row.expand(t, v).contiguous()
    x[-1, 5] = 20.0
    target = torch.full((t,), 5, device=DEV)
    o = token_logprobs(x, target, k=2)
    assert o.top_index[-1, 0] == 5 and (o.lse[:-1] == o.lse[0]).all()
    one = token_logprobs(x[-1:].clone(), target[-1:], k=2)
    # one row alone is split over workgroups: its sum is added up in another order
    assert (one.lse - o.lse[-1:]).abs() <= 2 * _terms(v) * U + 8 * U * 20
    assert torch.equal(one.top_index, o.top_index[-1:])
    xg = x.requires_grad_()
    g, = torch.autograd.grad(token_logprobs(xg, target, entropy=False).logprob.sum(), xg)
    assert torch.equal(g[0], g[t // 2]) and abs(g[-1, 5].item()) < 1e-3


def test_more_rows_than_a_launch(token_logprobs):
    """the rows behind the first 2^21 against a call of their own"""
    t, v, k = (1 << 21) + 1001, 65, 3
    x = torch.randn(t, v, device=DEV).half()
    target = torch.randint(0, v, (t,), device=DEV)
    gl, gt = torch.randn(t, device=DEV), torch.randn(t, k, device=DEV)
    def both(z, tg, a, b):
        z = z.detach().requires_grad_()
        o = token_logprobs(z, tg, k=k)
        g, = torch.autograd.grad((o.logprob, o.entropy, o.top_logprob), z, (a, a, b))
        return [e.detach() for e in o] + [g]
    whole = both(x, target, gl, gt)
    for cut in (slice(0, 700), slice((1 << 21) - 300, None)):
        part = both(x[cut], target[cut], gl[cut], gt[cut])
        assert all(torch.equal(a[cut], b) for a, b in zip(whole, part)), cut


def test_refusals(token_logprobs):
    x = torch.randn(3, 20, device=DEV)
    t = torch.zeros(3, dtype=torch.int64, device=DEV)
    for bad, err in ((lambda: token_logprobs(x.double()), TypeError), (lambda: token_logprobs(x, t.int()), TypeError),
                     (lambda: token_logprobs(x, t[:2]), ValueError), (lambda: token_logprobs(x, t.cpu()), ValueError),
                     (lambda: token_logprobs(x, k=21), ValueError), (lambda: token_logprobs(x, k=-1), ValueError),
                     (lambda: token_logprobs(torch.zeros(2, 100, device=DEV), k=65), ValueError),
                     (lambda: token_logprobs(x, temperature=0.0), ValueError),
                     (lambda: token_logprobs(x, temperature=math.inf), ValueError),
                     (lambda: token_logprobs(x, temperature=math.nan), ValueError),
                     (lambda: token_logprobs(x[:, :0]), ValueError)):
        with pytest.raises(err):
            bad()
