"""LayerNorm of any width (norm.layer_norm, scm_norm_fwd / scm_norm_bwd) against the formula in 64 bits.

Tolerances, with u = 2^-24 (half a step of f32) and e the half step of the stored type (bf16 2^-8, fp16 2^-11, f32 u):
  y   a sum of D terms over a tree of depth <= 16 + log2(64 * 16) < 27 additions per path bounds the error of the
      mean by 27 u mean|x| and that of the variance by 29 u relative plus the mean's; (x - mu) rstd then is within
      32 u (|xh| + rstd (|mu| + mean|x|)) of the exact value; gamma, beta add two more roundings.
  dx  the same for the two means over gamma dy and gamma dy xh, times rstd.
  dgamma, dbeta  sums over T rows: <= (T / workgroups + 40) additions a path, each term within the error of xh.
Every bound is taken twice as wide as counted, once for the products' own roundings."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def layer_norm():
    from scmomer_amd.norm import layer_norm as f
    return f


def _exact(x, w, b, eps, dy):
    x, dy = x.double(), dy.double()
    d = x.shape[-1]
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    rs = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * rs
    g = dy * w
    dx = rs * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dict(y=xh * w + b, dx=dx, dw=(dy * xh).sum(0), db=dy.sum(0), mu=mu, rs=rs, xh=xh, g=g, w=w, b=b, x=x, dy=dy)


def _check(got, r, out_dtype, x_dtype):
    spread = r["xh"].abs() + r["rs"] * (r["mu"].abs() + r["x"].abs().mean(-1, keepdim=True))   # error of xh / (32 u)
    exh = 64 * U * spread
    tol = exh * r["w"].abs() + 4 * U * r["b"].abs() + HALF[out_dtype] * r["y"].abs()
    tol = tol + (2.0 ** -25 if out_dtype == torch.float16 else 0)            # fp16's smallest step
    assert ((got["y"].double() - r["y"]).abs() <= tol).all(), "y"
    if "dx" in got:
        ga = r["g"].abs().mean(-1, keepdim=True)
        part = r["g"].abs() + ga + (1 + r["xh"].abs()) * (r["g"] * r["xh"]).abs().mean(-1, keepdim=True)
        tol = r["rs"] * (128 * U * part + exh * ga * (1 + r["xh"].abs()) + exh.mean(-1, keepdim=True) * r["g"].abs())
        tol = tol + HALF[x_dtype] * r["dx"].abs() + (2.0 ** -25 if x_dtype == torch.float16 else 0)
        assert ((got["dx"].double() - r["dx"]).abs() <= tol).all(), "dx"
    steps = 2 * (r["x"].shape[0] / 256 + 40) * U
    if "dw" in got:
        tol = steps * (r["dy"] * r["xh"]).abs().sum(0) + (exh * r["dy"].abs()).sum(0)
        assert ((got["dw"].double() - r["dw"]).abs() <= tol).all(), "dw"
    if "db" in got:
        assert ((got["db"].double() - r["db"]).abs() <= steps * r["dy"].abs().sum(0)).all(), "db"


def _case(t, d, dtype, seed, shift=0.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(t, d, generator=gen) * 1.7 + shift).to(dtype).to(DEV)
    dy = torch.randn(t, d, generator=gen).to(DEV)
    w = (1 + 0.3 * torch.randn(d, generator=gen)).to(DEV)
    b = (0.2 * torch.randn(d, generator=gen)).to(DEV)
    return x, dy, w, b


def _run(layer_norm, x, w, b, eps, dy, out_dtype=None):
    x = x.detach().requires_grad_()
    w, b = w.detach().requires_grad_(), b.detach().requires_grad_()
    y = layer_norm(x, w, b, eps, out_dtype=out_dtype)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy.to(y.dtype))
    return dict(y=y.detach(), dx=dx, dw=dw, db=db)


# every lane count and both of its sides, odd widths, one row to more rows than workgroups
@pytest.mark.parametrize("t,d", [(1, 1), (3, 2), (5, 7), (33, 127), (700, 128), (9000, 129), (257, 200), (16, 256), (64, 257),
                                 (100, 511), (2100, 640), (31, 1024), (1030, 1025), (7, 1111), (600, 2049), (3, 4096),
                                 (2, 4097), (520, 8191), (1, 8193), (3, 16384), (2, 16383)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_forward_and_gradients(layer_norm, t, d, dtype):
    x, dy, w, b = _case(t, d, dtype, 1000 * t + d)
    got = _run(layer_norm, x, w, b, 1e-5, dy)
    assert got["y"].dtype == dtype and got["dx"].dtype == dtype and got["dw"].dtype == torch.float32
    _check(got, _exact(x, w, b, 1e-5, dy.to(dtype)), dtype, dtype)
    with torch.no_grad():      # the form without statistics gives the same bits
        assert torch.equal(layer_norm(x, w, b, 1e-5), got["y"])


@pytest.mark.parametrize("t,d", [(5, 200), (300, 1001)])
def test_f32_in_bf16_out(layer_norm, t, d):
    x, dy, w, b = _case(t, d, torch.float32, 3)
    got = _run(layer_norm, x, w, b, 1e-5, dy, out_dtype=torch.bfloat16)
    assert got["y"].dtype == torch.bfloat16 and got["dx"].dtype == torch.float32
    _check(got, _exact(x, w, b, 1e-5, dy.bfloat16()), torch.bfloat16, torch.float32)


@pytest.mark.parametrize("shift", [0.0, 300.0])
def test_rows_far_from_zero_and_constant_rows(layer_norm, shift):
    """a mean much larger than the spread, and rows without any spread (y = beta, dx finite)"""
    x, dy, w, b = _case(40, 777, torch.float32, 5, shift)
    x[3] = 2.5
    x[4] = 0.0
    got = _run(layer_norm, x, w, b, 1e-5, dy)
    _check(got, _exact(x, w, b, 1e-5, dy), torch.float32, torch.float32)
    assert torch.equal(got["y"][4], b)


def test_large_and_small_values(layer_norm):
    x, dy, w, b = _case(20, 300, torch.float32, 6, 0.0)
    x[0] *= 1e15
    x[1] *= 1e-15
    got = _run(layer_norm, x, w, b, 1e-5, dy)
    _check(got, _exact(x, w, b, 1e-5, dy), torch.float32, torch.float32)
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    y = layer_norm(x, w, b)
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).any() and torch.isfinite(y[4:]).all()


def test_without_weight_or_bias_and_partial_gradients(layer_norm):
    x, dy, w, b = _case(70, 333, torch.bfloat16, 7)
    r = _exact(x, None, None, 1e-3, dy.bfloat16())
    xg = x.detach().requires_grad_()
    y = layer_norm(xg, eps=1e-3)
    dx, = torch.autograd.grad(y, (xg,), dy.bfloat16())
    _check(dict(y=y.detach(), dx=dx), r, torch.bfloat16, torch.bfloat16)
    r = _exact(x, w, None, 1e-3, dy.bfloat16())
    wg = w.detach().requires_grad_()
    dw, = torch.autograd.grad(layer_norm(x, wg, eps=1e-3), (wg,), dy.bfloat16())
    _check(dict(y=layer_norm(x, w, eps=1e-3), dw=dw), r, torch.bfloat16, torch.bfloat16)


def test_strides_batches_and_offsets(layer_norm):
    """a column slice (odd row stride, unaligned start), leading dimensions, an expanded batch, a transposed input"""
    gen = torch.Generator().manual_seed(9)
    wide = torch.randn(6, 11, 517, generator=gen).to(torch.bfloat16).to(DEV)
    w = (1 + torch.randn(301, generator=gen)).to(DEV)
    b = torch.randn(301, generator=gen).to(DEV)
    want = layer_norm(wide[..., 5:306].contiguous(), w, b)
    assert torch.equal(layer_norm(wide[..., 5:306], w, b), want)
    base = torch.randn(1, 301, generator=gen).to(DEV)
    xe = base.detach().requires_grad_()
    ye = layer_norm(xe.expand(13, 301), w, b)
    dy = torch.randn(13, 301, generator=gen).to(DEV)
    dxe, = torch.autograd.grad(ye, (xe,), dy)
    full = _exact(base.expand(13, 301), w, b, 1e-5, dy)
    _check(dict(y=ye.detach()), full, torch.float32, torch.float32)
    tol = 1e-5 * full["dx"].abs().sum(0) + 1e-5
    assert ((dxe[0].double() - full["dx"].sum(0)).abs() <= tol).all()
    xt = torch.randn(301, 20, generator=gen).to(DEV).t()
    assert torch.equal(layer_norm(xt, w, b), layer_norm(xt.contiguous(), w, b))
    dyw = torch.randn(4, 602, generator=gen).to(DEV)[:, ::2]      # an incoming gradient with a stride in the row
    x4 = torch.randn(4, 301, generator=gen).to(DEV)
    ga = _run(layer_norm, x4, w, b, 1e-5, dyw)
    gb = _run(layer_norm, x4, w, b, 1e-5, dyw.contiguous())
    assert all(torch.equal(ga[k], gb[k]) for k in ga)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_column(layer_norm, dtype):
    """x - mean is 0: the result is the bias and x has no gradient, exactly"""
    x, dy, w, b = _case(596, 1, dtype, 21)
    x, w = x.requires_grad_(), (w + 0.3).requires_grad_()
    y = layer_norm(x, w, b)
    assert torch.equal(y, b.to(dtype).expand(596, 1))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert not dx.any() and not dw.any()


def test_no_rows(layer_norm):
    x = torch.empty(0, 40, device=DEV, requires_grad=True)
    w = torch.ones(40, device=DEV, requires_grad=True)
    y = layer_norm(x, w)
    assert y.shape == (0, 40)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert dx.shape == (0, 40) and torch.equal(dw, torch.zeros_like(dw))


def test_many_rows(layer_norm):
    """more rows than a grid has groups, offsets past 2^31 bytes"""
    t, d = 1_100_000, 1024
    x = torch.randn(1, d, device=DEV).bfloat16().expand(t, d).contiguous()
    x[-1] = torch.arange(d, device=DEV).bfloat16()
    y = layer_norm(x)
    assert torch.equal(y[0], y[t // 2]) and torch.equal(y[-1], layer_norm(x[-1:])[0])
    xg = x.requires_grad_()
    dx, = torch.autograd.grad(layer_norm(xg), (xg,), y)
    one = x.detach()[-1:].requires_grad_()
    want, = torch.autograd.grad(layer_norm(one), (one,), y[-1:])
    assert torch.equal(dx[-1:], want)


def test_results_repeat_and_streams(layer_norm):
    x, dy, w, b = _case(3000, 640, torch.bfloat16, 11)
    want = _run(layer_norm, x, w, b, 1e-5, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(layer_norm, x, w, b, 1e-5, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want[k], got[k]) for k in want)


def test_captured_and_replayed(layer_norm):
    x, dy, w, b = _case(513, 200, torch.float32, 12)
    xs = x.clone()
    pool = torch.cuda.Stream()
    pool.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(pool):
        _run(layer_norm, xs, w, b, 1e-5, dy)
    torch.cuda.current_stream().wait_stream(pool)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(layer_norm, xs, w, b, 1e-5, dy)
    for k in range(3):
        xs.copy_(x * (1 + k))
        graph.replay()
        want = _run(layer_norm, x * (1 + k), w, b, 1e-5, dy)
        torch.cuda.synchronize()
        assert all(torch.equal(out[n], want[n]) for n in want), k


def test_gradient_against_differences(layer_norm):
    """dx . v = (f(x + h v) - f(x - h v)) / 2h for f = sum(y c): truncation h^2, rounding u |f| / h"""
    x, c, w, b = _case(2, 50, torch.float32, 13)
    v = torch.randn(2, 50, generator=torch.Generator().manual_seed(1)).to(DEV)
    dx = _run(layer_norm, x, w, b, 1e-5, c)["dx"].double()
    h = 2.0 ** -7
    f = lambda z: (layer_norm(z, w, b).double() * c.double()).sum()
    num = (f(x + h * v) - f(x - h * v)) / (2 * h)
    assert abs(num - (dx * v.double()).sum()) <= 100 * (h * h + 64 * U / h)


def test_refusals(layer_norm):
    x = torch.randn(3, 20, device=DEV)
    w = torch.ones(20, device=DEV)
    for bad, err in ((lambda: layer_norm(x.double()), TypeError), (lambda: layer_norm(x, w.half()), TypeError),
                     (lambda: layer_norm(x, w[:10]), ValueError), (lambda: layer_norm(x, w.cpu()), ValueError),
                     (lambda: layer_norm(x, w, torch.ones(40, device=DEV)[::2]), ValueError),
                     (lambda: layer_norm(x.half(), out_dtype=torch.float32), TypeError),
                     (lambda: layer_norm(torch.empty(2, 16385, device=DEV)), ValueError),
                     (lambda: layer_norm(torch.empty(3, 0, device=DEV)), ValueError),
                     (lambda: layer_norm(torch.tensor(1.0, device=DEV)), ValueError)):
        with pytest.raises(err):
            bad()
