"""Every kernel form that the host side of layer_norm, token_logprobs and topk_distillation chooses between, by the sizes that
choose it: threads per row, elements a thread, rows in one step or several, rows split into segments, results that stay in
the caches or stream past them (more than 32 MB), with and without entropy, alternatives and gradients, in every type.

The checks are those of test_gpu_layer_norm, test_gpu_logits and test_gpu_topk_distill.  Their count of additions per thread is
given here by the widest row that each number of threads takes (2-byte types; f32 rows have half the elements):
  scores        64 threads up to 8192 tokens, 128 up to 24576, 256 up to 98304, 512 beyond; the joins of waves and segments,
                the exponentials' roundings and 40 u for the exponents' own are the constant 104 that is counted there
  distillation  64 threads up to 8192 tokens, 256 beyond; 168 as counted there"""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HERE = os.path.dirname(os.path.abspath(__file__))


def _checks(name, terms=None):
    """a copy of that test module with its own count of additions"""
    spec = importlib.util.spec_from_file_location(f"checks_of_{name}", os.path.join(HERE, f"{name}.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    if terms:
        m._terms = terms
    return m


def _score_terms(v):
    return (v / 64 if v <= 8192 else v / 128 if v <= 24576 else v / 256 if v <= 98304 else v / 512) + 104


def _distill_terms(v):
    return (v / 64 if v <= 8192 else v / 256) + 168


@pytest.fixture(scope="module")
def scores():
    from scmomer_amd.logits import token_logprobs
    return _checks("test_gpu_logits", _score_terms), token_logprobs


@pytest.fixture(scope="module")
def distill():
    from scmomer_amd import logits
    return _checks("test_gpu_topk_distill", _distill_terms), logits


@pytest.fixture(scope="module")
def norm():
    from scmomer_amd.norm import layer_norm
    return _checks("test_gpu_layer_norm"), layer_norm


def _rows(size, v, dtype):
    """few: not many; many: no results above 32 MB; streamed: results above"""
    if size == "streamed":
        return (9_000_000 if dtype == torch.float32 else 18_000_000) // v
    return size


def _draw(t, v, dtype, seed, scale=3.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(t, v, generator=gen, device=DEV) * scale).to(dtype), torch.randint(0, v, (t,), generator=gen, device=DEV)


@pytest.mark.parametrize("t,v,k", [(700, 7, 3), (700, 13, 5), (8300, 64, 9),                       # a thread per row
                                   (3, 131072, 20), (15, 131072, 9), (60, 131072, 40),             # split rows
                                   (100, 1500, 20), (100, 3001, 20), (100, 8001, 64),              # few rows, one step
                                   (1100, 300, 8), (1100, 300, 40), (1100, 900, 8), (1100, 900, 40), (1100, 4000, 8),
                                   (150, 60000, 64), (600, 12000, 20), (300, 40000, 20), (260, 110000, 20)])
@pytest.mark.parametrize("entropy", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores(scores, t, v, k, entropy, dtype):
    m, f = scores
    x, target = _draw(t, v, dtype, t + v)
    for alternatives in (0, k):
        m._check(f(x, target, k=alternatives, entropy=entropy, temperature=0.7), x, target, alternatives, 0.7)


@pytest.mark.parametrize("size,v,k", [(3700, 7, 2), (33000, 64, 3), (200, 300, 4), ("streamed", 300, 4), (200, 900, 4),
                                      ("streamed", 900, 4), (200, 1800, 4), ("streamed", 1800, 4), (200, 5000, 4),
                                      ("streamed", 5000, 4)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_the_scores(scores, size, v, k, dtype):
    m, f = scores
    t = _rows(size, v, dtype)
    x, target = _draw(t, v, dtype, t + v, 2.0)
    target[2] = -100
    gen = torch.Generator(device=DEV).manual_seed(v)
    gl, gh, gz = (torch.randn(t, generator=gen, device=DEV) for _ in range(3))
    gt = torch.randn(t, k, generator=gen, device=DEV)
    m._check_grad(m._grad(f, x, target, k, 0.7, gl, gh, gz, gt), x, target, k, 0.7, gl, gh, gz, gt)


@pytest.mark.parametrize("size,v,k", [(3700, 7, 3), (33000, 64, 5),                                # a thread per row
                                      (3, 131072, 20), (15, 131072, 9), (60, 131072, 40),          # split rows
                                      (100, 1500, 20), (100, 3001, 20), (100, 8001, 64), (100, 16001, 9), (100, 32001, 9),
                                      (1030, 300, 8), ("streamed", 300, 8), (1030, 900, 8), ("streamed", 900, 8),
                                      (1030, 1800, 8), ("streamed", 1800, 8), (1030, 3000, 64), ("streamed", 3000, 8),
                                      (1030, 7000, 8), ("streamed", 7000, 8), (260, 16000, 33), ("streamed", 16000, 8),
                                      (257, 16385, 4), (257, 32000, 32), ("streamed", 32000, 32), (256, 32768, 64),
                                      (257, 32767, 64), (257, 32768, 64), (70, 60000, 20), ("streamed", 60000, 8),
                                      (70, 100000, 20), ("streamed", 100000, 8)])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_distillation(distill, size, v, k, tail, dtype):
    """with entries that are not used, named twice and named everywhere, and rows of weight 0"""
    m, lib = distill
    t = _rows(size, v, dtype)
    x, target = _draw(t, v, dtype, t + v, 2.5)
    gen = torch.Generator(device=DEV).manual_seed(k)
    start = torch.randint(0, v, (t, 1), generator=gen, device=DEV)
    step = torch.randint(1, max(2, v // k), (t, 1), generator=gen, device=DEV)
    idx = (start + step * torch.arange(k, device=DEV)) % v                                         # distinct
    lp = torch.log(0.9 * torch.softmax(2 * torch.randn(t, k, generator=gen, device=DEV), 1))
    w = 2 * torch.rand(t, generator=gen, device=DEV)
    w[1] = 0
    idx[0, k - 1] = idx[0, 0]
    idx[2, 1:] = -1
    idx[-1, 0] = v - 1
    m._check(lib, x, idx, lp, w, 1.3, tail)


@pytest.mark.parametrize("size", [33, "streamed"])
@pytest.mark.parametrize("d", [3, 5, 100, 200, 400, 900, 1500, 3000, 6000, 12000])
@pytest.mark.parametrize("dtype,out", [(t, t) for t in TYPES] + [(torch.float32, torch.bfloat16)])
def test_layer_norm(norm, size, d, dtype, out):
    m, f = norm
    t = _rows(size, d, out)
    gen = torch.Generator(device=DEV).manual_seed(d)
    x = (1.7 * torch.randn(t, d, generator=gen, device=DEV) + 0.5).to(dtype)
    dy = torch.randn(t, d, generator=gen, device=DEV)
    w, b = 1 + 0.3 * torch.randn(d, generator=gen, device=DEV), 0.2 * torch.randn(d, generator=gen, device=DEV)
    got = m._run(f, x, w, b, 1e-5, dy, out_dtype=out)
    assert got["y"].dtype == out and got["dx"].dtype == dtype
    m._check(got, m._exact(x, w, b, 1e-5, dy.to(out)), out, dtype)
