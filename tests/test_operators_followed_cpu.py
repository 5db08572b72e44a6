"""The operators at a model's end work on addresses: under whatever follows a call by its torch operations (forward-mode
differentiation, tracers, tensor subclasses with a dispatch of their own) they raise, before anything else is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx


def _entry(t=2, v=8, k=3):
    idx, lp, w = torch.zeros(t, k, dtype=torch.int64), torch.zeros(t, k), torch.ones(t)
    return idx, lp, w


def _calls():
    from scmomer_amd import logits as L, norm
    idx, lp, w = _entry()
    return {"norm": lambda x: norm.layer_norm(x), "norm_weight": lambda x: norm.layer_norm(torch.ones(2, 8), x[0]),
            "norm_bias": lambda x: norm.layer_norm(torch.ones(2, 8), None, x[0]), "score": lambda x: L.token_logprobs(x).lse,
            "distill": lambda x: L.topk_distillation(x, idx, lp), "teacher": lambda x: L.topk_distillation(torch.ones(2, 8), idx, x[:, :3]),
            "weight": lambda x: L.topk_distillation(torch.ones(2, 8), idx, lp, weight=x[:, 0]),
            "step": lambda x: L.topk_distillation_grad(x, idx, lp)}


NAMES = ["norm", "norm_weight", "norm_bias", "score", "distill", "teacher", "weight", "step"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_raises(name, grad):
    f = _calls()[name]
    with fwAD.dual_level():
        x = fwAD.make_dual(torch.randn(2, 8).requires_grad_(grad), torch.randn(2, 8))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(x)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(x)


@pytest.mark.parametrize("name", ["norm", "score", "distill", "step"])
def test_tracers_raise(name):
    f = _calls()[name]
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(f, (torch.randn(2, 8),), check_trace=False)
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(f, tracing_mode=mode)(torch.randn(2, 8))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(NotImplementedError):
        f(torch.randn(2, 8))


class Wrapper(torch.Tensor):
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func is torch.ops.aten.detach.default:
            return args[0]
        raise AssertionError(f"{func} reached the wrapper")


@pytest.mark.parametrize("name", ["norm", "score", "distill", "step"])
def test_tensors_with_a_dispatch_of_their_own_raise(name):
    with pytest.raises(NotImplementedError, match="plain tensors"):
        _calls()[name](Wrapper(torch.randn(2, 8)))


@pytest.mark.parametrize("name", ["norm", "score", "distill", "step"])
def test_a_mode_that_only_counts_is_no_tracer(name):
    """its call is as without: here the refusal of host tensors"""
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False), pytest.raises(ValueError, match="device"):
        _calls()[name](torch.randn(2, 8))


@pytest.mark.parametrize("name", ["norm", "score", "distill", "step"])
def test_function_transforms_raise(name):
    f = _calls()[name]
    with pytest.raises(NotImplementedError, match="plain tensors"):
        torch.func.vmap(f)(torch.randn(3, 2, 8))
    for transform in (torch.func.grad(lambda x: torch.as_tensor(f(x)).sum()), torch.func.jacrev(f)):
        with pytest.raises(NotImplementedError, match="plain tensors"):
            transform(torch.randn(2, 8))
    with pytest.raises(NotImplementedError):
        torch.func.jvp(f, (torch.randn(2, 8),), (torch.randn(2, 8),))
    with pytest.raises(NotImplementedError, match="plain tensors"):
        torch.func.functionalize(f)(torch.randn(2, 8))
