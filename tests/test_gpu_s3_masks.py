"""The S3 step with the tail and the optimizer on their kernels against the torch tail, for several dropout masks each.

Weights after Adam are no measure of the kernels' rounding: the first step divides a gradient by its own magnitude, so that an
entry near zero moves by a share of the learning rate that its rounding decides.  What the kernels owe is held apart here:
the gradients that reach the optimizer, and the optimizer's step from the gradients that it was given."""
import types

import numpy as np
import pytest
import torch

from oracle import performer_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
N, PEAKS, BSZ = 16906, 3000, 3
U = 2.0 ** -24


@pytest.fixture(scope="module")
def setup():
    import scmomer_amd as S
    from scmomer_amd import s3
    rng = np.random.default_rng(80)
    t = lambda *s_, sc=0.05: torch.from_numpy((rng.standard_normal(s_) * sc).astype(np.float32))
    state = {**O.make_scmomer_params(6), "RNA.output_mean.0.weight": t(N, 128), "RNA.output_mean.0.bias": t(N),
             "ATAC.output_mean.0.weight": t(PEAKS, 128), "ATAC.output_mean.0.bias": t(PEAKS)}
    batches = [(torch.from_numpy(O.synthetic_cells(81 + i, BSZ, N)).to(DEV),
                torch.from_numpy((rng.random((BSZ, PEAKS)) < 0.05).astype(np.float32)).to(DEV),
                t(BSZ, 128, sc=1.0).to(DEV)) for i in range(4)]

    def make(fused, lr):
        cfg = types.SimpleNamespace(projection_dim=128, normalize=True)
        m = S.scMomer(cfg, atac_config=None, encoder=S.StudentEncoder(N, 128, dropout=0.1),
                      rna_decoder=s3.ReconstructNet(N, 128), atac_decoder=s3.ReconstructNet(PEAKS, 128))
        m.load_state_dict(state, strict=False)
        m = m.to(DEV)
        s3.freeze_for_distillation(m)
        m.train()
        m.rna_model.model.performer.fix_projection_matrices_()
        return s3.S3Step(m, lr=lr, grad_acc=2, pos_weight=2.0, distill_weight=0.5, fused=fused)
    return make, batches


def _adam64(p, g, m, v, n, lr, b1=0.9, b2=0.999, eps=1e-8):
    """-> the weight after Adam's n-th step in 64 bits, and how far f32 may be from it.  m' = m + (g - m) (1 - b1): three
    roundings of parts no larger than |m| + |g|, and the rounded constant; v', a sum of positive terms: 4 u relative, half of
    it in its root; the root's two divisions, eps, the quotient and the step's factor: 6 u of the move; the weight's own
    rounding before and after."""
    p, g, m, v = (z.double() for z in (p, g, m, v))
    m1, v1 = m + (g - m) * (1 - b1), v * b2 + (1 - b2) * g * g
    step, denom = lr / (1 - b1 ** n), v1.sqrt() / (1 - b2 ** n) ** 0.5 + eps
    want = p - step * m1 / denom
    return want, step / denom * (4 * U * (m.abs() + g.abs()) + 10 * U * m1.abs()) + U * (p.abs() + want.abs())


@pytest.mark.parametrize("mask", range(8))
def test_gradients_and_optimizer_for_any_mask(setup, monkeypatch, mask):
    """Gradients before the first optimizer step: sums of up to n = 16,906 f32 terms in another order, three of them one after
    the other (the student's first layer, the decoders, the products back); terms of either sign leave u sqrt(n) = 130 u of
    such a sum's own scale: 390 u of the tensor's largest entry.  Losses likewise, 1e-5.  Optimizer: _adam64, for torch's
    first step and the kernel's second one."""
    make, batches = setup
    lr = 1e-3
    keep = (torch.rand((BSZ, 256), generator=torch.Generator().manual_seed(100 + mask)) >= 0.1).float().to(DEV) / 0.9
    monkeypatch.setattr(torch.nn.functional, "dropout", lambda x, p=0.5, training=True, inplace=False: x * keep)
    grads, losses = [], []
    for fused in (False, True):
        step = make(fused, lr)
        assert (step._tail_accs is not None) == fused
        seen = []
        after = step._after

        def checked():
            if step.index % step.grad_acc:
                return after()
            state = [step.optimizer.state.get(p, {}) for p in step.params]
            before = [(p.detach().clone(), a.clone(), s["exp_avg"].clone() if s else torch.zeros_like(p),
                       s["exp_avg_sq"].clone() if s else torch.zeros_like(p)) for p, a, s in zip(step.params, step.accs, state)]
            assert torch.stack([a.double().square().sum() for a in step.accs]).sum().sqrt() < 1e4     # nothing is clipped
            after()
            seen.append([b[1] for b in before])
            for p, (w, g, m, v) in zip(step.params, before):
                want, tol = _adam64(w, g.view_as(w), m, v, len(seen), lr)
                off = (p.detach().double() - want).abs()
                assert (off <= tol).all(), (fused, len(seen), float((off / tol).max()))
        step._after = checked
        losses.append([{k: float(v) for k, v in step.micro_step(*b).items()} for b in batches])
        assert len(seen) == 2 and (step._adam_table is not None) == fused
        grads.append(seen[0])
    for a, b in zip(*losses):
        for k in a:
            assert abs(a[k] - b[k]) <= 1e-5 * abs(a[k]), (k, a[k], b[k])
    worst = 0.0
    for a, b in zip(*grads):
        e = float((a - b).abs().max() / a.abs().max())
        worst = max(worst, e)
        assert e <= 390 * U, (tuple(a.shape), e / U)
    print(f"mask {mask}: worst gradient difference {worst / U:.0f} u of the largest entry")
