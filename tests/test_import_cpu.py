"""The package without the torch functions of norm.py and logits.py (csrc/torch_ops.cpp, tied to the torch they were built for):
everything else imports and runs, and only a call of theirs says what is missing."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import sys
sys.modules["scmomer_amd._torch_ops"] = None            # as if it were not there
import torch
import scmomer_amd as S
from scmomer_amd import extract, logits, norm, ops, s1, s3, train
from scmomer_amd._lib import lib
assert lib.scm_version() >= 1
S.PerformerLM(num_tokens=7, dim=200, depth=1, max_seq_len=64, heads=10, local_attn_heads=0)
idx, lp = torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1)
for f in (lambda x: S.layer_norm(x), lambda x: S.token_logprobs(x), lambda x: S.topk_distillation(x, idx, lp),
          lambda x: S.topk_distillation_grad(x, idx, lp)):
    try:
        f(torch.randn(2, 8))
    except ImportError as e:
        assert "_torch_ops.so" in str(e) and "make -C scmomer_amd/csrc" in str(e), e
    else:
        raise AssertionError("no ImportError")
print("imported without")
"""


def test_package_without_the_torch_functions():
    out = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True)
    assert out.returncode == 0 and "imported without" in out.stdout, out.stderr


def test_torch_functions_are_loaded_where_they_are_called():
    code = ("import sys, torch, scmomer_amd as S; assert 'scmomer_amd._torch_ops' not in sys.modules\n"
            "try: S.layer_norm(torch.randn(2, 8))\nexcept ValueError: pass\n"
            "assert 'scmomer_amd._torch_ops' in sys.modules")
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
