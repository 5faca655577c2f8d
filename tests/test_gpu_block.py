"""The operators of a gated recurrence block in processes and runs of their own."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), '..'))

FIRST_CALL = '''
import sys
sys.path.insert(0, 'flash-linear-attention_b200')
import torch, b200gdn
x = torch.randn(2, 300, 64, device='cuda', dtype=torch.bfloat16)
{make}
loss = y.sum()
loss.backward()
torch.cuda.synchronize()
print('done', torch.isfinite(leaf.grad).all().item())
'''


@pytest.mark.parametrize('make', ['leaf = -x.abs(); leaf.requires_grad_(True); y, _ = b200gdn.gated_recurrence(x, leaf)',
                                  'leaf = torch.randn(72, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True); y = b200gdn.fused_linear(x, leaf)',
                                  'leaf = x.clone().requires_grad_(True); y, _ = b200gdn.residual_rms_norm(leaf, residual=x)'])
def test_the_first_backward_pass_of_a_process(make):
    """It runs on a thread that has made no CUDA call yet."""
    out = subprocess.run([sys.executable, '-c', FIRST_CALL.format(make=make)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and 'done True' in out.stdout, out.stderr[-2000:]
