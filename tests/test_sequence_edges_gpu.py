"""The operators over whole sequences where there is nothing, or nothing finite, to compute with."""
import pytest
import torch

import brainpylib_b200 as bpl

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------------------------------------
# no channels
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('batched', [False, True])
def test_no_channels(cuda, batched, dtype):
  """The gradients of B and C are sums over no channels: zeros, whatever stood in the memory that they got."""
  lead, n = ((3, 40) if batched else (120,)), 16
  r = lambda *s: torch.randn(*s, device=cuda, generator=torch.Generator(cuda).manual_seed(0)).to(dtype).requires_grad_(True)
  x, delta, A = r(*lead, 0), r(*lead, 0), torch.zeros(0, n, device=cuda, requires_grad=True)
  B, C = r(*lead, 2, n), r(*lead, 2, n)
  y, last = bpl.state_scan(x, delta, A, B, C, return_state=True)
  assert y.shape == (*lead, 0) and last.shape == (3 if batched else 1, 0, n)
  rubbish = [torch.full_like(B, float('nan')) for _ in range(16)]
  torch.cuda.synchronize()
  del rubbish
  for g, of in zip(torch.autograd.grad([y, last], [x, delta, A, B, C], [torch.zeros_like(y), torch.zeros_like(last)]), (x, delta, A, B, C)):
    assert g.shape == of.shape and g.dtype == of.dtype and not g.any()
