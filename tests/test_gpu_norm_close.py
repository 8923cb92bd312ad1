"""Layer norm of costs that are so close together that their squares are below fp32, without eps or with one as small: the bounds
are those of tests/test_gpu_norm.py, which are relative to the deviation."""
import numpy as np
import pytest
import torch

from tests.test_gpu_norm import _check, _inputs

pytestmark = pytest.mark.gpu

COUNTS = [2, 3, 4, 8, 12, 16, 17, 21, 32, 48, 60, 96, 130, 192, 256]


def _close(n, labels_first):
  """Pixels of spreads from 1 down to the smallest numbers, beside each other; dy of a size that dx is within fp32."""
  x, weight, bias, dy = _inputs(2, 1, n, 3, 47, torch.float32, True, offset=0.0)
  spreads = torch.tensor([1.0, 1e-10, 1e-14, 1e-16, 3e-17, 1e-19, 1e-21, 1e-23, 1e-25, 1e-30, 1e-37, 1e-40, 1e10])
  spread = spreads[torch.arange(3 * 47) % len(spreads)].view(1, 1, 1, 3, 47).cuda()
  x = x.detach() * spread
  dy = dy * spread.clamp(min=1e-30).movedim(2, -1)
  x = (x if labels_first else x.movedim(2, -1).contiguous()).requires_grad_(True)
  return x, weight, bias, dy


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-33, 1e-28])
@pytest.mark.parametrize("n", COUNTS)
def test_costs_close_together(gpu, n, eps, labels_first):
  x, weight, bias, dy = _close(n, labels_first)
  eps = float(np.float32(eps))
  _check(x, weight, bias, eps, dy, labels_first)


@pytest.mark.parametrize("eps", [1e-44, 1e-38, 1e-31, 1e-29])
@pytest.mark.parametrize("n", [2, 7, 16, 21, 100, 251])
def test_equal_costs_with_a_small_eps(gpu, n, eps):
  """Whatever their size: the bias comes out, and no NaN where r is large."""
  from mplayers_amd import labels_last_norm
  g = torch.Generator().manual_seed(n)
  x = torch.randn(1, 2, 1, 5, 31, generator=g) * 10.0 ** torch.randint(-40, 37, (1, 2, 1, 5, 31), generator=g)
  x = x.expand(1, 2, n, 5, 31).cuda().requires_grad_(True)
  bias = torch.randn(n, generator=g).cuda()
  y = labels_last_norm(x, None, bias, eps)
  assert torch.equal(y, bias.expand_as(y))
  (dx,) = torch.autograd.grad(y, x, torch.zeros_like(y))
  assert not bool(dx.any())
