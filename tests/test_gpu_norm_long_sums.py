"""Layer norm's sums over many pixels: a lane adds a term per tile in 32 bits, N of them, then the lanes' sums are added (6 steps), those
of up to 4 wavefronts, and the workgroups' in 64 bits.  So dweight and dbias are off by at most (N + 6 + 4 + 1) u of the sums of
their terms' sizes, u = 2^-24, and dweight by what its terms are (e of tests/test_gpu_norm.py); (N + 16) u is taken, as there.
The terms have a sign in common, so that what is lost adds up.  Against 64 bits in torch."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _rounds(n, pixels):
  """Tiles of 64 pixels that a wavefront of the gradient goes over: tiles to a workgroup at a time, workgroups at most."""
  waves = 4 if n <= 4 else 2 if n <= 8 else 4 if n <= 16 else 3 if n <= 24 else 4 if n <= 32 else 6 if n <= 48 else 8
  at_a_time, most = 4 if n <= 4 else 1, 512 if waves == 8 else 1792 if waves == 4 else 2048
  return math.ceil(math.ceil(math.ceil(pixels / 64) / at_a_time) / most)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n,pixels", [(2, 46_000_037), (7, 13_200_011), (16, 11_500_003), (21, 11_500_001), (130, 3_300_005)])
def test_sums_over_many_tiles(gpu, n, pixels, labels_first):
  from mplayers_amd import labels_last_norm
  run = _rounds(n, pixels)
  assert 87 <= run <= 103
  g = torch.Generator(device="cuda").manual_seed(n)
  # (the first label has the greatest cost mostly, so xhat a mean that is not 0, and dy has one)
  x = torch.randn(1, 1, n, 1, pixels, device="cuda", generator=g)
  x[:, :, 0] += 2.0
  dy = torch.rand(1, 1, 1, pixels, n, device="cuda", generator=g).add_(0.5)
  weight, bias = (torch.rand(n, device="cuda", generator=g).add_(0.5).requires_grad_(True) for _ in range(2))
  leaf = x if labels_first else x.movedim(2, -1).contiguous()
  y = labels_last_norm(leaf, weight, bias, 1e-5, labels_first)
  dweight, dbias = torch.autograd.grad(y, (weight, bias), dy)
  del y, leaf
  sums = torch.zeros(4, n, dtype=torch.float64, device="cuda")
  for part in range(0, pixels, 1_000_000):
    c = x[0, 0, :, 0, part:part + 1_000_000].t().double()
    d = dy[0, 0, 0, part:part + 1_000_000].double()
    centred = c - c.mean(1, keepdim=True)
    r = 1 / ((centred * centred).mean(1, keepdim=True) + 1e-5).sqrt()
    xhat = centred * r
    e = 64 * U * (1 + xhat.abs()) * (1 + c.abs().amax(1, keepdim=True) * r)
    sums += torch.stack([(d * xhat).sum(0), (d * xhat).abs().sum(0), (d * e).sum(0), d.sum(0)])
  want, size, of_terms, plain = sums
  assert bool(((dweight.double() - want).abs() <= of_terms + (run + 16) * U * size).all())
  assert bool(((dbias.double() - plain).abs() <= (run + 16) * U * plain).all())
