"""Layer norm in the layout change of CPU tensors: the function that the kernels compute, at the costs where squares or sums in
32 bits would not do, with its gradients, against the plain form in 64 bits.

Both sides hold everything in 64 bits and round once, by half a step of the type: 2^-24 of a result in fp32, finfo.eps / 2 of a
gradient in a costs' type.  The sides differ in the order of at most 256 additions: with the tests' own bound for 32 bits (64 u (1 +
|xhat|) (1 + A r) per entry, in tests/test_gpu_norm.py) at u = 2^-53 and 256 for 64."""
import math

import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle

U = 2.0 ** -53
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _flat(t, labels_first):
  a = t.detach().double().numpy()
  a = np.moveaxis(a, 2, -1) if labels_first else a
  return a.reshape(-1, a.shape[-1])


def _check(x, weight, bias, eps, dy, labels_first):
  from mplayers_amd import labels_last_norm
  leaves = [t.detach().clone().requires_grad_(True) for t in (x, weight, bias)]
  y = labels_last_norm(*leaves, eps, labels_first)
  assert y.dtype == torch.float32 and y.is_contiguous()
  grads = torch.autograd.grad(y, leaves, dy)
  flat, d, w, b = _flat(x, labels_first), _flat(dy, False), weight.double().numpy(), bias.double().numpy()
  want, xhat, r = oracle.norm(flat, w, b, eps)
  dx, dweight, dbias = oracle.norm_grad(flat, w, eps, d)
  scale = 1 + np.abs(flat).max(1, keepdims=True) * r
  e = 256 * U * (1 + np.abs(xhat)) * scale
  half = 2.0 ** -24
  assert bool((np.abs(_flat(y, False) - want) <= e * np.abs(w) + 4 * U * np.abs(b) + half * np.abs(want) * (1 + 1e-6)).all())
  assert grads[0].dtype == x.dtype and grads[0].shape == x.shape
  largest = np.abs(d * w).max(1, keepdims=True)
  tolerance = 5 * 256 * U * r * largest * scale * (1 + np.abs(xhat).max(1, keepdims=True)) ** 2
  step, least = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
  assert bool((np.abs(_flat(grads[0], labels_first) - dx) <= tolerance + step * np.abs(dx) * (1 + 1e-6) + least).all())
  for got, want, parts in ((grads[1], dweight, np.abs(d * xhat)), (grads[2], dbias, np.abs(d))):
    assert got.dtype == torch.float32
    off = np.abs(got.double().numpy() - want)
    # (a sum over the pixels: an addition each)
    assert bool((off <= half * np.abs(want) * (1 + 1e-6) + (np.abs(d) * e).sum(0) + len(d) * U * parts.sum(0)).all())


def _inputs(n, dtype):
  g = torch.Generator().manual_seed(n * 7)
  x = (torch.randn(2, 1, n, 3, 17, generator=g) * (0.1 + 5 * torch.rand(2, 1, 1, 3, 17, generator=g)) + 3).to(dtype)
  return x, 1 + 0.3 * torch.randn(n, generator=g), torch.randn(n, generator=g), torch.randn(2, 1, 3, 17, n, generator=g)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 3, 8, 21, 60, 256])
def test_costs_far_apart(n, dtype, labels_first):
  """The type's largest number as a mask, and costs whose squares are beyond fp32."""
  x, weight, bias, dy = _inputs(n, dtype)
  largest = torch.finfo(dtype).max
  x[0, 0, 0, :, ::3] = largest
  x[0, 0, n - 1, :, 1::6] = -largest
  x[1, 0, n // 2, 0] = min(1e22, largest)
  x[1, 0, :, 1, ::2] *= min(1e20, largest / 1e3)
  x[1, 0, :, 2, ::5] = largest
  x = x if labels_first else x.movedim(2, -1).contiguous()
  _check(x, weight, bias, 1e-5, dy, labels_first)
  _check(x, weight, bias, 1e38, dy, labels_first)


@pytest.mark.parametrize("offset", [0.0, 1e3, -1e5])
@pytest.mark.parametrize("n", [3, 30, 150])
def test_large_means(n, offset):
  x, weight, bias, dy = _inputs(n, torch.float32)
  _check(x + offset, weight, bias, 1e-5, dy, True)


@pytest.mark.parametrize("n", [2, 3, 7, 13, 21, 47, 100, 133, 251])
def test_equal_costs_of_any_size(n):
  from mplayers_amd import labels_last_norm
  g = torch.Generator().manual_seed(n)
  x = torch.randn(1, 2, 1, 5, 31, generator=g) * 10.0 ** torch.randint(-3, 30, (1, 2, 1, 5, 31), generator=g)
  x[..., :3] = torch.tensor([1.2345e20, torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max])
  x, bias = x.expand(1, 2, n, 5, 31), torch.randn(n, generator=g)
  for labels_first in (True, False):
    y = labels_last_norm(x if labels_first else x.movedim(2, -1), None, bias, 1e-5, labels_first)
    assert torch.equal(y, bias.expand_as(y))


def test_costs_that_are_close_together_without_eps():
  x, weight, bias, dy = _inputs(21, torch.float32)
  for scale in (1e-19, 1e-24, 1e-30):
    _check((x - 3) * scale, weight, bias, 0.0, dy * scale, True)


def test_costs_that_are_no_numbers_stay_in_their_pixel():
  from mplayers_amd import labels_last_norm
  x, weight, bias, _ = _inputs(21, torch.float32)
  bad = x.clone()
  bad[0, 0, 9, 1, 3], bad[0, 0, 0, 2, 7], bad[1, 0, 20, 2, 16] = math.nan, math.inf, -math.inf
  y, z = (labels_last_norm(t, weight, bias) for t in (x, bad))
  spoilt = (bad != x).any(2)
  assert int(spoilt.sum()) == 3 and bool(z[spoilt].isnan().all()) and torch.equal(y[~spoilt], z[~spoilt])


def test_refusals_are_those_of_gpu_tensors():
  from mplayers_amd import labels_last_norm
  x, weight = torch.zeros(1, 1, 4, 4, 5), torch.ones(4)
  for wrong in [dict(weight=weight.double()), dict(weight=weight.half()), dict(weight=weight[:3]), dict(weight=weight[None]),
                dict(bias=weight.half()), dict(bias=weight[:1]), dict(eps=1e39), dict(eps=math.nan)]:
    with pytest.raises(RuntimeError):
      labels_last_norm(**{**dict(x=x, weight=weight, bias=weight), **wrong})
  empty = torch.zeros(0, 1, 4, 2, 2, requires_grad=True)
  y = labels_last_norm(empty, weight, weight)
  assert y.shape == (0, 1, 2, 2, 4) and torch.autograd.grad(y.sum(), empty)[0].shape == empty.shape
