"""A teacher's best labels where the list's type has no number for a cost: such a label is not in the list, and what it weighs is
in the rest, so that list and rest together are the teacher's distribution whatever the type.

Bounds: labels and costs are equal; those of rest and divergence as in tests/test_gpu_distill.py."""
import math

import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle

pytestmark = pytest.mark.gpu

INF = math.inf
U = 2.0 ** -24
# half a step above the largest number: from here on a cost is +inf in the type (ties go to the even number)
LIMITS = {torch.float32: INF, torch.float16: 65520.0, torch.bfloat16: float(np.float32((2 - 2.0 ** -8) * 2.0 ** 127))}


@pytest.mark.parametrize("dtype", list(LIMITS))
def test_the_limits_are_the_types(gpu, dtype):
  limit = min(LIMITS[dtype], float(np.finfo(np.float32).max))
  below = np.nextafter(np.float32(limit), np.float32(0))
  assert torch.isfinite(torch.tensor(float(below)).to(dtype))
  assert dtype == torch.float32 or torch.isinf(torch.tensor(limit).to(dtype))


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("dtype", list(LIMITS))
@pytest.mark.parametrize("n", [2, 4, 9, 16, 21, 40, 60, 96, 150, 256])
def test_costs_beyond_the_lists_type(gpu, n, dtype, labels_first):
  from mplayers_amd import best_labels
  rng = np.random.default_rng(n)
  # (pixels in turn: within fp16, around its end, beyond it, around bfloat16's end; a few masked)
  size = np.array([100.0, 65500.0, 65536.0, 1e6, 3.39e38, 3.3e38])[np.arange(48) % 6]
  cost = (rng.random((1, 1, n, 2, 48)) * size).astype(np.float32)
  cost[:, :, : (n + 1) // 2, :, 1::6] += np.float32(32.0)
  cost[rng.random(cost.shape) < 0.1] = INF
  cost[0, 0, 0] = 0.0
  cost[0, 0, n - 1, 0, 1::6] = 65520.0
  cost[0, 0, n - 1, 1, 1::6] = np.nextafter(np.float32(65520.0), np.float32(0))
  cost[0, 0, n - 1, 0, 4::6] = np.float32(min(LIMITS[torch.bfloat16], 3e39))
  t = torch.from_numpy(cost).cuda()
  t = t if labels_first else t.movedim(2, -1).contiguous()
  for k in sorted({1, min(n, 3), min(n, 13)}):
    temperature = 1e4
    labels, costs, rest = best_labels(t, k, temperature, labels_first, dtype)
    labels, costs = ((x if labels_first else x.movedim(-1, 2)).movedim(2, -1).reshape(-1, k).cpu() for x in (labels, costs))
    rest = rest.flatten().double().cpu().numpy()
    for p, row in enumerate(np.moveaxis(cost, 2, -1).reshape(-1, n)):
      want = oracle.best_labels(row, k, temperature, LIMITS[dtype])
      assert labels[p].tolist() == want[0], (p, labels[p].tolist(), want)
      assert torch.equal(costs[p], torch.tensor(want[1], dtype=torch.float32).to(dtype)), (p, costs[p], want)
      if want[2] == INF:
        assert rest[p] == INF
      else:
        others = [float(np.float32(c)) for c in row if c < INF]
        assert abs(rest[p] - want[2]) <= 64 * U * temperature + 4 * U * (abs(want[2]) + max(others) + temperature * 6), (p, rest[p], want)


@pytest.mark.parametrize("n,k", [(5, 4), (21, 7), (70, 7), (200, 7), (70, 40), (200, 100)])
def test_a_teacher_is_the_same_in_any_type(gpu, n, k):
  """Costs that go far beyond fp16 at a temperature as high: the divergence from the list and the rest is that from the whole
  teacher with the labels beyond the type taken as one class; a student that is the teacher has none."""
  from mplayers_amd import best_labels, distill_costs
  g = torch.Generator(device="cuda").manual_seed(n)
  cost = torch.rand(1, 1, n, 3, 40, device="cuda", generator=g) * 2e5
  cost[:, :, 0] = 0
  temperature = 5e4
  labels, costs, rest = best_labels(cost, k, temperature, dtype=torch.float16)
  # (a third of the labels and more are not within fp16: a list of that many has some beyond it, a short one of many labels none)
  assert bool((costs == INF).any()) == (3 * k >= n) and bool((costs[:, :, 1] < INF).any())
  leaf = cost.clone().requires_grad_(True)
  loss = distill_costs(leaf, labels, costs, rest, temperature)
  (grad,) = torch.autograd.grad(loss.sum(), leaf)
  # costs in fp16 are off by half a step, 2^-11 of up to 65504, so a class's logarithm by 32 / T = 6.4e-4 beside the roundings
  # of fp32 (bounds above at a reach of 8); a loss of two distributions whose logarithms differ by up to 2 d is at most 2 d^2
  # and those roundings, and the gradient is at most (e^(2 d) - 1) / T of a weight
  d = 32 / temperature
  assert float(loss.detach().abs().max()) <= 2 * d * d + U * ((5 * 8 + 2 * (k + 1) + 16) * 9 + 160)
  assert float(grad.abs().max()) <= (math.expm1(2 * d) + U * (5 * 1.45 * 8 + 2 * (k + 1) + 120) * 2) / temperature
