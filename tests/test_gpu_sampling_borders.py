"""Draws whose target falls on a running sum, with labels that weigh nothing beside it.

Where the target is a sum up to roundings, either label at that border is right.  A weight of the kernel is off by
four roundings of its exponent, at most 5 / 0.7 here, and by about 2^-51 of its own: 36 * 2^-53.  A sum of up to 256
is off by as many roundings more, and so is the total that the target is a product with: 2 * (36 + 255) + 1 < 2^10
of 2^-53, 2^-43 of the total in all."""
import numpy as np
import pytest
import torch

from oracle import around_oracle

pytestmark = pytest.mark.gpu

INF = float("inf")
NEAR = 2.0 ** -43


def _draw(cost, uniforms, labels_first=True, **parameters):
  """cost (batch, cv, labels, H, W) whichever layout is asked for."""
  from mplayers_amd import sample_labels
  cost = torch.from_numpy(np.ascontiguousarray(cost, np.float32)).cuda()
  if not labels_first:
    cost = cost.permute(0, 1, 3, 4, 2).contiguous()
  uniforms = torch.from_numpy(np.ascontiguousarray(uniforms, np.float32)).cuda()
  return sample_labels(cost, uniforms, labels_first=labels_first, **parameters).cpu().numpy()


def _borders(cost, temperature=1.0, top_k=0, min_p=0.0):
  """Per label the share of the total before it and up to it; NaN where it does not stay.  No top_p."""
  order = sorted((c, l) for l, c in enumerate(cost) if c < INF)
  order = order[:top_k] if top_k else order
  temperature = np.longdouble(np.float32(temperature))
  weight = np.zeros(len(cost), np.longdouble)
  for c, l in order:
    weight[l] = np.exp((order[0][0] - np.longdouble(c)) / temperature)
  weight[weight < np.float32(min_p)] = 0  # (no cost of these tests is next to the one where min_p cuts)
  upto = np.cumsum(weight)
  before = np.concatenate([[0], upto[:-1]])
  return np.where(weight > 0, before / upto[-1], np.nan), upto / upto[-1]


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("parameters", [dict(), dict(temperature=0.7), dict(top_k=9), dict(min_p=0.1),
                                        dict(top_k=12, min_p=0.02, temperature=0.7)])
@pytest.mark.parametrize("lead,half,gap", [(0, 7, 2), (0, 6, 9), (0, 12, 8), (4, 24, 8), (0, 25, 10), (12, 34, 16), (0, 70, 52),
                                           (5, 100, 51)])
def test_mirrored_costs_around_masked_labels(gpu, lead, half, gap, parameters, labels_first):
  """The sum of the first half is half the total, and the labels in the middle have no weight.  A draw has the same label
  whatever the number of draws beside it."""
  rng = np.random.default_rng(lead + half)
  pixels, n = 80, lead + 2 * half + gap
  side = rng.integers(0, 40, (half, pixels)) / 8.0
  cost = np.concatenate([np.full((lead, pixels), INF), side, np.full((gap, pixels), INF), side[::-1]])
  shares = [_borders(cost[:, p], **parameters) for p in range(pixels)]
  uniforms = np.array([0.5, 0.25, 0.75, 0.5, 0.0] + [k / 64 for k in range(1, 61)])
  labels = {}
  for draws in (1, 2, 4, 5, 65):
    u = np.broadcast_to(uniforms[:draws, None], (draws, pixels)).reshape(draws, 1, 1, 2, 40)
    labels[draws] = _draw(cost.reshape(1, 1, n, 2, 40), u, labels_first, **parameters).reshape(draws, pixels)
  for d, u in enumerate(uniforms):
    for p, (before, upto) in enumerate(shares):
      label = int(labels[65][d, p])
      assert before[label] <= u + NEAR and upto[label] > u - NEAR, (d, p, label, before[label], upto[label])
  for draws in (1, 2, 4, 5):
    wrong = np.argwhere(labels[draws] != labels[65][:draws])
    assert len(wrong) == 0, (draws, len(wrong), wrong[:4])


@pytest.mark.parametrize("masked", [0.0, 0.3, 0.97, 1.0])
@pytest.mark.parametrize("draws", [5, 70])
@pytest.mark.parametrize("n", [21, 96, 200])
def test_whole_sums_and_many_draws(gpu, n, draws, masked):
  """Costs that are all the same and mostly out: every sum is a whole number, exact in 64 bits, and every target here
  is one too or halfway."""
  rng = np.random.default_rng(int(100 * masked) + n + draws)
  cost = np.where(rng.random((1, 1, n, 1, 9)) < masked, INF, 0.75)
  u = rng.integers(0, 16, (draws, 1, 1, 1, 9)) / np.float32(16)
  for parameters in (dict(), dict(top_p=0.5), dict(top_k=4, top_p=0.25), dict(min_p=1.0)):
    want = around_oracle.draw_labels(cost.astype(np.float32), u, **parameters)
    assert np.array_equal(_draw(cost, u, **parameters), want), parameters


@pytest.mark.parametrize("n", [3, 16, 21, 60, 200])
def test_min_p_of_1_at_any_temperature(gpu, n):
  """min_p of 1 leaves the labels of the best cost, whatever the temperature: at an infinite one too, where a lesser min_p
  leaves all candidates."""
  from mplayers_amd import sample_labels
  rng = np.random.default_rng(n)
  cost = np.round(rng.standard_normal((2, 1, n, 2, 33)) * 3) / 2
  cost[rng.random(cost.shape) < 0.2] = INF
  cost = cost.astype(np.float32)
  u = rng.integers(0, 2 ** 24, (3, 2, 1, 2, 33)).astype(np.float32) * np.float32(2.0 ** -24)
  best = cost.min(2)
  for temperature in (INF, 1e30, 1.0, 1e-30):
    for more in (dict(), dict(top_p=0.5), dict(top_k=2)):
      parameters = dict(temperature=temperature, min_p=1.0, **more)
      got = _draw(cost, u, **parameters)
      assert np.array_equal(got, around_oracle.draw_labels(cost, u, **parameters)), parameters
      assert (np.take_along_axis(cost[None], got[:, :, :, None].astype(np.int64), 3)[:, :, :, 0] == best).all()
  # per image: an infinite temperature with min_p of 1 and just below it
  below = float(np.nextafter(np.float32(1), np.float32(0)))
  got = sample_labels(torch.from_numpy(cost).cuda(), torch.from_numpy(u).cuda(), temperature=torch.tensor([INF, INF]).cuda(),
                      min_p=torch.tensor([1.0, below]).cuda()).cpu().numpy()
  assert np.array_equal(got, around_oracle.draw_labels(cost, u, temperature=[INF, INF], min_p=[1.0, below]))
