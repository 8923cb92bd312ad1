"""A teacher's best labels and the divergence from them on the GPU against their plain forms in 64 bits.

best_labels   labels are equal, costs are one difference in fp32 and one rounding to their type: the same bits.
  rest: -T log of a sum of at most 256 weights.  A weight exp(-a) is off by the three roundings of a, 3 a u (u = 2^-24), and an
  ulp; sum(a w) <= ln(256) sum(w); 40 additions: a part of 19 u + 40 u of the sum.  So 59 u T, and roundings of the terms.

distill_costs, with R the largest (|c - M| + |t - m|) / T of a class that is there, and K classes:
  a class's p is off by a part of (3 * 1.45 R + 2 K + 10) u, the factor of p by two roundings: in all (5 R + 2 K + 16) u (1 + R);
  the logarithms of three sums, 59 u each of them, less their roundings: 160 u.
  The gradient is a difference of q, p and the rest's share, of which `size` is the sum: each a weight over a sum or two,
  off by a part of (5 A + 2 K + 120) u, A the largest exponent of its pixel; half a step of its type."""
import math

import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
INF, NAN = math.inf, math.nan
COUNTS = [1, 2, 3, 4, 5, 7, 8, 9, 11, 12, 13, 16, 17, 18, 20, 21, 24, 25, 28, 29, 32, 33, 48, 49, 64, 65, 80, 81, 96, 97, 112,
          113, 128, 129, 160, 161, 192, 193, 224, 225, 255, 256]


def _gpu(a, labels_first, dtype=torch.float32):
  """(batch, cv, labels, H, W) numpy -> the layout and type asked for."""
  t = torch.from_numpy(np.ascontiguousarray(a)).to(dtype)
  return (t if labels_first else t.movedim(2, -1)).contiguous().cuda()


def _rows(t, labels_first):
  """-> (pixels, labels) numpy"""
  a = t.detach().cpu()
  a = a.double().numpy() if a.is_floating_point() else a.numpy()
  a = np.moveaxis(a, 2, -1) if labels_first else a
  return a.reshape(-1, a.shape[-1])


# ------------------------------------------------------------------------------------------------------ best labels
def _check_best(cost, k, temperature, labels_first, dtype):
  from mplayers_amd import best_labels
  labels, costs, rest = best_labels(cost, k, temperature, labels_first, dtype)
  assert labels.dtype == torch.uint8 and costs.dtype == dtype and rest.dtype == torch.float32
  b, cv, h, w = (cost.shape[:2] + cost.shape[3:]) if labels_first else cost.shape[:4]
  assert labels.shape == costs.shape == ((b, cv, k, h, w) if labels_first else (b, cv, h, w, k)) and rest.shape == (b, cv, h, w)
  flat = _rows(cost, labels_first)
  got_labels, got_costs, got_rest = _rows(labels, labels_first), _rows(costs, labels_first), rest.cpu().double().numpy().reshape(-1)
  for p, row in enumerate(flat):
    want_labels, want_costs, want_rest = oracle.best_labels(row, k, temperature)
    rounded = torch.tensor(want_costs, dtype=torch.float32).to(dtype).double().numpy()
    assert got_labels[p].tolist() == want_labels and np.array_equal(got_costs[p], rounded), (p, got_costs[p], rounded)
    if want_rest == INF:
      assert got_rest[p] == INF
    else:
      least = max(want_costs)  # (no other candidate is below it)
      tolerance = 64 * U * temperature + 4 * U * (abs(want_rest) + least + temperature * 6)
      assert abs(got_rest[p] - want_rest) <= tolerance, (p, got_rest[p], want_rest)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n", COUNTS)
def test_best_of_label_counts(gpu, n, labels_first):
  rng = np.random.default_rng(n)
  cost = rng.standard_normal((1, 2, n, 3, 25)) * 3
  cost[..., ::2] = np.round(cost[..., ::2])  # ties
  cost[rng.random(cost.shape) < 0.1] = INF
  cost[rng.random(cost.shape) < 0.02] = NAN
  for k in sorted({1, min(n, 4), (n + 1) // 2, min(n, 17)}):
    _check_best(_gpu(cost, labels_first), k, 1.0, labels_first, torch.float32)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,kept", [(21, 5, torch.float16), (21, 21, torch.float32), (40, 33, torch.bfloat16), (97, 8, torch.float16),
                                      (256, 256, torch.float32), (192, 16, torch.bfloat16)])
def test_best_of_types(gpu, n, k, kept, dtype, labels_first):
  rng = np.random.default_rng(n + k)
  cost = rng.standard_normal((2, 1, n, 5, 14)) * 20
  _check_best(_gpu(cost, labels_first, dtype), k, 2.5, labels_first, kept)


@pytest.mark.parametrize("n", [2, 9, 21, 70, 150, 256])
def test_best_of_costs_that_are_no_numbers(gpu, n):
  big = float(np.finfo(np.float32).max)
  i = np.arange(n)
  rows = [np.full(n, INF), np.full(n, NAN), np.full(n, -INF), np.full(n, big), np.full(n, -big), np.where(i % 2, 0.0, -0.0),
          np.where(i % 3, big, -big), np.where(i % 2, -INF, 1.0), np.where(i % 2, NAN, 0.5), np.where(i == n - 1, 3.0, INF),
          np.where(i == 0, -INF, INF), i * 1e-42, i * 1e4, 2.0 ** (i % 120 - 60)]
  cost = np.stack(rows, 1).reshape(1, 1, n, 1, len(rows)).astype(np.float32)
  for labels_first in (True, False):
    for dtype in TYPES:
      _check_best(_gpu(cost, labels_first), min(n, 6), 0.7, labels_first, dtype)


@pytest.mark.parametrize("temperature", [1e-3, 0.1, 30.0, 1e6])
def test_best_at_other_temperatures(gpu, temperature):
  cost = np.random.default_rng(1).standard_normal((1, 1, 50, 2, 40)) * 3
  _check_best(_gpu(cost, True), 7, temperature, True, torch.float32)


# ------------------------------------------------------------------------------------------------------- divergence
def _check_distill(cost, labels, costs, rest, temperature, labels_first, dloss=None):
  """cost, labels, costs on the GPU, in the layout; the plain form takes their values as they are in their types."""
  from mplayers_amd import distill_costs
  leaf = cost.detach().clone().requires_grad_(True)
  loss = distill_costs(leaf, labels, costs, rest, temperature, labels_first)
  shape = (cost.shape[:2] + cost.shape[3:]) if labels_first else cost.shape[:4]
  assert loss.dtype == torch.float32 and loss.shape == shape
  if dloss is None:
    dloss = torch.randn(shape, generator=torch.Generator().manual_seed(5)).cuda()
  (grad,) = torch.autograd.grad(loss, leaf, dloss)
  assert grad.dtype == cost.dtype and grad.shape == cost.shape
  c, l, t = (_rows(x, labels_first) for x in (cost, labels, costs))
  r = None if rest is None else rest.double().cpu().numpy().reshape(-1)
  d, got, got_grad = dloss.double().cpu().numpy().reshape(-1), loss.detach().double().cpu().numpy().reshape(-1), _rows(grad, labels_first)
  step = 0 if cost.dtype == torch.float32 else torch.finfo(cost.dtype).eps / 2
  least = 1e-37 if cost.dtype == torch.float32 else torch.finfo(cost.dtype).smallest_normal * torch.finfo(cost.dtype).eps
  for p in range(len(c)):
    want, want_grad, size = oracle.distill(c[p], l[p], t[p], None if r is None else r[p], temperature)
    want_grad, size = np.array(want_grad) * d[p], np.array(size) * abs(d[p])
    if want != want:
      assert got[p] != got[p] and np.array_equal(np.isnan(got_grad[p]), np.isnan(want_grad)), p
      assert bool((got_grad[p][c[p] == INF] == 0).all())
      continue
    spread = [np.ptp(x[np.isfinite(x)]) if np.isfinite(x).any() else 0.0
              for x in (c[p], np.append(t[p], [] if r is None else r[p]))]
    reach, k = sum(spread) / temperature, t.shape[1] + 1
    assert abs(got[p] - want) <= U * ((5 * reach + 2 * k + 16) * (1 + reach) + 160), (p, got[p], want)
    tolerance = size * (5 * 1.45 * reach + 2 * k + 120) * U + least
    off = np.abs(got_grad[p] - want_grad)
    assert bool((off <= tolerance * (1 + step) + step * np.abs(want_grad)).all()), (p, off / tolerance)


def _problem(n, k, shape, seed, masked=0.1):
  b, cv, h, w = shape
  rng = np.random.default_rng(seed)
  cost = rng.standard_normal((b, cv, n, h, w)) * 3
  cost[rng.random(cost.shape) < masked] = INF
  labels = np.argsort(rng.random((b, cv, n, h, w)), axis=2)[:, :, :k].astype(np.uint8)
  costs = rng.random((b, cv, k, h, w)) * 5
  costs[rng.random(costs.shape) < 0.1] = INF
  rest = rng.random((b, cv, h, w)) * 6
  rest[rng.random(rest.shape) < 0.1] = INF
  return cost, labels, costs, rest


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("with_rest", [True, False])
@pytest.mark.parametrize("n", COUNTS)
def test_label_counts(gpu, n, with_rest, labels_first):
  for k in sorted({1, min(n, 5), min(n, 34)}):
    cost, labels, costs, rest = _problem(n, k, (1, 2, 3, 25), n + k)
    _check_distill(_gpu(cost, labels_first), _gpu(labels, labels_first, torch.uint8), _gpu(costs, labels_first),
                   torch.from_numpy(rest).float().cuda() if with_rest else None, 1.0, labels_first)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("kept", TYPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,temperature", [(7, 3, 0.5), (21, 4, 2.0), (60, 9, 1.0), (192, 8, 4.0)])
def test_types(gpu, n, k, temperature, dtype, kept, labels_first):
  cost, labels, costs, rest = _problem(n, k, (2, 1, 5, 14), n)
  _check_distill(_gpu(cost, labels_first, dtype), _gpu(labels, labels_first, torch.uint8), _gpu(costs, labels_first, kept),
                 torch.from_numpy(rest).float().cuda(), temperature, labels_first)


@pytest.mark.parametrize("n", [4, 21, 40, 100, 200])
@pytest.mark.parametrize("what", ["same label", "no such label", "none", "all masked", "all named", "one left", "named is masked"])
def test_lists(gpu, n, what):
  """Lists with a label twice or one that there is none of, without entries, or naming every label; a student without labels."""
  k = {"all named": n, "one left": n - 1}.get(what, 4)
  cost, labels, costs, rest = _problem(n, min(k, n), (1, 1, 2, 35), n)
  if what == "same label":
    labels[:, :, 1] = labels[:, :, 0]
    labels[:, :, 3, :, ::2] = labels[:, :, 0, :, ::2]
  if what == "no such label":
    labels[:, :, 1] = 255
    labels[:, :, 2] = n
  if what == "none":
    costs[...] = INF
    rest[:, :, :, ::2] = INF
  if what == "all masked":
    cost[..., ::2] = INF
  if what == "named is masked":
    np.put_along_axis(cost, labels[:, :, :2].astype(np.int64), INF, 2)
  for labels_first in (True, False):
    for with_rest in (True, False):
      _check_distill(_gpu(cost, labels_first), _gpu(labels, labels_first, torch.uint8), _gpu(costs, labels_first),
                     torch.from_numpy(rest).float().cuda() if with_rest else None, 1.5, labels_first)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n,k", [(1, 9), (5, 200), (21, 64), (40, 256), (100, 130), (200, 256)])
def test_lists_that_are_longer_than_the_labels(gpu, n, k, labels_first):
  """Labels named many times, and labels that there are none of between them."""
  rng = np.random.default_rng(n + k)
  cost, _, _, rest = _problem(n, 1, (1, 1, 2, 19), n)
  labels = rng.integers(0, min(n + 3, 256), (1, 1, k, 2, 19)).astype(np.uint8)
  costs = rng.random((1, 1, k, 2, 19)) * 5
  for with_rest in (True, False):
    _check_distill(_gpu(cost, labels_first), _gpu(labels, labels_first, torch.uint8), _gpu(costs, labels_first),
                   torch.from_numpy(rest).float().cuda() if with_rest else None, 1.0, labels_first)


@pytest.mark.parametrize("n", [3, 21, 50, 130])
def test_costs_that_are_no_numbers(gpu, n):
  """NaN and infinities of either sign on either side; they stay in their pixel."""
  cost, labels, costs, rest = _problem(n, 3, (1, 1, 2, 35), n, 0.0)
  cost[0, 0, n // 2, 0, 3] = NAN
  cost[0, 0, :, 0, 4] = NAN
  cost[0, 0, 0, 0, 5] = -INF
  cost[0, 0, :, 0, 6] = -INF
  costs[0, 0, 1, 0, 8] = NAN
  costs[0, 0, :, 0, 9] = NAN
  costs[0, 0, 0, 0, 10] = -INF
  rest[0, 0, 0, 12] = NAN
  rest[0, 0, 0, 13] = -INF
  costs[0, 0, :, 0, 14] = INF
  rest[0, 0, 0, 14] = INF
  cost[0, 0, 1, 0, 14] = NAN  # (no class is there)
  for labels_first in (True, False):
    for with_rest in (True, False):
      _check_distill(_gpu(cost, labels_first), _gpu(labels, labels_first, torch.uint8), _gpu(costs, labels_first),
                     torch.from_numpy(rest).float().cuda() if with_rest else None, 1.0, labels_first)


@pytest.mark.parametrize("n", [5, 21, 90])
def test_far_costs(gpu, n):
  """A student so sure that its other labels weigh nothing in fp32: what they weigh among themselves still tells, and the
  divergence is as large as the costs say.  Costs of the type's extremes make weights of 0 or a loss beyond it, no NaN."""
  from mplayers_amd import distill_costs
  cost, labels, costs, rest = _problem(n, 2, (1, 1, 2, 35), n, 0.0)
  cost += 500.0
  np.put_along_axis(cost, labels[:, :, :1].astype(np.int64), -300.0, 2)
  costs[np.isinf(costs)] = 1.0
  rest[np.isinf(rest)] = 1.0
  _check_distill(_gpu(cost, True), _gpu(labels, True, torch.uint8), _gpu(costs, True), torch.from_numpy(rest).float().cuda(), 1.0, True)
  big = float(np.finfo(np.float32).max)
  np.put_along_axis(cost, labels[:, :, 1:2].astype(np.int64), big, 2)
  leaf = _gpu(cost, True).requires_grad_(True)
  loss = distill_costs(leaf, _gpu(labels, True, torch.uint8), _gpu(costs, True), temperature=0.5)
  (grad,) = torch.autograd.grad(loss.sum(), leaf)
  # (the list's costs are in [0, 5]: at T = 0.5 that label has p of e^-10 / 2 = 2.2e-5 at least, and the loss p * 3.4e38 / T)
  assert bool((loss > 1e34).all()) and bool(torch.isfinite(grad).all())


def test_equal_distributions_have_no_divergence(gpu):
  """All labels listed with the student's own costs: nothing to learn."""
  from mplayers_amd import best_labels, distill_costs
  for n in (2, 21, 60, 192):
    cost = (torch.randn(1, 1, n, 9, 31, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) * 3)
    for k in sorted({n, min(n, 7)}):
      labels, costs, rest = best_labels(cost, k)
      leaf = cost.clone().requires_grad_(True)
      loss = distill_costs(leaf, labels, costs, rest if k < n else None)
      (grad,) = torch.autograd.grad(loss.sum(), leaf)
      # (costs relative to the best one are off by a rounding, and the bounds above at R < 40)
      assert float(loss.detach().abs().max()) <= U * ((5 * 40 + 2 * n + 16) * 41 + 160)
      assert float(grad.abs().max()) <= U * (5 * 1.45 * 40 + 2 * n + 120) * 2


def test_the_gradient_against_differences(gpu):
  from mplayers_amd import distill_costs
  cost, labels, costs, rest = _problem(21, 4, (1, 1, 2, 10), 3)
  t = 1.3
  leaf = _gpu(cost, True).requires_grad_(True)
  (grad,) = torch.autograd.grad(distill_costs(leaf, _gpu(labels, True, torch.uint8), _gpu(costs, True),
                                              torch.from_numpy(rest).float().cuda(), t).sum(), leaf)
  c, l, s = _rows(_gpu(cost, True), True), _rows(_gpu(labels, True, torch.uint8), True), _rows(_gpu(costs, True), True)
  r, g = torch.from_numpy(rest).float().double().numpy().reshape(-1), _rows(grad, True)
  h = np.random.default_rng(4).standard_normal(c.shape)
  for p in range(len(c)):
    ends = [oracle.distill(c[p] + e * h[p], l[p], s[p], r[p], t)[0] for e in (1e-5, -1e-5)]
    got = (np.where(np.isinf(c[p]), 0, g[p]) * h[p]).sum()
    # differences: 1e-10 of third derivatives, 1e5 * 2^-52 of a loss below 50; gradient: the bound above at a reach of 30
    assert abs((ends[0] - ends[1]) / 2e-5 - got) <= 1e-6 + 400 * U * np.abs(h[p]).max() * 2


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n", [24, 60])
def test_alignment_and_strides(gpu, n, labels_first):
  from mplayers_amd import best_labels, distill_costs
  cost, labels, costs, rest = _problem(n, 4, (1, 1, 5, 26), n)
  c, l, t = _gpu(cost, labels_first), _gpu(labels, labels_first, torch.uint8), _gpu(costs, labels_first)
  r, d = torch.from_numpy(rest).float().cuda(), torch.randn(1, 1, 5, 26, device="cuda")

  def step(c, l, t, r, d):
    leaf = c.detach().requires_grad_(True)
    loss = distill_costs(leaf, l, t, r, 1.0, labels_first)
    return (loss.detach(),) + torch.autograd.grad(loss, leaf, d) + best_labels(c, 3, labels_first=labels_first)

  def shifted(x):
    return torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)

  def strided(x):
    return torch.empty(x.shape + (2,), dtype=x.dtype, device="cuda")[..., 0].copy_(x)

  want = step(c, l, t, r, d)
  for other in (shifted, strided):
    assert all(torch.equal(a, b) for a, b in zip(step(*(other(x) for x in (c, l, t, r, d))), want))
  one = step(c, l, t, r, torch.ones((), device="cuda").expand(d.shape))
  assert all(torch.equal(a, b) for a, b in zip(one, step(c, l, t, r, torch.ones_like(d))))


def test_a_captured_step_and_two_streams(gpu):
  from mplayers_amd import best_labels, distill_costs
  g = torch.Generator(device="cuda").manual_seed(2)
  teacher = torch.randn(2, 1, 21, 13, 17, device="cuda", generator=g)
  student = torch.randn(2, 1, 21, 13, 17, device="cuda", generator=g).requires_grad_(True)
  dloss = torch.rand(2, 1, 13, 17, device="cuda", generator=g)

  def step():
    labels, costs, rest = best_labels(teacher, 4, 2.0, dtype=torch.float16)
    loss = distill_costs(student, labels, costs, rest, 2.0)
    return labels, costs, rest, loss.detach(), torch.autograd.grad(loss, student, dloss)[0]

  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    step()
  torch.cuda.current_stream().wait_stream(stream)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  for k in range(3):
    for t in out:
      t.fill_(7)
    teacher.mul_(1.25)
    with torch.no_grad():
      student.add_(teacher, alpha=0.1 * k)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))
  want = step()
  streams = [torch.cuda.Stream() for _ in range(2)]
  torch.cuda.synchronize()
  for _ in range(3):
    got = []
    for stream in streams:
      with torch.cuda.stream(stream):
        got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for s in got for a, b in zip(s, want))


def test_autograd_modes(gpu):
  from mplayers_amd import distill_costs
  cost, labels, costs, rest = _problem(9, 3, (1, 1, 4, 6), 1, 0.0)
  c, l, t, r = (_gpu(cost, True).requires_grad_(True), _gpu(labels, True, torch.uint8), _gpu(costs, True),
                torch.from_numpy(rest).float().cuda())
  want = distill_costs(c, l, t, r)
  with torch.no_grad():
    got = distill_costs(c, l, t, r)
  assert not got.requires_grad and torch.equal(got, want)
  with torch.inference_mode():
    assert torch.equal(distill_costs(c, l, t, r), want)
  (first,) = torch.autograd.grad(want.sum(), c, create_graph=True)
  (again,) = torch.autograd.grad(distill_costs(c, l, t, r).sum(), c)
  assert torch.equal(first, again)
  with pytest.raises(RuntimeError, match="differentiated twice"):
    torch.autograd.grad(first.sum(), c)
  loss = distill_costs(c, l, t, r)
  t.add_(1)
  with pytest.raises(RuntimeError, match="modified by an inplace"):
    loss.sum().backward()


def test_a_volume_beyond_32_bits(gpu):
  """More than 2^32 entries: the last pixels' results are theirs."""
  from mplayers_amd import best_labels, distill_costs
  n, pixels = 24, 180_000_011
  cost = torch.zeros(1, 1, n, 1, pixels, device="cuda", dtype=torch.float16)
  tail = torch.randn(1, 1, n, 1, 100, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
  cost[..., -100:] = tail
  labels, costs, rest = best_labels(cost, 2, dtype=torch.float16)
  want = best_labels(tail, 2, dtype=torch.float16)
  assert all(torch.equal(a[..., -100:], b) for a, b in zip((labels, costs, rest), want))
  assert bool((labels[0, 0, 0] == 0)[..., :-100].all()) and bool((labels[0, 0, 1] == 1)[..., :-100].all())
  loss = distill_costs(cost, labels, costs, rest)
  assert torch.equal(loss[..., -100:], distill_costs(tail, *want))
  leaf = cost.requires_grad_(True)
  d = torch.ones((), device="cuda").expand(loss.shape)
  (grad,) = torch.autograd.grad(distill_costs(leaf, labels, costs), leaf, d)
  small = tail.clone().requires_grad_(True)
  (part,) = torch.autograd.grad(distill_costs(small, *want[:2]).sum(), small)
  assert torch.equal(grad[..., -100:], part)


def test_refusals(gpu):
  from mplayers_amd import best_labels, distill_costs
  cost = torch.zeros(1, 1, 4, 5, 6, device="cuda")
  labels, costs = torch.zeros(1, 1, 2, 5, 6, dtype=torch.uint8, device="cuda"), torch.zeros(1, 1, 2, 5, 6, device="cuda")
  rest = torch.zeros(1, 1, 5, 6, device="cuda")
  good = dict(cost=cost, labels=labels, costs=costs, rest=rest)
  for wrong in [dict(cost=cost[0]), dict(cost=cost.double()), dict(labels=labels.int()), dict(labels=labels.cpu()),
                dict(costs=costs.double()), dict(costs=costs.cpu()), dict(labels=labels[..., :5]), dict(costs=costs[:, :, :1]),
                dict(costs=costs.clone().requires_grad_(True)), dict(rest=rest.double()), dict(rest=rest[0]), dict(rest=rest.cpu()),
                dict(rest=rest[..., :5]), dict(rest=rest.clone().requires_grad_(True)), dict(temperature=0.0), dict(temperature=-1.0),
                dict(temperature=INF), dict(temperature=NAN), dict(temperature=1e-45), dict(labels_first=False),
                dict(labels=labels[:, :, :0], costs=costs[:, :, :0]),
                dict(cost=torch.zeros(1, 1, 257, 5, 6, device="cuda")), dict(cost=torch.zeros(1, 1, 0, 5, 6, device="cuda")),
                dict(labels=labels[:, :, :1].expand(1, 1, 257, 5, 6), costs=costs[:, :, :1].expand(1, 1, 257, 5, 6))]:
    with pytest.raises(RuntimeError):
      distill_costs(**{**good, **wrong})
  for wrong in [dict(cost=cost[0]), dict(cost=cost.long()), dict(k=0), dict(k=5), dict(k=-1), dict(temperature=0.0),
                dict(temperature=INF), dict(dtype=torch.float64), dict(dtype=7)]:
    with pytest.raises(RuntimeError):
      best_labels(**{**dict(cost=cost, k=2), **wrong})
  empty = torch.zeros(0, 1, 4, 5, 6, device="cuda", requires_grad=True)
  kept = best_labels(empty, 2)
  assert [tuple(t.shape) for t in kept] == [(0, 1, 2, 5, 6), (0, 1, 2, 5, 6), (0, 1, 5, 6)]
  loss = distill_costs(empty, *kept)
  assert loss.shape == (0, 1, 5, 6) and torch.autograd.grad(loss.sum(), empty)[0].shape == empty.shape


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n", [3, 12, 21, 46, 60, 96, 130, 192, 256])
def test_a_rest_alone_has_no_gradient(gpu, n, labels_first):
  """The list names a masked label, so the teacher says nothing about the others: exactly none."""
  from mplayers_amd import distill_costs
  g = torch.Generator().manual_seed(n)
  cost = 4 * torch.randn(1, 1, n, 3, 40, generator=g)
  cost[:, :, n // 2] = INF
  labels = torch.full((1, 1, 1, 3, 40), n // 2, dtype=torch.uint8)
  rest = torch.randn(1, 1, 3, 40, generator=g).cuda()
  costs = torch.zeros(1, 1, 1, 3, 40)
  if not labels_first:
    cost, labels, costs = (t.movedim(2, -1).contiguous() for t in (cost, labels, costs))
  cost = cost.cuda().requires_grad_(True)
  loss = distill_costs(cost, labels.cuda(), costs.cuda(), rest, 0.7, labels_first)
  assert float(loss.detach().abs().max()) <= 12 * U  # (two logarithms of up to 256, half a step each)
  (grad,) = torch.autograd.grad(loss.sum(), cost)
  assert not bool(grad.any())


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n,k", [(3, 5), (4, 9), (8, 4), (8, 5), (12, 8), (21, 9), (32, 8), (40, 8), (40, 9), (60, 7), (60, 9), (130, 9)])
def test_lists_as_long_as_what_is_held_and_longer(gpu, n, k, labels_first):
  """Longer than the labels too: such a list names some twice."""
  cost, _, _, rest = _problem(n, 1, (2, 1, 3, 47), n + k)
  rng = np.random.default_rng(k)
  labels, costs = rng.integers(0, n, (2, 1, k, 3, 47)).astype(np.uint8), rng.random((2, 1, k, 3, 47)) * 5
  costs[rng.random(costs.shape) < 0.1] = INF
  _check_distill(_gpu(cost, labels_first), _gpu(labels, labels_first, torch.uint8), _gpu(costs, labels_first, torch.float16),
                 torch.from_numpy(rest).float().cuda(), 1.0, labels_first)
