"""Verified labels on the GPU against the plain form in 64 bits: equal, label by label, and kept alike.

Both sides hold weights and sums in 64 bits; they differ in the order of sums, by at most 256 * 2^-52 of one, and a result can
only differ where a uniform number of 24 bits falls that close to a border."""
import math

import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan
COUNTS = [1, 2, 3, 4, 5, 7, 8, 9, 11, 12, 13, 16, 17, 18, 20, 21, 24, 25, 28, 29, 32, 33, 40, 41, 47, 48, 49, 64, 65, 80, 81, 96,
          97, 112, 113, 128, 129, 160, 161, 192, 193, 224, 225, 255, 256]


def _verify(cost, draft, uniforms, draft_cost=None, labels_first=True, **temperatures):
  """cost, draft_cost (batch, cv, labels, H, W) whichever layout is asked for."""
  from mplayers_amd import verify_labels

  def volume(a):
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()
    return t if labels_first else t.permute(0, 1, 3, 4, 2).contiguous()

  temperatures = {k: (torch.as_tensor(np.asarray(v), dtype=torch.float32).cuda() if np.ndim(v) else v) for k, v in temperatures.items()}
  labels, kept = verify_labels(volume(cost), torch.from_numpy(draft).cuda(),
                               torch.from_numpy(np.ascontiguousarray(uniforms, np.float32)).cuda(),
                               None if draft_cost is None else volume(draft_cost), labels_first=labels_first, **temperatures)
  assert labels.dtype == torch.uint8 and kept.dtype == torch.bool
  return labels.cpu().numpy(), kept.cpu().numpy()


def _same(got, want):
  for g, w in zip(got, want):
    wrong = list(zip(*np.nonzero(g != w)))
    assert g.shape == w.shape and not wrong, "%d of %d: %s" % (len(wrong), w.size, wrong[:4])


def _uniforms(rng, shape):
  return rng.integers(0, 2 ** 24, shape).astype(np.float32) * np.float32(2.0 ** -24)


def _drawn(rng, cost, temperature, n):
  """n labels drawn from softmax(-cost / T), pixels without any get one at random; (n, batch, cv, H, W) uint8."""
  c = np.where(np.isnan(cost), INF, np.asarray(cost, np.float64))
  best = c.min(2, keepdims=True)
  weight = np.exp(-(c - np.where(np.isfinite(best), best, 0)) / temperature)
  target = rng.random((n,) + best.shape) * weight.sum(2, keepdims=True)
  label = (np.cumsum(weight, 2)[None] <= target).sum(3)
  return np.minimum(label, cost.shape[2] - 1).astype(np.uint8)


def _problem(n, shape, drafts, seed, masked=0.1, noise=0.7, t=1.0):
  rng = np.random.default_rng(seed)
  b, cv, h, w = shape
  cost = rng.standard_normal((b, cv, n, h, w)) * 2
  cost[..., ::2] = np.round(cost[..., ::2])  # ties
  draft_cost = cost + noise * rng.standard_normal(cost.shape)
  cost[rng.random(cost.shape) < masked] = INF
  draft_cost[rng.random(cost.shape) < masked] = INF
  cost, draft_cost = cost.astype(np.float32), draft_cost.astype(np.float32)
  draft = _drawn(rng, draft_cost, t, drafts)
  return cost, draft, _uniforms(rng, (2,) + draft.shape), draft_cost


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("with_costs", [True, False])
@pytest.mark.parametrize("n", COUNTS)
def test_label_counts(gpu, n, with_costs, labels_first):
  """Every number of labels that a kernel variant starts or ends with; one draft, and several; more pixels than a tile."""
  for drafts in (1, 3):
    cost, draft, u, draft_cost = _problem(n, (1, 2, 3, 25), drafts, 10 * n + drafts)
    draft_cost = draft_cost if with_costs else None
    _same(_verify(cost, draft, u, draft_cost, labels_first), oracle.verify_labels(cost, draft, u, draft_cost))


@pytest.mark.parametrize("n", [3, 16, 21, 60, 96, 192, 256])
@pytest.mark.parametrize("temperatures", [dict(temperature=2.5), dict(temperature=0.5, draft_temperature=3.0),
                                          dict(temperature=4.0, draft_temperature=0.3), dict(temperature=0.0),
                                          dict(temperature=1.0, draft_temperature=0.0), dict(temperature=INF),
                                          dict(temperature=1.0, draft_temperature=INF), dict(temperature=1e-30),
                                          dict(temperature=1e30, draft_temperature=1.0), dict(temperature=1e-38),
                                          dict(temperature=[0.5, 0.0, 2.0], draft_temperature=[1.0, 1.0, INF]),
                                          dict(temperature=[INF, 1.0, 0.1])])
def test_temperatures(gpu, n, temperatures):
  cost, draft, u, draft_cost = _problem(n, (3, 1, 2, 23), 2, n, t=2.0)
  for costs in (draft_cost, None):
    _same(_verify(cost, draft, u, costs, **temperatures), oracle.verify_labels(cost, draft, u, costs, **temperatures))


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n", [2, 9, 21, 70, 150, 256])
def test_costs_that_are_no_numbers(gpu, n, labels_first):
  """Pixels without candidates on either side, infinities, NaN, the type's extremes; drafted labels of every kind, those that
  the draft cannot have drawn among them; uniform numbers outside their range."""
  rng = np.random.default_rng(n)
  big = float(np.finfo(np.float32).max)
  i = np.arange(n)
  rows = [np.full(n, INF), np.full(n, NAN), np.full(n, -INF), np.full(n, big), np.full(n, -big), np.where(i % 2, 0.0, -0.0),
          np.where(i % 3, big, -big), np.where(i % 2, -INF, 1.0), np.where(i % 2, NAN, 0.5), np.where(i == n - 1, 3.0, INF),
          np.where(i == 0, -INF, INF), i * 1e-42, i * 50.0, rng.standard_normal(n), 2.0 ** (i % 120 - 60)]
  first, second = np.meshgrid(np.arange(len(rows)), np.arange(len(rows)))
  cost = np.stack([rows[k] for k in first.ravel()], 1).reshape(1, 1, n, 1, -1).astype(np.float32)
  other = np.stack([rows[k] for k in second.ravel()], 1).reshape(1, 1, n, 1, -1).astype(np.float32)
  draft = rng.integers(0, min(n + 2, 256), (3, 1, 1, 1, cost.shape[-1])).astype(np.uint8)
  u = _uniforms(rng, (2,) + draft.shape)
  u[:, 1, ..., ::7] = 0.0
  u[:, 1, ..., 1::7] = 1.0
  u[:, 1, ..., 2::7] = -1.0
  u[:, 1, ..., 3::7] = NAN
  u[:, 1, ..., 4::7] = INF
  u[:, 1, ..., 5::7] = 2.0
  for costs in (other, None):
    _same(_verify(cost, draft, u, costs, labels_first), oracle.verify_labels(cost, draft, u, costs))


@pytest.mark.parametrize("n", [4, 21, 60, 192])
def test_the_same_costs_keep_every_label(gpu, n):
  rng = np.random.default_rng(n)
  cost = (rng.standard_normal((1, 1, n, 5, 31)) * 3).astype(np.float32)
  draft = _drawn(rng, cost, 1.0, 2)
  u = _uniforms(rng, (2,) + draft.shape)
  u[0, 0] = np.float32(1 - 2.0 ** -24)
  labels, kept = _verify(cost, draft, u, cost)
  assert kept.all() and np.array_equal(labels, draft)
  # q 1 at the best label of a target at temperature 0
  best = cost.argmin(2)[None].astype(np.uint8)
  labels, kept = _verify(cost, best, u[:, :1], None, temperature=0.0)
  assert kept.all() and np.array_equal(labels, best)


@pytest.mark.parametrize("n", [8, 21, 60, 130, 256])
def test_targets_at_borders(gpu, n):
  """Costs of equal weights and uniform numbers that are their sums: 32 bits do not tell on which side a target lies."""
  rng = np.random.default_rng(n)
  cost = np.zeros((1, 1, n, 4, 33), np.float32)
  cost[..., 16:] = INF
  cost[:, :, : 1 << (n.bit_length() - 1), :, 16:] = 0.0  # a power of two of them: sums without rounding
  other = cost.copy()
  half = (1 << (n.bit_length() - 1)) // 2
  other[:, :, half:, :, 16:] = INF  # q is 2 p of the first half: a label stays where u < 1/2, else one of the second half
  draft = rng.integers(0, half, (3, 1, 1, 4, 33)).astype(np.uint8)
  u = (rng.integers(0, 64, (2,) + draft.shape) / 64).astype(np.float32)
  for costs in (other, None):
    for labels_first in (True, False):
      got, want = _verify(cost, draft, u, costs, labels_first), oracle.verify_labels(cost, draft, u, costs)
      _same([g[..., 16:] for g in got], [w[..., 16:] for w in want])


@pytest.mark.parametrize("n", [21, 60, 192])
@pytest.mark.parametrize("labels_first", [True, False])
def test_more_pixels_than_the_plain_form_can(gpu, n, labels_first):
  """Against 64 bits in torch: enough pixels that some need them."""
  from mplayers_amd import verify_labels
  g = torch.Generator(device="cuda").manual_seed(n)
  h, w = 201, 307
  cost = torch.randn(2, 1, n, h, w, device="cuda", generator=g) * 2
  other = cost + 0.4 * torch.randn(cost.shape, device="cuda", generator=g)
  for noise in (True, False):  # (no noise but a rounding: what is left of p is one)
    if not noise:
      other = (cost + 3.0) - 2.999
    p, q = (torch.softmax(-x.movedim(2, -1).double() / 1.5, -1) for x in (cost, other))
    draft = torch.multinomial(q.view(-1, n), 2, replacement=True, generator=g).t().reshape(2, 2, 1, h, w).to(torch.uint8).contiguous()
    u = torch.rand((2,) + draft.shape, device="cuda", generator=g)
    p_d, q_d = (x.expand(2, -1, -1, -1, -1, -1).gather(-1, draft.long()[..., None])[..., 0] for x in (p, q))
    border = (u[0].double() * q_d - p_d).abs() < 1e-13
    want_kept = u[0].double() * q_d < p_d
    left = (p - q).clamp(min=0).cumsum(-1)
    target = u[1].double() * left[..., -1]
    want = (left <= target[..., None]).sum(-1)
    border |= ~want_kept & ((left - target[..., None]).abs().amin(-1) < 1e-13)
    want = torch.where(want_kept, draft.long(), want.clamp(max=n - 1))
    volumes = [x if labels_first else x.movedim(2, -1).contiguous() for x in (cost, other)]
    labels, kept = verify_labels(volumes[0], draft, u, volumes[1], temperature=1.5, labels_first=labels_first)
    assert bool(((kept == want_kept) | border).all()) and bool(((labels == want) | border).all())
    if noise:
      assert float(border.float().mean()) < 1e-6 and 0.05 < float((~kept).float().mean()) < 0.5


def test_labels_are_distributed_as_the_target_says(gpu):
  """Drafted from q, verified against p: the frequencies are those of p, and no more labels change than have to."""
  from mplayers_amd import sample_labels, verify_labels
  g = torch.Generator(device="cuda").manual_seed(9)
  n, pixels = 7, 400_000
  one, two = torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g)
  cost, other = (x.view(1, 1, n, 1, 1).expand(1, 1, n, 1, pixels).contiguous() for x in (one, two))
  draft = sample_labels(other, torch.rand(1, 1, 1, pixels, device="cuda", generator=g))
  labels, kept = verify_labels(cost, draft, torch.rand(2, 1, 1, 1, pixels, device="cuda", generator=g), other)
  p, q = torch.softmax(-one.double(), 0), torch.softmax(-two.double(), 0)
  got = torch.bincount(labels.flatten().long(), minlength=n).double() / pixels
  # five standard deviations
  assert bool(((got - p).abs() <= 5 * (p * (1 - p) / pixels).sqrt()).all()), (got, p)
  stay = float(torch.minimum(p, q).sum())
  assert abs(float(kept.double().mean()) - stay) <= 5 * (stay * (1 - stay) / pixels) ** 0.5
  assert bool((labels == draft)[kept].all()) and bool((labels != draft)[~kept].all())


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n", [5, 24, 60, 200])
def test_the_number_of_drafts_changes_nothing(gpu, n, labels_first):
  cost, draft, u, draft_cost = _problem(n, (2, 1, 4, 37), 9, n)
  for costs in (draft_cost, None):
    labels, kept = _verify(cost, draft, u, costs, labels_first)
    for k in range(9):
      one = _verify(cost, draft[k], u[:, k], costs, labels_first)
      assert np.array_equal(one[0], labels[k]) and np.array_equal(one[1], kept[k])
    _same((labels, kept), oracle.verify_labels(cost, draft, u, costs))


@pytest.mark.parametrize("with_costs", [True, False])
@pytest.mark.parametrize("n,temperature", [(5, 1.0), (21, 1e-31), (40, 1e31), (130, 1.0), (21, INF)])
def test_many_drafts(gpu, n, temperature, with_costs):
  """More drafts than a wavefront has lanes, at temperatures that 32 bits leave to 64 as well; pixels at borders."""
  rng = np.random.default_rng(n)
  cost = np.round(rng.standard_normal((1, 1, n, 1, 9)) * 2).astype(np.float32) * np.float32(min(max(temperature, 1e-32), 1e32))
  other = np.roll(cost, 1, 2)
  draft = rng.integers(0, n + 1, (150, 1, 1, 1, 9)).astype(np.uint8)
  u = (rng.integers(0, 16, (2,) + draft.shape) / 16).astype(np.float32)
  costs = other if with_costs else None
  temperatures = dict(temperature=temperature)
  p = torch.softmax(-torch.from_numpy(cost).double().movedim(2, -1) / temperature, -1)
  q = torch.softmax(-torch.from_numpy(other).double().movedim(2, -1) / temperature, -1) if with_costs else None
  got, want = _verify(cost, draft, u, costs, **temperatures), oracle.verify_labels(cost, draft, u, costs, **temperatures)
  # (uniform numbers of four bits: a target may be a sum exactly, where 64 bits go by the order of their additions)
  told = np.ones(draft.shape, bool)
  d = torch.from_numpy(draft).long()
  p_d = p.expand(draft.shape + (n,)).gather(-1, d.clamp(max=n - 1)[..., None])[..., 0]
  q_d = torch.ones_like(p_d) if q is None else q.expand(draft.shape + (n,)).gather(-1, d.clamp(max=n - 1)[..., None])[..., 0]
  u0, u1 = torch.from_numpy(u[0]).double(), torch.from_numpy(u[1]).double()
  told &= ((u0 * q_d - p_d).abs() > 1e-12).numpy()
  left = (p - q).clamp(min=0).expand(draft.shape + (n,)) if with_costs else \
      torch.where(torch.arange(n) == d[..., None], 0.0, p.expand(draft.shape + (n,)))
  for weights in (left, p.expand(draft.shape + (n,))):
    sums = weights.cumsum(-1)
    told &= (((sums - u1[..., None] * sums[..., -1:]).abs().amin(-1) > 1e-12) | (sums[..., -1] == 0)).numpy()
  assert told.mean() > 0.3
  for g, w in zip(got, want):
    assert np.array_equal(g[told], w[told])


@pytest.mark.parametrize("n", [21, 24, 60, 192])
def test_alignment(gpu, n):
  from mplayers_amd import verify_labels
  cost, draft, u, draft_cost = (torch.from_numpy(a).cuda() for a in _problem(n, (1, 1, 5, 26), 2, n))

  def shifted(t):
    return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

  for labels_first in (True, False):
    volumes = [t if labels_first else t.movedim(2, -1).contiguous() for t in (cost, draft_cost)]
    want = verify_labels(volumes[0], draft, u, volumes[1], labels_first=labels_first)
    got = verify_labels(shifted(volumes[0]), shifted(draft), shifted(u), shifted(volumes[1]), labels_first=labels_first)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_captured_call_and_two_streams(gpu):
  from mplayers_amd import verify_labels
  cost, draft, u, draft_cost = (torch.from_numpy(a).cuda() for a in _problem(60, (2, 1, 13, 17), 2, 1))
  temperature = torch.tensor([1.0, 2.0], device="cuda")

  def step():
    return verify_labels(cost, draft, u, draft_cost, temperature=temperature) + verify_labels(cost, draft, u)

  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    step()
  torch.cuda.current_stream().wait_stream(stream)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  for _ in range(3):
    for t in out:
      t.fill_(1)
    u.copy_(u.flip(-1))
    temperature.mul_(1.5)
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


def test_a_volume_beyond_32_bits(gpu):
  from mplayers_amd import verify_labels
  n, pixels = 20, 215_000_009
  cost = torch.zeros(1, 1, n, 1, pixels, device="cuda")
  tail = torch.randn(1, 1, n, 1, 100, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
  cost[..., -100:] = tail
  draft = torch.full((1, 1, 1, pixels), 3, dtype=torch.uint8, device="cuda")
  u = torch.full((2, 1, 1, 1, pixels), 0.5, device="cuda")
  u[0, ..., :-100] = 0.01  # (p is 1/20 there)
  u[1, ..., -100:] = torch.rand(100, device="cuda")
  labels, kept = verify_labels(cost, draft, u)
  want = verify_labels(tail, draft[..., -100:].contiguous(), u[..., -100:].contiguous())
  assert torch.equal(labels[..., -100:], want[0]) and torch.equal(kept[..., -100:], want[1])
  assert bool(kept[..., :-100].all()) and bool((labels[..., :-100] == 3).all())


def test_refusals(gpu):
  from mplayers_amd import verify_labels
  cost = torch.zeros(2, 1, 4, 3, 5, device="cuda")
  draft = torch.zeros(2, 1, 3, 5, dtype=torch.uint8, device="cuda")
  u = torch.zeros(2, 2, 1, 3, 5, device="cuda")
  good = dict(cost=cost, draft=draft, uniforms=u, draft_cost=cost)
  each = torch.ones(2, device="cuda")
  for wrong in [dict(cost=cost.half()), dict(cost=cost.cpu()), dict(cost=cost[0], draft_cost=None), dict(draft=draft.int()),
                dict(draft=draft.cpu()), dict(draft=draft[..., :4]), dict(draft=draft[None, None]), dict(uniforms=u.double()),
                dict(uniforms=u.cpu()), dict(uniforms=u[0]), dict(uniforms=u[:1]), dict(uniforms=u[..., :4]),
                dict(draft_cost=cost.double()), dict(draft_cost=cost.cpu()), dict(draft_cost=cost[:, :, :3]),
                dict(cost=cost.transpose(3, 4).contiguous().transpose(3, 4)), dict(labels_first=False), dict(temperature=-1.0),
                dict(temperature=NAN), dict(temperature=each.cpu()), dict(temperature=each.double()), dict(temperature=each[:1]),
                dict(draft_temperature=-0.5), dict(draft_temperature=each.int()),
                dict(cost=torch.zeros(2, 1, 257, 3, 5, device="cuda"), draft_cost=None)]:
    with pytest.raises(RuntimeError):
      verify_labels(**{**good, **wrong})
  for wrong in [dict(cost=[0.0]), dict(draft=None), dict(temperature="1")]:
    with pytest.raises(TypeError):
      verify_labels(**{**good, **wrong})
  labels, kept = verify_labels(cost[:0], draft[:0], u[:, :0])
  assert labels.shape == kept.shape == (0, 1, 3, 5)
  labels, kept = verify_labels(cost, draft[None][:0], u[:, None][:, :0])
  assert labels.shape == kept.shape == (0, 2, 1, 3, 5)
