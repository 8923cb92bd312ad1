"""Labels drawn on the GPU against the plain form in 64 bits: equal, label by label.

Both sides hold weights and sums in 64 bits; their sums differ in order, by at most 256 * 2^-52 of the total, and a
label can only differ where a uniform number of 24 bits falls that close to a border."""
import math

import numpy as np
import pytest
import torch

from oracle import around_oracle

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan
COUNTS = [1, 2, 4, 5, 8, 11, 16, 17, 21, 24, 25, 32, 33, 48, 49, 64, 65, 96, 97, 128, 129, 192, 193, 255, 256]
FILTERS = [dict(), dict(top_k=3), dict(top_p=0.8), dict(min_p=0.1), dict(top_k=7, top_p=0.9, min_p=0.05, temperature=2.5)]


def _draw(cost, uniforms, labels_first=True, **parameters):
  """cost (batch, cv, labels, H, W) whichever layout is asked for."""
  from mplayers_amd import sample_labels
  cost = torch.from_numpy(np.ascontiguousarray(cost, np.float32)).cuda()
  if not labels_first:
    cost = cost.permute(0, 1, 3, 4, 2).contiguous()
  uniforms = torch.from_numpy(np.ascontiguousarray(uniforms, np.float32)).cuda()
  parameters = {k: (torch.as_tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32).cuda() if np.ndim(v) else v)
                for k, v in parameters.items()}
  return sample_labels(cost, uniforms, labels_first=labels_first, **parameters).cpu().numpy()


def _same(got, want):
  wrong = list(zip(*np.nonzero(got != want)))
  assert got.shape == want.shape and not wrong, "%d of %d: %s" % (len(wrong), want.size, wrong[:4])


def _uniforms(rng, shape):
  return rng.integers(0, 2 ** 24, shape).astype(np.float32) * np.float32(2.0 ** -24)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("which", range(len(FILTERS)))
@pytest.mark.parametrize("n", COUNTS)
def test_label_counts(gpu, n, which, labels_first):
  """Every number of labels that a kernel variant starts or ends with; costs with ties; more pixels than a tile."""
  rng = np.random.default_rng(100 * n + which)
  cost = rng.standard_normal((1, 1, n, 3, 25)) * 2
  cost[..., ::2] = np.round(cost[..., ::2])  # ties
  cost[rng.random(cost.shape) < 0.1] = INF
  u = _uniforms(rng, (2, 1, 1, 3, 25))
  want = around_oracle.draw_labels(cost.astype(np.float32), u, **FILTERS[which])
  _same(_draw(cost, u, labels_first, **FILTERS[which]), want)


@pytest.mark.parametrize("n", [3, 16, 21, 60, 96, 192, 256])
@pytest.mark.parametrize("parameters", [dict(top_p=0.0), dict(top_p=1e-6), dict(top_p=0.999999), dict(min_p=1.0),
                                        dict(min_p=1e-30), dict(top_k=1), dict(top_k=1000), dict(temperature=0.0),
                                        dict(temperature=1e-30), dict(temperature=1e30), dict(temperature=INF),
                                        dict(temperature=INF, top_p=0.5, top_k=5), dict(temperature=INF, min_p=0.5),
                                        dict(temperature=0.0, top_p=0.3, min_p=0.2)])
def test_extreme_parameters(gpu, n, parameters):
  rng = np.random.default_rng(n)
  cost = np.round(rng.standard_normal((1, 1, n, 2, 33)) * 4) / 2
  cost[rng.random(cost.shape) < 0.2] = INF
  u = _uniforms(rng, (1, 1, 1, 2, 33))
  want = around_oracle.draw_labels(cost.astype(np.float32), u, **parameters)
  _same(_draw(cost, u, **parameters), want)


@pytest.mark.parametrize("parameters", [dict(), dict(top_k=2), dict(top_p=0.7), dict(min_p=0.2),
                                        dict(top_k=4, top_p=0.9, min_p=0.01, temperature=0.5), dict(temperature=0.0)])
@pytest.mark.parametrize("n", [2, 9, 21, 70, 150, 256])
def test_costs_that_are_no_numbers(gpu, n, parameters):
  """Pixels without candidates, infinities of both signs, NaN, both zeros, the type's extremes, subnormal costs and
  costs that grow by factors; uniform numbers outside their range."""
  rng = np.random.default_rng(n)
  big = float(np.finfo(np.float32).max)
  rows = [np.full(n, INF), np.full(n, NAN), np.full(n, -INF), np.full(n, big), np.full(n, -big), np.zeros(n),
          np.where(np.arange(n) % 2, 0.0, -0.0), np.where(np.arange(n) % 3, big, -big), np.where(np.arange(n) % 2, -INF, 1.0),
          np.where(np.arange(n) % 2, NAN, 0.5), np.where(np.arange(n) == n - 1, 3.0, INF),
          np.where(np.arange(n) == n // 2, -INF, INF), np.arange(n) * 1e-42, 2.0 ** (np.arange(n) % 126 - 60),
          -2.0 ** (np.arange(n) % 126 - 60), np.where(np.arange(n) % 2, INF, -INF), np.where(np.arange(n) % 2, big, 0.0),
          1e-3 * 1.5 ** (np.arange(n) % 100)]
  uniforms = [0.0, 0.25, 0.5, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, NAN, INF, -INF, -0.0, 1e-40]
  with np.errstate(over="ignore"):
    cost = np.stack(rows, -1).astype(np.float32).reshape(1, 1, n, 1, len(rows))
  u = np.repeat(np.array(uniforms, np.float32), len(rows)).reshape(len(uniforms), 1, 1, 1, len(rows))
  u[2] = _uniforms(rng, u[2].shape)
  want = around_oracle.draw_labels(cost, u, **parameters)
  for labels_first in (True, False):
    _same(_draw(cost, u, labels_first, **parameters), want)


@pytest.mark.parametrize("parameters", [dict(), dict(top_k=2), dict(top_p=0.7), dict(min_p=0.2), dict(top_k=1, min_p=0.5),
                                        dict(top_k=4, top_p=0.9, min_p=0.01, temperature=0.5), dict(temperature=0.0),
                                        dict(temperature=[0.0], top_k=[3])])
@pytest.mark.parametrize("n", [2, 9, 21, 70, 150, 256])
def test_the_same_costs_with_ordinary_numbers(gpu, n, parameters):
  """Costs as above, but uniform numbers inside their range: those outside have a pixel drawn in 64 bits throughout."""
  rng = np.random.default_rng(n + 1)
  big = float(np.finfo(np.float32).max)
  odd = np.arange(n) % 2
  rows = [np.full(n, -INF), np.where(odd, -INF, 1.0), np.where(odd, 1.0, -INF), np.where(np.arange(n) == n - 1, -INF, np.arange(n)),
          np.where(odd, INF, -INF), np.where(odd, -INF, NAN), np.where(odd, -INF, -big), np.full(n, NAN), np.full(n, big),
          np.full(n, -big), np.where(odd, big, -big), np.where(odd, -big, INF), np.where(odd, big, 0.0), np.where(odd, 0.0, -0.0),
          np.arange(n) * 1e-42, np.where(odd, NAN, 0.5), 2.0 ** (np.arange(n) % 126 - 60), -2.0 ** (np.arange(n) % 126 - 60)]
  cost = np.stack(rows, -1).astype(np.float32).reshape(1, 1, n, 1, len(rows))
  for draws in (1, 3):
    u = _uniforms(rng, (draws, 1, 1, 1, len(rows)))
    want = around_oracle.draw_labels(cost, u, **parameters)
    for labels_first in (True, False):
      _same(_draw(cost, u, labels_first, **parameters), want)


@pytest.mark.parametrize("parameters", [dict(top_p=0.999, min_p=0.6), dict(top_p=0.95, min_p=0.8, temperature=0.3),
                                        dict(top_k=5, top_p=0.8, min_p=0.5), dict(top_p=0.5, temperature=20.0, min_p=0.99)])
@pytest.mark.parametrize("n", [4, 14, 41, 99, 250])
def test_min_p_at_a_cost_that_occurs(gpu, n, parameters):
  """Costs so large that all floats between them occur: the last cost that min_p leaves is one of them, beside pixels
  whose ties top_p cuts."""
  rng = np.random.default_rng(n)
  for offset in (1e6, -1e6, 3e4):
    cost = (offset + rng.standard_normal((1, 1, n, 3, 40))).astype(np.float32)
    for draws in (1, 2):
      u = _uniforms(rng, (draws, 1, 1, 3, 40))
      _same(_draw(cost, u, **parameters), around_oracle.draw_labels(cost, u, **parameters))


@pytest.mark.parametrize("n,labels_first", [(21, True), (21, False), (130, True)])
def test_parameters_of_each_image(gpu, n, labels_first):
  rng = np.random.default_rng(n)
  cost = rng.standard_normal((6, 2, n, 5, 7)) * 3
  u = _uniforms(rng, (3, 6, 2, 5, 7))
  parameters = dict(temperature=[1.0, 0.0, 0.3, 2.0, -1.0, 5.0], top_k=[0, 3, 1, 5, -2, 500], top_p=[1.0, 0.5, 0.9, 0.2, 2.0, -1.0],
                    min_p=[0.0, 0.1, 0.0, -3.0, 0.4, 1.5])
  want = around_oracle.draw_labels(cost.astype(np.float32), u, **parameters)
  _same(_draw(cost, u, labels_first, **parameters), want)
  _same(_draw(cost, u, labels_first, top_p=parameters["top_p"], temperature=2.0),
        around_oracle.draw_labels(cost.astype(np.float32), u, top_p=parameters["top_p"], temperature=2.0))


def test_temperatures_that_are_no_numbers(gpu):
  rng = np.random.default_rng(2)
  cost = rng.standard_normal((3, 1, 30, 4, 9))
  u = _uniforms(rng, (2, 3, 1, 4, 9))
  got = _draw(cost, u, temperature=[NAN, -NAN, -INF], top_k=[5, 0, 3], top_p=[0.5, 0.9, 1.0], min_p=[NAN, 0.5, NAN])
  _same(got, np.broadcast_to(cost.astype(np.float32).argmin(2), u.shape))


@pytest.mark.parametrize("masked", [0.0, 0.3, 0.97, 1.0])
@pytest.mark.parametrize("n", [21, 96, 200])
def test_masked_and_constant_images(gpu, n, masked):
  """Images whose labels are mostly out, and whose costs are all the same: every sum is a whole number, and a target
  may be one of them."""
  rng = np.random.default_rng(int(100 * masked) + n)
  cost = np.where(rng.random((1, 1, n, 6, 40)) < masked, INF, 0.75)
  u = _uniforms(rng, (2, 1, 1, 6, 40))
  u[1] = rng.integers(0, 8, u[1].shape) / 8
  for parameters in (dict(), dict(top_p=0.5), dict(top_k=4, top_p=0.25), dict(min_p=1.0), dict(top_p=0.75, min_p=0.5)):
    _same(_draw(cost, u, **parameters), around_oracle.draw_labels(cost.astype(np.float32), u, **parameters))


@pytest.mark.parametrize("n", [21, 70, 256])
def test_costs_close_together_in_a_wide_range(gpu, n):
  """Most costs within 1e-3 of each other and a few far away, or growing by factors: the thresholds are not found by
  halving the range."""
  rng = np.random.default_rng(n)
  cost = 1 + 1e-3 * rng.random((1, 1, n, 4, 33))
  cost[:, :, ::7] = 50 * rng.random(cost[:, :, ::7].shape)
  cost[..., 16:] = 2.0 ** rng.uniform(-100, 100, cost[..., 16:].shape)
  u = _uniforms(rng, (3, 1, 1, 4, 33))
  for parameters in (dict(top_k=n // 2), dict(top_p=0.6), dict(top_k=n - 1, top_p=0.3, min_p=0.2), dict(top_p=0.99, temperature=20)):
    _same(_draw(cost, u, **parameters), around_oracle.draw_labels(cost.astype(np.float32), u, **parameters))


@pytest.mark.parametrize("height,width", [(1, 1), (1, 63), (1, 64), (1, 65), (7, 19), (16, 16)])
@pytest.mark.parametrize("n", [12, 21, 192])
def test_image_sizes_and_items(gpu, n, height, width):
  rng = np.random.default_rng(height * width)
  cost = rng.standard_normal((2, 2, n, height, width))
  u = _uniforms(rng, (1, 2, 2, height, width))
  for labels_first in (True, False):
    for parameters in (dict(), dict(top_p=0.6)):
      _same(_draw(cost, u, labels_first, **parameters),
            around_oracle.draw_labels(cost.astype(np.float32), u, **parameters))


@pytest.mark.parametrize("draws", [1, 2, 7, 64, 300])
@pytest.mark.parametrize("n", [7, 21, 100, 256])
def test_many_draws(gpu, n, draws):
  rng = np.random.default_rng(draws)
  cost = rng.standard_normal((1, 1, n, 2, 5))
  u = _uniforms(rng, (draws, 1, 1, 2, 5))
  for parameters in (dict(), dict(top_k=5, top_p=0.95)):
    want = around_oracle.draw_labels(cost.astype(np.float32), u, **parameters)
    _same(_draw(cost, u, **parameters), want)


def test_frequencies(gpu):
  """The labels of many pixels with the same costs come as often as their probabilities say, within six standard
  deviations."""
  rng = np.random.default_rng(1)
  pixels = 200_000
  row = np.array([0.0, 0.7, 0.2, INF, 3.0, 0.2])
  u = _uniforms(rng, (1, 1, 1, 1, pixels))
  got = _draw(np.broadcast_to(row.reshape(1, 1, 6, 1, 1), (1, 1, 6, 1, pixels)), u, temperature=0.5)
  share = np.exp(-row / 0.5) / np.exp(-row / 0.5).sum()
  count = np.bincount(got.ravel(), minlength=6)
  assert (np.abs(count - pixels * share) <= 6 * np.sqrt(pixels * share * (1 - share)) + 1e-9).all()


def test_addresses_streams_and_replays(gpu):
  """Tensors one entry behind an aligned address; a stream of their own; a captured call replayed on new numbers,
  with eager work between the replays."""
  from mplayers_amd import sample_labels
  rng = np.random.default_rng(12)
  for n in (20, 96):
    cost = rng.standard_normal((1, 1, n, 8, 11)).astype(np.float32)
    u = _uniforms(rng, (2, 1, 1, 8, 11))
    want = around_oracle.draw_labels(cost, u, top_p=0.9)
    for labels_first in (True, False):
      flat = cost if labels_first else cost.transpose(0, 1, 3, 4, 2)
      shape = flat.shape
      flat = torch.from_numpy(np.concatenate([[0], np.ascontiguousarray(flat).ravel()]).astype(np.float32))
      stream = torch.cuda.Stream()
      with torch.cuda.stream(stream):
        on = flat.cuda()[1:].view(shape)
        uniforms = torch.from_numpy(np.concatenate([[0], u.ravel()]).astype(np.float32)).cuda()[1:].view(u.shape)
        got = sample_labels(on, uniforms, top_p=0.9, labels_first=labels_first)
      stream.synchronize()
      _same(got.cpu().numpy(), want)
  temperature = torch.ones(1, device="cuda")
  uniforms = torch.zeros(u.shape, device="cuda")
  cost_gpu = torch.from_numpy(cost).cuda()
  sample_labels(cost_gpu, uniforms, temperature=temperature, top_k=9)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = sample_labels(cost_gpu, uniforms, temperature=temperature, top_k=9)
  for t in (1.0, 0.25, 3.0):
    u = _uniforms(rng, u.shape)
    uniforms.copy_(torch.from_numpy(u))
    temperature.fill_(t)
    out.fill_(77)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    _same(out.cpu().numpy(), around_oracle.draw_labels(cost, u, temperature=t, top_k=9))


def test_nothing_but_the_labels_is_written(gpu):
  from mplayers_amd import _lib
  rng = np.random.default_rng(3)
  for n, pixels in ((21, 67), (192, 65)):
    cost = torch.from_numpy(rng.standard_normal((n, pixels)).astype(np.float32)).cuda()
    u = torch.rand(3, pixels, device="cuda")
    room = torch.full((3 * pixels + 64,), 201, dtype=torch.uint8, device="cuda")
    rc = _lib.load().mpl_sample_labels(1, cost.data_ptr(), u.data_ptr(), 1, 1, n, pixels, 3, None, 1.0, None, 0, None, 0.9,
                                       None, 0.0, room.data_ptr() + 32, torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "sample_labels")
    room = room.cpu()
    assert (room[:32] == 201).all() and (room[-32:] == 201).all() and (room[32:-32] < n).all()


def test_a_volume_beyond_32_bits(gpu):
  """More than 2^32 costs and, in the draws, more labels than 2^31: the last pixels are drawn as alone."""
  from mplayers_amd import sample_labels
  n, pixels = 3, 1_500_000_007
  cost = torch.zeros(1, 1, n, 1, pixels, device="cuda")
  rng = np.random.default_rng(6)
  tail = rng.standard_normal((1, 1, n, 1, 70)).astype(np.float32)
  cost[..., -70:] = torch.from_numpy(tail).cuda()
  u = torch.zeros(2, 1, 1, 1, pixels, device="cuda")
  tail_u = _uniforms(rng, (2, 1, 1, 1, 70))
  u[..., -70:] = torch.from_numpy(tail_u).cuda()
  for parameters in (dict(), dict(top_p=0.7)):
    got = sample_labels(cost, u, **parameters)
    _same(got[..., -70:].cpu().numpy(), around_oracle.draw_labels(tail, tail_u, **parameters))
    assert int(got[..., :-70].max()) == 0
    del got


def test_refusals(gpu):
  from mplayers_amd import sample_labels
  cost, u = torch.zeros(2, 1, 4, 3, 3, device="cuda"), torch.zeros(2, 1, 3, 3, device="cuda")
  two = torch.ones(2, device="cuda")
  for wrong in [dict(cost=cost.double()), dict(cost=cost.cpu()), dict(cost=cost.transpose(3, 4)[..., 1:]), dict(cost=cost[0]),
                dict(uniforms=u.cpu()), dict(uniforms=u.half()), dict(uniforms=u[:1]), dict(uniforms=u[..., ::2]),
                dict(uniforms=u[0]), dict(labels_first=False), dict(temperature=-1.0), dict(temperature=NAN), dict(top_k=-1),
                dict(top_k=1.5), dict(top_k=True), dict(top_p=1.5), dict(top_p=-0.5), dict(min_p=2.0), dict(min_p=NAN),
                dict(top_p=two.cpu()), dict(top_p=two[:1]), dict(top_p=two.double()), dict(top_k=two),
                dict(temperature=torch.ones(4, device="cuda")[::2]), dict(cost=torch.zeros(2, 1, 257, 3, 3, device="cuda")),
                dict(cost=torch.zeros(2, 1, 0, 3, 3, device="cuda"))]:
    with pytest.raises(RuntimeError):
      sample_labels(**{**dict(cost=cost, uniforms=u), **wrong})
  assert torch.equal(sample_labels(cost, u, temperature=np.float32(2), top_k=np.int64(2)), sample_labels(cost, u, temperature=2, top_k=2))
  assert sample_labels(cost[:0], u[:0]).shape == (0, 1, 3, 3)
  assert sample_labels(cost, u[None][:0]).shape == (0, 2, 1, 3, 3)
