"""Layer norm in the layout change on the GPU against its plain form in 64 bits.

Tolerances, with u = 2^-24 and, for each pixel, A = max |x|, r = 1 / sqrt(var + eps) and X = max |xhat|.  A mean is a sum of at
most 32 labels' differences, of up to 2 A, from a first one and of 8 wavefronts' such: 2 u A for the differences, the average
partial sum of 33 A u, 3 u A for the division and what is added again, and so 2 + 2 + 9 + 3 over the wavefronts, 54 u A.  So a
difference from it is off by 55 u A, r by a part of 54 u A r, and xhat by e = 64 u (1 + |xhat|) (1 + A r), its own roundings in it.
  y        e |weight| and two roundings more
  dx       with G = max |g|: r (46 u G + e G X + X (45 u G X + G e) + the part of r) <= 5 * 64 u r G (1 + A r) (1 + X)^2,
           and half a step of its type
  dweight  the e of each term, and a sum of `run` tiles of a workgroup, of 64 lanes and of 4 wavefronts:
           (run + 16) u sum |dy xhat|;  dbias (run + 16) u sum |dy|"""
import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
COUNTS = [1, 2, 4, 5, 8, 9, 11, 12, 13, 16, 17, 20, 21, 24, 25, 28, 29, 32, 33, 48, 49, 60, 64, 65, 96, 97, 128, 129, 192, 193,
          255, 256]


def _flat(t, labels_first):
  a = t.detach().double().cpu().numpy()
  a = np.moveaxis(a, 2, -1) if labels_first else a
  return a.reshape(-1, a.shape[-1])


def _within(name, got, want, tolerance):
  off = np.abs(got - want)
  assert got.shape == want.shape and bool((off <= tolerance).all()), \
      "%s: %g times the tolerance" % (name, np.max(off / np.maximum(tolerance, 1e-300)))


def _check(x, weight, bias, eps, dy, labels_first, run=1):
  from mplayers_amd import labels_last_norm
  y = labels_last_norm(x, weight, bias, eps, labels_first)
  assert y.dtype == torch.float32 and y.is_contiguous()
  leaves = [t for t in (x, weight, bias) if t is not None and t.requires_grad]
  grads = dict(zip((id(t) for t in leaves), torch.autograd.grad(y, leaves, dy)))
  n = y.shape[-1]
  flat, d = _flat(x, labels_first), _flat(dy, False)
  w = np.ones(n) if weight is None else weight.detach().double().cpu().numpy()
  b = np.zeros(n) if bias is None else bias.detach().double().cpu().numpy()
  want, xhat, r = oracle.norm(flat, w, b, eps)
  scale = 1 + np.abs(flat).max(1, keepdims=True) * r
  e = 64 * U * (1 + np.abs(xhat)) * scale
  _within("y", _flat(y, False), want, e * np.abs(w) + 4 * U * (np.abs(want) + np.abs(b)))
  dx, dweight, dbias = oracle.norm_grad(flat, w, eps, d)
  largest = np.abs(d * w).max(1, keepdims=True)
  if x.requires_grad:
    got = grads[id(x)]
    assert got.dtype == x.dtype and got.shape == x.shape
    tolerance = 5 * 64 * U * r * largest * scale * (1 + np.abs(xhat).max(1, keepdims=True)) ** 2
    step = 0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
    least = 0 if x.dtype == torch.float32 else torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    _within("dx", _flat(got, labels_first), dx, tolerance * (1 + step) + step * np.abs(dx) + least)
  if weight is not None and weight.requires_grad:
    _within("dweight", grads[id(weight)].double().cpu().numpy(), dweight,
            (np.abs(d) * e).sum(0) + (run + 16) * U * np.abs(d * xhat).sum(0))
  if bias is not None and bias.requires_grad:
    _within("dbias", grads[id(bias)].double().cpu().numpy(), dbias, (run + 16) * U * np.abs(d).sum(0))


def _inputs(b, cv, n, h, w, dtype, labels_first, offset=3.0):
  g = torch.Generator().manual_seed(n * 7 + h)
  x = torch.randn(b, cv, n, h, w, generator=g) * (0.1 + 5 * torch.rand(b, cv, 1, h, w, generator=g)) + offset
  x = (x if labels_first else x.movedim(2, -1).contiguous()).to(dtype).cuda().requires_grad_(True)
  weight = (1 + 0.3 * torch.randn(n, generator=g)).cuda().requires_grad_(True)
  bias = torch.randn(n, generator=g).cuda().requires_grad_(True)
  return x, weight, bias, torch.randn(b, cv, h, w, n, generator=g).cuda()


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", COUNTS)
def test_label_counts(gpu, n, dtype, labels_first):
  """Every number of labels that a kernel variant starts or ends with; a tile that is not full, and two images."""
  x, weight, bias, dy = _inputs(2, 1, n, 3, 47, dtype, labels_first)
  _check(x, weight, bias, 1e-5, dy, labels_first)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("b,cv,n,h,w", [(1, 1, 21, 1, 1), (3, 2, 21, 1, 64), (1, 1, 96, 1, 65), (2, 2, 40, 5, 13), (1, 1, 8, 1, 256),
                                        (1, 3, 6, 9, 31), (1, 1, 192, 2, 1), (7, 1, 3, 1, 1)])
def test_sizes(gpu, b, cv, n, h, w, labels_first):
  x, weight, bias, dy = _inputs(b, cv, n, h, w, torch.float32, labels_first)
  _check(x, weight, bias, 1e-5, dy, labels_first)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n,pixels", [(4, 600_001), (20, 530_011), (130, 133_000), (70, 140_003)])
def test_more_tiles_than_workgroups(gpu, n, pixels, labels_first):
  """A gradient's workgroups go over several tiles each (2048 of 64 or 256 pixels at a time)."""
  x, weight, bias, dy = _inputs(1, 1, n, 1, pixels, torch.float32, labels_first)
  _check(x, weight, bias, 1e-5, dy, labels_first, run=2)


@pytest.mark.parametrize("n", [5, 21, 96])
@pytest.mark.parametrize("which", ["neither", "weight", "bias", "fixed", "x fixed", "only bias"])
def test_which_gradients(gpu, n, which):
  x, weight, bias, dy = _inputs(1, 1, n, 5, 33, torch.float32, True)
  if which in ("neither", "bias"):
    weight = None
  if which in ("neither", "weight"):
    bias = None
  if which in ("fixed", "only bias"):
    weight = weight.detach()
  if which == "fixed":
    bias = bias.detach()
  if which in ("x fixed", "only bias"):
    x = x.detach()
  _check(x, weight, bias, 1e-5, dy, True)


@pytest.mark.parametrize("offset", [0.0, 1e3, -1e5])
@pytest.mark.parametrize("n", [3, 30, 150])
def test_large_means(gpu, n, offset):
  """Differences from the mean, not of squares: costs whose mean is far larger than their spread."""
  x, weight, bias, dy = _inputs(1, 1, n, 3, 25, torch.float32, True, offset)
  _check(x, weight, bias, 1e-5, dy, True)


@pytest.mark.parametrize("n", [1, 7, 21, 100])
def test_equal_costs(gpu, n):
  from mplayers_amd import labels_last_norm
  x = torch.full((1, 1, n, 2, 3), 2.0, device="cuda", requires_grad=True)
  bias = torch.arange(n, device="cuda", dtype=torch.float32)
  y = labels_last_norm(x, torch.full((n,), 3.0, device="cuda"), bias, 0.25)
  assert torch.equal(y.detach(), bias.expand_as(y))
  dy = torch.zeros(1, 1, 2, 3, n, device="cuda")
  dy[..., 0] = 1
  (dx,) = torch.autograd.grad(y, x, dy)
  want = torch.full((n,), -6.0 / n)
  want[0] += 6  # r = 2
  # (a mean and a difference of it)
  assert torch.allclose(dx.cpu(), want.view(1, 1, n, 1, 1).expand_as(dx), rtol=0, atol=6 * 4 * U)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n", [2, 3, 7, 13, 21, 47, 100, 133, 251])
def test_equal_costs_of_any_size(gpu, n, labels_first):
  """The mean of equal costs is that cost, whatever its bits: differences of 0, so the bias comes out."""
  from mplayers_amd import labels_last_norm
  g = torch.Generator().manual_seed(n)
  x = (torch.randn(1, 2, 1, 5, 31, generator=g) * 10.0 ** torch.randint(-3, 30, (1, 2, 1, 5, 31), generator=g)).cuda()
  x = x.expand(1, 2, n, 5, 31)
  bias = torch.randn(n, generator=g).cuda()
  y = labels_last_norm(x if labels_first else x.movedim(2, -1), None, bias, 1e-5, labels_first)
  assert torch.equal(y, bias.expand_as(y))


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 3, 8, 12, 16, 21, 32, 60, 130, 192, 256])
def test_costs_far_apart(gpu, n, dtype, labels_first):
  """The type's largest number as a mask, and costs whose squares are beyond fp32, in some of the pixels and not in others."""
  x, weight, bias, dy = _inputs(2, 1, n, 3, 47, dtype, True)
  largest = torch.finfo(dtype).max
  with torch.no_grad():
    x[0, 0, 0, :, ::3] = largest
    x[0, 0, n - 1, :, 1::6] = -largest
    x[1, 0, n // 2, 0] = min(1e22, largest)
    x[1, 0, :, 1, ::2] *= min(1e20, largest / 1e3)
    x[1, 0, :, 2, ::5] = largest
  if not labels_first:
    x = x.detach().movedim(2, -1).contiguous().requires_grad_(True)
  _check(x, weight, bias, 1e-5, dy, labels_first)
  _check(x, weight, bias, 1e38, dy, labels_first)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n", [4, 21, 50, 130])
def test_costs_that_are_no_numbers_stay_in_their_pixel(gpu, n, labels_first):
  from mplayers_amd import labels_last_norm
  x, weight, bias, dy = _inputs(1, 1, n, 5, 30, torch.float32, labels_first)
  dy = dy.requires_grad_(False)
  bad = x.detach().clone()
  at = bad if labels_first else bad.movedim(-1, 2)
  at[0, 0, n // 2, 1, 3] = float("nan")
  at[0, 0, 0, 2, 7] = float("inf")
  at[0, 0, n - 1, 4, 29] = -float("inf")
  bad.requires_grad_(True)
  spoilt = torch.zeros(5, 30, dtype=torch.bool, device="cuda")
  spoilt[1, 3] = spoilt[2, 7] = spoilt[4, 29] = True
  y, z = (labels_last_norm(t, weight, bias, labels_first=labels_first) for t in (x, bad))
  assert bool(z[0, 0][spoilt].isnan().all()) and torch.equal(y[0, 0][~spoilt], z[0, 0][~spoilt])
  (dx,), (dz,) = torch.autograd.grad(y, x, dy), torch.autograd.grad(z, bad, dy)
  if labels_first:
    dx, dz = dx.movedim(2, -1), dz.movedim(2, -1)
  assert bool(dz[0, 0][spoilt].isnan().all()) and torch.equal(dx[0, 0][~spoilt], dz[0, 0][~spoilt])


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_alignment_and_strides(gpu, dtype, labels_first):
  """Inputs one entry behind an aligned address, with other strides, a gradient that is broadcast, weights with gaps."""
  from mplayers_amd import labels_last_norm
  n, h, w = 24, 5, 26
  x, weight, bias, dy = _inputs(1, 1, n, h, w, dtype, labels_first)
  y = labels_last_norm(x, weight, bias, labels_first=labels_first)
  want = (y.detach(),) + torch.autograd.grad(y, (x, weight, bias), dy)
  room = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")
  shifted = room[1:].view(x.shape).copy_(x.detach()).requires_grad_(True)
  strided = torch.empty(x.shape[:3] + (w, h), dtype=dtype, device="cuda").transpose(3, 4) if labels_first else \
      torch.empty((1, 1, n, h, w), dtype=dtype, device="cuda").movedim(2, -1)
  strided = strided.copy_(x.detach()).requires_grad_(True)
  assert not strided.is_contiguous()
  for other in (shifted, strided):
    gaps = [torch.stack([t.detach(), t.detach()], 1)[:, 0].requires_grad_(True) for t in (weight, bias)]
    far = torch.empty(dy.numel() + 1, device="cuda")[1:].view(dy.shape).copy_(dy)
    z = labels_last_norm(other, gaps[0], gaps[1], labels_first=labels_first)
    got = (z.detach(),) + torch.autograd.grad(z, (other, gaps[0], gaps[1]), far)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
  y = labels_last_norm(x, weight, bias, labels_first=labels_first)
  one = torch.autograd.grad(y, (x, weight, bias), torch.ones((), device="cuda").expand(y.shape), retain_graph=True)
  all_of = torch.autograd.grad(y, (x, weight, bias), torch.ones(y.shape, device="cuda"))
  assert all(torch.equal(a, b) for a, b in zip(one, all_of))


def test_the_gradient_against_differences(gpu):
  """The directional derivative in 64 bits of the plain form, at a random direction: the gradient's own formula is not used."""
  x, weight, bias, dy = _inputs(1, 1, 21, 3, 20, torch.float32, True)
  from mplayers_amd import labels_last_norm
  y = labels_last_norm(x, weight, bias)
  grads = torch.autograd.grad(y, (x, weight, bias), dy)
  rng = np.random.default_rng(3)
  values = [_flat(x, True), weight.detach().double().cpu().numpy(), bias.detach().double().cpu().numpy()]
  flat = [_flat(grads[0], True), grads[1].double().cpu().numpy(), grads[2].double().cpu().numpy()]
  d = _flat(dy, False)
  for k in range(3):
    h = rng.standard_normal(values[k].shape)
    ends = []
    for step in (1e-5, -1e-5):
      moved = [v + step * h if i == k else v for i, v in enumerate(values)]
      ends.append((oracle.norm(moved[0], moved[1], moved[2], 1e-5)[0] * d).sum())
    want, got = (ends[0] - ends[1]) / 2e-5, (flat[k] * h).sum()
    # differences: third derivatives times 1e-10 and 2^-52 * 1e5 of sums of some thousands; the gradient: 2^-24 * 1e3
    assert abs(got - want) <= 1e-4 * (1 + np.abs(flat[k] * h).sum())


def test_same_bits_and_two_streams(gpu):
  """The sums have an order of their own: repeated calls, also two at once, give the same bits."""
  from mplayers_amd import labels_last_norm
  x, weight, bias, dy = _inputs(1, 1, 60, 300, 401, torch.bfloat16, True)

  def step():
    y = labels_last_norm(x, weight, bias)
    return (y.detach(),) + torch.autograd.grad(y, (x, weight, bias), dy)

  want = step()
  streams = [torch.cuda.Stream() for _ in range(2)]
  torch.cuda.synchronize()
  for _ in range(3):
    got = []
    for stream in streams:
      with torch.cuda.stream(stream):
        got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_a_captured_step(gpu):
  from mplayers_amd import labels_last_norm
  x, weight, bias, dy = _inputs(2, 1, 21, 13, 17, torch.float16, True)

  def step():
    y = labels_last_norm(x, weight, bias)
    return (y.detach(),) + torch.autograd.grad(y, (x, weight, bias), dy)

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
    with torch.no_grad():
      x.add_(0.25 * k)
      weight.mul_(1.5)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_autograd_modes(gpu):
  from mplayers_amd import labels_last_norm
  x, weight, bias, dy = _inputs(1, 1, 9, 4, 6, torch.float32, True)
  want = labels_last_norm(x, weight, bias)
  with torch.no_grad():
    got = labels_last_norm(x, weight, bias)
  assert not got.requires_grad and torch.equal(got, want)
  with torch.inference_mode():
    assert torch.equal(labels_last_norm(x, weight, bias), want)
  assert not labels_last_norm(x.detach(), weight.detach()).requires_grad
  # a gradient that is recorded is the same; one of it is refused, not silently zero
  first = torch.autograd.grad(want, (x, weight), dy, create_graph=True)
  again = torch.autograd.grad(labels_last_norm(x, weight, bias), (x, weight), dy)
  assert all(torch.equal(a, b) for a, b in zip(first, again))
  with pytest.raises(RuntimeError, match="differentiated twice"):
    torch.autograd.grad(first[0].sum(), x)
  y = labels_last_norm(x, weight, bias)
  with torch.no_grad():
    weight.add_(1)
  with pytest.raises(RuntimeError, match="modified by an inplace"):
    y.sum().backward()


def test_refusals(gpu):
  from mplayers_amd import labels_last_norm
  x, weight = torch.zeros(1, 1, 4, 4, 5, device="cuda"), torch.ones(4, device="cuda")
  good = dict(x=x, weight=weight, bias=weight)
  for wrong in [dict(x=x[0]), dict(x=x.double()), dict(x=x.int()), dict(weight=weight.cpu()), dict(weight=weight.double()),
                dict(weight=weight[:3]), dict(weight=weight[None]), dict(bias=weight.half()), dict(labels_first=False),
                dict(eps=-1e-9), dict(eps=float("nan")), dict(eps=float("inf")), dict(eps=1e39),
                dict(x=torch.zeros(1, 1, 257, 2, 2, device="cuda"), weight=None, bias=None),
                dict(x=torch.zeros(1, 1, 0, 2, 2, device="cuda"), weight=None, bias=None)]:
    with pytest.raises(RuntimeError):
      labels_last_norm(**{**good, **wrong})
  for shape in [(0, 1, 4, 2, 2), (2, 1, 4, 0, 3)]:
    empty = torch.zeros(shape, device="cuda", requires_grad=True)
    w = torch.ones(4, device="cuda", requires_grad=True)
    y = labels_last_norm(empty, w, w)
    assert y.shape == (shape[0], 1, shape[3], shape[4], 4)
    dx, dw = torch.autograd.grad(y.sum(), (empty, w))
    assert dx.shape == empty.shape and torch.equal(dw, torch.zeros(4, device="cuda"))
