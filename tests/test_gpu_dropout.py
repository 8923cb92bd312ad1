"""Dropout in the layout change on the GPU against its plain form.

What stays is one fp32 product, and rounded once more where the type is a half: the plain form makes the same two
roundings, so the values are equal bit for bit."""
import numpy as np
import pytest
import torch

from oracle import around_oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _state(seed, offset=0):
  return torch.tensor([seed, offset], dtype=torch.int64, device="cuda")


def _plain(x, dy, p, seed, offset, share):
  """y and dx as the plain form has them; x (b, cv, n, h, w), dy (b, cv, h, w, n), CPU tensors."""
  b, cv, n, h, w = x.shape
  keep = torch.from_numpy(around_oracle.kept(b * cv, n, h * w, p, seed, offset, share)).view(x.shape)
  scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=torch.float32)
  zero = torch.zeros(())
  y = torch.where(keep, x.float() * scale, zero).permute(0, 1, 3, 4, 2)
  return y, torch.where(keep, dy.permute(0, 1, 4, 2, 3) * scale, zero).to(x.dtype)


def _same(got, want):
  assert got.shape == want.shape and got.dtype == want.dtype
  bits = torch.int32 if got.dtype == torch.float32 else torch.int16
  got, want = got.detach().cpu().contiguous().view(bits), want.contiguous().view(bits)
  wrong = int((got != want).sum())
  assert wrong == 0, "%d of %d entries differ" % (wrong, got.numel())


@pytest.mark.parametrize("share", ["element", "pixel", "label"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,cv,n,h,w,p", [(1, 1, 1, 1, 1, 0.5), (2, 2, 3, 5, 7, 0.1), (1, 1, 4, 8, 8, 0.25), (3, 1, 21, 9, 15, 0.5),
                                          (1, 1, 64, 4, 16, 0.9), (1, 2, 97, 3, 43, 0.3), (1, 1, 192, 2, 65, 0.2),
                                          (2, 1, 255, 1, 67, 0.0), (1, 1, 256, 5, 26, 0.7), (1, 1, 16, 3, 300, 1.0)])
def test_against_the_plain_form(gpu, b, cv, n, h, w, p, dtype, share):
  from mplayers_amd import labels_last_dropout
  g = torch.Generator().manual_seed(n + h)
  x = torch.randn(b, cv, n, h, w, generator=g).to(dtype)
  dy = torch.randn(b, cv, h, w, n, generator=g)
  seed, offset = -(2 ** 61) - n, 2 ** 35 + w
  y, dx = _plain(x, dy, p, seed, offset, share)
  leaf = x.cuda().requires_grad_(True)
  got = labels_last_dropout(leaf, p, _state(seed, offset), share=share)
  _same(got, y)
  (grad,) = torch.autograd.grad(got, leaf, dy.cuda())
  _same(grad, dx)


@pytest.mark.parametrize("dtype", TYPES)
def test_alignment_and_strides(gpu, dtype):
  """Inputs one entry behind an aligned address, and with other strides; a gradient that is broadcast."""
  from mplayers_amd import labels_last_dropout
  g = torch.Generator().manual_seed(8)
  for n, h, w in ((32, 8, 16), (21, 8, 8)):
    flat = torch.randn(1 + n * h * w, generator=g).to(dtype)
    x = flat[1:].view(1, 1, n, h, w)
    dy = torch.randn(1 + n * h * w, generator=g)
    y, dx = _plain(x, dy[1:].view(1, 1, h, w, n), 0.4, 5, 6, "element")
    leaf = flat.cuda()[1:].view(1, 1, n, h, w).requires_grad_(True)
    got = labels_last_dropout(leaf, 0.4, _state(5, 6))
    _same(got, y)
    _same(torch.autograd.grad(got, leaf, dy.cuda()[1:].view(1, 1, h, w, n))[0], dx)
    turned = x.cuda().transpose(3, 4).contiguous().transpose(3, 4).requires_grad_(True)
    assert not turned.is_contiguous()
    got = labels_last_dropout(turned, 0.4, _state(5, 6))
    _same(got, y)
    one = torch.ones(1, device="cuda").expand(1, 1, h, w, n)
    _same(torch.autograd.grad(got, turned, one)[0], _plain(x, torch.ones(1, 1, h, w, n), 0.4, 5, 6, "element")[1])


def test_rates_and_seeds(gpu):
  """The share that stays is within five standard deviations of the rate's, and another seed, offset or item has
  another mask."""
  from mplayers_amd import labels_last_dropout
  x = torch.ones(2, 1, 64, 100, 100, device="cuda")
  for p in (0.1, 0.5, 0.9):
    y = labels_last_dropout(x, p, _state(3, 4))
    stays = y != 0
    count = stays.numel()
    assert abs(int(stays.sum()) - count * (1 - p)) <= 5 * (count * p * (1 - p)) ** 0.5
    for other in (_state(4, 4), _state(3, 5), _state(3 + 2 ** 32, 4), _state(3, 4 + 2 ** 32)):
      same = (labels_last_dropout(x, p, other) != 0) == stays
      assert abs(int(same.sum()) - count * (p * p + (1 - p) ** 2)) <= 6 * count ** 0.5 / 2
    assert torch.equal(y, labels_last_dropout(x, p, _state(3, 4)))
    assert not torch.equal(stays[0], stays[1])
  assert torch.equal(labels_last_dropout(x, 0, _state(1)), x.permute(0, 1, 3, 4, 2))


def test_dropped_entries_are_zero_whatever_they_were(gpu):
  from mplayers_amd import labels_last_dropout
  for value in (float("inf"), float("-inf"), float("nan")):
    x = torch.full((1, 1, 16, 8, 8), value, device="cuda")
    y = labels_last_dropout(x, 0.5, _state(9))
    keep = torch.from_numpy(around_oracle.kept(1, 16, 64, 0.5, 9, 0, "element")).view(16, 8, 8).permute(1, 2, 0)
    y = y[0, 0].cpu()
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    assert (labels_last_dropout(x, 1, _state(9)) == 0).all()


def test_gradients(gpu):
  """The gradient is the transpose of the map, its gradient the map; and by a difference: the map is linear, and
  with halves of whole numbers and a rate of one half exact."""
  from mplayers_amd import labels_last_dropout
  g = torch.Generator(device="cuda").manual_seed(2)
  x = torch.randint(-8, 8, (2, 1, 21, 5, 9), device="cuda", generator=g).float().requires_grad_(True)
  state = _state(11, 12)
  y = labels_last_dropout(x, 0.5, state, share="pixel")
  dy = torch.randint(-8, 8, y.shape, device="cuda", generator=g).float().requires_grad_(True)
  (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
  h = torch.randint(-8, 8, x.shape, device="cuda", generator=g).float()
  difference = labels_last_dropout(x.detach() + h, 0.5, state, share="pixel") - y.detach()
  assert float((difference * dy.detach()).sum()) == float((dx.detach() * h).sum())
  (second,) = torch.autograd.grad(dx, dy, h)
  assert torch.equal(second, labels_last_dropout(h, 0.5, state, share="pixel"))


def test_state_written_before_the_backward_pass_is_refused(gpu):
  from mplayers_amd import labels_last_dropout
  x = torch.randn(1, 1, 4, 4, 4, device="cuda").requires_grad_(True)
  state = _state(1)
  y = labels_last_dropout(x, 0.5, state)
  state += 1
  with pytest.raises(RuntimeError, match="modified by an inplace"):
    y.sum().backward()


def test_replays_read_the_state(gpu):
  """A captured forward and backward call has the mask of the state at each replay; eager work between them."""
  from mplayers_amd import labels_last_dropout
  g = torch.Generator().manual_seed(5)
  x = torch.randn(2, 1, 21, 13, 17, generator=g)
  dy = torch.randn(2, 1, 13, 17, 21, generator=g)
  state, dy_gpu = _state(0), dy.cuda()
  leaf = x.cuda().requires_grad_(True)

  def step():
    y = labels_last_dropout(leaf, 0.3, state)
    return y.detach(), torch.autograd.grad(y, leaf, dy_gpu)[0]

  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    step()
  torch.cuda.current_stream().wait_stream(stream)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  for seed in (4, 5, 4):
    for t in out:
      t.fill_(7)
    state.copy_(torch.tensor([seed, 2 * seed]))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(out, _plain(x, dy, 0.3, seed, 2 * seed, "element")):
      _same(got, want)


def test_another_stream(gpu):
  from mplayers_amd import labels_last_dropout
  x = torch.randn(1, 1, 96, 64, 64)
  stream = torch.cuda.Stream()
  with torch.cuda.stream(stream):
    on = x.cuda() * 2
    y = labels_last_dropout(on, 0.5, _state(3))
  stream.synchronize()
  _same(y, _plain(x * 2, torch.zeros(1, 1, 64, 64, 96), 0.5, 3, 0, "element")[0])


def test_a_volume_beyond_32_bits(gpu):
  """More than 2^32 entries in fp16, and of the masks' groups: the last pixels have the words of their own numbers."""
  from mplayers_amd import labels_last_dropout
  n, pixels = 3, 1_500_000_007
  x = torch.ones(1, 1, n, 1, pixels, device="cuda", dtype=torch.float16)
  y = labels_last_dropout(x, 0.5, _state(21, 22))
  last = list(range(pixels - 70, pixels))
  words = [around_oracle.random_words(p, 21, 22) for p in last]
  keep = torch.tensor([[w[l] >= 2 ** 31 for l in range(n)] for w in words])
  assert torch.equal(y[0, 0, 0, -70:].cpu(), 2.0 * keep.float())
  del x, y


def test_refusals(gpu):
  from mplayers_amd import labels_last_dropout
  x = torch.zeros(1, 1, 4, 4, 4, device="cuda")
  state = _state(1)
  good = dict(x=x, p=0.5, state=state)
  for wrong in [dict(x=x[0]), dict(x=x.double()), dict(x=x.cpu()), dict(p=-0.1), dict(p=1.1), dict(p=float("nan")),
                dict(state=state.cpu()), dict(state=state.int()), dict(state=state[:1]), dict(share="row"),
                dict(state=torch.zeros(4, dtype=torch.int64, device="cuda")[::2]),
                dict(x=torch.zeros(1, 1, 257, 2, 2, device="cuda")), dict(x=torch.zeros(1, 1, 0, 2, 2, device="cuda"))]:
    with pytest.raises(RuntimeError):
      labels_last_dropout(**{**good, **wrong})
  empty = torch.zeros(0, 1, 4, 2, 2, device="cuda", requires_grad=True)
  y = labels_last_dropout(empty, 0.5, state)
  assert y.shape == (0, 1, 2, 2, 4)
  assert torch.autograd.grad(y.sum(), empty)[0].shape == empty.shape
