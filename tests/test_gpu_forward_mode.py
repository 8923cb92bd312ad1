"""Derivatives of the forward mode, which the operators around the layers have none of: refused, not lost."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _dual(t):
  return forward_ad.make_dual(t.detach().clone(), torch.ones_like(t))


def _inputs(n):
  g = torch.Generator(device="cuda").manual_seed(n)
  x = torch.randn(1, 1, n, 3, 20, device="cuda", generator=g)
  weight, bias = torch.rand(n, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
  return x, weight, bias, torch.rand(1, 1, 3, 20, n, device="cuda", generator=g)


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("n", [5, 40])
def test_layer_norm(gpu, n, which, grad_mode):
  from mplayers_amd import labels_last_norm
  inputs = list(_inputs(n)[:3])
  want = labels_last_norm(*inputs)
  with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
    inputs[which] = _dual(inputs[which])
    with pytest.raises(RuntimeError):
      labels_last_norm(*inputs)
    # without the tangent, or outside of the level, as ever
    inputs[which] = forward_ad.unpack_dual(inputs[which]).primal
    assert torch.equal(labels_last_norm(*inputs), want)
  assert torch.equal(labels_last_norm(*inputs), want)


@pytest.mark.parametrize("grad_mode", [True, False])
def test_the_divergence(gpu, grad_mode):
  from mplayers_amd import best_labels, distill_costs
  cost = _inputs(21)[0]
  labels, costs, rest = best_labels(cost.flip(2), 4)
  good = dict(cost=cost, labels=labels, costs=costs, rest=rest)
  want = distill_costs(**good)
  with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
    for name in ("cost", "costs", "rest"):
      with pytest.raises(RuntimeError):
        distill_costs(**{**good, name: _dual(good[name])})
    assert torch.equal(distill_costs(**good), want)


def test_the_gradients(gpu):
  """A gradient that carries a tangent: none of what is made of it does."""
  from mplayers_amd import best_labels, bucket_context, distill_costs, label_buckets, labels_last_dropout, labels_last_norm
  x, weight, _, dy = _inputs(9)
  x, weight = x.requires_grad_(True), weight.requires_grad_(True)
  state = torch.tensor([1, 2], device="cuda")
  table = torch.rand(4, 3, device="cuda", requires_grad=True)
  starts = label_buckets(9, 3)
  calls = [(labels_last_norm(x, weight), (x, weight)), (labels_last_dropout(x, 0.5, state), (x,)),
           (distill_costs(x, *best_labels(x.detach().flip(2), 3)), (x,)), (bucket_context(table, starts), (table,))]
  for out, leaves in calls:
    g = torch.rand_like(out)
    want = torch.autograd.grad(out, leaves, g, retain_graph=True)
    with forward_ad.dual_level():
      with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaves, forward_ad.make_dual(g, torch.ones_like(g)), retain_graph=True)
    got = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
