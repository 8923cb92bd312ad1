"""Bucketed pairwise tables on the GPU against their plain form in 64 bits.

The forward call copies entries: equal bits.  A gradient is a sum in 64 bits, rounded once: it is off by half a step
of fp32, 2^-24 of the value, and what the 64-bit sum of up to 65 536 terms may be off, 65 536 * 2^-53 of the sum of
their magnitudes."""
import numpy as np
import pytest
import torch

from oracle import around_oracle

pytestmark = pytest.mark.gpu

FORMS = [(False, True), (True, True), (True, False)]


@pytest.mark.parametrize("square,symmetric", FORMS)
@pytest.mark.parametrize("tables,n,buckets,far", [((), 1, 1, None), ((1,), 2, 1, None), ((3,), 21, 8, 21), ((), 64, 64, None),
                                                  ((2, 2), 65, 9, 30), ((1,), 97, 200, None), ((5,), 256, 32, 128),
                                                  ((16,), 256, 2, None), ((1,), 256, 256, None)])
def test_against_the_plain_form(gpu, tables, n, buckets, far, square, symmetric):
  from mplayers_amd import bucket_context, label_buckets
  rng = np.random.default_rng(n + buckets)
  starts = label_buckets(n, buckets, far)
  table = torch.tensor(rng.standard_normal(tables + (buckets,)), dtype=torch.float32).cuda().requires_grad_(True)
  out = bucket_context(table, starts, square=square, symmetric=symmetric)
  want = around_oracle.bucket_context(table.detach().cpu(), starts, square, symmetric)
  assert out.shape == want.shape and np.array_equal(out.detach().cpu().numpy(), want)
  d = rng.standard_normal(want.shape).astype(np.float32)
  (grad,) = torch.autograd.grad(out, table, torch.from_numpy(d).cuda())
  want = around_oracle.bucket_sums(d, starts, square, symmetric)
  size = around_oracle.bucket_sums(np.abs(d), starts, square, symmetric)
  assert grad.shape == table.shape
  assert (np.abs(grad.cpu().numpy() - want) <= 2.0 ** -24 * np.abs(want) + 65536 * 2.0 ** -53 * size).all()


def test_gradient_against_differences(gpu):
  """A linear map of whole numbers: the differences are exact, and so is the gradient."""
  from mplayers_amd import bucket_context, label_buckets
  rng = np.random.default_rng(4)
  starts = label_buckets(21, 6)
  table = torch.tensor(rng.integers(-8, 8, 6), dtype=torch.float32).cuda().requires_grad_(True)
  d = torch.tensor(rng.integers(-8, 8, (21, 21)), dtype=torch.float32).cuda()

  def value(t):
    return float((bucket_context(t, starts, square=True) * d).sum())

  bucket_context(table, starts, square=True).backward(d)
  for b in range(6):
    step = torch.zeros(6).cuda()
    step[b] = 1
    assert value(table.detach() + step) - value(table.detach()) == float(table.grad[b])


def test_strides_second_gradients_and_an_infinite_entry(gpu):
  from mplayers_amd import bucket_context, label_buckets
  starts = label_buckets(40, 7)
  wide = torch.randn(3, 14, device="cuda")
  every = wide[:, ::2].requires_grad_(True)
  out = bucket_context(every, starts)
  assert torch.equal(out, bucket_context(every.detach().contiguous(), starts))
  d = torch.randn(40, 3, device="cuda").t().requires_grad_(True)
  (grad,) = torch.autograd.grad(out, every, d, create_graph=True)
  h = torch.randn_like(grad)
  (second,) = torch.autograd.grad(grad, d, h)  # the gradient's gradient is the table of h
  assert torch.equal(second, bucket_context(h, starts))
  # an entry that is not finite stays in its bucket
  bad = torch.zeros(3, 40, device="cuda")
  bad[1, 39], bad[2, 1] = float("inf"), float("nan")
  (grad,) = torch.autograd.grad(bucket_context(every, starts), every, bad)
  assert torch.isinf(grad).nonzero().tolist() == [[1, 6]] and torch.isnan(grad).nonzero().tolist() == [[2, 1]]
  assert bucket_context(torch.zeros(0, 7, device="cuda"), starts, square=True).shape == (0, 40, 40)


def test_refusals(gpu):
  from mplayers_amd import bucket_context, label_buckets
  starts = label_buckets(9, 4)
  table = torch.zeros(4, device="cuda")
  for t, s in [(table.half(), starts), (table, starts.cuda()), (torch.zeros(3, device="cuda"), starts),
               (table, torch.tensor([0, 3, 2, 4, 9], dtype=torch.int32)),
               (table, torch.tensor([0, 3, 4, 5, 257], dtype=torch.int32)),
               (table, torch.tensor([1, 3, 4, 5, 9], dtype=torch.int32))]:
    with pytest.raises(RuntimeError):
      bucket_context(t, s)
