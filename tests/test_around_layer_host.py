"""What stands around the layers, on the CPU: the buckets of label distances, the refusals of the entry points and
the plain forms that the GPU tests compare with."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import around_oracle


def test_generator_gives_the_published_words():
  """The known answers of the generator's authors for 4x32 with ten rounds."""
  ones = (1 << 64) - 1
  assert around_oracle.random_words(0, 0, 0) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
  assert around_oracle.random_words(ones, ones, ones) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def test_bucket_borders():
  from mplayers_amd import label_buckets
  assert label_buckets(5, 5).tolist() == [0, 1, 2, 3, 4, 5]
  assert label_buckets(7, 1).tolist() == [0, 7]
  assert label_buckets(1, 3).tolist() == [0, 1, 1, 1]
  # 4, 8, 16, 32, 64 are exact powers of the ratio 2: borders, where logarithms may fall on either side
  assert label_buckets(256, 8, 64).tolist() == [0, 1, 2, 3, 4, 8, 16, 32, 256]
  for n, b, far in [(256, 32, 128), (21, 8, 21), (192, 16, None), (96, 13, 50), (3, 200, 2), (256, 256, 1)]:
    starts = label_buckets(n, b, far).tolist()
    half, logs, far = b // 2, b - b // 2, max(far or n, b // 2)
    assert len(starts) == b + 1 and starts[0] == 0 and starts[-1] == n and starts == sorted(starts)
    assert starts[:half + 1] == [min(k, n) for k in range(half)] + [min(half, n)]
    for j in range(1, logs):
      # half * (far / half) ** (j / logs) <= start, and not one before it
      if half and half < starts[half + j] < n:
        assert starts[half + j] ** logs * half ** j >= half ** logs * far ** j
        assert (starts[half + j] == starts[half + j - 1] or
                (starts[half + j] - 1) ** logs * half ** j < half ** logs * far ** j)
  for wrong in [(0, 4), (257, 4), (4, 0), (4, 257), (4, 4, 0)]:
    with pytest.raises(ValueError):
      label_buckets(*wrong)


@pytest.mark.parametrize("n,buckets,square,symmetric", [(1, 1, False, True), (9, 4, False, True), (9, 12, True, True),
                                                         (21, 6, True, False)])
def test_bucket_context_on_the_cpu(n, buckets, square, symmetric):
  from mplayers_amd import bucket_context, label_buckets
  rng = np.random.default_rng(n)
  starts = label_buckets(n, buckets)
  table = torch.tensor(rng.standard_normal((2, buckets)), dtype=torch.float32, requires_grad=True)
  out = bucket_context(table, starts, square=square, symmetric=symmetric)
  assert np.array_equal(out.detach().numpy(), around_oracle.bucket_context(table.detach(), starts, square, symmetric))
  d = torch.tensor(rng.integers(-9, 9, out.shape), dtype=torch.float32)  # (whole numbers: sums are exact)
  out.backward(d)
  assert np.array_equal(table.grad.numpy(), around_oracle.bucket_sums(d, starts, square, symmetric))


def test_bucket_table_of_a_module():
  from mplayers_amd import MPModule
  from tests.test_capi_host import _args
  for n, shape in ((21, (21, 21)), (40, (40,))):
    args = _args(n_classes=n, mpnet_smoothness_mode="TL", mpnet_smoothness_trunct_value=3, mpnet_smoothness_buckets=8,
                 mpnet_smoothness_train="on")
    module = MPModule(args, enable_create_label_context=True)
    table, loc, diag = module.get_label_context()
    starts = module.label_buckets
    assert table.shape == (8,) and table.requires_grad and list(loc) == list(range(1, 8)) and list(diag) == [0]
    assert torch.equal(table.detach(), 2.0 * starts[:-1].float().clamp(max=3))
    assert module._effective_label_context().shape == shape
  module.set_label_context(torch.nn.Parameter(torch.zeros(40)), range(1, 40), range(1))
  assert module.label_buckets is None and module._effective_label_context().shape == (40,)


def test_bucket_context_refuses():
  from mplayers_amd import bucket_context, label_buckets
  starts = label_buckets(9, 4)
  table = torch.zeros(4)
  for t, s in [(torch.zeros(5), starts), (table.double(), starts), (table, starts.long()), (table, starts[None]),
               (table, torch.tensor([0, 3, 2, 4, 9], dtype=torch.int32)), (torch.zeros(()), starts),
               (table, torch.tensor([1, 2, 3, 4, 9], dtype=torch.int32)), (table, starts[:1]),
               (table, torch.tensor([0, 2, 3, 4, 257], dtype=torch.int32)),
               (table, torch.tensor([0, 0, 0, 0, 0], dtype=torch.int32))]:
    with pytest.raises(RuntimeError):
      bucket_context(t, s)
  with pytest.raises(TypeError):
    bucket_context(table, [0, 1, 2, 3, 9])


def test_entry_points_refuse_before_any_launch():
  from mplayers_amd import _lib
  lib = _lib.load()
  one = ctypes.c_void_p(256)  # never dereferenced: validation answers first
  starts = np.array([0, 2, 9], np.int32)
  at = starts.ctypes.data

  def refused(rc, word):
    assert rc == -1
    assert word in lib.mpl_last_error(), lib.mpl_last_error()

  for call in (lib.mpl_bucket_context, lib.mpl_bucket_sums):
    refused(call(None, at, 1, 2, 9, 0, one, None), b"null")
    refused(call(one, at, 1, 2, 9, 0, None, None), b"null")
    refused(call(one, None, 1, 2, 9, 0, one, None), b"null")
    refused(call(one, at, 1, 2, 8, 0, one, None), b"n_disp")
    refused(call(one, at, 1, 2, 257, 0, one, None), b"n_disp")
    refused(call(one, at, 1, 0, 9, 0, one, None), b"n_buckets")
    refused(call(one, at, -1, 2, 9, 0, one, None), b"n_tables")
    refused(call(one, at, 1, 2, 9, 3, one, None), b"square")
    unordered = np.array([0, 7, 5, 9], np.int32)
    refused(call(one, unordered.ctypes.data, 1, 3, 9, 0, one, None), b"order")
    assert call(one, at, 0, 2, 9, 0, one, None) == 0
  for call in (lib.mpl_dropout_labels_last, lib.mpl_dropout_labels_first):
    refused(call(0, 0, 0.5, None, one, one, 1, 4, 9, None), b"null")
    refused(call(0, 0, 0.5, one, None, one, 1, 4, 9, None), b"null")
    refused(call(3, 0, 0.5, one, one, one, 1, 4, 9, None), b"type")
    refused(call(0, 3, 0.5, one, one, one, 1, 4, 9, None), b"share")
    refused(call(0, 0, 1.5, one, one, one, 1, 4, 9, None), b"rate")
    refused(call(0, 0, math.nan, one, one, one, 1, 4, 9, None), b"rate")
    refused(call(0, 0, 0.5, one, one, one, 1, 257, 9, None), b"n_disp")
    refused(call(0, 0, 0.5, one, one, one, 1, 4, -9, None), b"negative")
    refused(call(0, 0, 0.5, one, one, one, 1 << 20, 4, 1 << 30, None), b"too many")
    refused(call(0, 0, 0.5, one, one, one, 1, 1, 1 << 32, None), b"too many")  # 2^33 threads
    assert call(0, 0, 0.5, one, one, one, 0, 4, 9, None) == 0

  def sample(cost=one, uniforms=one, batch=1, n_cv=1, n=4, pixels=9, draws=1, labels=one):
    return lib.mpl_sample_labels(1, cost, uniforms, batch, n_cv, n, pixels, draws, None, 1.0, None, 0, None, 1.0, None, 0.0,
                                 labels, None)

  refused(sample(cost=None), b"null")
  refused(sample(uniforms=None), b"null")
  refused(sample(labels=None), b"null")
  refused(sample(n=0), b"n_disp")
  refused(sample(n=257), b"n_disp")
  refused(sample(draws=-1), b"negative")
  refused(sample(batch=1 << 20, pixels=1 << 30), b"too many")
  refused(sample(n=200, pixels=1 << 30), b"too many")  # 2^33 threads
  assert sample(draws=0) == 0 and sample(batch=0) == 0 and sample(pixels=0) == 0


def test_python_entry_points_refuse_cpu_tensors():
  from mplayers_amd import labels_last_dropout, sample_labels
  with pytest.raises(RuntimeError, match="GPU"):
    sample_labels(torch.zeros(1, 1, 4, 2, 2), torch.zeros(1, 1, 2, 2))
  with pytest.raises(RuntimeError, match="GPU"):
    labels_last_dropout(torch.zeros(1, 1, 4, 2, 2), 0.5, torch.zeros(2, dtype=torch.int64))
  with pytest.raises(TypeError):
    sample_labels([0.0], torch.zeros(1, 1, 2, 2))
  with pytest.raises(TypeError):
    labels_last_dropout(torch.zeros(1, 1, 4, 2, 2), 0.5, 7)


def test_drawn_labels_of_the_plain_form():
  draw = around_oracle.draw_label
  assert draw([math.inf, math.nan], 0.5) == 0
  assert draw([1, 0, 0], 0.9, temperature=0) == 1
  assert [draw([0, 0, math.inf, 0], u) for u in (0, 0.3, 0.34, 0.67, 1.0)] == [0, 0, 1, 3, 3]
  assert [draw([2, 1, 0, 0], 0.99, top_k=k) for k in (1, 2, 3)] == [2, 3, 3]
  assert draw([0, -math.inf, 1, -math.inf], 0.6) == 3
  assert draw([0, 0, 0, 0], 0.99, top_p=0.5) == 1
  assert draw([0, 0.5, 1], 0.99, min_p=math.exp(-0.75)) == 1
