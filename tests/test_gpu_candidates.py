"""What is no candidate, bit by bit: quiet and signalling NaN of either sign and +inf are none, every other cost is one as it
is, denormal numbers and -0 included.  Labels are equal to the plain form's (both in 64 bits), costs the same bits."""

import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle

pytestmark = pytest.mark.gpu

# fp32: quiet and signalling NaN, +inf, and numbers at the ends of the type
NONE = [0x7fc00000, 0xffc00000, 0x7f800001, 0xff800001, 0x7fffffff, 0xffffffff, 0x7fbfffff, 0x7f800000]
SOME = [0x00000000, 0x80000000, 0x00000001, 0x80000001, 0x007fffff, 0x00800000, 0x3f800000, 0xbf800000, 0x40490fdb, 0xc0490fdb]


def _costs(n, seed):
  rng = np.random.default_rng(seed)
  bits = np.array(SOME, np.uint32)[rng.integers(0, len(SOME), (1, 2, n, 3, 45))]
  none = np.array(NONE, np.uint32)[rng.integers(0, len(NONE), bits.shape)]
  return np.where(rng.random(bits.shape) < 0.5, none, bits).astype(np.uint32).view(np.float32)


def _gpu(cost, labels_first):
  t = torch.from_numpy(cost.view(np.int32)).cuda()
  return (t if labels_first else t.movedim(2, -1)).contiguous().view(torch.float32)


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("n", [1, 3, 4, 8, 10, 16, 21, 24, 28, 32, 40, 60, 72, 96, 112, 128, 160, 192, 224, 256])
def test_every_kind_of_number(gpu, n, labels_first):
  from mplayers_amd import best_labels, verify_labels
  cost, other = _costs(n, n), _costs(n, n + 1000)
  flat = np.moveaxis(cost, 2, -1).reshape(-1, n)
  k = min(n, 5)
  labels, costs, _ = best_labels(_gpu(cost, labels_first), k, labels_first=labels_first)
  labels, costs = ((t if labels_first else t.movedim(-1, 2)).movedim(2, -1).reshape(-1, k).cpu().numpy() for t in (labels, costs))
  for p, row in enumerate(flat):
    want = oracle.best_labels(row, k, 1.0)
    assert labels[p].tolist() == want[0] and np.array_equal(costs[p], np.array(want[1], np.float32)), (p, labels[p], want)
  rng = np.random.default_rng(n)
  draft = rng.integers(0, min(n + 1, 256), (2, 1, 2, 3, 45)).astype(np.uint8)
  u = (rng.integers(0, 2 ** 24, (2,) + draft.shape) * 2.0 ** -24).astype(np.float32)
  for one in (other, None):
    got = verify_labels(_gpu(cost, labels_first), torch.from_numpy(draft).cuda(), torch.from_numpy(u).cuda(),
                        None if one is None else _gpu(one, labels_first), temperature=0.5, labels_first=labels_first)
    want = oracle.verify_labels(cost, draft, u, one, 0.5)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])


@pytest.mark.parametrize("labels_first", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [5, 21, 96, 200])
def test_signalling_nan_of_half_precision(gpu, n, dtype, labels_first):
  from mplayers_amd import best_labels
  rng = np.random.default_rng(n)
  signalling, infinite = (0x7c01, 0x7c00) if dtype == torch.float16 else (0x7f81, 0x7f80)
  cost = torch.from_numpy(rng.standard_normal((1, 1, n, 2, 40))).to(dtype).view(torch.int16).numpy()
  drop = rng.random(cost.shape)
  cost = np.where(drop < 0.3, signalling, np.where(drop < 0.4, infinite, cost)).astype(np.int16)
  t = torch.from_numpy(cost).cuda()
  t = (t if labels_first else t.movedim(2, -1)).contiguous().view(dtype)
  labels = best_labels(t, 3, labels_first=labels_first)[0]
  labels = (labels if labels_first else labels.movedim(-1, 2)).movedim(2, -1).reshape(-1, 3).cpu().numpy()
  flat = np.moveaxis(torch.from_numpy(cost).view(dtype).float().numpy(), 2, -1).reshape(-1, n)
  for p, row in enumerate(flat):
    assert labels[p].tolist() == oracle.best_labels(row, 3, 1.0)[0], p
