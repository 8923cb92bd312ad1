"""Dropout of volumes whose masks have more than 2^32 groups, so that the counter's second word counts too."""
import pytest
import torch

from oracle import around_oracle

pytestmark = pytest.mark.gpu


def test_groups_beyond_32_bits(gpu):
  """Two items of five labels, two groups to a pixel: 4.4e9 groups and 11e9 entries, forward and backward.  The pixels on
  both sides of group 2^32 and at the end of either item have the words of their own numbers."""
  from mplayers_amd import labels_last_dropout
  n, pixels, quads = 5, 1_100_000_009, 2
  assert 2 * pixels * quads > 2 ** 32
  state = torch.tensor([31, -5], device="cuda")
  x = torch.ones(2, 1, n, 1, pixels, device="cuda", dtype=torch.float16).requires_grad_(True)
  y = labels_last_dropout(x, 0.5, state)
  dy = torch.ones(1, device="cuda").expand(y.shape)
  (dx,) = torch.autograd.grad(y, x, dy)
  border = 2 ** 32 // quads - pixels
  assert 70 < border < pixels - 140
  for item, first in ((0, 0), (0, pixels - 70), (1, border - 35), (1, pixels - 70)):
    keep = []
    for p in range(first, first + 70):
      group = (item * pixels + p) * quads
      words = around_oracle.random_words(group, 31, -5 % 2 ** 64) + around_oracle.random_words(group + 1, 31, -5 % 2 ** 64)
      keep.append([word >= 2 ** 31 for word in words[:n]])
    want = 2.0 * torch.tensor(keep).float()
    assert torch.equal(y[item, 0, 0, first:first + 70].detach().cpu(), want), (item, first)
    assert torch.equal(dx[item, 0, :, 0, first:first + 70].cpu().t().float(), want), (item, first)
