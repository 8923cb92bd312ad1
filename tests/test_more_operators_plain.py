"""The plain form of verified labels that is measured beside the kernels, on the CPU against the plain form in 64 bits pixel by
pixel (oracle/more_around_oracle.py), where a rounding to 32 bits on the way would show.

Both sides hold differences, weights and sums in 64 bits; they differ in the order of at most 64 additions, so by 64 * 2^-53 of a
sum.  The uniform numbers are borders rounded to 24 bits, off by up to 2^-25 of them: one in four million is as close as the
orders differ, and the numbers are fixed.  A cost difference rounded to 24 bits moves a border by up to |difference| * 2^-24 of it,
as much as that or more for the differences that the costs have."""
import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle
from perf import more_operators


def _softmax64(cost, t):
  z = -cost.double() / t
  return torch.softmax(z, -1)


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("costs", [True, False])
@pytest.mark.parametrize("n,t,draft_t", [(3, 1.0, 1.0), (21, 1.0, 2.5), (60, 3.0, 1.0)])
def test_verified_labels_next_to_borders(n, t, draft_t, costs, last):
  g = torch.Generator().manual_seed(n)
  m, h, w = 2, 6, 40
  # (differences with more than 24 bits: a wide range of exponents)
  cost = 10 * torch.rand(1, 1, h, w, n, generator=g) * 2.0 ** torch.randint(-4, 2, (1, 1, h, w, n), generator=g)
  other = cost + 0.5 * torch.randn(cost.shape, generator=g)
  draft = torch.randint(0, n, (m, 1, 1, h, w), generator=g)
  p = _softmax64(cost, t).expand(m, 1, 1, h, w, n)
  q = _softmax64(other, draft_t).expand(m, 1, 1, h, w, n) if costs else torch.nn.functional.one_hot(draft, n).double()
  p_d, q_d = (x.gather(-1, draft[..., None])[..., 0] for x in (p, q))
  u0 = (p_d / q_d).clamp(max=1).float()  # the border itself, rounded
  u0[1] = 1.0                            # as many as may be are drawn anew
  left = (p - q).clamp(min=0).cumsum(-1)
  at = torch.randint(0, n, (m, 1, 1, h, w, 1), generator=g)
  u1 = (left.gather(-1, at)[..., 0] / left[..., -1]).float().nan_to_num(0.5)
  layout = (lambda x: x.contiguous()) if last else (lambda x: x.movedim(-1, 2).contiguous())
  state = dict(case=dict(kind="verify", batch=1, labels=n, height=h, width=w, last=last, drafts=m, costs=costs),
               cost=layout(cost), draft=draft.to(torch.uint8), draft_cost=layout(other) if costs else None, u=torch.stack([u0, u1]),
               T=t, draft_T=draft_t)
  device, more_operators.DEVICE = more_operators.DEVICE, "cpu"
  try:
    labels, kept = more_operators.run(state)
  finally:
    more_operators.DEVICE = device
  want = oracle.verify_labels(cost.movedim(-1, 2).numpy(), draft.numpy(), state["u"].numpy(),
                              other.movedim(-1, 2).numpy() if costs else None, t, draft_t)
  assert np.array_equal(kept.numpy(), want[1]) and np.array_equal(labels.numpy(), want[0])
  assert 0.2 < want[1][0].mean() < 0.9 and want[1][1].mean() < 0.9  # (both answers occur at the border)


def test_best_labels_beyond_the_lists_type():
  """The plain form of lists whose type has no number for a cost."""
  inf = float("inf")
  assert oracle.best_labels([0, 7e4, 5], 3, 1.0, 65520.0) == ([0, 2, 0], [0, 5, inf], 7e4)
  assert oracle.best_labels([0, 7e4, 5], 2, 1.0, 65520.0) == ([0, 2], [0, 5], 7e4)
  assert oracle.best_labels([0, 65519, 65520], 3, 1.0, 65520.0) == ([0, 1, 0], [0, 65519, inf], 65520)
