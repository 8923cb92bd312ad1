"""Plain forms in 64 bits of layer norm in the layout change, a teacher's best labels, the divergence from them and verified
labels (test infrastructure only): pixel by pixel from their definitions in include/mplayers_amd.h."""
import math

import numpy as np


# ------------------------------------------------------------------------------------------------------ layer norm
def norm(x, weight, bias, eps):
  """x (pixels, labels) -> y, xhat, r (pixels, 1)."""
  x = np.asarray(x, np.float64)
  centred = x - x.mean(1, keepdims=True)
  r = 1.0 / np.sqrt((centred ** 2).mean(1, keepdims=True) + eps)
  xhat = centred * r
  return xhat * np.asarray(weight, np.float64) + np.asarray(bias, np.float64), xhat, r


def norm_grad(x, weight, eps, dy):
  """-> dx, dweight, dbias."""
  dy = np.asarray(dy, np.float64)
  _, xhat, r = norm(x, weight, np.zeros(dy.shape[1]), eps)
  g = dy * np.asarray(weight, np.float64)
  dx = r * (g - g.mean(1, keepdims=True) - xhat * (g * xhat).mean(1, keepdims=True))
  return dx, (dy * xhat).sum(0), dy.sum(0)


# ------------------------------------------------------------------------------------------- a teacher's best labels
def softmin(costs, temperature):
  """-T log(sum of exp(-c / T)), +inf of nothing."""
  if not costs:
    return math.inf
  best = min(costs)
  if best == math.inf:
    return math.inf
  return best - temperature * math.log(math.fsum(math.exp(-(c - best) / temperature) for c in costs))


def best_labels(cost, k, temperature, limit=math.inf):
  """One pixel: k labels, their costs relative to the best one, and the softmin of the other candidates'.  limit: from here on
  a relative cost is +inf in the list's type, which then has not got it."""
  cost = [math.inf if c != c else float(c) for c in cost]
  order = sorted((c, l) for l, c in enumerate(cost) if c < math.inf)
  if order and order[0][0] == -math.inf:
    order = [(0.0, l) for c, l in order if c == -math.inf]
  elif order:
    with np.errstate(over="ignore"):  # (the difference is one of fp32)
      order = [(float(np.float32(c) - np.float32(order[0][0])), l) for c, l in order]
    order = [(c, l) for c, l in order if c < math.inf]
  kept = [(c, l) for c, l in order[:k] if c < limit]
  others = order[len(kept):]
  labels = [l for _, l in kept] + [0] * (k - len(kept))
  return labels, [c for c, _ in kept] + [math.inf] * (k - len(kept)), softmin([c for c, _ in others], temperature)


# ------------------------------------------------------------------------------------- the divergence from a teacher
def distill(cost, labels, costs, rest, temperature):
  """One pixel: the loss, its gradient with respect to the costs, and the sizes of what each of those is a difference of;
  rest None: no such class."""
  n = len(cost)
  cost = [float(c) for c in cost]
  candidates = [l for l in range(n) if cost[l] != math.inf]
  named = [(int(l), float(c)) for l, c in zip(labels, costs) if c != math.inf and l < n]
  listed = {l for l, _ in named}
  classes = [([l], c) for l, c in named if l in candidates]
  left = [l for l in candidates if l not in listed]
  if rest is not None and rest != math.inf and left:
    classes.append((left, float(rest)))
  if not classes:
    return 0.0, [0.0] * n, [0.0] * n
  if any(c != c or c == -math.inf for c in [cost[l] for l in candidates] + [c for _, c in classes]):
    return math.nan, [0.0 if c == math.inf else math.nan for c in cost], [0.0] * n
  total, mass = softmin([cost[l] for l in candidates], temperature), softmin([c for _, c in classes], temperature)
  loss, grad, size = [], [0.0] * n, [0.0] * n
  for l in candidates:
    size[l] = math.exp(-(cost[l] - total) / temperature) / temperature
    grad[l] -= size[l]
  for members, c in classes:
    p, own = math.exp(-(c - mass) / temperature), softmin([cost[l] for l in members], temperature)
    if p > 0:
      loss.append(p * ((mass - c) - (total - own)) / temperature)
    for l in members:
      share = p * math.exp(-(cost[l] - own) / temperature) / temperature
      grad[l] += share
      size[l] += share
  return math.fsum(loss), grad, size


# ------------------------------------------------------------------------------------------------- verified labels
def _weights(cost, temperature):
  """exp(-cost / T) over its sum, as drawn labels have it; None where there is no candidate."""
  temperature = float(np.float32(temperature))
  cost = [math.inf if c != c else float(c) for c in cost]
  best = min(cost)
  if best == math.inf:
    return None
  if not temperature > 0:
    first = cost.index(best)
    return [1.0 if l == first else 0.0 for l in range(len(cost))]
  weight = []
  for c in cost:
    if c == best:
      weight.append(1.0)
    elif c == math.inf or best == -math.inf:
      weight.append(0.0)
    else:
      weight.append(math.exp(max(-1e9, (best - c) / temperature)) if temperature < math.inf else 1.0)
  total = math.fsum(weight)
  return [w / total for w in weight]


def _first_past(weight, u):
  """The first label whose running sum exceeds u times the sum, or the last that weighs."""
  total = math.fsum(weight)
  run = []
  last = max(l for l, w in enumerate(weight) if w > 0)
  for l, w in enumerate(weight):
    run.append(w)
    if math.fsum(run) > u * total:
      return l
  return last


def verify_label(cost, label, u0, u1, draft_cost=None, temperature=1.0, draft_temperature=None):
  """One pixel: the label and whether the drafted one stayed."""
  n = len(cost)
  u0, u1 = (float(u) if u > 0 else 0.0 for u in (u0, u1))
  p = _weights(cost, temperature)
  if p is None:
    return 0, False
  if draft_cost is None:
    q = [1.0 if l == label else 0.0 for l in range(n)]
  else:
    q = _weights(draft_cost, temperature if draft_temperature is None else draft_temperature) or [0.0] * n
  drafted = label < n and q[label] > 0
  if not drafted:
    return _first_past(p, u1), False
  if u0 * q[label] < p[label]:
    return int(label), True
  left = [max(a - b, 0.0) for a, b in zip(p, q)]
  return _first_past(left if sum(left) > 0 else p, u1), False


def verify_labels(cost, draft, uniforms, draft_cost=None, temperature=1.0, draft_temperature=None):
  """cost, draft_cost (batch, cv, labels, H, W); draft (n, batch, cv, H, W); uniforms (2, n, ...); temperatures: numbers or
  one per image."""
  labels, kept = np.zeros(draft.shape, np.uint8), np.zeros(draft.shape, bool)
  for at in np.ndindex(*draft.shape):
    _, b, c, y, x = at
    t, dt = (v[b] if np.ndim(v) else v for v in (temperature, draft_temperature))
    labels[at], kept[at] = verify_label(cost[b, c, :, y, x], int(draft[at]), uniforms[(0,) + at], uniforms[(1,) + at],
                                        None if draft_cost is None else draft_cost[b, c, :, y, x], t, dt)
  return labels, kept
