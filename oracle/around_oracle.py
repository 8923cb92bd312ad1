"""Plain forms, in 64 bits and entry by entry, of what stands around the layers: the dropout masks, the bucketed
pairwise tables and the labels drawn from costs.  Test infrastructure only; nothing here is the reference's."""
import math

import numpy as np


def random_words(group, seed, offset):
  """Four words of the 4x32 generator (ten rounds) of Salmon, Moraes, Dror and Shaw, in Python's whole numbers."""
  c = [group & 0xffffffff, group >> 32, offset & 0xffffffff, (offset >> 32) & 0xffffffff]
  k0, k1 = seed & 0xffffffff, (seed >> 32) & 0xffffffff
  for _ in range(10):
    a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
    c = [(b >> 32) ^ c[1] ^ k0, b & 0xffffffff, (a >> 32) ^ c[3] ^ k1, a & 0xffffffff]
    k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
  return c


def kept(items, labels, pixels, rate, seed, offset, share):
  """(items, labels, pixels) truth values: what stays."""
  keep = np.zeros((items, labels, pixels), bool)
  bound = math.floor(rate * 2.0 ** 32)
  quads = -(-labels // 4)
  if share == "pixel":
    for i in range(items):
      for p in range(pixels):
        keep[i, :, p] = random_words(i * pixels + p, seed, offset)[0] >= bound
    return keep
  for i in range(items):
    for q in range(quads):
      if share == "label":
        words = [random_words(i * quads + q, seed, offset)] * pixels
      else:
        words = [random_words((i * pixels + p) * quads + q, seed, offset) for p in range(pixels)]
      for l in range(4 * q, min(labels, 4 * q + 4)):
        keep[i, l] = [w[l % 4] >= bound for w in words]
  return keep


def bucket_context(table, starts, square=False, symmetric=True):
  table = np.asarray(table, np.float64)
  n = int(starts[-1])
  bucket = [max(b for b in range(len(starts) - 1) if starts[b] <= k) for k in range(n)]
  if not square:
    return table[..., bucket]
  out = np.zeros(table.shape[:-1] + (n, n))
  for a in range(n):
    for b in range(n):
      if b >= a or symmetric:
        out[..., a, b] = table[..., bucket[abs(a - b)]]
  return out


def bucket_sums(dcontext, starts, square=False, symmetric=True):
  d = np.asarray(dcontext, np.float64)
  n = int(starts[-1])
  bucket = [max(b for b in range(len(starts) - 1) if starts[b] <= k) for k in range(n)]
  out = np.zeros(d.shape[:-2 if square else -1] + (len(starts) - 1,))
  if not square:
    for k in range(n):
      out[..., bucket[k]] += d[..., k]
    return out
  for a in range(n):
    for b in range(n):
      if b >= a or symmetric:
        out[..., bucket[abs(a - b)]] += d[..., a, b]
  return out


def draw_label(cost, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
  """The label of one pixel; cost: its labels' costs."""
  temperature, top_p, min_p = (float(np.float32(v)) for v in (temperature, top_p, min_p))
  cost = [math.inf if c != c else float(c) for c in cost]
  order = sorted((c, l) for l, c in enumerate(cost) if c < math.inf)
  if not order:
    return 0
  best = order[0][0]

  def weight(c):
    if c == best:
      return 1.0
    if best == -math.inf:
      return 0.0
    return math.exp(max(-1e9, (best - c) / temperature)) if temperature < math.inf else 1.0

  if not temperature > 0:
    return order[0][1]
  if 0 < top_k:
    order = order[:top_k]
  if top_p < 1:
    target = top_p * math.fsum(weight(c) for c, _ in order)
    left = []
    for c, l in order:
      if left and math.fsum(weight(x) for x, _ in left) >= target:
        break
      left.append((c, l))
    order = left
  if min_p > 0:
    reach = 0.0 if min_p >= 1 else -temperature * math.log(min_p)
    order = [(c, l) for c, l in order if c == best or c - best <= reach]
  stay = {l: weight(c) for c, l in order}
  total = math.fsum(stay.values())
  target = (float(u) if u > 0 else 0.0) * total
  run, last = [], 0
  for l in sorted(stay):
    if stay[l] > 0:
      last = l
    run.append(stay[l])
    if math.fsum(run) > target:  # (rounded once, as the total is: no part of it exceeds it)
      return l
  return last


def draw_labels(cost, uniforms, **parameters):
  """cost (batch, cv, labels, H, W); uniforms (n, batch, cv, H, W); parameters: numbers or one per image."""
  n, batch, cv, height, width = uniforms.shape
  out = np.zeros(uniforms.shape, np.uint8)
  for b in range(batch):
    own = {k: (v[b] if np.ndim(v) else v) for k, v in parameters.items()}
    for c in range(cv):
      for y in range(height):
        for x in range(width):
          for d in range(n):
            out[d, b, c, y, x] = draw_label(cost[b, c, :, y, x], uniforms[d, b, c, y, x], **own)
  return out
