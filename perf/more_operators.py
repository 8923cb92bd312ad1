"""More of what stands around a message-passing layer in training and in use, operator by operator, for measurement.

Four operators, each in a plain form of elementary torch operations and, where `own` is true, through the
framework's entry points:

  norm     layer norm of the unary costs over the labels of a pixel within the change to the layer's layout, forward
           and backward, with the gradients of its weight and bias (`labels_last_norm`)
  best     the labels of least cost of every pixel, their costs and what the others weigh: what is kept of a teacher
           (`best_labels`)
  distill  the divergence of a layer's costs from such a teacher's, and its gradient (`distill_costs`)
  verify   labels that were drafted from other costs, kept or drawn anew so that they are distributed as the layer's
           costs say, from given uniform numbers (`verify_labels`)

Definitions that the plain forms spell out:

  norm     y = (x - mean) / sqrt(var + eps) * weight + bias, mean and var over the labels of a pixel
  best     +inf and NaN are no candidates; equal costs order by label; costs are given relative to the best one.
           A place behind the last candidate has label 0 and cost +inf.  rest = -T log(sum over the other
           candidates of exp(-cost / T)), +inf where there are none.
  distill  q = softmax(-cost / T) over the labels.  Teacher's classes: the entries of its list, and the rest of the labels
           where `rest` is given; an entry is there where its cost is below +inf, its label exists and the student's
           cost of that label is below +inf; the rest where its cost is below +inf and such a label is left.
           p = softmax(-cost / T) over the classes that are there; loss = sum p (log p - log q of the class); 0 where no
           class is there.
  verify   p, q: softmax(-cost / T) of the target and the draft, as `sample_labels` has it (candidates, T <= 0); without
           costs of the draft q is 1 at the drafted label.  The label d stays where u0 q[d] < p[d]; else one is drawn from
           max(p - q, 0) with u1: the first whose running sum exceeds u1 * total.  Where q[d] is 0 (or there is no label d)
           one is drawn from p.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda"

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


# ------------------------------------------------------------------------------------------------- cases
def listed():
  return [
      # the smallest layer of the benchmark in training
      dict(name="norm 16x64x96", kind="norm", batch=1, labels=16, height=64, width=96, type="f32", last=False),
      # a segmentation network's logits in bf16 (batch and size of the reference's training options)
      dict(name="norm 12x21x129x129 bf16", kind="norm", batch=12, labels=21, height=129, width=129, type="bf16", last=False),
      # an odd crop of a stereo volume that is in the operators' layout already
      dict(name="norm 97x301x803 last", kind="norm", batch=1, labels=97, height=301, width=803, type="f32", last=True),
      # the headline configuration's cost volume
      dict(name="norm 192x1500x2000", kind="norm", batch=1, labels=192, height=1500, width=2000, type="f32", last=False),
      # what is kept of a segmentation teacher, for storing
      dict(name="best 12x21x129x129 k4", kind="best", batch=12, labels=21, height=129, width=129, type="f32", last=False,
           k=4, kept="f16", T=2.0, masked=False),
      # of a stereo teacher, labels outside the image masked
      dict(name="best 96x384x1248 k8", kind="best", batch=1, labels=96, height=384, width=1248, type="f32", last=False,
           k=8, kept="f32", T=1.0, masked=True),
      # a small student
      dict(name="distill 16x64x96 k3", kind="distill", batch=1, labels=16, height=64, width=96, type="f32", last=False,
           k=3, kept="f32", rest=False, T=1.0, masked=False),
      # a segmentation student, the teacher's list in fp16
      dict(name="distill 12x21x129x129 k4", kind="distill", batch=12, labels=21, height=129, width=129, type="f32",
           last=False, k=4, kept="f16", rest=True, T=2.0, masked=False),
      # the headline configuration in training
      dict(name="distill 192x1500x2000 k8", kind="distill", batch=1, labels=192, height=1500, width=2000, type="f32",
           last=False, k=8, kept="f16", rest=True, T=1.0, masked=True),
      # labels of a small layer
      dict(name="verify 16x64x96", kind="verify", batch=1, labels=16, height=64, width=96, last=False, drafts=1, T=1.0,
           draft_T=1.0, costs=True, masked=False, each=False),
      # the energy minimiser's 60-label image in the operators' layout, several labellings at once
      dict(name="verify 60x375x450 last", kind="verify", batch=1, labels=60, height=375, width=450, last=True, drafts=8,
           T=2.0, draft_T=3.0, costs=True, masked=True, each=False),
      # the headline configuration, labels of fewer iterations against the last one's costs
      dict(name="verify 192x1500x2000", kind="verify", batch=1, labels=192, height=1500, width=2000, last=False, drafts=1,
           T=1.0, draft_T=1.0, costs=True, masked=False, each=False),
  ]


def _spread(rng, low, high):
  return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _image(rng, labels, batch, low, high):
  """A height and a width that give the volume between low and high entries."""
  pixels = max(1.0, math.exp(rng.uniform(math.log(low), math.log(high))) / (labels * batch))
  height = max(1, int(round(math.sqrt(pixels) * math.exp(rng.uniform(-0.7, 0.7)))))
  return height, max(1, int(pixels / height))


def draw(rng):
  kind = rng.choice(["norm", "norm", "best", "distill", "distill", "verify", "verify"])
  labels, batch = _spread(rng, 2, 256), rng.choice([1, 1, 2, 3, 4, 7, 12])
  height, width = _image(rng, labels, batch, 2e3, 2e8 if kind == "norm" else 6e7)
  case = dict(kind=kind, batch=batch, labels=labels, height=height, width=width, last=rng.random() < 0.4)
  if kind != "verify":
    case["type"] = rng.choice(["f32", "f32", "f16", "bf16"])
  if kind != "norm":
    case["masked"] = rng.random() < 0.5
    case["T"] = rng.choice([1.0, round(rng.uniform(0.5, 4.0), 2)])
  if kind in ("best", "distill"):
    case["k"] = _spread(rng, 1, min(labels, 32))
    case["kept"] = rng.choice(["f32", "f16", "bf16"])
  if kind == "distill":
    case["rest"] = rng.random() < 0.5
  if kind == "verify":
    case.update(drafts=rng.choice([1, 1, 2, 5, 8]), draft_T=rng.choice([1.0, case["T"], round(rng.uniform(0.5, 4.0), 2)]),
                costs=rng.random() < 0.75, each=rng.random() < 0.4)
  return case


# ---------------------------------------------------------------------------------------------- the inputs
def _size(case):
  return tuple(case[k] for k in ("batch", "labels", "height", "width"))


def _centres(case, g):
  """The label that a pixel's costs have their valley around; it changes over the image."""
  b, n, h, w = _size(case)
  rows = torch.rand(b, 1, 1, h, 1, device=DEVICE, generator=g)
  cols = torch.rand(b, 1, 1, 1, w, device=DEVICE, generator=g)
  return (rows + cols) * (0.5 * n)


def _costs(case, g, centre):
  """Costs as the layer gives them: a valley, noise, and, where labels are masked, +inf for those that would lie left
  of the image, with a few pixels that have none left."""
  b, n, h, w = _size(case)
  label = torch.arange(n, device=DEVICE, dtype=torch.float32).view(1, 1, n, 1, 1)
  cost = torch.randn(b, 1, n, h, w, device=DEVICE, generator=g)
  cost += (label - centre).abs_().clamp_(max=20).mul_(0.4)
  if case.get("masked"):
    x = torch.arange(w, device=DEVICE, dtype=torch.float32).view(1, 1, 1, 1, w)
    cost.masked_fill_(label > x, math.inf)
    cost.masked_fill_(torch.rand(b, 1, 1, h, w, device=DEVICE, generator=g) < 0.001, math.inf)
  return cost


def _laid_out(case, t):
  return t.movedim(2, -1).contiguous() if case["last"] else t


def _prepare_norm(case, g):
  b, n, h, w = _size(case)
  x = _costs(case, g, _centres(case, g)).mul_(0.2 + 4 * torch.rand(b, 1, 1, h, w, device=DEVICE, generator=g))
  x = _laid_out(case, x.to(_TYPES[case["type"]]))
  return dict(case=case, x=x.requires_grad_(True),
              weight=(1 + 0.2 * torch.randn(n, device=DEVICE, generator=g)).requires_grad_(True),
              bias=(0.2 * torch.randn(n, device=DEVICE, generator=g)).requires_grad_(True),
              dy=torch.randn(b, 1, h, w, n, device=DEVICE, generator=g))


def _prepare_best(case, g):
  return dict(case=case, cost=_laid_out(case, _costs(case, g, _centres(case, g)).to(_TYPES[case["type"]])))


def _prepare_distill(case, g):
  """The teacher's list is around the student's valley, its costs rise from 0, and some of its ends are missing."""
  b, n, h, w = _size(case)
  centre, k = _centres(case, g), case["k"]
  cost = _costs(case, g, centre).to(_TYPES[case["type"]])
  place = torch.arange(k, device=DEVICE).view(1, 1, k, 1, 1)
  aside = torch.where(place % 2 == 0, -(place // 2), (place + 1) // 2)
  labels = ((centre + 0.5).long() + aside).remainder(n).to(torch.uint8)
  steps = torch.rand(b, 1, k, h, w, device=DEVICE, generator=g)
  costs = (steps.cumsum(2) - steps[:, :, :1]).mul_(1.5)
  missing = torch.rand(b, 1, 1, h, w, device=DEVICE, generator=g) < 0.01
  costs.masked_fill_(missing & (place >= k // 2), math.inf)
  rest = None
  if case["rest"]:
    rest = costs[:, :, 0] + 1.5 * k ** 0.5 + torch.randn(b, 1, h, w, device=DEVICE, generator=g)
  return dict(case=case, cost=_laid_out(case, cost).requires_grad_(True), labels=_laid_out(case, labels),
              costs=_laid_out(case, costs.to(_TYPES[case["kept"]])), rest=rest,
              dloss=torch.rand(b, 1, h, w, device=DEVICE, generator=g))


def _prepare_verify(case, g):
  """The draft's costs are the target's with noise, as those of fewer iterations, and its labels are drawn from them; some
  pixels have none."""
  b, n, h, w = _size(case)
  centre, m = _centres(case, g), case["drafts"]
  cost = _costs(case, g, centre)
  other = cost + 0.5 * torch.randn(cost.shape, device=DEVICE, generator=g)
  weight = torch.exp((other.amin(2, keepdim=True).clamp(max=3e38) - other) / case["draft_T"])
  sums = weight.cumsum_(2).movedim(2, -1)
  target = torch.rand(m, b, 1, h, w, 1, device=DEVICE, generator=g) * sums[..., -1:]
  draft = torch.searchsorted(sums.contiguous().expand(m, b, 1, h, w, n).contiguous() if m > 1 else sums.contiguous()[None],
                             target, right=True)[..., 0].clamp_(max=n - 1).to(torch.uint8)
  if n < 256:
    draft.masked_fill_(torch.rand(draft.shape, device=DEVICE, generator=g) < 0.002, 255)
  s = dict(case=case, cost=_laid_out(case, cost), draft=draft, draft_cost=_laid_out(case, other) if case["costs"] else None,
           u=torch.rand((2,) + draft.shape, device=DEVICE, generator=g))
  if case["each"]:
    spread = torch.linspace(0.5, 1.0, b, device=DEVICE)
    s.update(T=case["T"] * spread, draft_T=case["draft_T"] * spread)
  else:
    s.update(T=case["T"], draft_T=case["draft_T"])
  return s


def prepare(case, seed):
  g = torch.Generator(device=DEVICE).manual_seed(seed)
  return {"norm": _prepare_norm, "best": _prepare_best, "distill": _prepare_distill,
          "verify": _prepare_verify}[case["kind"]](case, g)


# ----------------------------------------------------------------------------------------- the plain forms
def _last(case, t):
  return t if case["last"] else t.movedim(2, -1)


def _plain_norm(s):
  case = s["case"]
  x, weight, bias, dy = _last(case, s["x"].detach()).float(), s["weight"].detach(), s["bias"].detach(), s["dy"]
  centred = x - x.mean(-1, keepdim=True)
  r = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
  xhat = centred * r
  y = (xhat * weight + bias).contiguous()
  g = dy * weight
  dx = r * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
  dx = (dx if case["last"] else dx.movedim(-1, 2)).to(s["x"].dtype).contiguous()
  over = (0, 1, 2, 3)
  return y, dx, (dy * xhat).sum(over, dtype=torch.float64).float(), dy.sum(over, dtype=torch.float64).float()


def _plain_best(s):
  case = s["case"]
  c = _last(case, s["cost"]).float()
  c = torch.where(c.isnan(), math.inf, c)
  c, order = torch.sort(c.contiguous(), dim=-1, stable=True)
  c = torch.where(c == c[..., :1], torch.where(c == math.inf, math.inf, 0.0), c - c[..., :1])
  k = case["k"]
  costs, labels = c[..., :k], torch.where(c[..., :k] == math.inf, 0, order[..., :k])
  others = torch.cat([c[..., k:], torch.full_like(c[..., :1], math.inf)], -1)
  least = others[..., :1].clamp(max=torch.finfo(torch.float32).max)
  rest = least[..., 0] - case["T"] * torch.log(torch.exp((least - others) / case["T"]).sum(-1))
  if not case["last"]:
    costs, labels = costs.movedim(-1, 2), labels.movedim(-1, 2)
  return labels.to(torch.uint8).contiguous(), costs.to(_TYPES[case["kept"]]).contiguous(), rest


def _plain_distill(s):
  case, t = s["case"], s["case"]["T"]
  n = case["labels"]
  c = _last(case, s["cost"].detach()).float()
  labels, costs = _last(case, s["labels"]).long(), _last(case, s["costs"]).float()
  candidate = c != math.inf
  best = c.amin(-1, keepdim=True).clamp(max=torch.finfo(torch.float32).max)
  z = (best - c) / t
  weight = torch.exp(z)
  total = weight.sum(-1, keepdim=True)
  log_q, q = z - torch.log(total), weight / total
  exists = (labels < n) & (costs != math.inf)
  labels = labels.clamp(max=n - 1)
  there = exists & candidate.gather(-1, labels)
  log_class = torch.where(there, log_q.gather(-1, labels), 0.0)
  listed_label = torch.zeros_like(candidate, dtype=torch.int32).scatter_add_(-1, labels, exists.int()) > 0
  others = torch.where(listed_label, 0.0, weight).sum(-1, keepdim=True)
  if s["rest"] is not None:
    costs = torch.cat([costs, s["rest"][..., None]], -1)
    there = torch.cat([there, (s["rest"][..., None] != math.inf) & (candidate & ~listed_label).any(-1, keepdim=True)], -1)
    log_class = torch.cat([log_class, torch.where(there[..., -1:], torch.log(others) - torch.log(total), 0.0)], -1)
  costs = torch.where(there, costs, math.inf)
  log_p = (costs.amin(-1, keepdim=True).clamp(max=torch.finfo(torch.float32).max) - costs) / t
  p = torch.exp(log_p)
  mass = p.sum(-1, keepdim=True)
  log_p, p = log_p - torch.log(mass), torch.where(there, p / mass, 0.0)
  loss = torch.where(p > 0, p * (log_p - log_class), 0.0).sum(-1)
  dz = -q
  dz.scatter_add_(-1, labels, p[..., :case["k"]])
  if s["rest"] is not None:
    dz += torch.where(listed_label | (p[..., -1:] == 0), 0.0, p[..., -1:] * weight / others)
  dcost = torch.where(candidate & there.any(-1, keepdim=True), dz / t * s["dloss"][..., None], 0.0)
  dcost = dcost if case["last"] else dcost.movedim(-1, 2)
  return loss, dcost.to(s["cost"].dtype).contiguous()


def _weights(c, temperature):
  """exp(-cost / T) relative to the best, in 64 bits."""
  c = torch.where(c.isnan(), math.inf, c)
  best = c.amin(-1, keepdim=True)
  weight = torch.exp((best.double() - c.double()) / temperature)  # (in 32 bits the difference would be rounded already)
  weight = torch.where(c == best, 1.0, torch.where(c == math.inf, 0.0, weight))
  return torch.where(best == math.inf, 0.0, weight)


def _plain_verify(s):
  case = s["case"]
  n = case["labels"]

  def per_image(v):
    return torch.as_tensor(v, dtype=torch.float32, device=DEVICE).double().view(-1, 1, 1, 1, 1)

  p = _weights(_last(case, s["cost"]), per_image(s["T"]))
  p /= p.sum(-1, keepdim=True).clamp(min=1)
  sums = p.cumsum(-1)
  d = s["draft"].long()
  exists, at = d < n, d.clamp(max=n - 1)[..., None]
  p_d = p.expand(d.shape + (n,)).gather(-1, at)[..., 0]
  if s["draft_cost"] is None:
    q_d = exists.double()
    left = torch.where(torch.arange(n, device=DEVICE) == at, 0.0, p)
  else:
    q = _weights(_last(case, s["draft_cost"]), per_image(s["draft_T"]))
    q /= q.sum(-1, keepdim=True).clamp(min=1)
    q_d = torch.where(exists, q.expand(d.shape + (n,)).gather(-1, at)[..., 0], 0.0)
    left = (p - q).clamp_(min=0)
  kept = exists & (q_d > 0) & (s["u"][0].double() * q_d < p_d)
  # what is drawn anew: from what is left, or from all of p
  left = left.cumsum(-1)
  whole = (q_d == 0) | (left[..., -1] == 0)
  u = s["u"][1].double()
  label = torch.where(whole, (sums <= (u * sums[..., -1])[..., None]).sum(-1), (left <= (u * left[..., -1])[..., None]).sum(-1))
  first = torch.where(whole, (sums < sums[..., -1:]).sum(-1), (left < left[..., -1:]).sum(-1))
  label = torch.where(kept, d, torch.minimum(label, first))
  label = torch.where(sums[..., -1] == 0, 0, label)
  return label.to(torch.uint8), kept


# ------------------------------------------------------------------------------------------ one pass of each
def _own_norm(s):
  from mplayers_amd import labels_last_norm
  y = labels_last_norm(s["x"], s["weight"], s["bias"], eps=_EPS, labels_first=not s["case"]["last"])
  return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])


def _own_best(s):
  from mplayers_amd import best_labels
  case = s["case"]
  return best_labels(s["cost"], case["k"], temperature=case["T"], dtype=_TYPES[case["kept"]], labels_first=not case["last"])


def _own_distill(s):
  from mplayers_amd import distill_costs
  loss = distill_costs(s["cost"], s["labels"], s["costs"], s["rest"], temperature=s["case"]["T"],
                       labels_first=not s["case"]["last"])
  return loss.detach(), torch.autograd.grad(loss, s["cost"], s["dloss"])[0]


def _own_verify(s):
  from mplayers_amd import verify_labels
  return verify_labels(s["cost"], s["draft"], s["u"], s["draft_cost"], temperature=s["T"], draft_temperature=s["draft_T"],
                       labels_first=not s["case"]["last"])


def run(state):
  kind = state["case"]["kind"]
  if own:
    return {"norm": _own_norm, "best": _own_best, "distill": _own_distill, "verify": _own_verify}[kind](state)
  return {"norm": _plain_norm, "best": _plain_best, "distill": _plain_distill, "verify": _plain_verify}[kind](state)


def work(case):
  b, n, h, w = _size(case)
  pixels = b * h * w
  entries = pixels * n
  wide = 4 if case.get("type", "f32") == "f32" else 2
  if case["kind"] == "norm":
    return dict(bytes=entries * (3 * wide + 8) + 16 * n, flops=20 * entries)
  kept = case.get("k", 0) * (1 + (4 if case.get("kept") == "f32" else 2))
  if case["kind"] == "best":
    return dict(bytes=entries * wide + pixels * (kept + 4), flops=3 * entries)
  if case["kind"] == "distill":
    # the costs are read for the loss and, as its gradient is asked for later, again for that
    return dict(bytes=entries * 3 * wide + pixels * (2 * kept + 8 + (8 if case["rest"] else 0)), flops=8 * entries)
  return dict(bytes=entries * (8 if case["costs"] else 4) + pixels * case["drafts"] * 11, flops=8 * entries)


# ---------------------------------------------------------------------------------------- in 64 bits, apart
def _numbers(case, t):
  """A (batch, cv, labels, H, W) or label-innermost tensor as pixels x labels in 64 bits."""
  a = t.detach().double().cpu().numpy()
  return (a if case["last"] else np.moveaxis(a, 2, -1)).reshape(-1, a.shape[-1 if case["last"] else 2])


def _as(case, a):
  """Pixels x labels in the case's layout."""
  b, _, h, w = _size(case)
  a = a.reshape(b, 1, h, w, -1)
  return a if case["last"] else np.ascontiguousarray(np.moveaxis(a, -1, 2))


def _exact_norm(s):
  case = s["case"]
  b, n, h, w = _size(case)
  x, dy = _numbers(case, s["x"]), s["dy"].double().cpu().numpy().reshape(-1, n)
  weight, bias = (s[k].detach().double().cpu().numpy() for k in ("weight", "bias"))
  deviation = np.sqrt(x.var(1) + _EPS)[:, None]
  xhat = (x - x.mean(1)[:, None]) / deviation
  g = dy * weight
  dx = (n * g - g.sum(1)[:, None] - xhat * (g * xhat).sum(1)[:, None]) / (n * deviation)
  return (xhat * weight + bias).reshape(b, 1, h, w, n), _as(case, dx), np.einsum("pl,pl->l", dy, xhat), dy.sum(0)


def _soft_least(c, t):
  """-t log(sum of exp(-c / t)) over the last axis."""
  least = np.minimum(c.min(-1), 1e300)
  with np.errstate(divide="ignore"):
    return least - t * np.log(np.exp((least[..., None] - c) / t).sum(-1))


def _exact_best(s):
  case = s["case"]
  b, _, h, w = _size(case)
  c = _numbers(case, s["cost"])
  c = np.sort(c, axis=1)
  best = np.where(np.isinf(c[:, :1]), 0.0, c[:, :1])
  c = c - best
  k = case["k"]
  rest = _soft_least(c[:, k:], case["T"]) if k < c.shape[1] else np.full(len(c), np.inf)
  return None, _as(case, c[:, :k]), rest.reshape(b, 1, h, w)


def _exact_distill(s):
  case, t, k = s["case"], s["case"]["T"], s["case"]["k"]
  b, n, h, w = _size(case)
  c, costs = _numbers(case, s["cost"]), _numbers(case, s["costs"])
  labels = _numbers(case, s["labels"]).astype(np.int64)
  rows = np.arange(len(c))[:, None]
  none = np.isinf(c).all(1)
  z = -c / t
  z[none] = 0
  q = np.exp(z - z.max(1)[:, None])
  q /= q.sum(1)[:, None]
  named = ~np.isinf(costs)
  there = named & ~np.isinf(c[rows, labels])
  taken = np.zeros(c.shape, bool)
  taken[rows.repeat(k, 1)[named], labels[named]] = True
  left = np.where(taken | np.isinf(c), 0.0, q).sum(1)
  classes = np.where(there, q[rows, labels], 1.0)
  costs = np.where(there, costs, np.inf)
  if s["rest"] is not None:
    rest = s["rest"].double().cpu().numpy().reshape(-1, 1)
    costs = np.concatenate([costs, np.where((~taken & ~np.isinf(c)).any(1)[:, None], rest, np.inf)], 1)
    classes = np.concatenate([classes, np.where(np.isinf(costs[:, -1]), 1.0, left)[:, None]], 1)
  none = np.isinf(costs).all(1)
  costs[none] = 0
  p = np.exp((costs.min(1)[:, None] - costs) / t)
  p /= p.sum(1)[:, None]
  p[none] = 0
  with np.errstate(divide="ignore", invalid="ignore"):
    loss = np.where(p > 0, p * (np.log(p) - np.log(classes)), 0.0).sum(1)
    share = np.where(taken, 0.0, q / left[:, None]) * p[:, -1:] if s["rest"] is not None else np.zeros(c.shape)
  share[np.isinf(c) | ~np.isfinite(share)] = 0
  d = share - q
  np.add.at(d, (rows.repeat(k, 1), labels), p[:, :k])
  d[np.isinf(c) | none[:, None]] = 0
  d *= s["dloss"].double().cpu().numpy().reshape(-1, 1) / t
  return loss.reshape(b, 1, h, w), _as(case, d)


def exact(case, seed):
  if case["kind"] == "verify":
    return None  # whole numbers: the plain form has them from 64 bits
  if math.prod(_size(case)) > (3e7 if case["kind"] == "norm" else 1.2e7):
    return None  # over 20 seconds
  s = prepare(case, seed)
  return {"norm": _exact_norm, "best": _exact_best, "distill": _exact_distill}[case["kind"]](s)
