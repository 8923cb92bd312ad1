"""What stands around a message-passing layer in training and in use, operator by operator, for measurement.

Three operators, each in a plain form of elementary torch operations and, where `own` is true, through the
framework's entry points:

  buckets  the learned pairwise table whose entries go by buckets of the label distance, and its gradient
           (`bucket_context`)
  dropout  dropout of the unary costs within the change to the layer's layout, forward and backward, its mask
           formed anew from (seed, offset) in both directions (`labels_last_dropout`)
  sample   labels drawn from the layer's costs with given uniform numbers, temperature, top-k, top-p and min-p
           (`sample_labels`)

Definitions that the plain forms spell out:

  buckets  distances below half the number of buckets have a bucket each; the others share logarithmic ones up
           to `max_distance`.  starts[b] is the first distance of bucket b.
  dropout  the ten-round 4x32 generator of Salmon, Moraes, Dror and Shaw (SC 2011).  Key: the seed's two words;
           counter: the two words of a group's number and the two of the offset.  A group is four labels of a
           pixel (share "element": number (item*P + pixel)*ceil(L/4) + label//4, word label%4), a pixel
           ("pixel": item*P + pixel, word 0) or four label planes of an item ("label": item*ceil(L/4) + label//4,
           word label%4).  An entry stays where its word is at least floor(p * 2^32), times 1/(1-p).
  sample   weights exp((best - cost) / T); +inf and NaN are no candidates; equal costs order by label.  Of the
           top_k best, of these the shortest run of best ones whose weight is at least top_p of theirs, of these
           the ones of at least min_p of the best one's weight; the label is the first whose running sum exceeds
           uniform * total.  T <= 0 takes the best label; a pixel without candidates gets label 0.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda"

_HALF = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------- cases
def listed():
  return [
      # a learned table of a 256-label denoiser: one vector, launches are all there is
      dict(name="buckets 256 labels", kind="buckets", tables=1, buckets=32, labels=256, far=128, square=False),
      # the 21-class segmentation layer's square table
      dict(name="buckets 21x21", kind="buckets", tables=1, buckets=8, labels=21, far=21, square=True),
      # one square table per direction, as the energy minimiser and the CPU operators take them
      dict(name="buckets 16x256x256", kind="buckets", tables=16, buckets=64, labels=256, far=256, square=True),
      # the smallest layer of the benchmark in training
      dict(name="dropout 16x64x96", kind="dropout", batch=1, labels=16, height=64, width=96, type="f32", share="element",
           p=0.1),
      # a segmentation network's logits in bf16 (batch and size of the reference's training options)
      dict(name="dropout 12x21x129x129 bf16", kind="dropout", batch=12, labels=21, height=129, width=129, type="bf16",
           share="element", p=0.5),
      # a KITTI frame's cost volume in fp16, whole pixels left to their neighbours
      dict(name="dropout 128x375x1242 f16 pixels", kind="dropout", batch=1, labels=128, height=375, width=1242,
           type="f16", share="pixel", p=0.15),
      # the headline configuration's cost volume
      dict(name="dropout 192x1500x2000", kind="dropout", batch=1, labels=192, height=1500, width=2000, type="f32",
           share="element", p=0.2),
      # one draw of a small layer's labels
      dict(name="sample 16x64x96", kind="sample", batch=1, labels=16, height=64, width=96, last=False, draws=1, T=1.0,
           k=0, top_p=1.0, min_p=0.0, masked=False, each=False),
      # a batch of segmentations, each image with parameters of its own
      dict(name="sample 12x21x129x129 top-p", kind="sample", batch=12, labels=21, height=129, width=129, last=False,
           draws=1, T=0.7, k=0, top_p=0.9, min_p=0.0, masked=False, each=True),
      # the energy minimiser's 60-label image in the operators' layout, labels outside the image masked
      dict(name="sample 60x375x450 top-k", kind="sample", batch=1, labels=60, height=375, width=450, last=True, draws=16,
           T=2.0, k=5, top_p=1.0, min_p=0.02, masked=True, each=False),
      # stereo inference, everything on
      dict(name="sample 96x384x1248 all", kind="sample", batch=1, labels=96, height=384, width=1248, last=False, draws=4,
           T=1.5, k=40, top_p=0.95, min_p=0.001, masked=True, each=False),
      # the headline configuration, no filter
      dict(name="sample 192x1500x2000", kind="sample", batch=1, labels=192, height=1500, width=2000, last=False, draws=1,
           T=1.0, k=0, top_p=1.0, min_p=0.0, masked=False, each=False),
  ]


def _spread(rng, low, high):
  return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _image(rng, labels, batch, low, high):
  """A height and a width that give the volume between low and high entries."""
  pixels = max(1.0, math.exp(rng.uniform(math.log(low), math.log(high))) / (labels * batch))
  height = max(1, int(round(math.sqrt(pixels) * math.exp(rng.uniform(-0.7, 0.7)))))
  return height, max(1, int(pixels / height))


def draw(rng):
  kind = rng.choice(["buckets", "dropout", "dropout", "sample", "sample", "sample"])
  if kind == "buckets":
    labels = _spread(rng, 2, 256)
    buckets = min(_spread(rng, 2, 128), labels)
    return dict(kind=kind, tables=_spread(rng, 1, 16), buckets=buckets, labels=labels,
                far=rng.randint(buckets, max(buckets, labels)), square=rng.random() < 0.5)
  labels, batch = _spread(rng, 2, 256), rng.choice([1, 1, 2, 3, 4, 7, 12])
  if kind == "dropout":
    height, width = _image(rng, labels, batch, 2e3, 2e8)
    return dict(kind=kind, batch=batch, labels=labels, height=height, width=width,
                type=rng.choice(["f32", "f16", "bf16"]), share=rng.choice(["element", "element", "pixel", "label"]),
                p=rng.choice([0.1, 0.5, round(rng.uniform(0.01, 0.9), 3)]))
  height, width = _image(rng, labels, batch, 2e3, 6e7)
  filtered = rng.random() < 0.75
  return dict(kind=kind, batch=batch, labels=labels, height=height, width=width, last=rng.random() < 0.4,
              draws=rng.choice([1, 1, 2, 5, 16]), T=rng.choice([1.0, round(rng.uniform(0.2, 4.0), 2)]),
              k=rng.choice([0, rng.randint(1, labels)]) if filtered else 0,
              top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]) if filtered else 1.0,
              min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]) if filtered else 0.0,
              masked=rng.random() < 0.5, each=rng.random() < 0.4)


# ---------------------------------------------------------------------------------------------- the inputs
def _starts(labels, buckets, far):
  """First distance of each bucket, and the number of labels behind them.  In whole numbers, so that a distance
  on a border is on its right side."""
  half = buckets // 2
  logs = buckets - half
  starts = list(range(half))
  for j in range(logs):
    if half == 0:
      starts.append(0)
      continue
    k = half
    while k < labels and k ** logs < half ** (logs - j) * max(far, half) ** j:
      k += 1
    starts.append(max(k, starts[-1]))
  return [min(s, labels) for s in starts] + [labels]


def _costs(case, g):
  """Costs as the layer gives them: a valley around a label that changes over the image, noise, and, where labels
  are masked, +inf for those that would lie left of the image, with a few pixels that have none left."""
  b, n, h, w = (case[k] for k in ("batch", "labels", "height", "width"))
  rows = torch.rand(b, 1, 1, h, 1, device=DEVICE, generator=g)
  cols = torch.rand(b, 1, 1, 1, w, device=DEVICE, generator=g)
  label = torch.arange(n, device=DEVICE, dtype=torch.float32).view(1, 1, n, 1, 1)
  cost = torch.randn(b, 1, n, h, w, device=DEVICE, generator=g)
  cost += (label - (rows + cols) * (0.5 * n)).abs_().clamp_(max=20).mul_(0.4)
  if case["masked"]:
    x = torch.arange(w, device=DEVICE, dtype=torch.float32).view(1, 1, 1, 1, w)
    cost.masked_fill_(label > x, math.inf)
    cost.masked_fill_(torch.rand(b, 1, 1, h, w, device=DEVICE, generator=g) < 0.001, math.inf)
  return cost.permute(0, 1, 3, 4, 2).contiguous() if case["last"] else cost


def prepare(case, seed):
  g = torch.Generator(device=DEVICE).manual_seed(seed)
  if case["kind"] == "buckets":
    n, t = case["labels"], case["tables"]
    context = (t, n, n) if case["square"] else (t, n)
    return dict(case=case, starts=torch.tensor(_starts(n, case["buckets"], case["far"]), dtype=torch.int32),
                table=torch.rand(t, case["buckets"], device=DEVICE, generator=g).requires_grad_(True),
                dcontext=torch.randn(context, device=DEVICE, generator=g))
  b, n, h, w = (case[k] for k in ("batch", "labels", "height", "width"))
  if case["kind"] == "dropout":
    x = torch.randn(b, 1, n, h, w, device=DEVICE, generator=g).to(_HALF[case["type"]])
    return dict(case=case, x=x.requires_grad_(True), dy=torch.randn(b, 1, h, w, n, device=DEVICE, generator=g),
                state=torch.randint(0, 2 ** 62, (2,), device=DEVICE, generator=g))
  s = dict(case=case, cost=_costs(case, g),
           u=torch.rand(case["draws"], b, 1, h, w, device=DEVICE, generator=g))
  if case["each"]:
    spread = torch.linspace(0.5, 1.0, b, device=DEVICE)
    s.update(T=case["T"] * spread, k=torch.full((b,), case["k"], device=DEVICE, dtype=torch.int32),
             top_p=case["top_p"] * spread if case["top_p"] < 1 else torch.ones(b, device=DEVICE),
             min_p=case["min_p"] * spread)
  else:
    s.update(T=case["T"], k=case["k"], top_p=case["top_p"], min_p=case["min_p"])
  return s


# ----------------------------------------------------------------------------------------- the plain forms
def _plain_buckets(s):
  n = s["case"]["labels"]
  starts = s["starts"].to(DEVICE)
  label = torch.arange(n, device=DEVICE)
  bucket = (label[:, None] >= starts[1:-1]).sum(-1)
  if s["case"]["square"]:
    bucket = bucket[(label[:, None] - label).abs()]
  context = s["table"].detach()[:, bucket]
  dtable = torch.zeros(s["table"].shape, dtype=torch.float64, device=DEVICE)
  dtable.index_add_(1, bucket.flatten(), s["dcontext"].double().flatten(1))
  return context, dtable.float()


def _times(a, b):
  """High and low word of a constant times 32-bit words held in int64."""
  return ((a >> 16) * b + ((a & 0xffff) * b >> 16)) >> 16, (a * b) & 0xffffffff


def _words(group, state):
  """The generator's four words for each group."""
  low = 0xffffffff
  c0, c1, c2, c3 = group & low, group >> 32, (state[1] & low).expand_as(group), (state[1] >> 32 & low).expand_as(group)
  k0, k1 = state[0] & low, state[0] >> 32 & low
  for _ in range(10):
    h0, l0 = _times(0xD2511F53, c0)
    h1, l1 = _times(0xCD9E8D57, c2)
    c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
    k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
  return c0, c1, c2, c3


def _plain_keep(case, state):
  """(batch, 1, H, W, labels) truth values, or a shape that broadcasts to it."""
  b, n, h, w = (case[k] for k in ("batch", "labels", "height", "width"))
  quads, bound = (n + 3) // 4, int(case["p"] * 2 ** 32)
  if case["share"] == "pixel":
    return (_words(torch.arange(b * h * w, device=DEVICE), state)[0] >= bound).view(b, 1, h, w, 1)
  pixels = (h, w) if case["share"] == "element" else (1, 1)
  words = _words(torch.arange(b * pixels[0] * pixels[1] * quads, device=DEVICE), state)
  keep = torch.stack([word >= bound for word in words], -1)
  return keep.view((b, 1) + pixels + (4 * quads,))[..., :n]


def _plain_dropout(s):
  case = s["case"]
  keep = _plain_keep(case, s["state"])
  scale = torch.tensor(1.0 / (1.0 - case["p"]), dtype=torch.float32, device=DEVICE)
  x = s["x"].detach().permute(0, 1, 3, 4, 2).float()
  y = torch.where(keep, x * scale, 0.0).contiguous()
  dx = torch.where(keep, s["dy"] * scale, 0.0).permute(0, 1, 4, 2, 3).to(s["x"].dtype).contiguous()
  return y, dx


def _plain_sample(s):
  case = s["case"]
  c = s["cost"] if case["last"] else s["cost"].permute(0, 1, 3, 4, 2)
  n = case["labels"]

  def per_image(v, **kw):
    return torch.as_tensor(v, device=DEVICE, **kw).view(-1, 1, 1, 1, 1)

  single = dict(dtype=torch.float32)
  temperature = per_image(s["T"], **single).double()
  top_p, min_p = per_image(s["top_p"], **single).double(), per_image(s["min_p"], **single).double()
  k = per_image(s["k"])
  k = torch.where((k <= 0) | (k > n), n, k)
  k = torch.where(temperature > 0, k, 1)
  temperature = temperature.clamp(min=0)
  c = torch.where(c.isnan(), math.inf, c) + 0.0
  best = c.amin(-1, keepdim=True)
  gap = c.double() - best.double()
  weight = torch.where(c == best, 1.0, torch.where(gap.isinf(), 0.0, torch.exp(-gap / temperature)))
  weight = torch.where(c == math.inf, 0.0, weight)
  if case["k"] or case["top_p"] < 1 or case["min_p"] > 0 or case["T"] <= 0:
    order = torch.sort(c.contiguous(), dim=-1, stable=True)[1]
    ranked = weight.gather(-1, order)
    rank = torch.arange(n, device=DEVICE)
    ranked = torch.where(rank < k, ranked, 0.0)
    sums = ranked.cumsum(-1)
    before = torch.cat([torch.zeros_like(sums[..., :1]), sums[..., :-1]], -1)
    keep = (top_p >= 1) | (before < top_p * sums[..., -1:]) | (rank == 0)
    reach = torch.where(min_p > 0, -temperature * torch.log(min_p.clamp(1e-300, 1)), math.inf)
    keep &= (gap.gather(-1, order) <= reach) | (rank == 0)
    weight = torch.zeros_like(weight).scatter_(-1, order, torch.where(keep, ranked, 0.0))
  sums = weight.cumsum(-1)
  target = s["u"].double().clamp(min=0) * sums[..., -1]
  label = (sums <= target[..., None]).sum(-1)
  last = torch.where(weight > 0, torch.arange(n, device=DEVICE), 0).amax(-1)
  return torch.minimum(label, last).to(torch.uint8)


# ------------------------------------------------------------------------------------------ one pass of each
def _own_buckets(s):
  from mplayers_amd import bucket_context
  context = bucket_context(s["table"], s["starts"], square=s["case"]["square"])
  return context.detach(), torch.autograd.grad(context, s["table"], s["dcontext"])[0]


def _own_dropout(s):
  from mplayers_amd import labels_last_dropout
  y = labels_last_dropout(s["x"], s["case"]["p"], s["state"], share=s["case"]["share"])
  return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]


def _own_sample(s):
  from mplayers_amd import sample_labels
  return sample_labels(s["cost"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["top_p"], min_p=s["min_p"],
                       labels_first=not s["case"]["last"])


def run(state):
  kind = state["case"]["kind"]
  if own:
    return {"buckets": _own_buckets, "dropout": _own_dropout, "sample": _own_sample}[kind](state)
  return {"buckets": _plain_buckets, "dropout": _plain_dropout, "sample": _plain_sample}[kind](state)


def work(case):
  if case["kind"] == "buckets":
    entries = case["tables"] * case["labels"] ** (2 if case["square"] else 1)
    return dict(bytes=8 * entries + 8 * case["tables"] * case["buckets"], flops=entries)
  pixels = case["batch"] * case["height"] * case["width"]
  entries = pixels * case["labels"]
  if case["kind"] == "dropout":
    return dict(bytes=2 * entries * (4 + (4 if case["type"] == "f32" else 2)), flops=2 * entries)
  return dict(bytes=4 * entries + 5 * pixels * case["draws"], flops=4 * entries)


# ---------------------------------------------------------------------------------------- in 64 bits, apart
def _exact_buckets(s):
  case, starts = s["case"], s["starts"].numpy()
  n, of = case["labels"], np.zeros(case["labels"], np.int64)
  for b in range(case["buckets"]):
    of[starts[b]:starts[b + 1]] = b
  label = np.arange(n)
  of = of[np.abs(label[:, None] - label)] if case["square"] else of
  table, d = (s[k].detach().cpu().numpy().astype(np.float64) for k in ("table", "dcontext"))
  dtable = np.zeros(table.shape)
  for t in range(case["tables"]):
    dtable[t] = np.bincount(of.ravel(), d[t].ravel(), case["buckets"])
  return table[:, of], dtable


def _exact_dropout(s):
  case = s["case"]
  b, n, h, w = (case[k] for k in ("batch", "labels", "height", "width"))
  seed, offset = (int(v) for v in s["state"].cpu())
  quads = -(-n // 4)
  count = {"element": b * h * w * quads, "pixel": b * h * w, "label": b * quads}[case["share"]]
  low = np.uint64(0xffffffff)
  shift = np.uint64(32)
  group = np.arange(count, dtype=np.uint64)
  c = [group & low, group >> shift, np.full(count, offset & 0xffffffff, np.uint64),
       np.full(count, offset >> 32, np.uint64)]
  key = [seed & 0xffffffff, seed >> 32]
  for _ in range(10):
    a, d = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
    c = [(d >> shift) ^ c[1] ^ np.uint64(key[0]), d & low, (a >> shift) ^ c[3] ^ np.uint64(key[1]), a & low]
    key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
  kept = [word.astype(np.float64) >= np.floor(case["p"] * 2.0 ** 32) for word in c]
  if case["share"] == "pixel":
    keep = kept[0].reshape(b, 1, h, w, 1)
  else:
    keep = np.stack(kept, -1).reshape((b, 1) + ((h, w) if case["share"] == "element" else (1, 1)) + (4 * quads,))[..., :n]
  scale = 1.0 / (1.0 - case["p"])
  x = s["x"].detach().double().cpu().numpy().transpose(0, 1, 3, 4, 2)
  dy = s["dy"].double().cpu().numpy()
  return np.where(keep, x * scale, 0.0), np.ascontiguousarray(np.where(keep, dy * scale, 0.0).transpose(0, 1, 4, 2, 3))


def exact(case, seed):
  if case["kind"] == "sample":
    return None  # whole numbers: the plain form has them from 64 bits
  if case["kind"] == "dropout" and case["batch"] * case["labels"] * case["height"] * case["width"] > 3e7:
    return None  # over 20 seconds
  s = prepare(case, seed)
  return _exact_buckets(s) if case["kind"] == "buckets" else _exact_dropout(s)
