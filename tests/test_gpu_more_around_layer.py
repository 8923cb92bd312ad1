"""Layer norm, a teacher's best labels, the divergence from them and verified labels together around the layers, as a program
uses them: a student that learns from a teacher with more iterations, and labels drafted from the student's costs."""
import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle
from tests.test_capi_host import _args

pytestmark = pytest.mark.gpu


def _module(mode, n, n_iter, **more):
  from mplayers_amd import MPModule, MP_module_hard_soft
  args = _args(mpnet_mrf_mode="TRWP" if mode == "soft" else mode, n_classes=n, mpnet_max_iter=n_iter, mpnet_smoothness_mode="TL",
               mpnet_smoothness_train="on", mpnet_term_weight=0.3, mpnet_smoothness_trunct_value=4, enable_cuda=True,
               mpnet_enable_soft=True, **more)
  kind = MP_module_hard_soft.MPModule if mode == "soft" else MPModule
  return kind(args, enable_create_label_context=True).cuda()


@pytest.mark.parametrize("dropout", [False, True])
@pytest.mark.parametrize("mode,n", [("TRWP", 21), ("ISGMR", 21), ("TRWP", 40), ("ISGMR", 70), ("soft", 12)])
def test_a_student_and_its_labels(gpu, mode, n, dropout):
  from mplayers_amd import best_labels, distill_costs, labels_last_dropout, labels_last_norm, sample_labels, verify_labels
  fields = dict(mpnet_unary_dropout=0.3) if dropout else dict()
  student = _module(mode, n, 1, mpnet_unary_norm=True, mpnet_unary_norm_eps=1e-3, **fields).train()
  teacher = _module("TRWP", n, 5).eval()
  g = torch.Generator(device="cuda").manual_seed(n)
  with torch.no_grad():
    student.unary_norm_weight.copy_(1 + 0.2 * torch.randn(n, device="cuda", generator=g))
    student.unary_norm_bias.copy_(0.2 * torch.randn(n, device="cuda", generator=g))
  unary = torch.randn(2, 1, n, 13, 18, device="cuda", generator=g).requires_grad_(True)
  with torch.no_grad():
    kept = best_labels(teacher(unary)[0], 4, temperature=2.0, dtype=torch.float16)
  leaves = (unary, student.label_context, student.unary_norm_weight, student.unary_norm_bias)
  torch.manual_seed(7)
  cost = student(unary)[0]
  loss = distill_costs(cost, *kept, temperature=2.0)
  got = torch.autograd.grad(loss.mean(), leaves, retain_graph=True)
  # the same layer without, on costs that were normalised by hand, and the divergence's gradient by hand
  torch.manual_seed(7)
  if dropout:
    state = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), device="cuda")
    x = labels_last_norm(labels_last_dropout(unary, 0.3, state), *leaves[2:], 1e-3, labels_first=False)
  else:
    x = labels_last_norm(unary, *leaves[2:], 1e-3)
  plain = _module(mode, n, 1).train()
  table = student.label_context
  plain.set_label_context(table, student.label_context_loc, student.label_context_diag_loc)
  by_hand = plain(x.permute(0, 1, 4, 2, 3))[0]
  assert torch.equal(cost, by_hand)
  flat = cost.detach().movedim(2, -1).reshape(-1, n).double().cpu().numpy()
  lists = [t.movedim(2, -1).reshape(-1, 4).double().cpu().numpy() for t in kept[:2]]
  rest = kept[2].reshape(-1).double().cpu().numpy()
  pixels = [oracle.distill(flat[p], lists[0][p].astype(int), lists[1][p], rest[p], 2.0) for p in range(len(flat))]
  # (the bounds of the divergence's own tests at a reach below 50 and a list of 4 and the rest)
  bound = 2.0 ** -24 * ((5 * 50 + 26) * 51 + 160)
  assert np.abs(loss.detach().cpu().numpy().reshape(-1) - [p[0] for p in pixels]).max() <= bound
  dcost = torch.tensor(np.array([p[1] for p in pixels]) / len(pixels), dtype=torch.float32, device="cuda")
  dcost = dcost.view(2, 1, 13, 18, n).movedim(-1, 2).contiguous()
  (direct,) = torch.autograd.grad(loss.mean(), cost, retain_graph=True)
  assert float((direct - dcost).abs().max()) <= 2.0 ** -24 * (5 * 1.45 * 50 + 130) * 2 / len(pixels)
  want = torch.autograd.grad(by_hand, leaves, direct)
  for a, b, name in zip(got, want, ("unary", "table", "weight", "bias")):
    # (the layer's dcontext is summed with atomics: 1e-4 of the largest, as its own tests have it)
    assert torch.equal(a, b) if name != "table" else float((a - b).abs().max()) <= 1e-4 * float(b.abs().max()), name
  # in use: labels of the student, drafted, and verified against the teacher's costs
  student.eval()
  with torch.no_grad():
    draft_cost, target = student(unary)[0], teacher(unary)[0]
  u = torch.rand(3, 3, 2, 1, 13, 18, device="cuda", generator=g)
  draft = sample_labels(draft_cost, u[0])
  labels, stay = verify_labels(target, draft, u[1:], draft_cost)
  want = oracle.verify_labels(target.cpu().numpy(), draft.cpu().numpy(), u[1:].cpu().numpy(), draft_cost.cpu().numpy())
  assert np.array_equal(labels.cpu().numpy(), want[0]) and np.array_equal(stay.cpu().numpy(), want[1])
  # the teacher's labels of least cost, as a draft that is certain of them
  certain = best_labels(target, 1)[0][:, :, 0]
  assert torch.equal(certain, sample_labels(target, u[0, 0], temperature=0.0))
  labels, stay = verify_labels(draft_cost, certain, u[1:, 0].contiguous())
  want = oracle.verify_labels(draft_cost.cpu().numpy(), certain[None].cpu().numpy(), u[1:, :1].cpu().numpy())
  assert np.array_equal(labels[None].cpu().numpy(), want[0]) and np.array_equal(stay[None].cpu().numpy(), want[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_half_precision_costs(gpu, dtype):
  """A network's fp16 or bf16 costs, normalised: the layer's costs are those of the same values in fp32."""
  module = _module("ISGMR", 21, 2, mpnet_unary_norm=True)
  half = torch.randn(1, 1, 21, 7, 10, device="cuda").to(dtype).requires_grad_(True)
  whole = half.detach().float().requires_grad_(True)
  dcost = torch.randn(1, 1, 21, 7, 10, device="cuda")
  got = []
  for x in (half, whole):
    for training in (True, False):
      cost = module.train(training)(x)[0]
      got.append(cost.detach())
      if training:
        got.append(torch.autograd.grad(cost, x, dcost)[0])
  assert torch.equal(got[0], got[3]) and torch.equal(got[2], got[5])
  assert got[1].dtype == dtype and torch.equal(got[1], got[4].to(dtype))


def test_a_captured_step(gpu):
  """The student's step and its labels captured and replayed, with eager work between the replays."""
  from mplayers_amd import best_labels, distill_costs, sample_labels, verify_labels
  student = _module("TRWP", 40, 1, mpnet_unary_norm=True).train()
  teacher = _module("ISGMR", 40, 3).eval()
  unary = torch.randn(1, 1, 40, 9, 12, device="cuda").requires_grad_(True)
  u = torch.rand(3, 1, 1, 9, 12, device="cuda")
  leaves = (unary, student.unary_norm_weight, student.unary_norm_bias)

  def step():
    with torch.no_grad():
      target = teacher(unary)[0]
      kept = best_labels(target, 5)
    cost = student(unary)[0]
    loss = distill_costs(cost, *kept)
    grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    draft = sample_labels(cost.detach(), u[0])
    return (loss.detach(),) + grads + kept + verify_labels(target, draft, u[1:], cost.detach())

  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    step()
  torch.cuda.current_stream().wait_stream(stream)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  for _ in range(3):
    with torch.no_grad():
      unary.mul_(1.25)
      student.unary_norm_bias.add_(0.1)
    u.copy_(u.flip(-1))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_layouts_give_the_same(gpu):
  """The operators' layout and the network's: the same labels, and numbers that differ by roundings only, where a product and a
  sum are one instruction in one and two in the other.
  Layer norm, costs and gradients below 6, so |xhat| < 6 as well: y by 2 roundings of numbers below 36; dx by a rounding of each
  product in a mean, 36 u, times |xhat|, and of four numbers below 36 + 12: 512 u.  The divergence: a rounding of each of
  its terms, which weigh 1 together, and is below 64; its gradient one of three numbers below 1."""
  u24 = 2.0 ** -24

  def near(a, b, steps):
    return float((a - b).detach().abs().max()) <= steps * u24

  from mplayers_amd import best_labels, distill_costs, labels_last_norm, verify_labels
  g = torch.Generator(device="cuda").manual_seed(3)
  for n in (7, 21, 48, 64, 100, 192, 250):
    x = torch.randn(2, 1, n, 11, 19, device="cuda", generator=g).requires_grad_(True)
    y = x.detach().movedim(2, -1).contiguous().requires_grad_(True)
    d = torch.randn(2, 1, 11, 19, n, device="cuda", generator=g)
    one, two = labels_last_norm(x), labels_last_norm(y, labels_first=False)
    (dx,), (dy,) = torch.autograd.grad(one, x, d), torch.autograd.grad(two, y, d)
    assert float(x.detach().abs().max()) < 6 and float(d.abs().max()) < 6
    assert near(one, two, 72) and near(dx.movedim(2, -1), dy, 512)
    k = min(5, n)
    one, two = best_labels(x, k), best_labels(y, k, labels_first=False)
    assert torch.equal(one[0].movedim(2, -1), two[0]) and torch.equal(one[1].movedim(2, -1), two[1]) and torch.equal(one[2], two[2])
    losses = distill_costs(x, *one), distill_costs(y, *two, labels_first=False)
    dloss = torch.rand(2, 1, 11, 19, device="cuda", generator=g)
    (dx,), (dy,) = (torch.autograd.grad(loss, leaf, dloss) for loss, leaf in zip(losses, (x, y)))
    assert near(*losses, 64) and near(dx.movedim(2, -1), dy, 8)
    u = torch.rand(2, 2, 1, 11, 19, device="cuda", generator=g)
    one = verify_labels(x.detach(), one[0][:, :, 0].contiguous(), u)
    two = verify_labels(y.detach(), two[0][..., 0].contiguous(), u, labels_first=False)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
