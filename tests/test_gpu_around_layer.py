"""The operators around a layer together, as a program uses them: a bucketed table, dropout of the unary costs, the
layer, its gradients, and labels drawn from its costs with their energies."""
import argparse

import numpy as np
import pytest
import torch

from oracle import around_oracle
from tests.test_capi_host import _args

pytestmark = pytest.mark.gpu


def _module_args(mode, n, **more):
  return _args(mpnet_mrf_mode=mode, n_classes=n, mpnet_max_iter=2, mpnet_smoothness_mode="TL", mpnet_smoothness_train="on",
               mpnet_term_weight=0.3, mpnet_smoothness_trunct_value=4, enable_cuda=True, mpnet_smoothness_buckets=6, **more)


@pytest.mark.parametrize("share", ["element", "pixel", "label"])
@pytest.mark.parametrize("mode,n", [("TRWP", 21), ("ISGMR", 21), ("TRWP", 40), ("ISGMR", 70), ("soft", 12)])
def test_a_training_step_and_draws(gpu, mode, n, share):
  from mplayers_amd import MPModule, MP_module_hard_soft, bucket_context, labels_last_dropout, sample_labels
  from mplayers_amd.compute_terms import mrf_energy
  args = _module_args("TRWP" if mode == "soft" else mode, n, mpnet_unary_dropout=0.3, mpnet_unary_dropout_share=share,
                      mpnet_enable_soft=True)
  kind = MP_module_hard_soft.MPModule if mode == "soft" else MPModule
  module = kind(args, enable_create_label_context=True).cuda().train()
  table = module.label_context
  g = torch.Generator(device="cuda").manual_seed(n)
  unary = torch.randn(2, 1, n, 13, 18, device="cuda", generator=g).requires_grad_(True)
  dcost = torch.randn(2, 1, n, 13, 18, device="cuda", generator=g)
  torch.manual_seed(7)
  cost, context, _, _, _ = module(unary)
  got = (cost, context) + torch.autograd.grad(cost, (unary, table), dcost)
  # the same layer on the unary dropped out and the table laid out by hand
  torch.manual_seed(7)
  state = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), device="cuda")
  plain = kind(_module_args("TRWP" if mode == "soft" else mode, n, mpnet_enable_soft=True))
  whole = bucket_context(table.detach(), module.label_buckets, square=n == 21).requires_grad_(True)
  plain.set_label_context(whole, None, None)
  plain.train()
  dropped = labels_last_dropout(unary, 0.3, state, share=share).permute(0, 1, 4, 2, 3)
  by_hand, effective, _, _, _ = plain(dropped)
  du, dwhole = torch.autograd.grad(by_hand, (unary, whole), dcost)
  if mode == "soft":  # (this module's term weight scales the stored table)
    assert torch.allclose(context, effective, rtol=1e-6, atol=0)
  else:
    assert torch.equal(context, effective)
  assert torch.equal(got[0], by_hand) and torch.equal(got[2], du)
  assert int((got[2] == 0).sum()) > 0
  want = around_oracle.bucket_sums(dwhole.cpu().numpy(), module.label_buckets, n == 21)
  # (the layer's dcontext is summed with atomics: 1e-4 of the largest, as its own tests have it)
  assert np.abs(got[3].cpu().numpy() - want).max() <= 1e-4 * max(1.0, np.abs(want).max())
  # another step has another mask, evaluation has none
  assert not torch.equal(module(unary)[0], cost)
  module.eval()
  plain.eval()
  cost = module(unary.detach())[0]
  assert torch.equal(cost, plain(unary.detach())[0])
  # labellings drawn from the costs, and their energies
  u = torch.rand(3, 2, 1, 13, 18, device="cuda", generator=g)
  parameters = dict(temperature=0.5, top_k=8, top_p=0.9, min_p=0.01)
  labels = sample_labels(cost.detach(), u, **parameters)
  assert np.array_equal(labels.cpu().numpy(), around_oracle.draw_labels(cost.detach().cpu().numpy(), u.cpu().numpy(), **parameters))
  flat = unary.detach().permute(0, 1, 3, 4, 2).reshape(2, 13, 18, n).contiguous()
  energy = mrf_energy(flat, whole.detach(), labels.view(3, 2, 13, 18), None, 4)
  picked = torch.gather(flat.expand(3, -1, -1, -1, -1), -1, labels.view(3, 2, 13, 18, 1).long()).double().sum((1, 2, 3, 4))
  assert torch.allclose(energy[:, 0], picked, rtol=1e-12, atol=1e-9)


def test_a_bucketed_table_under_the_sigmoid(gpu):
  from mplayers_amd import MPModule, bucket_context
  args = _module_args("TRWP", 40)
  args.mpnet_smoothness_train = "sigmoid"
  module = MPModule(args, enable_create_label_context=True).cuda().train()
  unary = torch.randn(1, 1, 40, 5, 6, device="cuda")
  context = module(unary)[1][0].detach()
  entry = 2 * 0.3 * torch.sigmoid(module.label_context.detach())
  entry[0] = 0  # mpnet_diag_value
  assert torch.allclose(context, bucket_context(entry, module.label_buckets), rtol=1e-6, atol=0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_half_precision_costs(gpu, dtype):
  """A network's fp16 or bf16 costs with dropout, in training and in evaluation: the layer's costs are those of the
  same values in fp32, the gradient comes in the network's type."""
  from mplayers_amd import MPModule
  module = MPModule(_module_args("ISGMR", 21, mpnet_unary_dropout=0.4), enable_create_label_context=True).cuda()
  half = torch.randn(1, 1, 21, 7, 10, device="cuda").to(dtype).requires_grad_(True)
  whole = half.detach().float().requires_grad_(True)
  dcost = torch.randn(1, 1, 21, 7, 10, device="cuda")
  got = []
  for x in (half, whole):
    torch.manual_seed(3)
    module.train()
    cost = module(x)[0]
    (dx,) = torch.autograd.grad(cost, x, dcost)
    module.eval()
    got.append((cost, dx, module(x.detach())[0]))
  assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][2], got[1][2])
  assert got[0][1].dtype == dtype and torch.equal(got[0][1], got[1][1].to(dtype))


def test_a_captured_step(gpu):
  """The whole step captured and replayed: every replay has a mask of its own, from torch's generator."""
  from mplayers_amd import MPModule
  module = MPModule(_module_args("TRWP", 40, mpnet_unary_dropout=0.5), enable_create_label_context=True).cuda().train()
  unary = torch.randn(1, 1, 40, 9, 12, device="cuda").requires_grad_(True)
  dcost = torch.randn(1, 1, 40, 9, 12, device="cuda")

  def step():
    cost, _, _, _, _ = module(unary)
    return (cost.detach(),) + torch.autograd.grad(cost, (unary, module.label_context), dcost)

  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    step()
  torch.cuda.current_stream().wait_stream(stream)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  seen = []
  for _ in range(3):
    graph.replay()
    torch.cuda.synchronize()
    seen.append([t.clone() for t in out])
    assert all(bool(torch.isfinite(t).all()) for t in out)
    step()  # eager work between the replays
  assert not torch.equal(seen[0][0], seen[1][0]) and not torch.equal(seen[1][0], seen[2][0])
  dropped = [float((s[1] == 0).float().mean()) for s in seen]
  # 4320 entries, half of them dropped: within five standard deviations
  assert all(abs(d - 0.5) <= 5 * 0.5 / 4320 ** 0.5 for d in dropped), dropped


def test_inference_mode_and_two_streams(gpu):
  """The three without autograd, and on two streams at once: the results of a call alone."""
  from mplayers_amd import bucket_context, label_buckets, labels_last_dropout, sample_labels
  starts = label_buckets(60, 9)
  table = torch.randn(9, device="cuda", requires_grad=True)
  x = torch.randn(1, 1, 60, 200, 300, device="cuda", requires_grad=True)
  u = torch.rand(2, 1, 1, 200, 300, device="cuda")
  states = [torch.tensor([k, 5], device="cuda") for k in range(2)]

  def step(state):
    context = bucket_context(table, starts)
    y = labels_last_dropout(x, 0.2, state)
    return context, y, sample_labels((y + context).detach(), u, top_p=0.8, top_k=20, labels_first=False)

  want = [step(state) for state in states]
  with torch.inference_mode():
    got = step(states[0])
  assert not got[0].requires_grad and not got[1].requires_grad
  assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
  streams = [torch.cuda.Stream() for _ in states]
  torch.cuda.synchronize()
  for _ in range(3):
    got = []
    for stream, state in zip(streams, states):
      with torch.cuda.stream(stream):
        got.append(step(state))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
      assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_the_energy_minimiser_draws(gpu, tmp_path):
  import scipy.io as scio
  from mplayers_amd import energy_min
  command = ["--synthetic", "30", "41", "--mode", "TRWP", "--n_dir", "4", "--n_iter", "3", "--n_disp", "12", "--context", "TL",
             "--truncated", "2", "--p_weight", "10", "--enable_saving_label", "--save_dir"]
  plain = energy_min.main(command + [str(tmp_path / "plain")])
  assert "draws" not in plain
  got = energy_min.main(command + [str(tmp_path / "drawn"), "--n_draws", "5", "--temperature", "4", "--top_p", "0.95"])
  assert torch.equal(got["labels"], plain["labels"]) and torch.equal(got["cost_final"], plain["cost_final"])
  assert got["draws"].shape == (5, 30, 41) and got["draws_energy"].shape == (5, 2)
  u = torch.rand((5, 1, 1, 30, 41), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2019))
  want = around_oracle.draw_labels(got["cost_final"].view(1, 1, 12, 30, 41).cpu().numpy(), u.cpu().numpy(), temperature=4, top_p=0.95)
  assert np.array_equal(got["draws"].cpu().numpy(), want.reshape(5, 30, 41))
  # at temperature 0 the draws are the labelling of the last iteration
  cold = energy_min.main(command + [str(tmp_path / "cold"), "--n_draws", "1", "--temperature", "0"])
  file = scio.loadmat(cold["file_path"])
  assert file["draws"].shape == (1, 30, 41) and np.array_equal(file["draws_energy"], cold["draws_energy"].cpu().numpy())
  costs = cold["cost_final"]
  assert torch.equal(torch.gather(costs, 0, cold["draws"].long())[0], costs.amin(0))
