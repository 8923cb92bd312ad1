"""The modules with dropout and bucketed tables, on the CPU: half-precision costs at a rate of 0, which entries of a
table are learned, and tables that are saved and loaded."""
import pytest
import torch

from tests.test_capi_host import _args


def _module(soft=False, **fields):
  from mplayers_amd import MPModule, MP_module_hard_soft
  kind = MP_module_hard_soft.MPModule if soft else MPModule
  return kind(_args(mpnet_smoothness_mode="TL", mpnet_smoothness_trunct_value=3, **fields), enable_create_label_context=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rate", [0, 0.0])
def test_half_precision_costs_at_a_rate_of_0(rate, dtype):
  """A rate that is scheduled from or to 0: the same network runs at 0, without dropout, as at any other rate."""
  half = torch.randn(2, 1, 9, 4, 5).to(dtype)
  for soft in (False, True):
    module = _module(soft, n_classes=9, mpnet_unary_dropout=rate)
    for training in (True, False):
      for x in (half, half.float()):
        last = module.train(training)._labels_last(x)
        assert last.dtype == torch.float32 and torch.equal(last, half.float().permute(0, 1, 3, 4, 2))
  # (the CPU operators take a table of all pairs of labels for each direction)
  table = (torch.arange(9)[:, None] - torch.arange(9)).abs().clamp(max=3).float().expand(4, 9, 9).contiguous()
  modules = [_module(n_classes=9, mpnet_unary_dropout=rate).eval(), _module(n_classes=9).eval()]
  for module in modules:
    module.set_label_context(torch.nn.Parameter(table), None, None)
  assert torch.equal(modules[0](half)[0], modules[1](half.float())[0])
  # without the field the costs are the operators' fp32 ones, as ever
  with pytest.raises(RuntimeError, match="float32"):
    modules[1](half)


@pytest.mark.parametrize("train", ["", "on", "sigmoid", "softmax"])
def test_one_bucket_is_refused(train):
  """The first entry is pinned, as the table's of distance 0 is: it has to be of that distance alone."""
  from mplayers_amd.label_context import create_bucket_table
  with pytest.raises(ValueError, match="distance 0"):
    _module(n_classes=9, mpnet_smoothness_train=train, mpnet_smoothness_buckets=1)
  with pytest.raises(ValueError, match="distance 0"):
    create_bucket_table(_args(n_classes=21, mpnet_smoothness_train=train), 1)
  module = _module(n_classes=9, mpnet_smoothness_train=train, mpnet_smoothness_buckets=2)
  context = module._effective_label_context()
  context = context.detach()
  assert context.shape == (9,) and float(context[0]) == 0 and bool((context[1:] == context[1]).all())
  # (one label has no other distance)
  assert create_bucket_table(_args(n_classes=1, mpnet_smoothness_train=train), 1)[3].tolist() == [0, 1]


@pytest.mark.parametrize("n,buckets,far", [(5, 8, None), (40, 9, 2), (40, 9, 20), (21, 30, None), (1, 3, None)])
def test_entries_of_empty_buckets_take_no_part(n, buckets, far):
  """The softmax is over the entries that a distance has: whatever the others hold, the table is the same, and they have
  no gradient."""
  module = _module(n_classes=n, mpnet_smoothness_train="softmax", mpnet_smoothness_buckets=buckets,
                   mpnet_smoothness_bucket_far=far)
  starts = module.label_buckets
  full = (starts[1:] > starts[:-1]).tolist()
  learned = [b for b in range(1, buckets) if full[b]]
  assert list(module.label_context_loc) == learned and list(module.label_context_diag_loc) == [0]
  entries = torch.linspace(-1, 1, buckets).double().tolist()
  module.label_context.data.copy_(torch.tensor(entries))
  # by the definition: e_b / max(e) * max of what is stored, e the softmax
  stored = [entries[b] for b in learned]
  want = torch.zeros(buckets, dtype=torch.float64)
  if learned:
    e = torch.exp(torch.tensor(stored, dtype=torch.float64))
    want[learned] = e / e.max() * max(stored)
  distance = torch.arange(n)
  bucket = (distance[:, None] >= starts[None, 1:-1]).sum(-1)
  want = want[bucket]
  if n == 21:
    want = want[(distance[:, None] - distance).abs()]
  for other in (0.0, 100.0):
    for b in range(buckets):
      if not full[b]:
        module.label_context.data[b] = other
    context = module._effective_label_context()
    # (fp32: a softmax of at most 30 entries and two products, some tens of roundings of 2^-24 of values up to 1)
    assert torch.allclose(context.detach().double(), want, rtol=0, atol=64 * 2.0 ** -24)
    (grad,) = torch.autograd.grad(context.sum(), module.label_context)
    assert all(float(grad[b]) == 0 for b in range(buckets) if not full[b])


@pytest.mark.parametrize("strict", [True, False])
def test_a_learned_table_is_loaded_with_its_borders(strict):
  """Entries that were learned for other distances are refused; a state without borders, or of a table without buckets,
  is loaded as ever."""
  from mplayers_amd import MP_module_hard_soft, label_buckets
  fields = dict(n_classes=40, mpnet_smoothness_train="on", mpnet_smoothness_buckets=8)
  module = _module(mpnet_smoothness_bucket_far=30, **fields)
  module.label_context.data.copy_(torch.rand(8))
  network = torch.nn.Sequential(torch.nn.Linear(2, 3), module)
  state = network.state_dict()
  assert torch.equal(state["1.label_buckets"], label_buckets(40, 8, 30))

  def other(**more):
    return torch.nn.Sequential(torch.nn.Linear(2, 3), _module(**{**fields, **more}))

  for soft in (False, True):
    same = torch.nn.Sequential(torch.nn.Linear(2, 3), _module(soft, mpnet_smoothness_bucket_far=30, **fields))
    same.load_state_dict(state, strict=strict)
    assert torch.equal(same[1].label_context, module.label_context) and isinstance(same[1], MP_module_hard_soft.MPModule) == soft
  for wrong in (other(mpnet_smoothness_bucket_far=20), other(n_classes=50, mpnet_smoothness_bucket_far=30),
                other(n_classes=8, mpnet_smoothness_buckets=0)):
    kept = wrong[1].label_context.detach().clone()
    with pytest.raises(RuntimeError, match="buckets"):
      wrong.load_state_dict(state, strict=strict)
    assert torch.equal(wrong[1].label_context, kept)
  before = {k: v for k, v in state.items() if k != "1.label_buckets"}
  loaded = other(mpnet_smoothness_bucket_far=30)
  loaded.load_state_dict(before, strict=strict)
  assert torch.equal(loaded[1].label_context, module.label_context)
  plain = other(mpnet_smoothness_buckets=0)
  assert set(plain.state_dict()) == {"0.weight", "0.bias", "1.label_context"}
  plain.load_state_dict(plain.state_dict(), strict=strict)


def test_layers_that_share_their_borders_are_saved(tmp_path):
  """Formats that refuse tensors of one memory under two names take them."""
  safetensors = pytest.importorskip("safetensors.torch")
  fields = dict(n_classes=40, mpnet_smoothness_train="on", mpnet_smoothness_buckets=8)
  first, second = _module(**fields), _module(**fields)
  second.set_label_context(second.label_context, second.label_context_loc, second.label_context_diag_loc, first.label_buckets)
  network = torch.nn.ModuleList([first, second])
  safetensors.save_file(network.state_dict(), str(tmp_path / "net.safetensors"))
  first.label_context.data.add_(1)
  network.load_state_dict(safetensors.load_file(str(tmp_path / "net.safetensors")))
  assert torch.equal(first.label_context, second.label_context)
