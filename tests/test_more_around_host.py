"""Layer norm in the layout change, a teacher's best labels, the divergence from them and verified labels on the CPU: the
refusals of the entry points, the plain forms that the GPU tests compare with, and the modules with them."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import more_around_oracle as oracle
from tests.test_capi_host import _args


@pytest.fixture(scope="module")
def lib():
  from mplayers_amd import _lib
  return _lib.load()


def _refused(lib, rc, words):
  assert rc == -1 and words in lib.mpl_last_error(), (rc, lib.mpl_last_error())


# (refused before a pointer is looked at, and nothing is launched)
ONE = ctypes.c_void_p(1 << 20)


def test_norm_refusals(lib):
  def last(dtype=0, src=ONE, eps=1e-5, dst=ONE, batch=1, n=4, pixels=9):
    return lib.mpl_norm_labels_last(dtype, 1, src, None, None, eps, dst, None, batch, n, pixels, None)

  def grad(dtype=0, src=ONE, eps=1e-5, stats=ONE, ddst=ONE, dsrc=ONE, dweight=None, workspace=None, batch=1, n=4, pixels=9):
    return lib.mpl_norm_labels_last_grad(dtype, 1, src, None, eps, stats, ddst, dsrc, dweight, None, workspace, batch, n, pixels, None)

  for call in (last, grad):
    _refused(lib, call(src=None), b"null")
    _refused(lib, call(dtype=3), b"type")
    _refused(lib, call(dtype=-1), b"type")
    _refused(lib, call(n=0), b"n_disp")
    _refused(lib, call(n=257), b"n_disp")
    _refused(lib, call(pixels=-1), b"negative")
    _refused(lib, call(batch=-1), b"negative")
    _refused(lib, call(batch=1 << 20, pixels=1 << 30), b"too many")
    _refused(lib, call(pixels=1 << 32), b"too many")
    assert call(batch=0) == 0 and call(pixels=0) == 0
    for eps in (-1e-9, math.nan, math.inf):
      _refused(lib, call(eps=eps), b"eps")
  _refused(lib, last(dst=None), b"null")
  # what the forward call keeps for the gradient: nothing up to 16 labels
  assert [lib.mpl_norm_stats(n) for n in (1, 16, 17, 256)] == [0, 0, 2, 2]
  _refused(lib, grad(stats=None, n=17), b"null")
  _refused(lib, grad(ddst=None), b"null")
  _refused(lib, grad(dweight=ONE), b"null")  # no workspace
  assert grad(dsrc=None) == 0  # nothing wanted
  # a row of 2 * n sums for each workgroup, 2048 at most
  assert lib.mpl_norm_workspace(1, 21, 64) == 42 and lib.mpl_norm_workspace(3, 21, 65) == 6 * 42
  assert lib.mpl_norm_workspace(1, 256, 1 << 30) == 2048 * 512 and lib.mpl_norm_workspace(1 << 30, 2, 1 << 30) == 2048 * 4
  assert lib.mpl_norm_workspace(0, 21, 9) == 0 and lib.mpl_norm_workspace(1, 21, 0) == 0


def test_norm_of_the_plain_form():
  x = np.array([[1.0, 3.0], [5.0, 5.0]])
  y, xhat, r = oracle.norm(x, [2.0, 1.0], [0.0, 10.0], 0.0 + 1e-30)
  assert np.allclose(y[0], [-2, 11]) and np.allclose(xhat[1], 0) and np.isclose(r[0, 0], 1)
  # against torch's, in 64 bits
  g = torch.Generator().manual_seed(1)
  x, w, b, dy = (torch.randn(s, dtype=torch.float64, generator=g, requires_grad=True) for s in ((7, 5), (5,), (5,), (7, 5)))
  y = torch.nn.functional.layer_norm(x, (5,), w, b, 1e-5)
  grads = torch.autograd.grad(y, (x, w, b), dy)
  x, w, b, dy = (t.detach().numpy() for t in (x, w, b, dy))
  assert np.allclose(oracle.norm(x, w, b, 1e-5)[0], y.detach().numpy(), rtol=0, atol=1e-12)
  for got, want in zip(oracle.norm_grad(x, w, 1e-5, dy), grads):
    assert np.allclose(got, want.numpy(), rtol=0, atol=1e-12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_of_cpu_tensors(dtype):
  from mplayers_amd import labels_last_norm
  x = torch.randn(2, 1, 6, 3, 4).to(dtype).requires_grad_(True)
  w, b = torch.rand(6).requires_grad_(True), torch.rand(6)
  y = labels_last_norm(x, w, b, 1e-3)
  assert y.shape == (2, 1, 3, 4, 6) and y.dtype == torch.float32 and y.is_contiguous()
  flat = np.moveaxis(x.detach().double().numpy(), 2, -1)
  want = oracle.norm(flat.reshape(-1, 6), w.detach().numpy(), b.numpy(), 1e-3)[0]
  # fp32: some tens of roundings of values below 32
  assert np.abs(y.detach().double().numpy().reshape(-1, 6) - want).max() <= 64 * 2.0 ** -24 * 32
  assert torch.equal(labels_last_norm(x.movedim(2, -1), w, b, 1e-3, labels_first=False), y)
  dx, dw = torch.autograd.grad(y.sum(), (x, w))
  assert dx.shape == x.shape and dx.dtype == dtype and dw.shape == (6,)
  for wrong in (dict(x=x[0]), dict(x=x.double()), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(weight=w[:5]),
                dict(labels_first=False), dict(x=torch.zeros(1, 1, 257, 2, 2), weight=None, bias=None),
                dict(x=torch.zeros(1, 1, 0, 2, 2), weight=None, bias=None)):
    with pytest.raises(RuntimeError):
      labels_last_norm(**{**dict(x=x, weight=w, bias=b), **wrong})


@pytest.mark.parametrize("soft", [False, True])
def test_a_module_that_normalises(soft):
  """mpnet_unary_norm: learned weights in the module's state, fp16 and bf16 costs taken, after dropout where there is any."""
  from mplayers_amd import MPModule, MP_module_hard_soft, labels_last_norm
  kind = MP_module_hard_soft.MPModule if soft else MPModule
  fields = dict(mpnet_smoothness_mode="TL", mpnet_smoothness_trunct_value=3, n_classes=9)
  module = kind(_args(mpnet_unary_norm=True, mpnet_unary_norm_eps=1e-2, **fields), enable_create_label_context=True)
  assert {"unary_norm_weight", "unary_norm_bias"} <= {name for name, _ in module.named_parameters()}
  with torch.no_grad():
    module.unary_norm_weight.copy_(torch.rand(9))
    module.unary_norm_bias.copy_(torch.rand(9))
  x = torch.randn(2, 1, 9, 4, 5)
  want = labels_last_norm(x, module.unary_norm_weight, module.unary_norm_bias, 1e-2)
  for training in (True, False):
    assert torch.equal(module.train(training)._labels_last(x), want)
  assert module._labels_last(x.half()).dtype == torch.float32
  other = kind(_args(mpnet_unary_norm=True, **fields), enable_create_label_context=True)
  other.load_state_dict(module.state_dict())
  assert torch.equal(other.unary_norm_weight, module.unary_norm_weight)
  for off in (dict(), dict(mpnet_unary_norm=False), dict(mpnet_unary_norm=None)):
    plain = kind(_args(**fields, **off), enable_create_label_context=True)
    assert set(plain.state_dict()) == {"label_context"} and torch.equal(plain._labels_last(x), x.permute(0, 1, 3, 4, 2))
  # copies, files, weights that are made of others, and modules of files from before
  import copy
  import pickle
  for other in (copy.deepcopy(module), pickle.loads(pickle.dumps(module))):
    assert torch.equal(other._labels_last(x), want)
  double = copy.deepcopy(module)
  torch.nn.utils.parametrize.register_parametrization(double, "unary_norm_weight", torch.nn.Softplus())
  assert torch.equal(double._labels_last(x), labels_last_norm(x, torch.nn.functional.softplus(module.unary_norm_weight),
                                                              module.unary_norm_bias, 1e-2))
  del plain.__dict__["unary_norm"]
  assert torch.equal(plain._labels_last(x), x.permute(0, 1, 3, 4, 2))
  # in evaluation a rate of dropout changes nothing
  dropped = kind(_args(mpnet_unary_norm=True, mpnet_unary_norm_eps=1e-2, mpnet_unary_dropout=0.5, **fields),
                 enable_create_label_context=True).eval()
  dropped.load_state_dict(module.state_dict())
  assert torch.equal(dropped._labels_last(x), want)


def test_a_cpu_layer_on_normalised_costs():
  """The CPU operators run on them as on any costs."""
  from mplayers_amd import MPModule
  fields = dict(mpnet_smoothness_mode="TL", mpnet_smoothness_trunct_value=3, n_classes=9)
  table = (torch.arange(9)[:, None] - torch.arange(9)).abs().clamp(max=3).float().expand(4, 9, 9).contiguous()
  modules = [MPModule(_args(mpnet_unary_norm=on, **fields), enable_create_label_context=True).eval() for on in (True, False)]
  for module in modules:
    module.set_label_context(torch.nn.Parameter(table), None, None)
  x = torch.randn(1, 1, 9, 4, 5)
  normalised = torch.nn.functional.layer_norm(x.movedim(2, -1), (9,)).movedim(-1, 2)
  assert torch.allclose(modules[0](x)[0], modules[1](normalised)[0], rtol=1e-5, atol=1e-5)


def test_distill_refusals(lib):
  def best(dtype=0, cost=ONE, k=2, t=1.0, kept=0, labels=ONE, costs=ONE, batch=1, n=4, pixels=9):
    return lib.mpl_best_labels(dtype, 1, cost, k, t, kept, labels, costs, None, batch, n, pixels, None)

  def loss(dtype=0, cost=ONE, k=2, t=1.0, kept=0, labels=ONE, costs=ONE, batch=1, n=4, pixels=9, out=ONE):
    return lib.mpl_distill_costs(dtype, 1, cost, kept, labels, costs, None, t, out, batch, n, k, pixels, None)

  def grad(dtype=0, cost=ONE, k=2, t=1.0, kept=0, labels=ONE, costs=ONE, batch=1, n=4, pixels=9, dloss=ONE, out=ONE):
    return lib.mpl_distill_costs_grad(dtype, 1, cost, kept, labels, costs, None, t, dloss, out, batch, n, k, pixels, None)

  for call in (best, loss, grad):
    for name in ("cost", "labels", "costs"):
      _refused(lib, call(**{name: None}), b"null")
    for wrong in (3, -1):
      _refused(lib, call(dtype=wrong), b"type")
      _refused(lib, call(kept=wrong), b"type")
    for n in (0, 257):
      _refused(lib, call(n=n), b"n_disp")
    for t in (0.0, -1.0, math.inf, math.nan, 1e-45):
      _refused(lib, call(t=t), b"temperature")
    _refused(lib, call(k=0), b"list")
    _refused(lib, call(k=257), b"list")
    _refused(lib, call(batch=-1), b"negative")
    _refused(lib, call(pixels=-1), b"negative")
    _refused(lib, call(batch=1 << 20, pixels=1 << 30), b"too many")
    _refused(lib, call(pixels=1 << 41), b"too many")
    assert call(batch=0) == 0 and call(pixels=0) == 0
  _refused(lib, best(k=5), b"list")
  _refused(lib, loss(out=None), b"null")
  _refused(lib, grad(out=None), b"null")
  _refused(lib, grad(dloss=None), b"null")


def test_temperatures_at_the_end_of_fp32(lib):
  """log2(e) / T is what exponents are multiplied by: beside an infinite one a difference of 0 is no number."""
  for t, taken in ((2.95e-39, False), (4.2e-39, False), (4.3e-39, True), (3e38, True)):
    for rc in (lib.mpl_best_labels(0, 1, ONE, 1, t, 0, ONE, ONE, None, 0, 2, 1, None),
               lib.mpl_distill_costs(0, 1, ONE, 0, ONE, ONE, None, t, ONE, 0, 2, 1, 1, None),
               lib.mpl_distill_costs_grad(0, 1, ONE, 0, ONE, ONE, None, t, ONE, ONE, 0, 2, 1, 1, None)):
      assert (rc == 0) == taken, t


def test_best_labels_of_the_plain_form():
  inf, nan = math.inf, math.nan
  assert oracle.best_labels([3, 1, 1, nan, 2], 3, 1.0)[:2] == ([1, 2, 4], [0, 0, 1])
  assert oracle.best_labels([3, 1, 1, nan, 2], 3, 1.0)[2] == 2
  assert oracle.best_labels([inf, 1, nan], 2, 1.0) == ([1, 0], [0, inf], inf)
  assert oracle.best_labels([5, -inf, 0, -inf], 1, 1.0) == ([1], [0.0], 0.0)
  assert abs(oracle.best_labels([0, 2, 2, 2], 1, 0.5)[2] - (2 - 0.5 * math.log(3))) < 1e-12


@pytest.mark.parametrize("with_rest", [True, False])
def test_distill_of_the_plain_form(with_rest):
  """Against autograd through the definition, in 64 bits."""
  g = torch.Generator().manual_seed(2)
  for _ in range(30):
    n, k, t = 9, 3, 1.7
    cost = torch.randn(n, dtype=torch.float64, generator=g).mul(2).requires_grad_(True)
    labels = torch.randperm(n, generator=g)[:k]
    costs, rest = torch.rand(k, dtype=torch.float64, generator=g) * 3, 2.0
    log_q = torch.log_softmax(-cost / t, 0)
    log_class, class_cost = log_q[labels], costs
    if with_rest:
      left = [l for l in range(n) if l not in labels.tolist()]
      log_class = torch.cat([log_class, torch.logsumexp(log_q[left], 0)[None]])
      class_cost = torch.cat([costs, torch.tensor([rest], dtype=torch.float64)])
    log_p = torch.log_softmax(-class_cost / t, 0)
    want = (log_p.exp() * (log_p - log_class)).sum()
    (grad,) = torch.autograd.grad(want, cost)
    loss, got, _ = oracle.distill(cost.tolist(), labels.tolist(), costs.tolist(), rest if with_rest else None, t)
    assert abs(loss - float(want.detach())) <= 1e-12 and np.allclose(got, grad.numpy(), rtol=0, atol=1e-12)
  inf, nan = math.inf, math.nan
  # entries that are not there; a pixel without any; what is no number
  assert oracle.distill([0, 1], [0, 1], [inf, inf], None, 1.0)[0] == 0
  assert oracle.distill([0, inf], [1, 7], [0, 0], None, 1.0)[:2] == (0.0, [0.0, 0.0])
  assert oracle.distill([0, 1], [0, 1], [0, 1], 5.0, 1.0)[0] == oracle.distill([0, 1], [0, 1], [0, 1], None, 1.0)[0]
  loss, grad, _ = oracle.distill([0, nan, inf], [0], [0], None, 1.0)
  assert math.isnan(loss) and math.isnan(grad[0]) and grad[2] == 0


def test_verify_refusals(lib):
  def call(cost=ONE, draft=ONE, uniforms=ONE, batch=1, n_cv=1, n=4, pixels=9, drafts=1, labels=ONE, kept=ONE):
    return lib.mpl_verify_labels(1, cost, draft, None, uniforms, batch, n_cv, n, pixels, drafts, None, 1.0, None, 1.0, labels, kept,
                                 None)

  for name in ("cost", "draft", "uniforms", "labels", "kept"):
    _refused(lib, call(**{name: None}), b"null")
  for n in (0, 257):
    _refused(lib, call(n=n), b"n_disp")
  for name in ("batch", "n_cv", "pixels", "drafts"):
    _refused(lib, call(**{name: -1}), b"negative")
    assert call(**{name: 0}) == 0
  _refused(lib, call(batch=1 << 20, pixels=1 << 30), b"too many")
  _refused(lib, call(n=200, pixels=1 << 30), b"too many")


def test_verified_labels_of_the_plain_form():
  inf = math.inf
  verify = oracle.verify_label
  log = [0.0, math.log(2), math.log(4), inf]  # p: 4/7, 2/7, 1/7
  assert verify(log, 1, 0.28, 0.5) == (1, True) and verify(log, 1, 0.29, 0.79) == (0, False)
  assert verify(log, 1, 0.29, 0.81) == (2, False) and verify(log, 3, 0.0, 0.9) == (2, False)
  # nothing drafted: from p
  assert [verify(log, 9, 0.0, u)[0] for u in (0.5, 0.6, 0.9, 1.0)] == [0, 1, 2, 2]
  assert verify(log, 1, 0.0, 0.6, [0, inf, 0, 0]) == (1, False)
  # q 1/2 each of labels 1 and 2: what is left is label 0 alone
  assert verify(log, 1, 0.57, 0.99, [inf, 0, 0, inf]) == (1, True) and verify(log, 1, 0.58, 0.99, [inf, 0, 0, inf]) == (0, False)
  assert verify([inf, inf], 1, 0.0, 0.5) == (0, False) and verify([1, 0], 0, 0.5, 0.5, temperature=0.0) == (1, False)
  assert verify([0, 1], 0, 0.999, 0.5, [0, 1]) == (0, True)


def test_python_entry_points_refuse_cpu_tensors():
  from mplayers_amd import best_labels, distill_costs, verify_labels
  cost = torch.zeros(1, 1, 4, 2, 2)
  with pytest.raises(RuntimeError, match="GPU"):
    best_labels(cost, 2)
  with pytest.raises(RuntimeError, match="GPU"):
    distill_costs(cost, torch.zeros(1, 1, 2, 2, 2, dtype=torch.uint8), torch.zeros(1, 1, 2, 2, 2))
  with pytest.raises(RuntimeError, match="GPU"):
    verify_labels(cost, torch.zeros(1, 1, 2, 2, dtype=torch.uint8), torch.zeros(2, 1, 1, 2, 2))
