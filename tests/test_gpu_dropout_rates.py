"""Modules whose dropout rate changes from step to step."""
import pytest
import torch

from tests.test_capi_host import _args

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mode", ["TRWP", "ISGMR"])
def test_a_rate_that_is_scheduled_to_0(gpu, mode, dtype):
  """Steps at 0.4 and at 0 by the same module: at 0 the costs are those without dropout, and the gradient is theirs in
  the network's type."""
  from mplayers_amd import MPModule
  fields = dict(mpnet_mrf_mode=mode, n_classes=12, mpnet_max_iter=2, mpnet_smoothness_mode="TL", mpnet_smoothness_train="on",
                mpnet_term_weight=0.3, mpnet_smoothness_trunct_value=4, enable_cuda=True)
  module = MPModule(_args(mpnet_unary_dropout=0.4, **fields), enable_create_label_context=True).cuda().train()
  plain = MPModule(_args(**fields), enable_create_label_context=True).cuda().train()
  x = torch.randn(2, 1, 12, 6, 7, device="cuda").to(dtype).requires_grad_(True)
  whole = x.detach().float().requires_grad_(True)
  dcost = torch.randn(2, 1, 12, 6, 7, device="cuda")
  want = plain(whole)[0]
  (dwhole,) = torch.autograd.grad(want, whole, dcost)
  for rate in (0.4, 0.0, 0.1, 0):
    module.args.mpnet_unary_dropout = rate
    cost = module(x)[0]
    (dx,) = torch.autograd.grad(cost, x, dcost)
    assert dx.dtype == dtype
    if rate:
      assert not torch.equal(cost, want)
    else:
      assert torch.equal(cost, want) and torch.equal(dx, dwhole.to(dtype))
