"""Labels drawn from the layers' costs (no counterpart in the reference, which takes the label of least cost only).

A layer's costs are energies: with a temperature they are a distribution over the labels of every pixel.
`sample_labels` draws from it through mpl_sample_labels.  The random numbers are the caller's.
"""
import torch

from . import _lib


def _parameter(name, value, batch, cost, dtype, low, high):
  """(pointer or None, number) of a parameter: a number, or a tensor with one per image."""
  if isinstance(value, torch.Tensor):
    if not value.is_cuda or value.device != cost.device:
      raise RuntimeError("sample_labels: %s must be on the device of the costs" % name)
    if value.dtype != dtype or value.shape != (batch,) or not value.is_contiguous():
      raise RuntimeError("sample_labels: %s must be a number or a contiguous %s tensor of one per image (%d)" %
                         (name, dtype, batch))
    return value.data_ptr(), 0
  if dtype == torch.int32 and (isinstance(value, bool) or not hasattr(value, "__index__")):
    raise RuntimeError("sample_labels: %s must be a whole number" % name)
  if not low <= value <= high:
    raise RuntimeError("sample_labels: %s must be in [%g, %g], got %r" % (name, low, high, value))
  return None, int(value) if dtype == torch.int32 else float(value)


def sample_labels(cost, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, labels_first=True):
  """Draws a label per pixel from softmax(-cost / temperature).

  cost       (batch, cv, labels, H, W) fp32 as MPModule returns it; with labels_first=False
             (batch, cv, H, W, labels) as the operators do.  +inf and NaN are no candidates.
  uniforms   (batch, cv, H, W), or (n, batch, cv, H, W) for n draws, fp32 in [0, 1)
  temperature, top_k, top_p, min_p
             numbers, or tensors of one per image on the device of the costs (fp32, top_k int32; these are not
             looked at).  top_k best labels (0: all), of these the best ones that weigh top_p together, of
             these the ones of min_p of the best one's weight.  temperature 0: the label of least cost.
  -> uint8 labels of the shape of uniforms.

  Equal costs order by label.  A pixel without candidates gets label 0."""
  for name, t in (("cost", cost), ("uniforms", uniforms)):
    if not isinstance(t, torch.Tensor):
      raise TypeError("sample_labels: %s must be a tensor" % name)
    if not t.is_cuda:
      raise RuntimeError("sample_labels: %s must be a GPU tensor" % name)
    if t.dtype != torch.float32:
      raise RuntimeError("sample_labels: %s must be float32, got %s" % (name, t.dtype))
    if not t.is_contiguous():
      raise RuntimeError("sample_labels: %s must be contiguous" % name)
  if uniforms.device != cost.device:
    raise RuntimeError("sample_labels: uniforms must be on the device of the costs")
  if cost.dim() != 5:
    raise RuntimeError("sample_labels: cost must be (batch, cv, labels, H, W) or (batch, cv, H, W, labels)")
  if labels_first:
    batch, cv, n, height, width = cost.shape
  else:
    batch, cv, height, width, n = cost.shape
  draws = uniforms.size(0) if uniforms.dim() == 5 else 1
  if tuple(uniforms.shape[-4:]) != (batch, cv, height, width) or uniforms.dim() not in (4, 5):
    raise RuntimeError("sample_labels: uniforms must be ([n,] %d, %d, %d, %d)" % (batch, cv, height, width))
  f32, inf = torch.float32, float("inf")
  ts, t = _parameter("temperature", temperature, batch, cost, f32, 0.0, inf)
  ks, k = _parameter("top_k", top_k, batch, cost, torch.int32, 0, 2 ** 31 - 1)
  ps, p = _parameter("top_p", top_p, batch, cost, f32, 0.0, 1.0)
  ms, m = _parameter("min_p", min_p, batch, cost, f32, 0.0, 1.0)
  labels = torch.empty(uniforms.shape, dtype=torch.uint8, device=cost.device)
  _lib.launch("mpl_sample_labels", cost, int(bool(labels_first)), cost.data_ptr(), uniforms.data_ptr(), batch, cv, n,
              height * width, draws, ts, t, ks, k, ps, p, ms, m, labels.data_ptr())
  return labels
