"""Labels drawn from the layers' costs (no counterpart in the reference, which takes the label of least cost only).

A layer's costs are energies: with a temperature they are a distribution over the labels of every pixel.
`sample_labels` draws from it through mpl_sample_labels.  The random numbers are the caller's.
"""
from . import _lib


def sample_labels(cost, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, labels_first=True):
  """Draws a label per pixel from softmax(-cost / temperature).

  cost       (batch, cv, labels, H, W) fp32 as MPModule returns it; with labels_first=False
             (batch, cv, H, W, labels) as the operators do.  +inf and NaN are no candidates.
  uniforms   (batch, cv, H, W), or (n, batch, cv, H, W) for n draws, fp32 in [0, 1)
  temperature, top_k, top_p, min_p
             numbers, or tensors of one per image on the device of the costs (fp32, top_k int32; these are not
             looked at).  top_k best labels (0: all), of these the best ones that weigh top_p together, of
             these the ones of min_p of the best one's weight (1: those of the best cost, at any temperature).
             temperature 0: the label of least cost; infinite: all candidates weigh the same.
  -> uint8 labels of the shape of uniforms.

  Equal costs order by label.  A pixel without candidates gets label 0."""
  return _lib.autograd().sample_labels(cost, uniforms, temperature, top_k, top_p, min_p, labels_first)
