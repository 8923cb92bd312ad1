"""Labels drawn from the layers' costs (no counterpart in the reference, which takes the label of least cost only).

A layer's costs are energies: with a temperature they are a distribution over the labels of every pixel.
`sample_labels` draws from it through mpl_sample_labels.  `verify_labels` takes labels that were drawn from other costs and makes
them labels of these, keeping as many as that allows, through mpl_verify_labels.  The random numbers are the caller's.
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


def verify_labels(cost, draft, uniforms, draft_cost=None, temperature=1.0, draft_temperature=None, labels_first=True):
  """Labels drafted from other costs, kept or drawn anew so that they are distributed as softmax(-cost / temperature).

  Labels of a layer with fewer iterations, say, or of the last frame: what still fits the costs stays, so that
  labellings change no more than the costs ask for.

  cost        as sample_labels takes it
  draft       (batch, cv, H, W) uint8, or (n, batch, cv, H, W) for n labellings; a number that is no label: nothing drafted
  uniforms    (2,) + draft's size, fp32 in [0, 1): for keeping a label, and for drawing another one
  draft_cost  like cost, the costs whose labels the draft has, drawn at draft_temperature without filters; None: the draft is
              certain of its labels (those of least cost, or given ones)
  temperature, draft_temperature
              numbers, or fp32 tensors of one per image on the device of the costs, as in sample_labels; draft_temperature None:
              as temperature
  -> labels (uint8) and kept (bool), of draft's size.  With p and q the distributions of the target and the draft (q 1 at the
     drafted label without draft_cost), a label d stays where uniforms[0] * q[d] < p[d]; else one is drawn from max(p - q, 0),
     or from p where nothing is left or nothing was drafted (there is no label d, or q[d] is 0).

  A pixel without candidates gets label 0, not kept."""
  return _lib.autograd().verify_labels(cost, draft, uniforms, draft_cost, temperature, draft_temperature, labels_first)
