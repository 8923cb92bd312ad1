"""Layers that learn from another layer's costs (no counterpart in the reference, whose layers learn from labels only).

A teacher (more iterations, more directions, a larger network) is run once and the labels of its least costs are kept:
`best_labels`, through mpl_best_labels.  `distill_costs` is the divergence of a student's costs from them, through
mpl_distill_costs and mpl_distill_costs_grad.
"""
import torch

from . import _lib


def best_labels(cost, k, temperature=1.0, labels_first=True, dtype=torch.float32):
  """The k labels of least cost of every pixel, in order of cost, equal costs in order of label.

  cost   (batch, cv, labels, H, W) fp32, fp16 or bf16, as MPModule returns it; with labels_first=False
         (batch, cv, H, W, labels) as the operators do.  +inf and NaN are no candidates.
  -> labels  uint8, (batch, cv, k, H, W) or (batch, cv, H, W, k)
     costs   of `dtype`, relative to the least cost of the pixel (so the first is 0); +inf, and label 0, where there is no
             candidate left, or none near enough for `dtype` (65504 in fp16)
     rest    (batch, cv, H, W) fp32, what the other candidates weigh together (all that the list has not got), as a cost: -T log(sum of exp(-cost / T)) with
             the temperature T, which is for this alone; +inf where there are none

  No gradients."""
  return _lib.autograd().best_labels(cost, k, temperature, labels_first, dtype)


def distill_costs(cost, labels, costs, rest=None, temperature=1.0, labels_first=True):
  """The divergence of softmax(-cost / T) from a teacher's, for every pixel, with a gradient for cost.

  cost     the student's, as best_labels takes it
  labels, costs
           a list for every pixel in the same layout, uint8 and fp32, fp16 or bf16 (as best_labels returns it, or of one's
           own: 1 to 256 entries in any order); an entry of cost +inf, or of a label that there is none of, is not there
  rest     (batch, cv, H, W) fp32, the cost of all labels that the list does not name, or None: those have no part in the
           teacher's distribution
  temperature
           T; the gradient has a factor 1 / T (times T twice where it is to have the size of one at T = 1)
  -> (batch, cv, H, W) fp32: sum of p (log p - log q), p the teacher's distribution over its entries (and the rest), q the
     student's of the same classes.

  A label of cost +inf is none of the student's: the teacher's entries of it are left out.  A pixel without entries has loss 0
  and no gradient.  NaN goes through to the loss and the gradient of its pixel."""
  return _lib.autograd().distill_costs(cost, labels, costs, rest, temperature, labels_first)
