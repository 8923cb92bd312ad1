"""Label-context (pairwise potential) construction, after utils/label_context.py:6-90.

create_label_context(args, enable_seg=None, enable_symmetric=False) returns
(nn.Parameter, loc, diag_loc): a (n_classes, n_classes) table for segmentation (n_classes == 21)
or a (n_classes,) vector indexed by |label difference| otherwise; `loc` indexes the learnable
entries (upper triangle / k >= 1), `diag_loc` the pinned ones (diagonal / k == 0).

args fields read: n_classes, mpnet_smoothness_mode ('Potts' | 'potts' | 'TL' | 'TQ' | 'NPotts'),
mpnet_smoothness_train, mpnet_smoothness_trunct_value, mpnet_smoothness_trunct_loc,
mpnet_term_weight, enable_cuda.

Tables whose entries go by buckets of the label distance (no counterpart in the reference): label_buckets
says which distances share an entry, bucket_context makes the table of a layer of such entries, on the GPU
through mpl_bucket_context with mpl_bucket_sums as its gradient, and create_bucket_table the parameter.
"""
import argparse

import numpy as np
import torch
import torch.nn as nn

from . import _lib


def _gap_cost(mode, gap):
  if mode in ('Potts', 'potts'):
    return 1.0
  if mode == 'TL':
    return float(gap)
  if mode == 'TQ':
    return float(gap) ** 2
  raise ValueError(mode)


def create_label_context(args, enable_seg=None, enable_symmetric=False):
  n = args.n_classes
  mode = args.mpnet_smoothness_mode
  train = args.mpnet_smoothness_train
  trunc_value = args.mpnet_smoothness_trunct_value
  trunc_loc = args.mpnet_smoothness_trunct_loc
  if enable_seg is None:
    enable_seg = (n == 21)
  potts = mode in ('Potts', 'potts')

  if enable_seg:
    table = np.zeros((n, n), dtype=np.float32)
    if mode == 'NPotts':
      table[np.arange(n), np.arange(n)] = -1
    elif mode in ('TL', 'TQ') or (potts and train != 'sigmoid'):
      for i in range(n):
        for j in range(n):
          gap = abs(j - i) if enable_symmetric else j - i
          if gap > 0:
            table[i, j] = _gap_cost(mode, gap)
    if trunc_value >= 0:
      if trunc_loc >= 0:
        # The reference tests the `gap` left over from the last cell of the construction loops
        # (utils/label_context.py:45-47), which is 0: a location of 0 truncates everything, any
        # positive location truncates nothing.  Kept as is.
        if not (mode in ('TL', 'TQ') or (potts and train != 'sigmoid')):
          raise NameError("name 'gap' is not defined")
        if 0 >= trunc_loc:
          table = np.minimum(table, np.float32(trunc_value))
      else:
        table = np.minimum(table, np.float32(trunc_value))
  else:
    table = np.zeros((n,), dtype=np.float32)
    if mode == 'NPotts':
      table[0] = -1
    elif potts:
      if train != 'sigmoid':
        table[1:] = 1
    elif mode in ('TL', 'TQ'):
      table = np.array([_gap_cost(mode, d) for d in range(n)], dtype=np.float32)
    if trunc_value >= 0:
      lo = trunc_loc if trunc_loc >= 0 else 0
      table[lo:] = np.minimum(table[lo:], np.float32(trunc_value))

  label_context = torch.from_numpy(table) * args.mpnet_term_weight
  if getattr(args, 'enable_cuda', False) and (not label_context.is_cuda):
    label_context = label_context.cuda()
  enable_grad = train in {'softmax', 'sigmoid', 'on'}
  label_context = nn.Parameter(label_context, requires_grad=enable_grad)
  if label_context.dim() == 2:
    loc = np.triu_indices(n, k=1)
    diag_loc = [range(n), range(n)]
  else:
    loc = range(1, n)
    diag_loc = range(1)
  return label_context, loc, diag_loc


def label_buckets(n_classes, n_buckets, max_distance=None):
  """int32 CPU tensor `starts` of n_buckets + 1: bucket b is the label distances starts[b] <= k < starts[b + 1].
  The first half of the buckets hold one distance each, the others widen in equal ratios up to max_distance
  (default n_classes); the last one goes on to n_classes.  The borders are found in whole numbers."""
  if not (1 <= n_classes <= 256 and 1 <= n_buckets <= 256):
    raise ValueError('label_buckets: 1 to 256 labels and buckets, got %r and %r' % (n_classes, n_buckets))
  half = n_buckets // 2
  far = n_classes if max_distance is None else int(max_distance)
  if far < 1:
    raise ValueError('label_buckets: max_distance must be positive, got %r' % (max_distance,))
  far = max(far, half)
  logs = n_buckets - half
  starts = list(range(half)) + [half if half else 0]
  for j in range(1, logs):
    k = max(starts[-1], 1)
    # k >= half * (far / half) ** (j / logs)
    while k < n_classes and k ** logs * half ** j < half ** logs * far ** j:
      k += 1
    starts.append(k)
  return torch.tensor([min(k, n_classes) for k in starts] + [n_classes], dtype=torch.int32)


def bucket_context(table, starts, square=False, symmetric=True):
  """The pairwise table of a layer from one entry per bucket of label distances.

  table   (..., n_buckets) fp32; leading axes are tables of their own (one per direction, say)
  starts  as label_buckets returns it
  square  False: (..., n) indexed by |a - b|; True: (..., n, n), with symmetric=False zeros below the diagonal
  -> the table, with autograd; the gradient of an entry is the sum over the distances of its bucket."""
  if not isinstance(table, torch.Tensor) or not isinstance(starts, torch.Tensor):
    raise TypeError('bucket_context: table and starts must be tensors')
  if table.is_cuda:
    return _lib.autograd().bucket_context(table, starts, square, symmetric)
  if starts.is_cuda or starts.dtype != torch.int32 or starts.dim() != 1 or not starts.is_contiguous():
    raise RuntimeError('bucket_context: starts must be an int32 CPU tensor, as label_buckets returns it')
  if table.dtype != torch.float32:
    raise RuntimeError('bucket_context: table must be float32, got %s' % table.dtype)
  if table.dim() < 1 or starts.numel() < 2 or table.size(-1) != starts.numel() - 1:
    raise RuntimeError('bucket_context: table has %s entries for %d buckets' %
                       (table.size(-1) if table.dim() else 'no', starts.numel() - 1))
  if not 1 <= int(starts[-1]) <= 256:
    raise RuntimeError('bucket_context: 1 to 256 labels, got %d' % int(starts[-1]))
  if int(starts[0]) != 0 or bool((starts[1:] < starts[:-1]).any()):
    raise RuntimeError('bucket_context: the buckets must be in order, from distance 0')
  bucket = torch.repeat_interleave(torch.arange(starts.numel() - 1), (starts[1:] - starts[:-1]).long())
  if not square:
    return table[..., bucket]
  label = torch.arange(bucket.numel())
  context = table[..., bucket[(label[:, None] - label).abs()]]
  return context if symmetric else context.triu()


def create_bucket_table(args, n_buckets, max_distance=None):
  """(nn.Parameter (n_buckets,), loc, diag_loc, starts): create_label_context's vector at the first distance of
  each bucket, loc the buckets that hold a distance; the reads of args are its own.  The first entry is the pinned one, so a single bucket of all distances
  is refused."""
  starts = label_buckets(args.n_classes, n_buckets, max_distance)
  if starts[1] != 1:
    raise ValueError('create_bucket_table: the first bucket must hold distance 0 alone, two buckets at least, got %r' %
                     (n_buckets,))
  plain = argparse.Namespace(**vars(args))
  vector, _, _ = create_label_context(plain, enable_seg=False)
  first = starts[:-1].long().clamp(max=args.n_classes - 1).to(vector.device)
  # (what an empty bucket's entry holds reaches no label: it is not to weigh in a softmax over the others)
  loc = [b for b in range(1, n_buckets) if starts[b] < starts[b + 1]]
  return nn.Parameter(vector.detach()[first].clone(), requires_grad=vector.requires_grad), loc, range(1), starts
