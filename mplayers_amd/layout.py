"""Layout changes of the modules as HIP transposes with autograd support.

The reference's modules move the label axis with permute().contiguous()
(pytorch/MP_module.py:199,203,233, pytorch/MP_module_hard_soft.py); these functions return the same
contiguous tensors through mpl_transpose (a batched 2-D transpose bound by HBM), and their backward
passes are the opposite transposes.

`labels_last_dropout` is dropout of the unary costs within that change (no counterpart in the
reference, whose networks have their dropout in front of the layer): mpl_dropout_labels_last and
mpl_dropout_labels_first, which form the mask anew from a seed instead of storing it.
"""
import ctypes

import torch

from . import _lib


def _transpose(src, batch, rows, cols, out_shape):
  dst = src.new_empty(out_shape)
  if src.numel() == 0:
    return dst
  with torch.cuda.device(src.device):
    rc = _lib.load().mpl_transpose(ctypes.c_void_p(src.data_ptr()), ctypes.c_void_p(dst.data_ptr()),
                                   int(batch), int(rows), int(cols),
                                   ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
  _lib.check(rc, "transpose")
  return dst


def _usable(t):
  return t.is_cuda and t.dtype == torch.float32 and t.dim() == 5


class _LabelsLast(torch.autograd.Function):
  """(batch, cv, labels, H, W) -> (batch, cv, H, W, labels), contiguous."""

  @staticmethod
  def forward(ctx, x):
    b, cv, n, h, w = x.shape
    return _transpose(x.contiguous(), b * cv, n, h * w, (b, cv, h, w, n))

  @staticmethod
  def backward(ctx, grad):
    b, cv, h, w, n = grad.shape
    return _transpose(grad.contiguous(), b * cv, h * w, n, (b, cv, n, h, w))


class _LabelsFirst(torch.autograd.Function):
  """(batch, cv, H, W, labels) -> (batch, cv, labels, H, W), contiguous."""

  @staticmethod
  def forward(ctx, x):
    b, cv, h, w, n = x.shape
    return _transpose(x.contiguous(), b * cv, h * w, n, (b, cv, n, h, w))

  @staticmethod
  def backward(ctx, grad):
    b, cv, n, h, w = grad.shape
    return _transpose(grad.contiguous(), b * cv, n, h * w, (b, cv, h, w, n))


def gradient_labels_last(grad):
  """The gradient of a (batch, cv, labels, H, W) result as (batch, cv, H, W, labels), contiguous."""
  return _LabelsFirst.backward(None, grad)


def labels_last(x):
  """x.permute(0, 1, 3, 4, 2).contiguous() for a (batch, cv, labels, H, W) tensor."""
  if _usable(x):
    return _LabelsLast.apply(x)
  return x.permute(0, 1, 3, 4, 2).contiguous()


def labels_first(x):
  """x.permute(0, 1, 4, 2, 3).contiguous() for a (batch, cv, H, W, labels) tensor."""
  if _usable(x):
    return _LabelsFirst.apply(x)
  return x.permute(0, 1, 4, 2, 3).contiguous()


_DROPOUT_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # MPL_F32, MPL_F16, MPL_BF16
_DROPOUT_SHARES = {"element": 0, "pixel": 1, "label": 2}  # MPL_DROPOUT_*


def _dropout_last(x, state, p, share):
  b, cv, n, h, w = x.shape
  x = x.contiguous()
  out = torch.empty((b, cv, h, w, n), dtype=torch.float32, device=x.device)
  if out.numel():
    _lib.launch("mpl_dropout_labels_last", x, _DROPOUT_TYPES[x.dtype], share, p, state.data_ptr(), x.data_ptr(),
                out.data_ptr(), b * cv, n, h * w)
  return out


def _dropout_first(grad, state, p, share, dtype):
  b, cv, h, w, n = grad.shape
  grad = grad.contiguous()
  out = torch.empty((b, cv, n, h, w), dtype=dtype, device=grad.device)
  if out.numel():
    _lib.launch("mpl_dropout_labels_first", grad, _DROPOUT_TYPES[dtype], share, p, state.data_ptr(), grad.data_ptr(),
                out.data_ptr(), b * cv, n, h * w)
  return out


class _DropoutLast(torch.autograd.Function):
  """(batch, cv, labels, H, W) -> (batch, cv, H, W, labels) fp32 with dropout."""

  @staticmethod
  def forward(ctx, x, state, p, share):
    ctx.save_for_backward(state)
    ctx.rest = (p, share, x.dtype)
    return _dropout_last(x, state, p, share)

  @staticmethod
  def backward(ctx, grad):
    call = _DropoutFirst.apply if torch.is_grad_enabled() else _dropout_first
    return call(grad, ctx.saved_tensors[0], *ctx.rest), None, None, None


class _DropoutFirst(torch.autograd.Function):
  """The gradient of _DropoutLast, back in the type of its input; linear, so its gradient is _DropoutLast."""

  @staticmethod
  def forward(ctx, grad, state, p, share, dtype):
    ctx.save_for_backward(state)
    ctx.rest = (p, share)
    return _dropout_first(grad, state, p, share, dtype)

  @staticmethod
  def backward(ctx, grad):
    return _DropoutLast.apply(grad, ctx.saved_tensors[0], *ctx.rest), None, None, None, None


def labels_last_dropout(x, p, state, share="element"):
  """labels_last(dropout(x)) in one pass over the costs, in fp32.

  x      (batch, cv, labels, H, W) fp32, fp16 or bf16 on the GPU, at most 256 labels
  p      rate in [0, 1]; what stays is multiplied by 1 / (1 - p)
  state  int64 tensor of two on the device of x, (seed, offset): the mask follows from it and is formed
         again in the backward pass, so it must not be written to before that.  A captured call reads it
         at every replay.
  share  'element': every entry by itself; 'pixel': all labels of a pixel (its neighbours' messages then
         decide); 'label': all pixels of a label's plane"""
  if not isinstance(x, torch.Tensor) or not isinstance(state, torch.Tensor):
    raise TypeError("labels_last_dropout: x and state must be tensors")
  if not x.is_cuda or x.dim() != 5:
    raise RuntimeError("labels_last_dropout: x must be a (batch, cv, labels, H, W) GPU tensor")
  if x.dtype not in _DROPOUT_TYPES:
    raise RuntimeError("labels_last_dropout: x must be float32, float16 or bfloat16, got %s" % x.dtype)
  if not 1 <= x.size(2) <= 256:
    raise RuntimeError("labels_last_dropout: 1 to 256 labels, got %d" % x.size(2))
  if state.device != x.device or state.dtype != torch.int64 or state.shape != (2,) or not state.is_contiguous():
    raise RuntimeError("labels_last_dropout: state must be two int64 numbers (seed, offset) on the device of x")
  if not 0 <= p <= 1:
    raise RuntimeError("labels_last_dropout: p must be in [0, 1], got %r" % (p,))
  if share not in _DROPOUT_SHARES:
    raise RuntimeError("labels_last_dropout: share must be 'element', 'pixel' or 'label', got %r" % (share,))
  call = _DropoutLast.apply if x.requires_grad and torch.is_grad_enabled() else _dropout_last
  return call(x, state, float(p), _DROPOUT_SHARES[share])
