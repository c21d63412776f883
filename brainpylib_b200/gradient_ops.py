"""The norm over all gradients of a training step, and clipping (no counterpart in brainpylib): what back-propagation through
many time steps needs between the gradients (of CSR weights, of the operators over whole sequences, of anything else) and the
update.

    N = (sum of g^2 over all elements of all tensors)^(1/2), or max |g|;   g = g * min(1, max_norm / (N + 1e-6))

Two launches for up to a thousand tensors, of any mix of float16, bfloat16, float32 and float64; nothing is copied to or read
from the host, so a call can be captured into a CUDA graph.  The squares of 16 bytes of float32, float16 or bfloat16 are added in 32
bits (their sum is off by 8 * 2^-24 of itself at most), everything else in 64 bits, in an order that depends on the sizes alone: a
norm of float64 tensors has 64 bits throughout, one of several types what its parts have.  Products are rounded once.  A norm that
is no finite number makes the factor what the formula says: 0 for an infinite norm (infinite elements become NaN), NaN for NaN.

Neither has a gradient itself: operands that require one are refused where gradients are recorded (a norm without one in a loss
would train on nothing).
"""
import torch

from . import _lib
from ._checks import unwrap
from .errors import GPUOperatorNotFound

__all__ = ['gradient_norm', 'clip_gradients']

_TYPES = (torch.float32, torch.float16, torch.bfloat16, torch.float64)


def _norm_kind(norm_type):
  kind = float(norm_type)
  if kind not in (2.0, float('inf')):
    raise ValueError(f'norm_type must be 2 or infinity. But we got {norm_type!r}.')
  return 2 if kind == 2.0 else 0


def _list(name, tensors):
  tensors = [unwrap(t) for t in ([tensors] if isinstance(tensors, torch.Tensor) else tensors)]
  for t in tensors:
    if t is not None and not isinstance(t, torch.Tensor):
      raise TypeError(f'{name} must be tensors. But we got {type(t).__name__}.')
  return tensors


def _no_gradient(op, tensors):
  if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
    what = 'has no gradient' if op == 'gradient_norm' else 'writes in place and has no gradient'
    raise ValueError(f'{op} {what}: call it under torch.no_grad(), or on tensors that require none.')


def _checked(op, tensors):
  for t in tensors:
    if t.layout != torch.strided:
      raise TypeError(f'{op}: only dense tensors are supported. But we got {t.layout}.')
    if t.dtype not in _TYPES:
      raise TypeError(f'{op}: only float32, float16, bfloat16 and float64 are supported. But we got {t.dtype}.')
    if t.device.type != 'cuda':
      raise GPUOperatorNotFound(f'{op} (operands are on {t.device}, a CUDA device is required)')
    if t.device != tensors[0].device:
      raise ValueError(f'{op}: operands are on several devices: {tensors[0].device}, {t.device}')


def _plain(t):
  return t if type(t) is torch.Tensor else t.detach().as_subclass(torch.Tensor)


def _dense(t):
  """Whether the elements fill a run of memory, in whatever order of the dimensions."""
  return t.permute(sorted(range(t.dim()), key=lambda i: -t.stride(i))).is_contiguous()


def _run(op, grads, out, max_norm, kind):
  norm = _lib.fast.clip_gradients(grads, out, max_norm, kind)
  if norm is None:
    raise RuntimeError(f'{op} runs on plain CUDA tensors only: not under torch.func transforms, forward-mode differentiation, '
                       f'dispatch modes or tracing.')
  return norm


def gradient_norm(grads, *, norm_type=2.0):
  """The norm over all elements of all tensors.

  Parameters
  ----------
  grads: tensors
    The gradients (or one); ``None`` entries are left out.
  norm_type: float
    2, or infinity for the largest magnitude.

  Returns
  -------
  norm : tensor
    Of no dimension, on the device of the gradients: float32, or float64 if one of them is.
  """
  kind = _norm_kind(norm_type)
  norm = (_lib.fast or _lib.load_fast()).clip_gradients(grads, None, 0.0, kind)
  if norm is not None:
    return norm
  every = _list('grads', grads)
  _no_gradient('gradient_norm', every)
  grads = [_plain(t) for t in every if t is not None]
  if not grads:
    return torch.zeros((), device='cuda' if torch.cuda.is_available() else 'cpu')
  _checked('gradient_norm', grads)
  # (memory order does not matter to a norm; what has gaps, or an element at several places, is copied first)
  return _run('gradient_norm', [t if _dense(t) else t.contiguous() for t in grads],
              None, 0.0, kind)


def clip_gradients(grads, max_norm, *, norm_type=2.0, out=None):
  """Scales all tensors by one factor so that their common norm is at most ``max_norm``.

  Parameters
  ----------
  grads: tensors
    The gradients (or one); ``None`` entries are left out.
  max_norm: float
    Zero or more.
  norm_type: float
    2, or infinity for the largest magnitude.
  out: tensors, optional
    Where to put the results: one like each of ``grads`` (``None`` where it is).  By default the gradients are overwritten, and not
    touched where their norm is small enough.  Results must not share memory with one another or with other gradients.

  Returns
  -------
  norm : tensor
    The norm before clipping, as :func:`gradient_norm` returns it.
  """
  kind = _norm_kind(norm_type)
  max_norm = float(max_norm)
  if not max_norm >= 0.0:
    raise ValueError(f'max_norm must be zero or more. But we got {max_norm}.')
  norm = (_lib.fast or _lib.load_fast()).clip_gradients(grads, grads if out is None else out, max_norm, kind)
  if norm is not None:
    return norm
  every = _list('grads', grads)
  targets = every if out is None else _list('out', out)
  if len(every) != len(targets) or any((g is None) != (o is None) for g, o in zip(every, targets)):
    raise ValueError('out must have one tensor for each gradient.')
  _no_gradient('clip_gradients', every + targets)
  grads = [_plain(t) for t in every if t is not None]
  if not grads:
    return torch.zeros((), device='cuda' if torch.cuda.is_available() else 'cpu')
  _checked('clip_gradients', [t for t in targets if t is not None])
  _checked('clip_gradients', grads)
  targets = grads if out is None else [_plain(t) for t in targets if t is not None]
  reads, writes, back = [], [], []
  for g, o in zip(grads, targets):
    if o.shape != g.shape or o.dtype != g.dtype or o.device != g.device:
      raise ValueError(f'out must be like the gradients: {tuple(o.shape)} {o.dtype} on {o.device} for {tuple(g.shape)} {g.dtype} '
                       f'on {g.device}.')
    if torch._debug_has_internal_overlap(o) == 1:
      raise ValueError('clip_gradients: a result holds several elements at one place.')
    if _dense(g) and _dense(o) and o.stride() == g.stride():
      reads.append(g)
      writes.append(o)
    else:                                     # gaps, or another order than the gradient's: by way of a copy
      copy = g.clone(memory_format=torch.contiguous_format)
      reads.append(copy)
      writes.append(copy)
      back.append((o, copy))
  norm = _run('clip_gradients', reads, writes, max_norm, kind)
  for o, c in back:
    o.copy_(c)
  return norm
