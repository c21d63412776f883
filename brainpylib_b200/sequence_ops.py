"""Leaky units over whole sequences (no counterpart in brainpylib, whose operators know one time step): a short causal
convolution of the input and leaky states whose decay and input are selected by the data, for packed sequences with their
gradients, and for one new token per running sequence against a pool of states.

    conv   p[t, c] = bias[c] + sum_j weight[c, j] x[t - W + 1 + j, c];   y = p, or p / (1 + e^-p) (``'silu'``)
    scan   dt = delta + delta_bias, or log(1 + e^(delta + delta_bias));   h[t] = exp(dt A) h[t - 1] + dt x B[t]
           y = sum_n C[t, n] h[t, n] + D x;   y = y z / (1 + e^-z) where a gate z is given

Every channel is on its own (channels of a group share ``B`` and ``C``), as the neurons of ``lif_exp_step`` are: a whole run
of a leaky unit whose decay is the same at every step is the scan with a constant ``delta``.

Batches.  ``x`` is ``(tokens, channels)`` with ``indptr`` (int32, the ``n + 1`` ascending bounds of ``n`` packed sequences, any of
them empty; without it the rows are one sequence), or ``(batch, length, channels)``.  Rows outside all sequences are not read;
outputs and gradients are zero there.  ``initial_state`` is the state that each sequence comes with (default: zeros), and
``return_state=True`` also returns the one it leaves.

Types.  ``x``, ``delta``, ``z``, ``B``, ``C`` are float32, float16 or bfloat16, all the same; parameters of the scan and its
states are float32.  Exponents, states and sums are held in 32 bits and every output is rounded once.  Rows may be strided (a
part of a wider projection is read in place); what the kernels cannot read in place is copied.

The prompt forms are differentiable in every floating argument, once (a second derivative, forward mode and torch.func
transforms are refused); the single-step forms are for inference, write their states in place and refuse operands that
require a gradient.
"""
import math

import torch

from . import _lib
from ._checks import unwrap
from .errors import GPUOperatorNotFound

__all__ = ['short_conv', 'short_conv_step', 'state_scan', 'state_scan_step']

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_STATE = 128         # states of a channel
MAX_WIDTH = 8           # taps of the convolution
MAX_STEP_ROWS = 65535   # rows of a single-step call


def _tensor(name, t, optional=False):
  t = unwrap(t)
  if t is None and optional:
    return None
  if not isinstance(t, torch.Tensor):
    raise TypeError(f'{name} must be a tensor. But we got {type(t).__name__}.')
  return t


def _same_type(name, t, dtype):
  if t is not None and t.dtype != dtype:
    raise TypeError(f'{name} must be {dtype}. But we got {t.dtype}.')


def _shape(name, t, shape):
  if t is not None and tuple(t.shape) != tuple(shape):
    raise ValueError(f'{name} must have shape {tuple(shape)}. But we got {tuple(t.shape)}.')


def _on_gpu(op, *tensors):
  for t in tensors:
    if t is not None and t.device.type != 'cuda':
      raise GPUOperatorNotFound(f'{op} (operands are on {t.device}, a CUDA device is required)')
  devices = {t.device for t in tensors if t is not None}
  if len(devices) > 1:
    raise ValueError(f'{op}: operands are on several devices: {sorted(map(str, devices))}')


def _rows(t, inner=1):
  """``t`` with evenly spaced rows and contiguous channels: itself where it has them, else a copy."""
  if type(t) is not torch.Tensor and not isinstance(t, torch.nn.Parameter):
    t = t.as_subclass(torch.Tensor)
  lead = t.dim() - inner
  even = lead == 1 or t.size(0) <= 1 or t.size(1) == 1 or t.stride(0) == t.size(1) * t.stride(1)
  return t if even and (t.size(-1) <= 1 or t.stride(-1) == 1) else t.contiguous()


def _whole(t):
  if t is None:
    return None
  if type(t) is not torch.Tensor and not isinstance(t, torch.nn.Parameter):
    t = t.as_subclass(torch.Tensor)
  return t.contiguous()


def _batch(op, x, indptr):
  """Checks of ``x`` and ``indptr``; the number of sequences."""
  if x.dtype not in _TYPES:
    raise TypeError(f'{op}: only float32, float16 and bfloat16 are supported. But we got {x.dtype}.')
  if x.dim() not in (2, 3):
    raise ValueError(f'x must be (tokens, channels) or (batch, length, channels). But we got {tuple(x.shape)}.')
  if math.prod(x.shape[:-1]) >= 2 ** 31:
    raise ValueError(f'{op}: fewer than 2^31 tokens are supported. But we got {tuple(x.shape)}.')
  if indptr is None:
    if x.dim() == 3 and x.size(0) >= 2 ** 31:
      raise ValueError(f'{op}: fewer than 2^31 sequences are supported. But we got {x.size(0)}.')
    return x.size(0) if x.dim() == 3 else 1
  if x.dim() == 3:
    raise ValueError('indptr goes with packed sequences: x must be (tokens, channels).')
  if indptr.dtype != torch.int32:
    raise TypeError(f'indptr must be int32. But we got {indptr.dtype}.')
  if indptr.dim() != 1 or indptr.numel() < 1:
    raise ValueError(f'indptr must be a vector of n + 1 bounds. But we got {tuple(indptr.shape)}.')
  if indptr.numel() > 2 ** 31:
    raise ValueError(f'{op}: fewer than 2^31 sequences are supported. But we got {indptr.numel() - 1}.')
  return indptr.numel() - 1


def _no_gradient(op, *tensors):
  if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
    raise ValueError(f'{op} has no gradient and writes its state in place: call it under torch.no_grad(), or use the form '
                     f'over whole sequences.')


def _done(op, result):
  if result is None:
    raise RuntimeError(f'{op} runs on plain CUDA tensors only: not under torch.func transforms, forward-mode '
                       f'differentiation, dispatch modes or tracing.')
  return result


# ---------------------------------------------------------------------------------------------------------
# short causal convolution
# ---------------------------------------------------------------------------------------------------------
def _silu(activation):
  if activation not in (None, 'silu'):
    raise ValueError(f"activation must be None or 'silu'. But we got {activation!r}.")
  return activation == 'silu'


def _conv_operands(x, weight, bias):
  if weight.dim() != 2 or weight.size(0) != x.size(-1) or not 1 <= weight.size(1) <= MAX_WIDTH:
    raise ValueError(f'weight must be (channels, width) with {x.size(-1)} channels and 1..{MAX_WIDTH} taps. '
                     f'But we got {tuple(weight.shape)}.')
  if weight.dtype not in (x.dtype, torch.float32):
    raise TypeError(f'weight must be {x.dtype} or torch.float32. But we got {weight.dtype}.')
  _same_type('bias', bias, weight.dtype)
  _shape('bias', bias, (x.size(-1),))


def short_conv(x, weight, bias=None, *, activation=None, indptr=None, initial_state=None, return_state=False):
  """Causal convolution of every channel with its own few taps over whole sequences.

  Parameters
  ----------
  x: tensor
    ``(tokens, channels)`` or ``(batch, length, channels)``.
  weight: tensor
    ``(channels, width)``, 1 to 8 taps, the last one for the token itself; of the type of ``x`` or float32.
  bias: tensor, optional
    ``(channels,)`` of the type of ``weight``.
  activation: str, optional
    ``'silu'``: the result is multiplied by its own sigmoid.
  indptr: tensor, optional
    int32 bounds of packed sequences.
  initial_state: tensor, optional
    ``(sequences, channels, width - 1)`` of the type of ``x``: the inputs before each sequence, the latest last.
  return_state: bool
    Whether to return the last ``width - 1`` inputs of every sequence, like ``initial_state``, as well.

  Returns
  -------
  y : tensor
    Like ``x``; with ``return_state`` the pair ``(y, last_state)``.
  """
  silu = _silu(activation)
  done = (_lib.fast or _lib.load_fast()).short_conv(x, weight, bias, silu, indptr, initial_state, return_state)
  if done is not None:
    return done
  x, weight = _tensor('x', x), _tensor('weight', weight)
  bias, indptr, initial_state = (_tensor(n, t, True) for n, t in (('bias', bias), ('indptr', indptr),
                                                                  ('initial_state', initial_state)))
  n = _batch('short_conv', x, indptr)
  _conv_operands(x, weight, bias)
  _same_type('initial_state', initial_state, x.dtype)
  _shape('initial_state', initial_state, (n, x.size(-1), weight.size(1) - 1))
  _on_gpu('short_conv', x, weight, bias, indptr, initial_state)
  return _done('short_conv', _lib.fast.short_conv(_rows(x), _whole(weight), _whole(bias), silu, _whole(indptr),
                                                  _whole(initial_state), bool(return_state)))


def short_conv_step(x, state, weight, bias=None, *, activation=None, slots=None):
  """One more token of ``n`` running sequences; their last inputs are updated in place.

  ``x`` is ``(n, channels)``; ``state`` the pool ``(pool, channels, width - 1)`` of the type of ``x``; ``weight``, ``bias`` and
  ``activation`` as for :func:`short_conv`.  Row ``i`` continues ``slots[i]`` (int32; without ``slots``, row ``i`` state ``i`` and the
  pool has ``n``).  A negative slot marks a row of padding: its output is 0.  A row whose slot lies beyond the pool, or was taken
  by an earlier row of the same call, gets NaN and leaves the pool alone.  At most 65,535 rows; every row looks through the slots of
  those in front of it, which counts from some thousand rows on (1024 channels, 4 taps, 4000 rows: 33 us, 22 without slots; 65,535
  rows: 2.9 ms and 0.3).  Returns ``y`` ``(n, channels)``."""
  silu = _silu(activation)
  done = (_lib.fast or _lib.load_fast()).short_conv_step(x, weight, bias, silu, state, slots)
  if done is not None:
    return done
  x, state, weight = _tensor('x', x), _tensor('state', state), _tensor('weight', weight)
  bias, slots = _tensor('bias', bias, True), _tensor('slots', slots, True)
  _step_rows('short_conv_step', x, state, slots)
  _conv_operands(x, weight, bias)
  _same_type('state', state, x.dtype)
  _shape('state', state, (state.size(0), x.size(1), weight.size(1) - 1))
  _on_gpu('short_conv_step', x, state, weight, bias, slots)
  _no_gradient('short_conv_step', x, state, weight, bias)
  return _done('short_conv_step', _lib.fast.short_conv_step(_rows(x), _whole(weight), _whole(bias), silu, state, _whole(slots)))


# ---------------------------------------------------------------------------------------------------------
# leaky states
# ---------------------------------------------------------------------------------------------------------
def _scan_operands(op, x, delta, A, B, C, D, z, delta_bias, lead):
  """Checks of the operands that the scan and its single step share."""
  if A.dim() != 2 or A.size(0) != x.size(-1) or not 1 <= A.size(1) <= MAX_STATE:
    raise ValueError(f'A must be (channels, state) with {x.size(-1)} channels and 1..{MAX_STATE} states. '
                     f'But we got {tuple(A.shape)}.')
  channels, state = A.shape
  for name, t in (('delta', delta), ('z', z), ('B', B), ('C', C)):
    _same_type(name, t, x.dtype)
  for name, t in (('A', A), ('D', D), ('delta_bias', delta_bias)):
    _same_type(name, t, torch.float32)
  _shape('delta', delta, x.shape)
  _shape('z', z, x.shape)
  _shape('D', D, (channels,))
  _shape('delta_bias', delta_bias, (channels,))
  inner = B.dim() - lead
  if inner not in (1, 2) or B.shape[:lead] != x.shape[:lead] or B.size(-1) != state:
    raise ValueError(f'B must be {tuple(x.shape[:lead])} rows of (state,) or (groups, state). But we got {tuple(B.shape)}.')
  _shape('C', C, B.shape)
  if inner == 2 and (B.size(lead) < 1 or channels % B.size(lead) != 0):
    raise ValueError(f'{channels} channels cannot be shared out to {B.size(lead)} groups.')
  return inner


def state_scan(x, delta, A, B, C, D=None, *, z=None, delta_bias=None, delta_softplus=False, indptr=None, initial_state=None,
               return_state=False):
  """Leaky states with input-dependent decay over whole sequences.

  Parameters
  ----------
  x, delta: tensor
    ``(tokens, channels)`` or ``(batch, length, channels)``: input and time step of every token and channel.
  A: tensor
    float32 ``(channels, state)``, 1 to 128 states: the rate of every state (negative for a decay).
  B, C: tensor
    Input weights and read-out of every token: the rows of ``x`` by ``(state,)``, or by ``(groups, state)``, group ``g`` for the
    ``g``-th run of ``channels / groups`` channels.
  D: tensor, optional
    float32 ``(channels,)``: what of ``x`` is added to the read-out.
  z: tensor, optional
    Like ``x``: the gate; the read-out is multiplied by ``z / (1 + e^-z)``.
  delta_bias: tensor, optional
    float32 ``(channels,)``, added to ``delta``.
  delta_softplus: bool
    Whether the time step is ``log(1 + e^(delta + delta_bias))``.
  indptr: tensor, optional
    int32 bounds of packed sequences.
  initial_state: tensor, optional
    float32 ``(sequences, channels, state)``.
  return_state: bool
    Whether to return the states that the sequences leave, float32 ``(sequences, channels, state)``, as well.

  Returns
  -------
  y : tensor
    Like ``x``; with ``return_state`` the pair ``(y, last_state)``.

  Memory.  Where a gradient is wanted, the states in front of every 16 tokens are kept: ``channels * state / 4`` bytes a token.  The
  backward pass takes scratch memory: ``8 * groups * state`` bytes a token for every block of channels (64 of them for up to 8
  states, 32, 16, 8, 4 for up to 16, 32, 64, 128), as many blocks as the card holds at once, or up to 2 GiB.
  """
  done = (_lib.fast or _lib.load_fast()).state_scan(x, delta, A, B, C, D, z, delta_bias, delta_softplus, indptr,
                                                    initial_state, return_state)
  if done is not None:
    return done
  x, delta, A, B, C = (_tensor(n, t) for n, t in (('x', x), ('delta', delta), ('A', A), ('B', B), ('C', C)))
  D, z, delta_bias, indptr, initial_state = (_tensor(n, t, True) for n, t in (
    ('D', D), ('z', z), ('delta_bias', delta_bias), ('indptr', indptr), ('initial_state', initial_state)))
  n = _batch('state_scan', x, indptr)
  inner = _scan_operands('state_scan', x, delta, A, B, C, D, z, delta_bias, x.dim() - 1)
  _same_type('initial_state', initial_state, torch.float32)
  _shape('initial_state', initial_state, (n,) + tuple(A.shape))
  _on_gpu('state_scan', x, delta, A, B, C, D, z, delta_bias, indptr, initial_state)
  return _done('state_scan', _lib.fast.state_scan(
    _rows(x), _rows(delta), _whole(A), _rows(B, inner), _rows(C, inner), _whole(D), None if z is None else _rows(z),
    _whole(delta_bias), bool(delta_softplus), _whole(indptr), _whole(initial_state), bool(return_state)))


def state_scan_step(x, delta, A, B, C, state, D=None, *, z=None, delta_bias=None, delta_softplus=False, slots=None):
  """One more token of ``n`` running sequences; their states are updated in place.

  Operands as for :func:`state_scan`, with one row per sequence: ``x``, ``delta``, ``z`` ``(n, channels)``, ``B``, ``C``
  ``(n, state)`` or ``(n, groups, state)``.  ``state`` is the float32 pool ``(pool, channels, state)``; row ``i`` continues state
  ``slots[i]`` (int32; without ``slots``, row ``i`` state ``i`` and the pool has ``n``).  A negative slot marks a row of padding: its
  output is 0.  A row whose slot lies beyond the pool, or was taken by an earlier row of the same call, gets NaN and leaves the
  pool alone.  At most 65,535 rows; every row looks through the slots of those in front of it, which counts from some thousand rows
  on (1024 channels, 16 states, 4000 rows: 150 us, 121 without slots; 65,535 rows: 6.7 ms and 1.9).  Returns ``y`` ``(n, channels)``."""
  done = (_lib.fast or _lib.load_fast()).state_scan_step(x, delta, A, B, C, D, z, delta_bias, delta_softplus, state, slots)
  if done is not None:
    return done
  x, delta, A, B, C, state = (_tensor(n, t) for n, t in (('x', x), ('delta', delta), ('A', A), ('B', B), ('C', C),
                                                         ('state', state)))
  D, z, delta_bias, slots = (_tensor(n, t, True) for n, t in (('D', D), ('z', z), ('delta_bias', delta_bias),
                                                              ('slots', slots)))
  _step_rows('state_scan_step', x, state, slots)
  inner = _scan_operands('state_scan_step', x, delta, A, B, C, D, z, delta_bias, 1)
  _same_type('state', state, torch.float32)
  _shape('state', state, (state.size(0),) + tuple(A.shape))
  _on_gpu('state_scan_step', x, delta, A, B, C, D, z, delta_bias, state, slots)
  _no_gradient('state_scan_step', x, delta, A, B, C, D, z, delta_bias, state)
  return _done('state_scan_step', _lib.fast.state_scan_step(
    _rows(x), _rows(delta), _whole(A), _rows(B, inner), _rows(C, inner), _whole(D), None if z is None else _rows(z),
    _whole(delta_bias), bool(delta_softplus), state, _whole(slots)))


def _step_rows(op, x, state, slots):
  if x.dtype not in _TYPES:
    raise TypeError(f'{op}: only float32, float16 and bfloat16 are supported. But we got {x.dtype}.')
  if x.dim() != 2 or x.size(0) > MAX_STEP_ROWS:
    raise ValueError(f'x must be (rows, channels) with at most {MAX_STEP_ROWS} rows. But we got {tuple(x.shape)}.')
  if state.dim() != 3 or not state.is_contiguous():
    raise ValueError(f'state must be contiguous and of three dimensions: it is written in place. But we got '
                     f'{tuple(state.shape)} with strides {state.stride()}.')
  if slots is None:
    if state.size(0) != x.size(0):
      raise ValueError(f'without slots there must be a state for every row. But we got {state.size(0)} states, '
                       f'{x.size(0)} rows.')
    return
  if slots.dtype != torch.int32:
    raise TypeError(f'slots must be int32. But we got {slots.dtype}.')
  _shape('slots', slots, (x.size(0),))
