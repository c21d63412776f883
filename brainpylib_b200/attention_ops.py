"""Layers of language models on leaky states (no counterpart in brainpylib): the rows of a table that tokens name, queries and keys
normed and rotated head by head, and linear attention with a decay for each head, over packed sequences with their gradients and for
one new token per running sequence against a pool of states.

    embedding   y[t] = scale weight[ids[t]]
    rotation    n = x (mean x^2 + eps)^(-1/2) w;   (a, b) -> (a cos - b sin, a sin + b cos),  angle = position * frequency
    attention   S[t] = exp(log_decay) S[t - 1] + k[t] v[t]^T;   y[t] = scale S[t]^T q[t],  for every head

The state of a head is a matrix that leaks as a whole, where :func:`state_scan` has vectors whose elements leak by themselves.

Batches.  Rows are ``(tokens, heads, size)`` with ``indptr`` (int32, the ``n + 1`` ascending bounds of ``n`` packed sequences, any of
them empty; without it the rows are one sequence), or ``(batch, length, heads, size)``.  Rows outside all sequences are not read;
outputs and gradients are zero there.

Types.  Rows are float32, float16 or bfloat16, all the same; states are float32.  Sums, norms and states are held in 32 bits, angles
in 64, and every output is rounded once (:func:`decay_attention` says what its products on tensor cores lose on the way).  Rows and heads
may be strided (parts of one projection are read in place); what the kernels cannot read in place is copied.

The forms over whole sequences are differentiable, once (a second derivative, forward mode and torch.func transforms are refused);
the single-step form is for inference, writes its states in place and refuses operands that require a gradient.
"""
import math

import torch

from . import _lib
from .sequence_ops import MAX_STEP_ROWS, _TYPES, _batch, _done, _no_gradient, _on_gpu, _rows, _same_type, _shape, _tensor, _whole

__all__ = ['embedding', 'norm_rotate', 'decay_attention', 'decay_attention_step']

MAX_HEAD = 256          # elements of a head
MAX_HEADS = 65535


def _number(name, v):
  v = float(v)
  if math.isnan(v):
    raise ValueError(f'{name} must be a number. But we got {v}.')
  return v


# ---------------------------------------------------------------------------------------------------------
# rows of a table
# ---------------------------------------------------------------------------------------------------------
def embedding(ids, weight, *, scale=1.0):
  """The rows of a table that tokens name, scaled.

  Parameters
  ----------
  ids: tensor
    int32 or int64, of any shape.  A negative id marks padding: its row is 0.  An id beyond the table gives NaN.
  weight: tensor
    ``(vocabulary, width)``, float32, float16 or bfloat16.
  scale: float
    What the rows are multiplied by.

  Returns
  -------
  y : tensor
    ``ids.shape + (width,)`` of the type of ``weight``.

  The gradient of ``weight`` is the whole table: sums in 32 bits over the tokens of each row in their order, so the same call gives the
  same bits; padding and ids beyond the table count nowhere.  It takes 16 bytes of scratch memory a token, and up to
  ``width / 2`` for parts of sums.
  """
  done = (_lib.fast or _lib.load_fast()).embedding(ids, weight, scale)
  if done is not None:
    return done
  ids, weight = _tensor('ids', ids), _tensor('weight', weight)
  scale = _number('scale', scale)
  if ids.dtype not in (torch.int32, torch.int64):
    raise TypeError(f'ids must be int32 or int64. But we got {ids.dtype}.')
  if weight.dtype not in _TYPES:
    raise TypeError(f'embedding: only float32, float16 and bfloat16 are supported. But we got {weight.dtype}.')
  if weight.dim() != 2:
    raise ValueError(f'weight must be (vocabulary, width). But we got {tuple(weight.shape)}.')
  if ids.numel() >= 2 ** 31 or weight.size(0) >= 2 ** 31 or weight.size(1) >= 2 ** 28:
    raise ValueError(f'embedding: fewer than 2^31 tokens and rows, and 2^28 columns are supported. But we got {tuple(ids.shape)} '
                     f'and {tuple(weight.shape)}.')
  _on_gpu('embedding', ids, weight)
  return _done('embedding', _lib.fast.embedding(_whole(ids), _rows(weight), scale))


# ---------------------------------------------------------------------------------------------------------
# queries and keys
# ---------------------------------------------------------------------------------------------------------
def _heads(name, t):
  """``t`` as (tokens, heads, size) or (batch, length, heads, size)."""
  if t.dtype not in _TYPES:
    raise TypeError(f'{name}: only float32, float16 and bfloat16 are supported. But we got {t.dtype}.')
  if t.dim() not in (3, 4):
    raise ValueError(f'{name} must be (tokens, heads, size) or (batch, length, heads, size). But we got {tuple(t.shape)}.')
  if math.prod(t.shape[:-2]) >= 2 ** 31 or t.size(-2) > MAX_HEADS:
    raise ValueError(f'{name}: fewer than 2^31 tokens and at most {MAX_HEADS} heads are supported. But we got {tuple(t.shape)}.')


def norm_rotate(q, k, positions, frequencies, q_weight=None, k_weight=None, *, eps=1e-6, interleaved=False):
  """Queries and keys normed head by head and rotated by their positions.

  Parameters
  ----------
  q, k: tensor
    ``(tokens, heads, size)`` or ``(batch, length, heads, size)``; the numbers of heads may differ.  Heads have 2 to 256 elements, an
    even number.
  positions: tensor
    int32 or int64, ``(tokens,)`` or ``(batch, length)``.
  frequencies: tensor
    float32, at most ``size / 2``: the angle of pair ``i`` is ``position * frequencies[i]``, taken in 64 bits.  Elements behind the
    first ``2 * len(frequencies)`` are normed and not rotated.
  q_weight, k_weight: tensor, optional
    ``(size,)`` of the type of ``q`` or float32 (both the same): what the normed heads are multiplied by.
  eps: float
    Added to the mean of the squares.
  interleaved: bool
    Pairs are neighbouring elements; by default, element ``i`` of the first and of the second half of what is rotated.

  Returns
  -------
  q, k : tensor
    Like the operands.
  """
  done = (_lib.fast or _lib.load_fast()).norm_rotate(q, k, positions, frequencies, q_weight, k_weight, eps, interleaved)
  if done is not None:
    return done
  q, k, positions, frequencies = (_tensor(n, t) for n, t in (('q', q), ('k', k), ('positions', positions),
                                                             ('frequencies', frequencies)))
  q_weight, k_weight = _tensor('q_weight', q_weight, True), _tensor('k_weight', k_weight, True)
  eps = _number('eps', eps)
  _heads('q', q)
  _same_type('k', k, q.dtype)
  _heads('k', k)
  if k.shape[:-2] != q.shape[:-2] or k.size(-1) != q.size(-1):
    raise ValueError(f'q and k must have the same rows and elements of a head. But we got {tuple(q.shape)} and {tuple(k.shape)}.')
  size = q.size(-1)
  if not 2 <= size <= MAX_HEAD or size % 2:
    raise ValueError(f'heads must have 2..{MAX_HEAD} elements, an even number. But we got {size}.')
  if positions.dtype not in (torch.int32, torch.int64):
    raise TypeError(f'positions must be int32 or int64. But we got {positions.dtype}.')
  _shape('positions', positions, q.shape[:-2])
  _same_type('frequencies', frequencies, torch.float32)
  if frequencies.dim() != 1 or 2 * frequencies.numel() > size:
    raise ValueError(f'frequencies must be a vector of at most {size // 2}. But we got {tuple(frequencies.shape)}.')
  for name, w in (('q_weight', q_weight), ('k_weight', k_weight)):
    if w is not None and w.dtype not in (q.dtype, torch.float32):
      raise TypeError(f'{name} must be {q.dtype} or torch.float32. But we got {w.dtype}.')
    _shape(name, w, (size,))
  if q_weight is not None:
    _same_type('k_weight', k_weight, q_weight.dtype)
  if torch.is_grad_enabled() and frequencies.requires_grad:
    raise ValueError('norm_rotate has no gradient by its frequencies: detach them.')
  _on_gpu('norm_rotate', q, k, positions, frequencies, q_weight, k_weight)
  return _done('norm_rotate', _lib.fast.norm_rotate(_rows(q, 2), _rows(k, 2), _whole(positions), _whole(frequencies), _whole(q_weight),
                                                    _whole(k_weight), eps, bool(interleaved)))


# ---------------------------------------------------------------------------------------------------------
# linear attention
# ---------------------------------------------------------------------------------------------------------
def _attention_operands(op, q, k, v, log_decay, scale):
  _heads('q', q)
  for name, t in (('k', k), ('v', v)):
    _same_type(name, t, q.dtype)
    _heads(name, t)
    if t.shape[:-2] != q.shape[:-2]:
      raise ValueError(f'{name} must have the rows of q. But we got {tuple(t.shape)} for {tuple(q.shape)}.')
  if k.size(-1) != q.size(-1) or not 1 <= q.size(-1) <= MAX_HEAD or not 1 <= v.size(-1) <= MAX_HEAD:
    raise ValueError(f'{op}: heads of q and k must have the same 1..{MAX_HEAD} elements, those of v 1..{MAX_HEAD}. But we got '
                     f'{q.size(-1)}, {k.size(-1)} and {v.size(-1)}.')
  if v.size(-2) != k.size(-2) or k.size(-2) < 1 or q.size(-2) < 1 or q.size(-2) % k.size(-2) != 0:
    raise ValueError(f'{q.size(-2)} heads cannot share {k.size(-2)} heads of k and {v.size(-2)} of v.')
  _same_type('log_decay', log_decay, torch.float32)
  _shape('log_decay', log_decay, (q.size(-2),))
  if torch.is_grad_enabled() and log_decay.requires_grad:
    raise ValueError(f'{op} has no gradient by log_decay, the decays are constants of the layer: detach it.')
  return None if scale is None else _number('scale', scale)


def decay_attention(q, k, v, log_decay, *, scale=None, indptr=None, initial_state=None, return_state=False):
  """Linear attention with a decay for each head over whole sequences.

  Parameters
  ----------
  q, k, v: tensor
    ``(tokens, heads, size)`` or ``(batch, length, heads, size)``, 1 to 256 elements to a head (``k`` as many as ``q``).  ``k`` and ``v``
    may have fewer heads: ``heads / kv_heads`` neighbouring heads of ``q`` share one.
  log_decay: tensor
    float32 ``(heads,)``: the logarithm of what is left of a state after a token (0 keeps it, minus infinity forgets it).  A constant:
    it has no gradient.
  scale: float, optional
    What the outputs are multiplied by; by default ``size ** -0.5`` of ``q``.
  indptr: tensor, optional
    int32 bounds of packed sequences.
  initial_state: tensor, optional
    float32 ``(sequences, heads, size of k, size of v)``: the states that the sequences come with (default: zeros).
  return_state: bool
    Whether to return the states that the sequences leave, like ``initial_state``, as well.

  Returns
  -------
  y : tensor
    ``q.shape[:-1] + (size of v,)``; with ``return_state`` the pair ``(y, last_state)``.

  bfloat16 with heads of a multiple of 8 elements (of ``q`` and of ``v``) and rows at 16-byte boundaries runs on tensor cores, in chunks of
  64 tokens.  Products of tokens of a chunk and the state that a chunk reads go there as sums of two numbers of 16 bits, which lose 2^-17 of
  them; results are off by as much as those of 32-bit arithmetic, rounded once.  States keep 32 bits.  An element of ``v`` that is not
  finite makes its column NaN from its token on there, keys that are not finite do so to all columns and queries to their token, and
  infinite initial states may do so to theirs; elsewhere infinities stay what they are.  In no case does a token reach those in front of it.

  Memory.  Heads that share keys and values take ``4 * heads * size`` bytes a token in the backward pass, heads of more than 128 elements
  on tensor cores twice that in both passes; states between the segments that long sequences are cut into 4 bytes an element, for two
  blocks on every SM at most.
  """
  done = (_lib.fast or _lib.load_fast()).decay_attention(q, k, v, log_decay, scale, indptr, initial_state, return_state)
  if done is not None:
    return done
  q, k, v, log_decay = (_tensor(n, t) for n, t in (('q', q), ('k', k), ('v', v), ('log_decay', log_decay)))
  indptr, initial_state = _tensor('indptr', indptr, True), _tensor('initial_state', initial_state, True)
  scale = _attention_operands('decay_attention', q, k, v, log_decay, scale)
  n = _batch('decay_attention', q.select(-1, 0), indptr)
  _same_type('initial_state', initial_state, torch.float32)
  _shape('initial_state', initial_state, (n, q.size(-2), q.size(-1), v.size(-1)))
  _on_gpu('decay_attention', q, k, v, log_decay, indptr, initial_state)
  return _done('decay_attention', _lib.fast.decay_attention(_rows(q, 2), _rows(k, 2), _rows(v, 2), _whole(log_decay), scale, _whole(indptr),
                                                            _whole(initial_state), bool(return_state)))


def decay_attention_step(q, k, v, log_decay, state, *, scale=None, slots=None):
  """One more token of ``n`` running sequences; their states are updated in place.

  Operands as for :func:`decay_attention`, with one row per sequence: ``q`` ``(n, heads, size)``, ``k`` and ``v`` accordingly.  ``state`` is
  the float32 pool ``(pool, heads, size of k, size of v)``; row ``i`` continues state ``slots[i]`` (int32; without ``slots``, row ``i``
  state ``i`` and the pool has ``n``).  A negative slot marks a row of padding: its output is 0.  A row whose slot lies beyond the pool,
  or was taken by an earlier row of the same call, gets NaN and leaves the pool alone.  At most 65,535 rows; every row looks through
  the slots of those in front of it.  Returns ``y`` ``(n, heads, size of v)``."""
  done = (_lib.fast or _lib.load_fast()).decay_attention_step(q, k, v, log_decay, state, scale, slots)
  if done is not None:
    return done
  q, k, v, log_decay, state = (_tensor(n, t) for n, t in (('q', q), ('k', k), ('v', v), ('log_decay', log_decay), ('state', state)))
  slots = _tensor('slots', slots, True)
  scale = _attention_operands('decay_attention_step', q, k, v, log_decay, scale)
  if q.dim() != 3 or q.size(0) > MAX_STEP_ROWS:
    raise ValueError(f'q must be (rows, heads, size) with at most {MAX_STEP_ROWS} rows. But we got {tuple(q.shape)}.')
  if state.dim() != 4 or not state.is_contiguous():
    raise ValueError(f'state must be contiguous and of four dimensions: it is written in place. But we got {tuple(state.shape)} with '
                     f'strides {state.stride()}.')
  _same_type('state', state, torch.float32)
  _shape('state', state, (state.size(0), q.size(1), q.size(2), v.size(2)))
  if slots is None:
    if state.size(0) != q.size(0):
      raise ValueError(f'without slots there must be a state for every row. But we got {state.size(0)} states, {q.size(0)} rows.')
  else:
    _same_type('slots', slots, torch.int32)
    _shape('slots', slots, (q.size(0),))
  _on_gpu('decay_attention_step', q, k, v, log_decay, state, slots)
  _no_gradient('decay_attention_step', q, k, v, log_decay, state)
  return _done('decay_attention_step', _lib.fast.decay_attention_step(_rows(q, 2), _rows(k, 2), _rows(v, 2), _whole(log_decay), state, scale,
                                                                      _whole(slots)))
