"""Plain statements in 64 bits of the layers of language models, and bounds for what a computation in 32 bits may be off.

As in ``sequence_reference``, every function also runs with ``absolute=True``: the same sums over the absolute values of all terms.
A computation that makes a relative error of 2^-24 per operation is off by at most the number of operations that a term passes
through, times 2^-24, times that majorant."""
import math
from fractions import Fraction

import torch

from sequence_reference import U, check, half_step          # noqa: F401  (the tests use them from here)


def embedding(ids, weight, scale):
  """``ids`` int64 of any shape, ``weight`` float64."""
  good = (ids >= 0) & (ids < weight.shape[0])
  y = weight[ids.clamp(0, max(weight.shape[0] - 1, 0))] * scale if weight.shape[0] else weight.new_zeros(*ids.shape, weight.shape[1])
  y = torch.where(good[..., None], y, float('nan'))
  return torch.where((ids < 0)[..., None], 0.0, y)


def embedding_gradient(ids, dy, vocabulary, scale, absolute=False):
  ids, dy = ids.reshape(-1), dy.reshape(-1, dy.shape[-1])
  good = (ids >= 0) & (ids < vocabulary)
  d = dy.abs() if absolute else dy
  return torch.zeros(vocabulary, dy.shape[1], dtype=torch.float64).index_add_(0, ids[good], d[good]) * scale


def turn(x, angle, interleaved):
  """The leading parts of the last dimension rotated: ``angle`` is (..., pairs)."""
  n = angle.shape[-1]
  c, s = angle.cos(), angle.sin()
  y = x.clone()
  a = slice(0, 2 * n, 2) if interleaved else slice(0, n)
  b = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
  y[..., a] = x[..., a] * c - x[..., b] * s
  y[..., b] = x[..., a] * s + x[..., b] * c
  return y


PI = Fraction('3.14159265358979323846264338327950288419716939937510582097494459230781640628620899')


def angles(positions, frequencies):
  """Positions times float32 numbers, exactly, without whole turns: (rows, 1, pairs) in float64."""
  turn_of = lambda p, f: float((p * f / (2 * PI) + Fraction(1, 2)) % 1 - Fraction(1, 2))       # noqa: E731
  f = [Fraction(float(v)) for v in frequencies]
  rows = [[turn_of(int(p), v) for v in f] for p in positions]
  return 2 * math.pi * torch.tensor(rows, dtype=torch.float64).reshape(len(positions), 1, len(f))


def rotation(x, angle, weight, eps, interleaved):
  """``x`` (rows, heads, size) and so on in float64; differentiable."""
  r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
  n = x * r if weight is None else x * r * weight
  return turn(n, angle, interleaved)


def attention(q, k, v, log_decay, scale, bounds, initial, dy=None, d_last=None, absolute=False):
  """``q`` (tokens, heads, size) and so on in float64, ``bounds`` pairs (begin, end).  Returns a dict of ``y``, ``last`` and, with
  ``dy`` or ``d_last``, the gradients."""
  if absolute:
    q, k, v, initial, dy, d_last = (None if t is None else t.abs() for t in (q, k, v, initial, dy, d_last))
    scale = abs(scale)
  heads, group = q.shape[1], q.shape[1] // k.shape[1]
  kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
  size = (len(bounds), heads, q.shape[2], v.shape[2])
  y, last = q.new_zeros(q.shape[0], heads, v.shape[2]), q.new_zeros(size)
  gradients = dy is not None or d_last is not None
  dy = torch.zeros_like(y) if dy is None else dy
  dq, dk, dv, d_initial = torch.zeros_like(q), torch.zeros_like(kk), torch.zeros_like(vv), q.new_zeros(size)
  for s, (b, e) in enumerate(bounds):
    n = torch.arange(e - b, dtype=torch.float64)
    first = initial[s] if initial is not None else q.new_zeros(size[1:])
    end = d_last[s] if d_last is not None else q.new_zeros(size[1:])
    for h in range(heads):
      a = math.exp(float(log_decay[h]))
      power = lambda m: torch.where(m == 0, 1.0, a ** m)           # noqa: E731
      counts = torch.tril(power((n[:, None] - n).clamp(min=0))) * scale
      enter, leave = power(n + 1)[:, None], power(e - b - 1 - n)[:, None]
      Q, K, V, G = q[b:e, h], kk[b:e, h], vv[b:e, h], dy[b:e, h]
      whole = power(torch.tensor(float(e - b), dtype=torch.float64))
      y[b:e, h] = ((Q @ K.t()) * counts) @ V + scale * enter * (Q @ first[h])
      last[s, h] = (K * leave).t() @ V + whole * first[h]
      if gradients:
        scores, d_scores = (Q @ K.t()) * counts, (G @ V.t()) * counts
        dq[b:e, h] = d_scores @ K + scale * enter * (G @ first[h].t())
        dk[b:e, h] = d_scores.t() @ Q + leave * (V @ end[h].t())
        dv[b:e, h] = scores.t() @ G + leave * (K @ end[h])
        d_initial[s, h] = scale * (Q * enter).t() @ G + whole * end[h]
  out = dict(y=y, last=last)
  if gradients:
    out.update(d_q=dq, d_k=dk.unflatten(1, (k.shape[1], group)).sum(2), d_v=dv.unflatten(1, (k.shape[1], group)).sum(2),
               d_initial=d_initial)
  return out
