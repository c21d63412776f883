"""Plain statements in 64 bits of the operators over whole sequences, and bounds for what a computation in 32 bits may be off.

Every function also runs with ``absolute=True``: the same sums of products over the absolute values of all terms, decays as they
are.  A computation that makes a relative error of u = 2^-24 per operation is off by at most the number of operations that a
term passes through, times u, times that majorant (Higham's running bound).  A term of the scan passes through every token of
its sequence once (state: product, sum, decay with its exponent: 8 roundings, the exponential counted as 4), and through a
fixed number of further operations."""
import torch

U = 2.0 ** -24


def sequences_of(n_rows, indptr, batch):
  """(begin, end) of every sequence."""
  if indptr is not None:
    p = [int(v) for v in indptr]
    return list(zip(p[:-1], p[1:]))
  length = n_rows // batch if batch else 0
  return [(i * length, (i + 1) * length) for i in range(batch)]


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


def _abs(absolute, *ts):
  return [t if t is None or not absolute else t.abs() for t in ts]


def sigmoid(v):
  return 1 / (1 + torch.exp(-v))


def conv(x, weight, bias, bounds, initial, silu, dy=None, d_last=None, absolute=False):
  """``x`` (tokens, channels) float64 and so on; returns a dict of ``y``, ``last`` and, with ``dy``, the gradients."""
  T, c = x.shape
  w = weight.shape[1]
  out = {'y': torch.zeros_like(x), 'last': x.new_zeros(len(bounds), c, w - 1)}
  if dy is not None:
    out.update(d_x=torch.zeros_like(x), d_weight=torch.zeros_like(weight), d_bias=x.new_zeros(c),
               d_initial=x.new_zeros(len(bounds), c, w - 1))
  for s, (b, e) in enumerate(bounds):
    first = initial[s].t() if initial is not None else x.new_zeros(w - 1, c)
    rows = torch.cat([first, x[b:e]])
    p = sum(rows[j:j + e - b] * weight[:, j] for j in range(w)) + (bias if bias is not None else 0)
    a_rows, a_weight, a_bias = _abs(absolute, rows, weight, bias)
    p_abs = sum(a_rows[j:j + e - b] * a_weight[:, j] for j in range(w)) + (a_bias if bias is not None else 0)
    sg = sigmoid(p)
    # silu'(p) is at most 1.1, so |silu(p + d) - silu(p)| <= 1.1 |d|
    out['y'][b:e] = (1.1 * p_abs if absolute else p * sg) if silu else p_abs
    out['last'][s] = a_rows[e - b:].t()
    if dy is None:
      continue
    slope = sg * (1 + p * (1 - sg)) if silu else torch.ones_like(p)
    # silu' is a sum of terms of at most 1.3 in all, and |silu''| <= 1/2
    dp = dy[b:e].abs() * (1.3 + p_abs if silu else 1) if absolute else dy[b:e] * slope
    d_rows = torch.zeros_like(rows)
    for j in range(w):
      d_rows[j:j + e - b] += dp * a_weight[:, j]
      out['d_weight'][:, j] += (dp * a_rows[j:j + e - b]).sum(0)
    if d_last is not None:
      d_rows[e - b:] += _abs(absolute, d_last[s])[0].t()
    out['d_bias'] += dp.sum(0)
    out['d_x'][b:e] = d_rows[w - 1:]
    out['d_initial'][s] = d_rows[:w - 1].t()
  return out


def scan(x, delta, A, B, C, D, z, delta_bias, softplus, bounds, initial, dy=None, d_last=None, absolute=False):
  """``B``, ``C``: (tokens, groups, state).  Returns a dict of ``y``, ``last`` and, with ``dy``, the gradients."""
  T, c = x.shape
  n, G = A.shape[1], B.shape[1]
  per = c // G
  raw = delta + (delta_bias if delta_bias is not None else 0)
  dt = torch.logaddexp(raw, torch.zeros((), dtype=raw.dtype)) if softplus else raw
  slope = sigmoid(raw) if softplus else torch.ones_like(raw)
  gate = z * sigmoid(z) if z is not None else torch.ones_like(x)
  if z is not None:
    sg = sigmoid(z)
    d_gate = sg * (1 + z * (1 - sg))
  rate = A
  # (the decay's exponent dt A is off by a few u times itself: the terms carry 1 + |dt A|)
  ax, adt, aB, aC, aD, ady, agate, ainit, ad_last, aA = _abs(absolute, x, dt, B, C, D, dy, gate, initial, d_last, A)
  aB, aC = aB.repeat_interleave(per, 1), aC.repeat_interleave(per, 1)
  out = {'y': torch.zeros_like(x), 'last': x.new_zeros(len(bounds), c, n)}
  if dy is not None:
    out.update(d_x=torch.zeros_like(x), d_delta=torch.zeros_like(x), d_A=torch.zeros_like(A), d_B=torch.zeros_like(B),
               d_C=torch.zeros_like(C))
    if D is not None:
      out['d_D'] = torch.zeros_like(D)
    if z is not None:
      out['d_z'] = torch.zeros_like(x)
    if delta_bias is not None:
      out['d_delta_bias'] = torch.zeros_like(delta_bias)
    if initial is not None:
      out['d_initial'] = torch.zeros_like(initial)
  for s, (b, e) in enumerate(bounds):
    h = ainit[s].clone() if initial is not None else x.new_zeros(c, n)
    hs, keeps, y0s = [h], [], []
    for t in range(b, e):
      ex = dt[t][:, None] * rate
      keep = torch.exp(ex)
      keeps.append(keep)
      grow = 1 + ex.abs() if absolute else 1
      h = h * keep * grow + (adt[t] * ax[t])[:, None] * aB[t]
      hs.append(h)
      y0 = (h * aC[t]).sum(1) + (aD * ax[t] if D is not None else 0)
      y0s.append(y0)
      out['y'][t] = y0 * agate[t]
    out['last'][s] = h
    if dy is None:
      continue
    g = ad_last[s].clone() if d_last is not None else x.new_zeros(c, n)
    for t in range(e - 1, b - 1, -1):
      dY = ady[t] * agate[t]
      ex = dt[t][:, None] * rate
      keep = keeps[t - b] * (1 + ex.abs() if absolute else 1)
      q = g + dY[:, None] * aC[t]
      qB = (q * aB[t]).sum(1)
      through = q * keep
      w = through * hs[t - b]
      out['d_x'][t] = qB * adt[t] + (aD * dY if D is not None else 0)
      d_dt = qB * ax[t] + (w * aA).sum(1)
      d_raw = d_dt * slope[t]
      out['d_delta'][t] = d_raw
      out['d_A'] += w * adt[t][:, None]
      out['d_B'][t] = (q * (adt[t] * ax[t])[:, None]).reshape(G, per, n).sum(1)
      out['d_C'][t] = (dY[:, None] * hs[t - b + 1]).reshape(G, per, n).sum(1)
      if D is not None:
        out['d_D'] += dY * ax[t]
      if z is not None:
        out['d_z'][t] = ady[t] * y0s[t - b] * (d_gate[t].abs() + 0.5 if absolute else d_gate[t])
      if delta_bias is not None:
        out['d_delta_bias'] += d_raw
      g = through
    if initial is not None:
      out['d_initial'][s] = g
  return out


def check(got, want, majorant, operations, what=''):
  """Every value of ``got`` is within half a step of its type and ``operations`` roundings of the majorant."""
  assert tuple(got.shape) == tuple(want.shape), (what, tuple(got.shape), tuple(want.shape))
  g = got.detach().double().cpu()
  tol = half_step(got.dtype) * want.abs() + operations * U * majorant
  if got.dtype == torch.float16:
    tol = tol + 2.0 ** -25                 # half a step of the subnormal numbers
  off = (g - want).abs()
  bad = ~(off <= tol * (1 + 1e-9))
  assert not bad.any(), (f'{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off / (tol + 1e-300)).max()):.3g} '
                         f'times the tolerance')
