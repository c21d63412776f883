"""Operators over whole sequences, as timed cases: leaky states, short convolutions and clipped gradients.

Five kinds of work, as a program that trains or serves a layer of leaky units gives it to this library:

  conv       a short causal convolution over packed sequences (``short_conv``), alone or with its gradients
  conv_step  the same for one new token per running request, against a pool of states (``short_conv_step``)
  scan       leaky states with input-dependent decay over packed sequences (``state_scan``), alone or with gradients
  scan_step  the same for one new token per running request (``state_scan_step``)
  clip       the global norm over all gradients of a training step, and clipping (``clip_gradients``)

Where ``own`` is true, ``run`` calls the library; otherwise it computes the same in elementary torch operations, in 32
bits, over the whole sequence at once: the recurrence by doubling (pairs of decay and input, log2 of the length rounds).
"""
import math
import random

import torch

own = False

_DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
_BYTES = {'float32': 4, 'bfloat16': 2, 'float16': 2}


def listed():
  return [
    # one request, one token: latency and launches are all there is
    dict(name='conv_step_one', kind='conv_step', rows=1, pool=1, channels=2048, width=4, dtype='bfloat16', silu=True),
    # a full serving batch, some rows of it padding, states of a larger pool
    dict(name='conv_step_pool', kind='conv_step', rows=200, pool=256, channels=5120, width=4, dtype='float16', silu=True),
    # prompts of different lengths in one packed batch, their last inputs kept for the steps that follow
    dict(name='conv_prompts', kind='conv', tokens=16_384, sequences=11, channels=4096, width=4, dtype='bfloat16', silu=True,
         grad=False),
    # a training step of odd sizes in 32 bits
    dict(name='conv_training', kind='conv', tokens=3109, sequences=4, channels=1003, width=3, dtype='float32', silu=False,
         grad=True),
    # one request, one token
    dict(name='scan_step_one', kind='scan_step', rows=1, pool=1, channels=2048, state=16, groups=1, dtype='bfloat16', gate=True),
    # a full serving batch: the states are read and written once
    dict(name='scan_step_pool', kind='scan_step', rows=250, pool=300, channels=4096, state=16, groups=1, dtype='bfloat16',
         gate=True),
    # one short prompt: few tokens, few channels, little to share out
    dict(name='scan_short_prompt', kind='scan', tokens=200, sequences=1, channels=1536, state=16, groups=1, dtype='bfloat16',
         gate=True, grad=False),
    # one long prompt
    dict(name='scan_long_prompt', kind='scan', tokens=16_384, sequences=1, channels=4096, state=16, groups=1,
         dtype='bfloat16', gate=True, grad=False),
    # a training step over packed sequences of different lengths
    dict(name='scan_training', kind='scan', tokens=8192, sequences=7, channels=2048, state=16, groups=1, dtype='bfloat16',
         gate=True, grad=True),
    # a training step of odd sizes in 32 bits, inputs and read-outs shared by groups of channels
    dict(name='scan_training_odd', kind='scan', tokens=1545, sequences=3, channels=750, state=10, groups=2, dtype='float32',
         gate=False, grad=True),
    # the gradients of a small network: a handful of matrices and their vectors
    dict(name='clip_small', kind='clip', tensors=24, elements=1_300_000, dtype='float32'),
    # the gradients of a large one: hundreds of tensors, weights in 16 bits and the rest in 32
    dict(name='clip_large', kind='clip', tensors=390, elements=600_000_000, dtype='bfloat16'),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  kind = rng.choice(['conv', 'conv', 'conv_step', 'scan', 'scan', 'scan', 'scan_step', 'clip'])
  dtype = rng.choice(['bfloat16', 'bfloat16', 'float16', 'float32'])
  if kind == 'conv':
    channels, tokens = _log(rng, 100, 8192), _log(rng, 64, 32_768)
    tokens = max(1, min(tokens, 16_384 * 4096 // channels // (2 if dtype == 'float32' else 1)))
    grad = rng.random() < 0.5
    return dict(kind=kind, tokens=tokens // 3 + 1 if grad else tokens, sequences=_log(rng, 1, 40), channels=channels,
                width=rng.choice([2, 3, 4, 4, 5]), dtype=dtype, silu=rng.random() < 0.7, grad=grad)
  if kind == 'conv_step':
    rows = _log(rng, 1, 250)
    return dict(kind=kind, rows=rows, pool=rows + rows // 4, channels=_log(rng, 100, 8192), width=rng.choice([2, 3, 4, 4, 5]),
                dtype=dtype, silu=rng.random() < 0.7)
  if kind == 'clip':
    return dict(kind=kind, tensors=_log(rng, 3, 600), elements=_log(rng, 100_000, 500_000_000), dtype=dtype)
  groups = rng.choice([1, 1, 1, 2, 4])
  state = rng.choice([8, 16, 16, 16, 24, 32, 64, rng.randint(3, 40)])
  channels = groups * _log(rng, 128 // groups, 8192 // groups)
  if kind == 'scan_step':
    rows = _log(rng, 1, max(1, min(250, 16_000_000 // (channels * state))))
    return dict(kind=kind, rows=rows, pool=rows + rows // 4, channels=channels, state=state, groups=groups, dtype=dtype,
                gate=rng.random() < 0.6)
  tokens, grad = _log(rng, 50, 16_384), rng.random() < 0.5
  tokens = max(1, min(tokens, (250_000_000 if grad else 1_000_000_000) // (channels * state)))
  return dict(kind=kind, tokens=tokens, sequences=_log(rng, 1, 12), channels=channels, state=state, groups=groups, dtype=dtype,
              gate=rng.random() < 0.6, grad=grad)


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
def _lengths(case, seed):
  """Sequence lengths that fill the tokens, cut at places drawn from the seed."""
  rng = random.Random(seed)
  cuts = sorted(rng.randint(0, case['tokens']) for _ in range(case['sequences'] - 1))
  return [b - a for a, b in zip([0] + cuts, cuts + [case['tokens']])]


def prepare(case, seed):
  g = torch.Generator(device='cuda').manual_seed(int(seed))
  return {'conv': _prepare_conv, 'conv_step': _prepare_conv_step, 'scan': _prepare_scan, 'scan_step': _prepare_scan_step,
          'clip': _prepare_clip}[case['kind']](case, int(seed), g)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
  return (torch.randn(*shape, device='cuda', generator=g) * scale).to(dtype)


def _packing(case, seed):
  lengths = _lengths(case, seed)
  indptr = torch.zeros(len(lengths) + 1, dtype=torch.int32)
  indptr[1:] = torch.tensor(lengths).cumsum(0)
  return dict(lengths=lengths, longest=max(lengths), indptr=indptr.cuda())


def _leaves(state, names):
  for name in names:
    state[name].requires_grad_(True)
  state['leaves'] = names
  return state


def _prepare_conv(case, seed, g):
  dtype, c, w = _DTYPES[case['dtype']], case['channels'], case['width']
  state = dict(_packing(case, seed), kind='conv', silu=case['silu'], grad=case['grad'],
               x=_randn(g, case['tokens'], c, dtype=dtype), weight=_randn(g, c, w, dtype=dtype, scale=w ** -0.5),
               bias=_randn(g, c, dtype=dtype, scale=0.1))
  if case['grad']:
    state['initial'] = _randn(g, case['sequences'], c, w - 1, dtype=dtype)
    state['dy'] = _randn(g, case['tokens'], c, dtype=dtype)
    _leaves(state, ['x', 'weight', 'bias', 'initial'])
  return state


def _slots(case, g):
  """A different state of the pool for every row; in a batch of more than 8 rows the last few rows are padding."""
  slots = torch.randperm(case['pool'], device='cuda', generator=g)[:case['rows']].to(torch.int32)
  if case['rows'] > 8:
    slots[-(case['rows'] // 16 + 1):] = -1
  return slots


def _prepare_conv_step(case, seed, g):
  dtype, c, w = _DTYPES[case['dtype']], case['channels'], case['width']
  return dict(kind='conv_step', silu=case['silu'], x=_randn(g, case['rows'], c, dtype=dtype),
              state=_randn(g, case['pool'], c, w - 1, dtype=dtype), weight=_randn(g, c, w, dtype=dtype, scale=w ** -0.5),
              bias=_randn(g, c, dtype=dtype, scale=0.1), slots=_slots(case, g))


def _scan_inputs(case, g, rows):
  """Decay rates of 1 to 16 per unit of time, time steps around 1e-3 to 0.1 once through the softplus."""
  dtype, c, n, groups = _DTYPES[case['dtype']], case['channels'], case['state'], case['groups']
  rate = torch.exp(torch.rand(c, n, device='cuda', generator=g) * math.log(16.0))
  dt = torch.exp(torch.rand(c, device='cuda', generator=g) * math.log(100.0)) * 1e-3
  state = dict(x=_randn(g, rows, c, dtype=dtype), delta=_randn(g, rows, c, dtype=dtype, scale=0.5), A=-rate,
               B=_randn(g, rows, groups, n, dtype=dtype), C=_randn(g, rows, groups, n, dtype=dtype),
               D=1 + _randn(g, c, scale=0.1), delta_bias=dt + torch.log(-torch.expm1(-dt)), z=None)
  if case['gate']:
    state['z'] = _randn(g, rows, c, dtype=dtype)
  return state


def _prepare_scan(case, seed, g):
  state = dict(_packing(case, seed), kind='scan', grad=case['grad'], **_scan_inputs(case, g, case['tokens']))
  if case['grad']:
    state['initial'] = _randn(g, case['sequences'], case['channels'], case['state'])
    state['dy'] = _randn(g, case['tokens'], case['channels'], dtype=_DTYPES[case['dtype']])
    _leaves(state, [k for k in ('x', 'delta', 'A', 'B', 'C', 'D', 'delta_bias', 'z', 'initial') if state[k] is not None])
  return state


def _prepare_scan_step(case, seed, g):
  return dict(kind='scan_step', slots=_slots(case, g), **_scan_inputs(case, g, case['rows']),
              state=_randn(g, case['pool'], case['channels'], case['state']))


def _sizes(case):
  """Sizes of the tensors of a network: most are vectors, a third are matrices and hold nearly all elements.  Every third
  tensor is one in 32 bits whatever the type of the matrices."""
  n, total = case['tensors'], case['elements']
  vectors = [max(1, total // (400 * n)) + i % 7 for i in range(n - n // 3)]
  rest = max(n // 3, total - sum(vectors))
  weights = [1 + i % 5 for i in range(n // 3)]
  matrices = [max(1, rest * w // sum(weights)) for w in weights]
  return matrices, vectors


def _prepare_clip(case, seed, g):
  """Gradients as a training program holds them: in two buckets, one per type, each tensor a part of its bucket."""
  matrices, vectors = _sizes(case)
  buckets = [_randn(g, sum(matrices), dtype=_DTYPES[case['dtype']], scale=0.02), _randn(g, sum(vectors), scale=0.05)]
  out = [torch.empty_like(b) for b in buckets]
  return dict(kind='clip', buckets=buckets, out=out, max_norm=1.0, sizes=(matrices, vectors),
              grads=[t for b, s in zip(buckets, (matrices, vectors)) for t in b.split(s)],
              clipped=[t for b, s in zip(out, (matrices, vectors)) for t in b.split(s)])


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------
def run(state):
  if own:
    return {'conv': _own_conv, 'conv_step': _own_conv_step, 'scan': _own_scan, 'scan_step': _own_scan_step,
            'clip': _own_clip}[state['kind']](state)
  with torch.no_grad():
    return {'conv': _plain_conv, 'conv_step': _plain_conv_step, 'scan': _plain_scan, 'scan_step': _plain_scan_step,
            'clip': _plain_clip}[state['kind']](state)


def _gradients(s, y):
  return dict(zip(('d_' + k for k in s['leaves']), torch.autograd.grad(y, [s[k] for k in s['leaves']], s['dy'])))


def _own_conv(s):
  import brainpylib_b200 as bpl
  activation = 'silu' if s['silu'] else None
  if s['grad']:
    y = bpl.short_conv(s['x'], s['weight'], s['bias'], activation=activation, indptr=s['indptr'], initial_state=s['initial'])
    return dict(_gradients(s, y), y=y)
  y, last = bpl.short_conv(s['x'], s['weight'], s['bias'], activation=activation, indptr=s['indptr'], return_state=True)
  return dict(y=y, last=last)


def _own_conv_step(s):
  import brainpylib_b200 as bpl
  y = bpl.short_conv_step(s['x'], s['state'], s['weight'], s['bias'], activation='silu' if s['silu'] else None,
                          slots=s['slots'])
  return dict(y=y, state=s['state'])


def _own_scan(s):
  import brainpylib_b200 as bpl
  args = dict(z=s['z'], delta_bias=s['delta_bias'], delta_softplus=True, indptr=s['indptr'])
  if s['grad']:
    y = bpl.state_scan(s['x'], s['delta'], s['A'], s['B'], s['C'], s['D'], initial_state=s['initial'], **args)
    return dict(_gradients(s, y), y=y)
  y, last = bpl.state_scan(s['x'], s['delta'], s['A'], s['B'], s['C'], s['D'], return_state=True, **args)
  return dict(y=y, last=last)


def _own_scan_step(s):
  import brainpylib_b200 as bpl
  y = bpl.state_scan_step(s['x'], s['delta'], s['A'], s['B'], s['C'], s['state'], s['D'], z=s['z'],
                          delta_bias=s['delta_bias'], delta_softplus=True, slots=s['slots'])
  return dict(y=y, state=s['state'])


def _own_clip(s):
  import brainpylib_b200 as bpl
  norm = bpl.clip_gradients(s['grads'], s['max_norm'], out=s['clipped'])
  return dict(norm=norm, clipped=s['out'])


# ---------------------------------------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits, rounded once at the end
# ---------------------------------------------------------------------------------------------------------
def _silu(v):
  return v * torch.sigmoid(v)


def _d_silu(v):
  s = torch.sigmoid(v)
  return s * (1 + v * (1 - s))


def _sequence_of(s):
  """Sequence of every token, and the token's place in it."""
  start = s['indptr'][:-1].long()
  lengths = s['indptr'][1:].long() - start
  total = sum(s['lengths'])
  seq = torch.repeat_interleave(torch.arange(len(s['lengths']), device=start.device), lengths, output_size=total)
  return seq, torch.arange(total, device=start.device) - start[seq]


def _plain_conv(s):
  x, weight = s['x'].float(), s['weight'].float()
  c, w = weight.shape
  n = len(s['lengths'])
  seq, _ = _sequence_of(s)
  row = torch.arange(x.shape[0], device=x.device) + (seq + 1) * (w - 1)      # every sequence behind its w - 1 earlier inputs
  first = s['indptr'][:-1].long() + torch.arange(n, device=x.device) * (w - 1)
  before = first[:, None] + torch.arange(w - 1, device=x.device)
  xp = x.new_zeros(x.shape[0] + n * (w - 1), c)
  xp[row] = x
  if s['grad']:
    xp[before] = s['initial'].float().transpose(1, 2)
  p = s['bias'].float() + sum(xp[row - (w - 1 - j)] * weight[:, j] for j in range(w))
  y = (_silu(p) if s['silu'] else p).to(s['x'].dtype)
  if not s['grad']:
    end = s['indptr'][1:].long() + (torch.arange(n, device=x.device) + 1) * (w - 1)
    last = xp[end[:, None] - (w - 1) + torch.arange(w - 1, device=x.device)].transpose(1, 2)
    return dict(y=y, last=last.to(s['x'].dtype).contiguous())
  dp = s['dy'].float() * (_d_silu(p) if s['silu'] else 1)
  d_weight = torch.stack([(dp * xp[row - (w - 1 - j)]).sum(0) for j in range(w)], 1)
  d_xp = torch.zeros_like(xp)
  d_xp[row] = dp * weight[:, w - 1]
  d_xp = d_xp + sum(torch.zeros_like(xp).index_copy_(0, row - (w - 1 - j), dp * weight[:, j]) for j in range(w - 1))
  return dict(y=y, d_x=d_xp[row].to(s['x'].dtype), d_weight=d_weight.to(s['weight'].dtype),
              d_bias=dp.sum(0).to(s['bias'].dtype), d_initial=d_xp[before].transpose(1, 2).to(s['initial'].dtype))


def _rows(s):
  """The rows that are not padding, and their states."""
  live = s['slots'] >= 0
  return live, s['slots'].clamp(min=0).long()


def _write_back(s, live, new):
  """The rows' new states into the pool, padding rows' nowhere."""
  pool, rows = s['state'].shape[0], new.shape[0]
  owner = torch.full((pool + 1,), -1, device=new.device)
  owner[torch.where(live, s['slots'].long(), pool)] = torch.arange(rows, device=new.device)
  owner = owner[:pool]
  s['state'].copy_(torch.where((owner >= 0)[:, None, None], new[owner.clamp(min=0)], s['state']))


def _plain_conv_step(s):
  live, at = _rows(s)
  x, weight, bias = s['x'], s['weight'].float(), s['bias'].float()
  window = torch.cat([s['state'][at], x[:, :, None]], 2)
  p = (window.float() * weight).sum(2) + bias
  y = torch.where(live[:, None], _silu(p) if s['silu'] else p, 0.0).to(x.dtype)
  _write_back(s, live, window[:, :, 1:])
  return dict(y=y, state=s['state'])


def _recurrence(a, b, longest):
  """h[t] = a[t] h[t - 1] + b[t] for all t at once, by doubling; a is 0 where a sequence starts."""
  step = 1
  while step < longest:
    b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
    a = torch.cat([a[:step], a[step:] * a[:-step]])
    step *= 2
  return b


def _long_sum(v):
  """Over all tokens."""
  return v.sum(0, dtype=torch.float64).float()


def _softplus(v):
  return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _scan_terms(s):
  c = s['A'].shape[0]
  repeat = c // s['B'].shape[1]
  raw = s['delta'].float() + s['delta_bias']
  dt = _softplus(raw)
  B, C = (s[k].float().repeat_interleave(repeat, 1) for k in ('B', 'C'))
  return s['x'].float(), raw, dt, B, C


def _plain_scan(s):
  x, raw, dt, B, C = _scan_terms(s)
  seq, place = _sequence_of(s)
  first = (place == 0)[:, None, None]
  decay = torch.exp(dt[:, :, None] * s['A'])
  b = (dt * x)[:, :, None] * B
  if s['grad']:
    initial = s['initial'].float()
    b = b + torch.where(first, decay * initial[seq], 0.0)
  h = _recurrence(torch.where(first, 0.0, decay), b, s['longest'])
  y0 = (h * C).sum(2) + s['D'] * x
  z = None if s['z'] is None else s['z'].float()
  y = (y0 if z is None else y0 * _silu(z)).to(s['x'].dtype)
  if not s['grad']:
    end, some = s['indptr'][1:].long() - 1, s['indptr'][1:] > s['indptr'][:-1]
    return dict(y=y, last=torch.where(some[:, None, None], h[end.clamp(min=0)], 0.0))
  dy = s['dy'].float()
  out = {}
  if z is not None:
    out['d_z'] = (dy * y0 * _d_silu(z)).to(s['z'].dtype)
    dy = dy * _silu(z)
  final = torch.cat([first[1:], torch.ones_like(first[:1])])
  after = torch.where(final, 0.0, torch.cat([decay[1:], decay[:1]]))
  q = _recurrence(after.flip(0), (dy[:, :, None] * C).flip(0), s['longest']).flip(0)
  earlier = torch.where(first, initial[seq], torch.cat([h[:1], h[:-1]]))
  qa = q * decay * earlier
  d_dt = (q * (x[:, :, None] * B) + qa * s['A']).sum(2)
  d_raw = d_dt * torch.sigmoid(raw)
  d_b = (q * (dt * x)[:, :, None]).unflatten(1, (s['B'].shape[1], -1)).sum(2)
  d_c = (dy[:, :, None] * h).unflatten(1, (s['B'].shape[1], -1)).sum(2)
  d_initial = torch.zeros_like(initial).index_add_(0, seq, torch.where(first, q * decay, 0.0))
  t = s['x'].dtype
  return dict(out, y=y, d_x=((q * B).sum(2) * dt + s['D'] * dy).to(t), d_delta=d_raw.to(t), d_A=_long_sum(qa * dt[:, :, None]),
              d_B=d_b.to(t), d_C=d_c.to(t), d_D=_long_sum(dy * x), d_delta_bias=_long_sum(d_raw),
              d_initial=d_initial)


def _plain_scan_step(s):
  live, at = _rows(s)
  x, _, dt, B, C = _scan_terms(s)
  h = s['state'][at] * torch.exp(dt[:, :, None] * s['A']) + (dt * x)[:, :, None] * B
  y = (h * C).sum(2) + s['D'] * x
  if s['z'] is not None:
    y = y * _silu(s['z'].float())
  _write_back(s, live, h)
  return dict(y=torch.where(live[:, None], y, 0.0).to(s['x'].dtype), state=s['state'])


def _plain_clip(s):
  squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s['grads']])
  norm = squares.sum().sqrt()
  scale = torch.clamp(s['max_norm'] / (norm + 1e-6), max=1.0).float()
  # (tensor by tensor, as the calls for the norm)
  done = [o.copy_(g.float() * scale) for g, o in zip(s['grads'], s['clipped'])]
  return dict(norm=norm.float(), clipped=s['out'] if done else [])


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------
def work(case):
  e = _BYTES[case['dtype']]
  if case['kind'] == 'clip':
    matrices, vectors = _sizes(case)
    return dict(bytes=2 * (e * sum(matrices) + 4 * sum(vectors)), flops=3 * (sum(matrices) + sum(vectors)))
  c = case['channels']
  if case['kind'] == 'conv':
    t, w = case['tokens'], case['width']
    passes = 4 if case['grad'] else 2                # x and y; with gradients dy and dx too
    edges = case['sequences'] * c * (w - 1) * e * (2 if case['grad'] else 1)
    return dict(bytes=passes * t * c * e + edges + c * (w + 1) * e * (2 if case['grad'] else 1),
                flops=(6 if case['grad'] else 2) * t * c * w)
  if case['kind'] == 'conv_step':
    live = case['rows'] - (case['rows'] // 16 + 1 if case['rows'] > 8 else 0)
    return dict(bytes=e * c * (live + case['rows'] + 2 * live * (case['width'] - 1) + case['width'] + 1),
                flops=2 * live * c * case['width'])
  n, groups, gate = case['state'], case['groups'], 1 if case['gate'] else 0
  if case['kind'] == 'scan_step':
    live = case['rows'] - (case['rows'] // 16 + 1 if case['rows'] > 8 else 0)
    return dict(bytes=live * c * (2 * 4 * n + e * (2 + gate)) + case['rows'] * c * e + live * 2 * groups * n * e + c * 4 * (n + 2),
                flops=7 * live * c * n)
  t = case['tokens']
  if case['grad']:                                   # x, delta, z, y and dy; dx, ddelta, dz; B and C and theirs; both states' ends
    return dict(bytes=t * c * e * (6 + 2 * gate) + 4 * t * groups * n * e + 2 * 4 * c * (n + 2) + 2 * 4 * case['sequences'] * c * n,
                flops=25 * t * c * n)
  return dict(bytes=t * c * e * (3 + gate) + 2 * t * groups * n * e + 4 * c * (n + 2) + 4 * case['sequences'] * c * n,
              flops=7 * t * c * n)


# ---------------------------------------------------------------------------------------------------------
# the definition, in 64 bits: token after token, gradients by differentiating it
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
  state = prepare(case, seed)
  return {'conv': _exact_conv, 'conv_step': _exact_conv_step, 'scan': _exact_scan, 'scan_step': _exact_scan_step,
          'clip': _exact_clip}[case['kind']](state)


def _doubles(s):
  d = {}
  for k, v in s.items():
    if isinstance(v, torch.Tensor) and v.is_floating_point():
      v = v.detach().double()
      v = v.requires_grad_(True) if k in s.get('leaves', ()) else v
    d[k] = v
  return d


def _by_definition(s, d, forward):
  """``forward`` over every sequence: outputs one behind the other, last states, and the gradients of the leaves."""
  with torch.enable_grad() if s['grad'] else torch.no_grad():
    ys, lasts, at = [], [], 0
    for i, length in enumerate(s['lengths']):
      y, last = forward(i, at, length)
      ys.append(y)
      lasts.append(last)
      at += length
    y = torch.cat(ys)
  if not s['grad']:
    return dict(y=y, last=torch.stack(lasts))
  return dict(_gradients(d, y), y=y.detach())


def _exact_conv(s):
  d = _doubles(s)
  c, w = d['weight'].shape

  def forward(i, at, length):
    before = d['initial'][i] if s['grad'] else d['x'].new_zeros(c, w - 1)
    row = torch.cat([before.t(), d['x'][at:at + length]])
    windows = torch.stack([row[j:j + length] for j in range(w)], 2)
    p = torch.einsum('tcw,cw->tc', windows, d['weight']) + d['bias']
    return (p / (1 + torch.exp(-p)) if s['silu'] else p), row[length:].t()

  return _by_definition(s, d, forward)


def _exact_conv_step(s):
  d = _doubles(s)
  y, state = torch.zeros_like(d['x']), d['state'].clone()
  for i, slot in enumerate(s['slots'].tolist()):
    if slot >= 0:
      window = torch.cat([state[slot], d['x'][i][:, None]], 1)
      p = torch.einsum('cw,cw->c', window, d['weight']) + d['bias']
      y[i] = p / (1 + torch.exp(-p)) if s['silu'] else p
      state[slot] = window[:, 1:]
  return dict(y=y, state=state)


def _exact_scan(s):
  d = _doubles(s)
  c, n = d['A'].shape
  repeat = c // d['B'].shape[1]

  def forward(i, at, length):
    h = d['initial'][i] if s['grad'] else d['x'].new_zeros(c, n)
    tokens = slice(at, at + length)
    dt = torch.logaddexp(d['delta'][tokens] + d['delta_bias'], torch.zeros((), dtype=torch.float64, device=h.device))
    B, C = (d[k][tokens].repeat_interleave(repeat, 1) for k in ('B', 'C'))
    rows = []
    for step, x, b, r in zip(dt.unbind(0), d['x'][tokens].unbind(0), B.unbind(0), C.unbind(0)):
      h = h * torch.exp(step[:, None] * d['A']) + (step * x)[:, None] * b
      rows.append(torch.einsum('cn,cn->c', h, r) + d['D'] * x)
    y = torch.stack(rows) if rows else d['x'][tokens]
    z = d['z'][tokens] if d['z'] is not None else None
    return (y if z is None else y * z / (1 + torch.exp(-z))), h

  return _by_definition(s, d, forward)


def _exact_scan_step(s):
  d = _doubles(s)
  c, n = d['A'].shape
  groups = d['B'].shape[1]
  y, state = torch.zeros_like(d['x']), d['state'].clone()
  for i, slot in enumerate(s['slots'].tolist()):
    if slot >= 0:
      dt = torch.logaddexp(d['delta'][i] + d['delta_bias'], torch.zeros((), dtype=torch.float64, device=y.device))
      B, C = (d[k][i][:, None].expand(groups, c // groups, n).reshape(c, n) for k in ('B', 'C'))
      state[slot] = torch.exp(dt[:, None] * d['A']) * state[slot] + torch.einsum('c,cn->cn', dt * d['x'][i], B)
      v = torch.einsum('cn,cn->c', state[slot], C) + d['D'] * d['x'][i]
      y[i] = v if d['z'] is None else v * d['z'][i] / (1 + torch.exp(-d['z'][i]))
  return dict(y=y, state=state)


def _exact_clip(s):
  norm = math.sqrt(sum(torch.linalg.vector_norm(b, dtype=torch.float64).item() ** 2 for b in s['buckets']))
  scale = min(1.0, s['max_norm'] / (norm + 1e-6))
  return dict(norm=torch.tensor(norm, dtype=torch.float64), clipped=[b.double() * scale for b in s['buckets']])
