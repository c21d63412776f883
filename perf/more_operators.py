"""Operators of a language model's layers with leaky matrix states, as timed cases.

Four kinds of work, as a program that trains or serves such a model gives it to this library:

  embed        the rows of a table that tokens name, scaled (``embedding``), alone or with the gradient of the table
  rotate       queries and keys normed head by head and rotated by their positions (``norm_rotate``), alone or with gradients
  attend       linear attention with a decay for each head over packed sequences (``decay_attention``), alone or with gradients
  attend_step  the same for one new token per running request, against a pool of states (``decay_attention_step``)

Where ``own`` is true, ``run`` calls the library; otherwise it computes the same in elementary torch operations, in 32
bits: attention as masked products of all pairs of tokens, the table's gradient by adding rows, angles in 64 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
_BYTES = {'float32': 4, 'bfloat16': 2, 'float16': 2}


def listed():
  return [
    # the tokens of one decoding step of a full serving batch
    dict(name='embed_step', kind='embed', tokens=64, vocabulary=50_000, width=2048, dtype='bfloat16', grad=False),
    # packed prompts
    dict(name='embed_prompts', kind='embed', tokens=16_384, vocabulary=50_000, width=2048, dtype='bfloat16', grad=False),
    # a training step: the whole table's gradient, frequent tokens in it thousands of times
    dict(name='embed_training', kind='embed', tokens=32_768, vocabulary=64_000, width=2048, dtype='bfloat16', grad=True),
    # one request, one token, far into its text
    dict(name='rotate_step', kind='rotate', tokens=1, far=100_000, heads=16, kv_heads=4, size=128, rotated=128,
         interleaved=False, dtype='bfloat16', grad=False),
    # packed prompts, keys shared by groups of queries, half of each head rotated
    dict(name='rotate_prompts', kind='rotate', tokens=16_384, far=16_384, heads=32, kv_heads=8, size=128, rotated=64,
         interleaved=False, dtype='bfloat16', grad=False),
    # a training step
    dict(name='rotate_training', kind='rotate', tokens=8192, far=4096, heads=16, kv_heads=16, size=128, rotated=128,
         interleaved=True, dtype='bfloat16', grad=True),
    # one request, one token
    dict(name='attend_step_one', kind='attend_step', rows=1, pool=1, heads=16, kv_heads=16, key=128, value=128,
         dtype='bfloat16'),
    # a serving batch, some rows of it padding, states of a larger pool
    dict(name='attend_step_pool', kind='attend_step', rows=100, pool=128, heads=16, kv_heads=8, key=128, value=128,
         dtype='float16'),
    # one short prompt
    dict(name='attend_short_prompt', kind='attend', tokens=300, sequences=1, heads=16, kv_heads=16, key=128, value=128,
         dtype='bfloat16', grad=False),
    # prompts of different lengths in one packed batch, their states kept for the tokens that follow
    dict(name='attend_prompts', kind='attend', tokens=16_384, sequences=7, heads=16, kv_heads=16, key=128, value=128,
         dtype='bfloat16', grad=False),
    # a training step over packed sequences, keys and values shared by groups of queries
    dict(name='attend_training', kind='attend', tokens=8192, sequences=4, heads=16, kv_heads=8, key=128, value=128,
         dtype='bfloat16', grad=True),
    # a training step of odd sizes in 32 bits
    dict(name='attend_training_odd', kind='attend', tokens=1501, sequences=3, heads=5, kv_heads=5, key=75, value=90,
         dtype='float32', grad=True),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  kind = rng.choice(['embed', 'embed', 'rotate', 'rotate', 'attend', 'attend', 'attend', 'attend_step'])
  dtype = rng.choice(['bfloat16', 'bfloat16', 'bfloat16', 'float16', 'float32'])
  grad = rng.random() < 0.5
  if kind == 'embed':
    width, vocabulary = _log(rng, 64, 8192), _log(rng, 300, 200_000)
    vocabulary = min(vocabulary, 64_000 * 2048 // width // (2 if dtype == 'float32' else 1))
    tokens = max(1, min(_log(rng, 1, 65_536), 32_768 * 2048 // width // (2 if dtype == 'float32' else 1)))
    return dict(kind=kind, tokens=tokens, vocabulary=vocabulary, width=width, dtype=dtype, grad=grad)
  kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
  heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
  if kind == 'rotate':
    size = 2 * _log(rng, 16, 128) if rng.random() < 0.3 else rng.choice([64, 80, 96, 128, 128, 128, 256])
    rotated = size if rng.random() < 0.7 else 2 * rng.randint(4, size // 2)
    tokens = min(_log(rng, 1, 32_768), (48 if grad else 120) * 1_000_000 // ((heads + kv_heads) * size))
    tokens = max(1, tokens // (2 if dtype == 'float32' else 1))
    return dict(kind=kind, tokens=tokens, far=_log(rng, 1000, 1_000_000), heads=heads, kv_heads=kv_heads, size=size,
                rotated=rotated, interleaved=rng.random() < 0.4, dtype=dtype, grad=grad)
  if rng.random() < 0.3:
    key, value = _log(rng, 16, 256), _log(rng, 16, 256)
  else:
    key, value = rng.choice([(64, 64), (64, 128), (128, 64), (128, 128), (128, 128), (96, 96), (256, 256)])
  if kind == 'attend_step':
    rows = _log(rng, 1, max(1, min(250, 25_000_000 // (heads * key * value))))
    return dict(kind=kind, rows=rows, pool=rows + rows // 4, heads=heads, kv_heads=kv_heads, key=key, value=value, dtype=dtype)
  tokens = min(_log(rng, 30, 16_384), int(math.sqrt((1.0e9 if grad else 4.0e9) / heads)))
  tokens = min(tokens, (8192 if grad else 16_384) * 16 * 128 * 128 // (heads * key * value))
  tokens = max(1, tokens // (2 if dtype == 'float32' else 1))
  return dict(kind=kind, tokens=tokens, sequences=_log(rng, 1, 12), heads=heads, kv_heads=kv_heads, key=key, value=value,
              dtype=dtype, grad=grad)


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
  return {'embed': _prepare_embed, 'rotate': _prepare_rotate, 'attend': _prepare_attend,
          'attend_step': _prepare_attend_step}[case['kind']](case, int(seed), g)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
  return (torch.randn(*shape, device='cuda', generator=g) * scale).to(dtype)


def _leaves(state, names):
  for name in names:
    state[name].requires_grad_(True)
  state['leaves'] = names
  return state


def _prepare_embed(case, seed, g):
  """Tokens as text has them: the r-th most frequent one about 1 / r as often as the first, anywhere in the table."""
  dtype, v = _DTYPES[case['dtype']], case['vocabulary']
  rank = torch.exp(torch.rand(case['tokens'], device='cuda', generator=g, dtype=torch.float64) * math.log(v + 1)).long() - 1
  ids = torch.randperm(v, device='cuda', generator=g)[rank.clamp(0, v - 1)]
  state = dict(kind='embed', grad=case['grad'], ids=ids, scale=math.sqrt(case['width']),
               weight=_randn(g, v, case['width'], dtype=dtype, scale=case['width'] ** -0.5))
  if case['grad']:
    state['dy'] = _randn(g, case['tokens'], case['width'], dtype=dtype)
    _leaves(state, ['weight'])
  return state


def _prepare_rotate(case, seed, g):
  """Queries and keys are parts of one projection's rows, as a layer has them."""
  dtype, t, size = _DTYPES[case['dtype']], case['tokens'], case['size']
  h, hk = case['heads'], case['kv_heads']
  rows = _randn(g, t, (h + 2 * hk) * size, dtype=dtype)
  start = random.Random(seed).randint(0, case['far'])
  state = dict(kind='rotate', grad=case['grad'], interleaved=case['interleaved'],
               q=rows[:, :h * size].unflatten(1, (h, size)), k=rows[:, h * size:(h + hk) * size].unflatten(1, (hk, size)),
               q_weight=1 + _randn(g, size, scale=0.1), k_weight=1 + _randn(g, size, scale=0.1),
               positions=(torch.arange(t, device='cuda') + start).to(torch.int32),
               frequencies=10_000.0 ** -(torch.arange(0, case['rotated'], 2, device='cuda') / case['rotated']))
  if case['grad']:
    state['q'], state['k'] = state['q'].contiguous(), state['k'].contiguous()
    state['dq_out'], state['dk_out'] = _randn(g, t, h, size, dtype=dtype), _randn(g, t, hk, size, dtype=dtype)
    _leaves(state, ['q', 'k', 'q_weight', 'k_weight'])
  return state


def _heads(case, g, rows):
  """Queries and keys of about unit length, decays from a few tokens to some hundreds."""
  dtype, h, hk = _DTYPES[case['dtype']], case['heads'], case['kv_heads']
  place = (torch.arange(h, device='cuda') + torch.rand(h, device='cuda', generator=g)) / h
  return dict(q=_randn(g, rows, h, case['key'], dtype=dtype, scale=case['key'] ** -0.25),
              k=_randn(g, rows, hk, case['key'], dtype=dtype, scale=case['key'] ** -0.25),
              v=_randn(g, rows, hk, case['value'], dtype=dtype), log_decay=-torch.exp2(-8 * place),
              scale=case['key'] ** -0.5)


def _prepare_attend(case, seed, g):
  lengths = _lengths(case, seed)
  indptr = torch.zeros(len(lengths) + 1, dtype=torch.int32)
  indptr[1:] = torch.tensor(lengths).cumsum(0)
  state = dict(kind='attend', grad=case['grad'], lengths=lengths, indptr=indptr.cuda(), **_heads(case, g, case['tokens']))
  if case['grad']:
    state['initial'] = _randn(g, case['sequences'], case['heads'], case['key'], case['value'])
    state['dy'] = _randn(g, case['tokens'], case['heads'], case['value'], dtype=_DTYPES[case['dtype']])
    _leaves(state, ['q', 'k', 'v', 'initial'])
  return state


def _prepare_attend_step(case, seed, g):
  """A different state of the pool for every row; in a batch of more than 8 rows the last few rows are padding."""
  slots = torch.randperm(case['pool'], device='cuda', generator=g)[:case['rows']].to(torch.int32)
  if case['rows'] > 8:
    slots[-(case['rows'] // 16 + 1):] = -1
  return dict(kind='attend_step', slots=slots, **_heads(case, g, case['rows']),
              state=_randn(g, case['pool'], case['heads'], case['key'], case['value']))


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------
def run(state):
  if own:
    return {'embed': _own_embed, 'rotate': _own_rotate, 'attend': _own_attend, 'attend_step': _own_attend_step}[state['kind']](state)
  with torch.no_grad():
    return {'embed': _plain_embed, 'rotate': _plain_rotate, 'attend': _plain_attend,
            'attend_step': _plain_attend_step}[state['kind']](state)


def _gradients(s, outputs, cotangents):
  return dict(zip(('d_' + k for k in s['leaves']), torch.autograd.grad(outputs, [s[k] for k in s['leaves']], cotangents)))


def _own_embed(s):
  import brainpylib_b200 as bpl
  y = bpl.embedding(s['ids'], s['weight'], scale=s['scale'])
  return dict(_gradients(s, y, s['dy']), y=y) if s['grad'] else dict(y=y)


def _own_rotate(s):
  import brainpylib_b200 as bpl
  q, k = bpl.norm_rotate(s['q'], s['k'], s['positions'], s['frequencies'], s['q_weight'], s['k_weight'],
                         interleaved=s['interleaved'])
  return dict(_gradients(s, [q, k], [s['dq_out'], s['dk_out']]), q=q, k=k) if s['grad'] else dict(q=q, k=k)


def _own_attend(s):
  import brainpylib_b200 as bpl
  if s['grad']:
    y = bpl.decay_attention(s['q'], s['k'], s['v'], s['log_decay'], scale=s['scale'], indptr=s['indptr'],
                            initial_state=s['initial'])
    return dict(_gradients(s, y, s['dy']), y=y)
  y, last = bpl.decay_attention(s['q'], s['k'], s['v'], s['log_decay'], scale=s['scale'], indptr=s['indptr'],
                                return_state=True)
  return dict(y=y, last=last)


def _own_attend_step(s):
  import brainpylib_b200 as bpl
  y = bpl.decay_attention_step(s['q'], s['k'], s['v'], s['log_decay'], s['state'], scale=s['scale'], slots=s['slots'])
  return dict(y=y, state=s['state'])


# ---------------------------------------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits, rounded once at the end
# ---------------------------------------------------------------------------------------------------------
def _plain_embed(s):
  y = (s['weight'][s['ids']].float() * s['scale']).to(s['weight'].dtype)
  if not s['grad']:
    return dict(y=y)
  d = torch.zeros(s['weight'].shape, device=y.device).index_add_(0, s['ids'], s['dy'].float())
  return dict(y=y, d_weight=(d * s['scale']).to(s['weight'].dtype))


def _turn(x, cos, sin, interleaved):
  """The leading parts of all heads rotated in the planes of their pairs."""
  n = cos.shape[-1]
  part, rest = x[..., :2 * n], x[..., 2 * n:]
  a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n], part[..., n:])
  turned = (a * cos - b * sin, a * sin + b * cos)
  return torch.cat([torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1), rest], -1)


def _norm(x):
  return torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def _plain_rotate(s):
  angle = s['positions'].double()[:, None] * s['frequencies'].double()
  cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
  t, out = s['q'].dtype, {}
  q, k = s['q'].float(), s['k'].float()
  rq, rk = _norm(q), _norm(k)
  out['q'] = _turn(q * rq * s['q_weight'], cos, sin, s['interleaved']).to(t)
  out['k'] = _turn(k * rk * s['k_weight'], cos, sin, s['interleaved']).to(t)
  if s['grad']:
    out['d_q'], out['d_q_weight'] = _d_rotate(q, rq, s['q_weight'], _turn(s['dq_out'].float(), cos, -sin, s['interleaved']))
    out['d_k'], out['d_k_weight'] = _d_rotate(k, rk, s['k_weight'], _turn(s['dk_out'].float(), cos, -sin, s['interleaved']))
    out['d_q'], out['d_k'] = out['d_q'].to(t), out['d_k'].to(t)
  return out


def _d_rotate(x, r, weight, dz):
  n = x * r
  dn = dz * weight
  return r * (dn - n * (dn * n).mean(-1, keepdim=True)), (dz * n).sum((0, 1), dtype=torch.float64).float()


def _pairs(s):
  """What token j still counts for token i of the same sequence, by head; what an initial state counts for a token, and a token
  for the state its sequence leaves; which tokens a sequence has."""
  start, end = s['indptr'][:-1].long(), s['indptr'][1:].long()
  place = torch.arange(s['q'].shape[0], device=start.device)
  member = (place >= start[:, None]) & (place < end[:, None])
  seq = member.long().argmax(0)
  apart = place[:, None] - place
  decay = torch.exp(apart.clamp(min=0) * s['log_decay'][:, None, None]).masked_fill_((apart < 0) | (seq[:, None] != seq), 0.0)
  before = torch.exp((place - start[seq] + 1) * s['log_decay'][:, None])
  behind = torch.exp((end[seq] - 1 - place) * s['log_decay'][:, None])
  return decay, before, behind, member.float(), end - start


def _by_head(x, heads):
  """(tokens, heads, size) as (heads, tokens, size), shared heads repeated."""
  return x.float().repeat_interleave(heads // x.shape[1], 1).transpose(0, 1).contiguous()


def _shared(x, like):
  """The sum over the heads that share one, in its place and type."""
  return x.transpose(0, 1).unflatten(1, (like.shape[1], -1)).sum(2).to(like.dtype)


def _plain_attend(s):
  h, scale, t = s['q'].shape[1], s['scale'], s['q'].dtype
  q, k, v = (_by_head(s[n], h) for n in ('q', 'k', 'v'))
  decay, before, behind, member, lengths = _pairs(s)
  scores = (q @ k.transpose(1, 2)).mul_(decay).mul_(scale)
  y = scores @ v
  if not s['grad']:
    last = ((k * behind[:, :, None]) * member[:, None, :, None]).transpose(2, 3) @ v
    return dict(y=y.transpose(0, 1).to(t), last=last)
  initial = s['initial'].float()
  mine = member[:, None, :, None]                                                 # (sequences, 1, tokens, 1)
  y += (((q * before[:, :, None]) * mine) @ initial).sum(0) * scale
  dy = _by_head(s['dy'], h)
  d_scores = (dy @ v.transpose(1, 2)).mul_(decay).mul_(scale)
  from_initial = ((dy * before[:, :, None]) * mine)
  d_q = d_scores @ k + (from_initial @ initial.transpose(2, 3)).sum(0) * scale
  d_initial = ((q * mine).transpose(2, 3) @ from_initial) * scale
  return dict(y=y.transpose(0, 1).to(t), d_q=d_q.transpose(0, 1).to(t), d_k=_shared(d_scores.transpose(1, 2) @ q, s['k']),
              d_v=_shared(scores.transpose(1, 2) @ dy, s['v']), d_initial=d_initial)


def _plain_attend_step(s):
  h = s['q'].shape[1]
  live, at = s['slots'] >= 0, s['slots'].clamp(min=0).long()
  q, k, v = (s[n].float().repeat_interleave(h // s[n].shape[1], 1) for n in ('q', 'k', 'v'))
  new = s['state'][at] * torch.exp(s['log_decay'])[:, None, None] + k[:, :, :, None] * v[:, :, None]
  y = (q[:, :, :, None] * new).sum(2) * s['scale']
  pool, rows = s['state'].shape[0], new.shape[0]
  owner = torch.full((pool + 1,), -1, device=new.device)                          # padding rows' states go nowhere
  owner[torch.where(live, at, pool)] = torch.arange(rows, device=new.device)
  owner = owner[:pool]
  s['state'].copy_(torch.where((owner >= 0)[:, None, None, None], new[owner.clamp(min=0)], s['state']))
  return dict(y=torch.where(live[:, None, None], y, 0.0).to(s['q'].dtype), state=s['state'])


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------
def work(case):
  e = _BYTES[case['dtype']]
  if case['kind'] == 'embed':
    t, v, w = case['tokens'], case['vocabulary'], case['width']
    place = torch.arange(1, v + 1, dtype=torch.float64)                           # rows that at least one token names
    distinct = float(-torch.expm1(t * torch.log1p(-torch.log1p(1 / place) / math.log(v + 1))).sum())
    grad = t * w * e + v * w * e if case['grad'] else 0
    return dict(bytes=8 * t + distinct * w * e + t * w * e + grad, flops=t * w * (2 if case['grad'] else 1))
  if case['kind'] == 'rotate':
    n = case['tokens'] * (case['heads'] + case['kv_heads']) * case['size']
    return dict(bytes=n * e * (5 if case['grad'] else 2) + 4 * case['tokens'], flops=n * (24 if case['grad'] else 8))
  h, hk, key, value = case['heads'], case['kv_heads'], case['key'], case['value']
  if case['kind'] == 'attend_step':
    live = case['rows'] - (case['rows'] // 16 + 1 if case['rows'] > 8 else 0)
    row = e * (h * key + hk * (key + value))
    return dict(bytes=live * (8 * h * key * value + row) + case['rows'] * h * value * e, flops=5 * live * h * key * value)
  t, states = case['tokens'], 4 * case['sequences'] * h * key * value
  row = e * (h * key + hk * (key + value))
  if case['grad']:             # q, k, v and their gradients, y and dy; both initial states
    return dict(bytes=t * (2 * row + 2 * e * h * value) + 2 * states, flops=14 * t * h * key * value)
  return dict(bytes=t * (row + e * h * value) + states, flops=4 * t * h * key * value)


# ---------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
  state = prepare(case, seed)
  return {'embed': _exact_embed, 'rotate': _exact_rotate, 'attend': _exact_attend,
          'attend_step': _exact_attend_step}[case['kind']](state)


def _doubles(s):
  d = {}
  for k, v in s.items():
    if isinstance(v, torch.Tensor) and v.is_floating_point():
      v = v.detach().double()
      v = v.requires_grad_(True) if k in s.get('leaves', ()) else v
    d[k] = v
  return d


def _exact_embed(s):
  d = _doubles(s)
  y = torch.nn.functional.embedding(s['ids'], d['weight']) * s['scale']
  return dict(_gradients(d, y, d['dy']), y=y.detach()) if s['grad'] else dict(y=y)


def _exact_rotate(s):
  """Pairs as complex numbers, gradients by differentiating."""
  d = _doubles(s)
  turn = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'), d['positions'][:, None] * d['frequencies'])[:, None]
  n = d['frequencies'].numel()
  out = {}
  for name in ('q', 'k'):
    x = d[name]
    x = x / torch.linalg.vector_norm(torch.cat([x / math.sqrt(x.shape[-1]), torch.full_like(x[..., :1], 1e-3)], -1), dim=-1,
                                     keepdim=True) * d[name + '_weight']
    pairs = x[..., :2 * n].unflatten(-1, (n, 2)) if s['interleaved'] else x[..., :2 * n].unflatten(-1, (2, n)).transpose(-1, -2)
    turned = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
    out[name] = torch.cat([(turned if s['interleaved'] else turned.transpose(-1, -2)).flatten(-2), x[..., 2 * n:]], -1)
  if not s['grad']:
    return out
  return dict(_gradients(d, [out['q'], out['k']], [d['dq_out'], d['dk_out']]), **{n: v.detach() for n, v in out.items()})


def _exact_attend(s):
  """Token after token; with gradients, sequence after sequence and head after head as a sum over the tokens so far."""
  d = _doubles(s)
  h = s['q'].shape[1]
  group, a = h // s['k'].shape[1], torch.exp(d['log_decay'])
  y, at, lasts = torch.zeros(*s['q'].shape[:2], s['v'].shape[2], dtype=torch.float64, device='cuda'), 0, []
  if not s['grad']:
    for length in s['lengths']:
      state = y.new_zeros(h, s['q'].shape[2], s['v'].shape[2])
      for i in range(at, at + length):
        state = torch.baddbmm(state * a[:, None, None], d['k'][i].repeat_interleave(group, 0)[:, :, None],
                              d['v'][i].repeat_interleave(group, 0)[:, None])
        y[i] = torch.bmm(d['q'][i][:, None], state)[:, 0] * s['scale']
      lasts.append(state)
      at += length
    return dict(y=y, last=torch.stack(lasts))
  grads = {k: torch.zeros_like(d[k]) for k in s['leaves']}
  for n, length in enumerate(s['lengths']):
    rows = slice(at, at + length)
    power = torch.arange(length, device='cuda', dtype=torch.float64)
    for i in range(h if length else 0):
      with torch.enable_grad():
        part = [d[k][rows, i // (1 if k == 'q' else group)].detach().requires_grad_(True) for k in ('q', 'k', 'v')]
        first = d['initial'][n, i].detach().requires_grad_(True)
        counts = torch.tril(a[i] ** (power[:, None] - power).clamp(min=0))
        out = (torch.einsum('ik,jk,ij->ij', part[0], part[1], counts) @ part[2] +
               a[i] ** (power + 1)[:, None] * (part[0] @ first)) * s['scale']
        got = torch.autograd.grad(out, part + [first], d['dy'][rows, i])
      y[rows, i] = out.detach()
      for k, v in zip(('q', 'k', 'v'), got):
        grads[k][rows, i // (1 if k == 'q' else group)] += v
      grads['initial'][n, i] = got[3]
    at += length
  return dict(y=y, **{'d_' + k: v.detach() for k, v in grads.items()})


def _exact_attend_step(s):
  d = _doubles(s)
  h = s['q'].shape[1]
  group = h // s['k'].shape[1]
  y, state = torch.zeros(*s['q'].shape[:2], s['v'].shape[2], dtype=torch.float64, device='cuda'), d['state'].clone()
  for i, slot in enumerate(s['slots'].tolist()):
    if slot >= 0:
      for j in range(h):
        state[slot, j] = torch.exp(d['log_decay'][j]) * state[slot, j] + torch.outer(d['k'][i, j // group], d['v'][i, j // group])
        y[i, j] = d['q'][i, j] @ state[slot, j] * s['scale']
  return dict(y=y, state=state)
