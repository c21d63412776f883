"""``decay_attention`` and ``decay_attention_step`` against the plain statement in 64 bits: sizes of heads, types, packed sequences whose
ends lie anywhere, states, decays from nothing to everything, strides, shared heads."""
import math
import struct

import pytest
import torch

import brainpylib_b200 as bpl
import language_reference as ref
from brainpylib_b200 import _lib

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inputs(tokens, heads, kv_heads, key, value, dtype=F32, *, sequences=1, initial=True, seed=0, decays=None):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
  if decays is None:
    decays = -torch.exp2(-8 * torch.rand(heads, generator=g, dtype=torch.float64))
  return dict(q=r(tokens, heads, key).to(dtype), k=r(tokens, kv_heads, key).to(dtype), v=r(tokens, kv_heads, value).to(dtype),
              log_decay=torch.as_tensor(decays, dtype=F32), initial=r(sequences, heads, key, value).to(F32) if initial else None)


def call(d, cuda, bounds=None, leaf=False, **kw):
  g = {k: v if v is None else v.to(cuda) for k, v in d.items()}
  leaves = [k for k in ('q', 'k', 'v', 'initial') if leaf and g[k] is not None]
  for k in leaves:
    g[k].requires_grad_(True)
  p = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=cuda)
  kw.setdefault('scale', 0.3)
  out = bpl.decay_attention(g['q'], g['k'], g['v'], g['log_decay'], indptr=p, initial_state=g['initial'], return_state=True, **kw)
  return out, leaves, [g[k] for k in leaves]


# Roundings of a term, beside half a step of the result.  32-bit arithmetic: the product, and for every token that it stays in the
# state one of the state and one of the decay (whose own rounding counts once a token); the read-out adds up the elements of a head;
# joins of segments and shared heads are 16 more.  bfloat16 on tensor cores: the products of tokens of a chunk and the state that it
# reads are rounded to 8 bits once each on their way into a product (half a step of 2^-8); what goes into a state keeps 24 bits where
# it is returned (three such numbers) and 16 where it is only read out (2^-16 of itself, less than another half step); sums are kept in
# 32 bits, and accumulators that cut off instead of rounding count as two.
def operations(d, length):
  return 4 * length + 2 * max(d['q'].shape[2], d['v'].shape[2]) + 32


def check(d, cuda, bounds=None, scale=0.3):
  T = d['q'].shape[0]
  pairs = list(zip(bounds[:-1], bounds[1:])) if bounds is not None else [(0, T)]
  g = torch.Generator().manual_seed(7)
  heads, key, value = d['q'].shape[1], d['q'].shape[2], d['v'].shape[2]
  dy = torch.randn(T, heads, value, generator=g, dtype=torch.float64).to(d['q'].dtype)
  d_last = torch.randn(len(pairs), heads, key, value, generator=g).to(F32)
  args = (d['q'].double(), d['k'].double(), d['v'].double(), d['log_decay'].double(), scale, pairs,
          None if d['initial'] is None else d['initial'].double(), dy.double(), d_last.double())
  want, most = ref.attention(*args), ref.attention(*args, absolute=True)
  (y, last), _, _ = call(d, cuda, bounds, scale=scale)
  n = operations(d, max((e - b for b, e in pairs), default=0))
  rows = n + (3 * 2 ** 16 if d['q'].dtype == BF16 else 0)           # 3 * 2^16 * 2^-24 = 3 * 2^-8
  ref.check(y, want['y'], most['y'], rows, 'y')
  ref.check(last, want['last'], most['last'], n, 'last')
  (y2, last2), names, leaves = call(d, cuda, bounds, True, scale=scale)
  assert torch.equal(y, y2) and torch.equal(last, last2)
  got = torch.autograd.grad([y2, last2], leaves, [dy.to(cuda), d_last.to(cuda)])
  for name, v in zip(names, got):
    ref.check(v, want['d_' + name], most['d_' + name], n if name == 'initial' else rows, 'd_' + name)
  return y, last


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('key,value', [(1, 1), (3, 70), (16, 16), (64, 64), (64, 128), (128, 64), (128, 128), (96, 96), (75, 90), (40, 200), (129, 8), (192, 136), (64, 144),
                                       (256, 256)])
def test_sizes_and_types(cuda, key, value, dtype):
  for tokens, heads, kv_heads in ((1, 2, 1), (37, 2, 2), (150, 1, 1)):
    check(inputs(tokens, heads, kv_heads, key, value, dtype, seed=tokens), cuda)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('bounds', [[0, 1, 2, 3, 60], [0, 0, 64, 128, 128, 128, 129, 300], [3, 66, 130], [7, 7, 7], [5, 70, 71, 200], [0, 63, 128],
                                    [0], [40], [0, 0, 0, 500, 500]], ids=str)
def test_packed_sequences(cuda, bounds, dtype):
  """Sequences of no token, one token, and whose ends lie at, in front of and behind those of tiles; rows outside are not read."""
  for initial, heads in ((True, 2), (False, 3)):
    d = inputs(bounds[-1] + 21, heads, 1, 64, 64, dtype, sequences=len(bounds) - 1, initial=initial, seed=bounds[-1])
    for t in (d['q'], d['k'], d['v']):
      t[:bounds[0]] = float('nan')
      t[bounds[-1]:] = float('inf')
    (y, last), names, leaves = call(d, cuda, bounds, True)
    assert not y[:bounds[0]].any() and not y[bounds[-1]:].any()
    dy = torch.full_like(y, float('nan'))
    dy[bounds[0]:bounds[-1]] = 1
    for v in torch.autograd.grad(y, leaves, dy):
      assert torch.isfinite(v).all()
    for t in (d['q'], d['k'], d['v']):
      t[:bounds[0]] = 0
      t[bounds[-1]:] = 0
    check(d, cuda, bounds)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_long_sequences_in_segments(cuda, dtype):
  """Few heads, many tokens: sequences that begin, end and go on across segments."""
  check(inputs(3000, 1, 1, 64, 64, dtype, sequences=1, seed=1), cuda)
  check(inputs(2500, 2, 1, 32, 48, dtype, sequences=5, seed=2), cuda, [2, 130, 131, 1900, 1900, 2490])
  check(inputs(1700, 2, 2, 128, 128, dtype, sequences=3, initial=False, seed=3), cuda, [0, 64, 640, 1700])
  check(inputs(1900, 1, 1, 256, 136, dtype, sequences=2, seed=4), cuda, [0, 1100, 1900])


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_decays(cuda, dtype):
  """Nothing forgotten, everything forgotten after each token, decays that leave the range, a state that grows a little."""
  check(inputs(300, 5, 5, 64, 64, dtype, decays=[0.0, float('-inf'), -50.0, -1e-7, 0.01], seed=4), cuda)
  check(inputs(200, 2, 1, 16, 33, dtype, decays=[-1e30, -3e-39], seed=5), cuda)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_steep_decays_of_large_and_small_products(cuda, dtype):
  """Products of tokens of 2^13 and of 2^-40, scales of 2^-100, with decays whose powers over a few tokens come near the ends of the range."""
  decays = [-5.5, -4.0, -1.5, -1.38, 1.3, 2.0, 4.0]
  for size in (30.0, 2.0 ** -20):
    d = inputs(20, 7, 7, 64, 64, dtype, decays=decays, seed=11)
    for name in ('q', 'k'):
      d[name] = (d[name].double() * size).to(dtype)
    check(d, cuda)
  check(inputs(20, 7, 7, 64, 64, dtype, decays=decays, seed=12), cuda, scale=2.0 ** -100)


def test_scales(cuda):
  d = inputs(70, 2, 2, 64, 64, BF16)
  for scale in (0.0, -1.7, 1e-3):
    check(d, cuda, scale=scale)
  (y, _), _, _ = call(d, cuda, scale=None)
  (z, _), _, _ = call(d, cuda, scale=0.125)
  assert torch.equal(y, z)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_shared_heads(cuda, dtype):
  check(inputs(130, 6, 2, 64, 64, dtype, seed=8), cuda)
  check(inputs(40, 8, 1, 24, 16, dtype, seed=9), cuda)
  check(inputs(100, 4, 2, 200, 160, dtype, seed=10), cuda)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_strides_and_batches_are_the_packed_call(cuda, dtype):
  b, length, h = 3, 50, 2
  d = inputs(b * length, h, h, 64, 64, dtype, sequences=b, seed=6)
  bounds = [i * length for i in range(b + 1)]
  g = {k: v.to(cuda) for k, v in d.items()}
  args = (*(d[n].double() for n in ('q', 'k', 'v', 'log_decay')), 0.3, list(zip(bounds[:-1], bounds[1:])), d['initial'].double())
  want, most = ref.attention(*args), ref.attention(*args, absolute=True)
  n = operations(d, length)

  def same(y, last):
    ref.check(y.flatten(0, 1), want['y'], most['y'], n + (3 * 2 ** 16 if dtype == BF16 else 0), 'y')
    ref.check(last, want['last'], most['last'], n, 'last')

  kw = dict(scale=0.3, initial_state=g['initial'], return_state=True)
  for shift in (0, 1, 8):
    rows = torch.zeros(b, length, 3 * h * 64 + 16, dtype=dtype, device=cuda)
    parts = [rows[..., shift + i * h * 64:shift + (i + 1) * h * 64].unflatten(-1, (h, 64)).copy_(g[n].unflatten(0, (b, length)))
             for i, n in enumerate('qkv')]
    same(*bpl.decay_attention(*parts, g['log_decay'], **kw))
  mixed = [g[n].unflatten(0, (b, length)).transpose(1, 2).contiguous().transpose(1, 2) for n in 'qkv']     # heads in front of tokens
  same(*bpl.decay_attention(*mixed, g['log_decay'], **kw))
  one = g['q'][:, :1].expand(-1, h, -1)
  y, z = (bpl.decay_attention(t, g['k'], g['v'], g['log_decay']) for t in (one, one.contiguous()))
  assert torch.equal(y, z)


def test_only_one_of_the_results_has_a_gradient(cuda):
  d = inputs(90, 2, 2, 64, 64, F32)
  (y, last), names, leaves = call(d, cuda, None, True)
  got = torch.autograd.grad(last, leaves, torch.ones_like(last), allow_unused=True)
  want = ref.attention(*(d[n].double() for n in ('q', 'k', 'v', 'log_decay')), 0.3, [(0, 90)], d['initial'].double(),
                       d_last=torch.ones_like(last).double().cpu())
  most = ref.attention(*(d[n].double() for n in ('q', 'k', 'v', 'log_decay')), 0.3, [(0, 90)], d['initial'].double(),
                       d_last=torch.ones_like(last).double().cpu(), absolute=True)
  for name, v in zip(names, got):
    ref.check(v, want['d_' + name], most['d_' + name], operations(d, 90), name)


def test_against_differences(cuda):
  """Along a random way through one operand at a time the result is linear, so differences over a whole step are exact but for
  roundings: 2^-24 of sums of some thousand terms."""
  d = inputs(40, 2, 1, 8, 12, F32, seed=11)
  (y, last), names, leaves = call(d, cuda, None, True)
  gy, gl = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)), torch.randn(last.shape, generator=torch.Generator().manual_seed(2))
  got = torch.autograd.grad([y, last], leaves, [gy.to(cuda), gl.to(cuda)])

  def loss(e):
    (a, b), _, _ = call(e, cuda)
    return float((a.double().cpu() * gy.double()).sum() + (b.double().cpu() * gl.double()).sum())

  for name, v in zip(names, got):
    way = torch.randn(d[name].shape, generator=torch.Generator().manual_seed(3))
    slope = (loss(dict(d, **{name: d[name] + way})) - loss(dict(d, **{name: d[name] - way}))) / 2
    terms = v.double().cpu() * way.double()
    assert abs(slope - float(terms.sum())) <= 1e-4 * (1 + float(terms.abs().sum())), name


@pytest.mark.parametrize('dtype', [F32, F16])
def test_an_infinite_state_stays_infinite_in_segments(cuda, dtype):
  """Infinity times a decay that is left of many tokens is infinity, as it is token by token, whatever that decay's power rounds to."""
  d = inputs(1500, 1, 1, 64, 64, dtype, decays=[-3.0], seed=2)
  (y, last), _, _ = call(d, cuda)
  d['initial'][0, 0, 5, 7] = float('inf')
  (z, z_last), _, _ = call(d, cuda)
  keep = [i for i in range(64) if i != 7]
  assert torch.equal(z[..., keep], y[..., keep]) and torch.equal(z_last[..., keep], last[..., keep])
  assert float(z_last[0, 0, 5, 7]) == float('inf') and torch.equal(z_last[0, 0, 6:, 7], last[0, 0, 6:, 7])
  assert torch.equal(z[:, 0, 7].cpu(), torch.where(d['q'][:, 0, 5] > 0, float('inf'), -float('inf')).to(dtype))


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_tokens_do_not_reach_those_in_front_of_them(cuda, dtype):
  """What is not finite in a token's operands changes no bit of earlier outputs, of other sequences and (in v) of other columns; a
  gradient that is not finite, none of later tokens'."""
  d = inputs(150, 2, 1, 64, 64, dtype, sequences=2)
  bounds = [0, 100, 150]
  (y, last), _, _ = call(d, cuda, bounds)
  bad = torch.tensor([float('nan'), float('inf'), -float('inf')])
  for at in (0, 20, 63, 64, 90, 99):
    for name in ('q', 'k', 'v'):
      e = dict(d, **{name: d[name].clone()})
      e[name][at, 0, 5:8] = bad.to(dtype)
      (z, z_last), _, _ = call(e, cuda, bounds)
      assert torch.equal(z[:at], y[:at]) and torch.equal(z[100:], y[100:]) and torch.equal(z_last[1], last[1]), (at, name)
      keep = [i for i in range(64) if not 5 <= i < 8]
      if name == 'q':
        assert torch.equal(z[at + 1:], y[at + 1:]) and torch.equal(z_last, last) and not torch.isfinite(z[at]).all()
      elif name == 'v':
        assert torch.equal(z[..., keep], y[..., keep]) and torch.equal(z_last[..., keep], last[..., keep])
        assert not torch.isfinite(z[at:100, :, 5:8]).any() and not torch.isfinite(z_last[0, :, :, 5:8]).any()
      else:
        assert not torch.isfinite(z[at:100]).any(dim=-1).all()
  (y, _), names, leaves = call(d, cuda, bounds, True)
  clean = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
  for at in (0, 35, 36, 70, 99):
    dy = torch.ones_like(y)
    dy[at, 0, 3] = float('inf')
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for name, a, b in zip(names[1:3], got[1:3], clean[1:3]):
      assert torch.equal(a[at + 1:], b[at + 1:]), (at, name)
    keep = [i for i in range(150) if i != at]
    assert torch.equal(got[0][keep], clean[0][keep])


def test_no_wait_of_a_block_ran_out(cuda):
  """(behind all of the above)"""
  from brainpylib_b200 import _lib
  check(inputs(700, 3, 1, 128, 64, BF16, sequences=3), cuda, [0, 100, 101, 700])
  torch.cuda.synchronize()
  assert _lib.lib().bpl_tensor_walk_failures() == 0


def test_no_rows(cuda):
  d = inputs(0, 2, 1, 64, 64, BF16, sequences=2)
  (y, last), names, leaves = call(d, cuda, [0, 0, 0], True)
  assert y.shape == (0, 2, 64) and torch.equal(last, leaves[3])
  d_last = torch.randn_like(last)
  assert torch.equal(torch.autograd.grad(last, leaves, d_last, allow_unused=True)[3], d_last)
  d = inputs(0, 2, 1, 64, 64, F32, sequences=2, initial=False)
  assert not call(d, cuda, [0, 0, 0])[0][1].any()


# ---- one token ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('key,value', [(1, 1), (64, 64), (128, 128), (75, 90), (256, 256), (130, 4), (5, 33)])
def test_steps(cuda, key, value, dtype):
  rows, heads, kv_heads, pool = 5, 4, 2, 7
  d = inputs(rows, heads, kv_heads, key, value, dtype, sequences=pool, seed=key)
  slots = torch.tensor([3, -1, 0, 6, 2], dtype=torch.int32)
  state = d['initial'].to(cuda)
  args = [d[n].to(cuda) for n in ('q', 'k', 'v', 'log_decay')]
  y = bpl.decay_attention_step(*args, state, scale=0.3, slots=slots.to(cuda))
  live = [i for i in range(rows) if slots[i] >= 0]
  at = slots[live].long()
  ref_args = (d['q'][live].double(), d['k'][live].double(), d['v'][live].double(), d['log_decay'].double(), 0.3,
              [(i, i + 1) for i in range(len(live))], d['initial'][at].double())
  want, most = ref.attention(*ref_args), ref.attention(*ref_args, absolute=True)
  ref.check(y[live], want['y'], most['y'], key + 16, 'y')
  ref.check(state[at.to(cuda)], want['last'], most['last'], 4, 'state')
  assert not y[1].any()
  rest = [i for i in range(pool) if i not in at.tolist()]
  assert torch.equal(state[rest].cpu(), d['initial'][rest])


def test_steps_continue_a_prompt(cuda):
  d = inputs(40, 2, 1, 64, 64, BF16, sequences=1, initial=False)
  head = {k: v if k in ('log_decay', 'initial') else v[:30] for k, v in d.items()}
  (_, state), _, _ = call(head, cuda)
  args = lambda i: [d[n][i:i + 1].to(cuda) for n in 'qkv'] + [d['log_decay'].to(cuda)]
  rows = [bpl.decay_attention_step(*args(i), state, scale=0.3) for i in range(30, 40)]
  ref_args = (d['q'].double(), d['k'].double(), d['v'].double(), d['log_decay'].double(), 0.3, [(0, 40)], None)
  want, most = ref.attention(*ref_args), ref.attention(*ref_args, absolute=True)
  ref.check(torch.cat(rows), want['y'][30:], most['y'][30:], operations(d, 40), 'y')
  ref.check(state, want['last'], most['last'], operations(d, 40), 'state')


def test_slots_that_are_taken_or_not_there(cuda):
  d = inputs(6, 2, 2, 64, 40, F32, sequences=3)
  slots = torch.tensor([1, 1, 3, -5, 2 ** 31 - 1, 0], dtype=torch.int32, device=cuda)
  state = d['initial'].to(cuda)
  y = bpl.decay_attention_step(*[d[n].to(cuda) for n in ('q', 'k', 'v', 'log_decay')], state, slots=slots)
  assert torch.isnan(y[[1, 2, 4]]).all() and not y[3].any() and torch.isfinite(y[[0, 5]]).all()
  assert torch.equal(state[2].cpu(), d['initial'][2])
  again = d['initial'].to(cuda)
  bpl.decay_attention_step(*[d[n].to(cuda)[[0, 5]] if n != 'log_decay' else d[n].to(cuda) for n in ('q', 'k', 'v', 'log_decay')], again,
                           slots=slots[[0, 5]])
  assert torch.equal(again, state)


def test_step_strides_and_no_slots(cuda):
  d = inputs(4, 4, 2, 64, 64, BF16, sequences=4)
  rows = torch.zeros(4, 3, 4 * 64, dtype=BF16, device=cuda)
  q = rows[:, 0].unflatten(1, (4, 64)).copy_(d['q'])
  k, v = (rows[:, i, :128].unflatten(1, (2, 64)).copy_(d[n]) for i, n in ((1, 'k'), (2, 'v')))
  states = [d['initial'].to(cuda) for _ in range(2)]
  a = bpl.decay_attention_step(q, k, v, d['log_decay'].to(cuda), states[0])
  b = bpl.decay_attention_step(*[d[n].to(cuda) for n in ('q', 'k', 'v', 'log_decay')], states[1],
                               slots=torch.arange(4, dtype=torch.int32, device=cuda))
  assert torch.equal(a, b) and torch.equal(*states)


# ---- norms of errors ---------------------------------------------------------------------------------------------------
def chunked(q, k, v, log_decay, scale, first, decayed=1):
  """``attention`` of one sequence in 64 bits on the device of the operands, chunk by chunk, a head of k and v for every head of q.  A
  token reads the state in front of it decayed ``decayed`` times, plus its own product: 1, or 0 for walks from the end."""
  a, s = log_decay.double(), first
  y = torch.zeros(*q.shape[:2], v.shape[2], dtype=torch.float64, device=q.device)
  for b in range(0, q.shape[0], 64):
    Q, K, V = (t[b:b + 64].transpose(0, 1) for t in (q, k, v))
    n = torch.arange(Q.shape[1], device=q.device, dtype=torch.float64)
    counts = torch.exp((n[:, None] - n).clamp(min=0) * a[:, None, None]).tril()
    y[b:b + 64] = (scale * ((Q @ K.mT * counts) @ V) + torch.exp((n + decayed) * a[:, None])[..., None] * (Q @ s)).transpose(0, 1)
    weights = torch.exp((len(n) - decayed - n) * a[:, None])[..., None]
    s = torch.exp(len(n) * a)[:, None, None] * s + scale * (K * weights).mT @ V
  return y, s


def exactly(d, scale, dy, d_last):
  """All results and gradients of one sequence in 64 bits: the walk and, with its operands exchanged, its gradients."""
  t = {k: v.double() for k, v in d.items()}
  group = t['q'].shape[1] // t['k'].shape[1]
  q, k, v = t['q'], t['k'].repeat_interleave(group, 1), t['v'].repeat_interleave(group, 1)
  # (the state holds the scale here, so that one function does for all)
  y, last = chunked(q, k, v, d['log_decay'], scale, scale * t['initial'][0])
  d_q, _ = chunked(dy, v, k, d['log_decay'], scale, scale * t['initial'][0].mT)
  back = lambda x: x.flip(0)
  d_v, d_initial = chunked(back(k), back(q), back(dy), d['log_decay'], scale, d_last[0], 0)
  d_k, _ = chunked(back(v), back(dy), back(q), d['log_decay'], scale, d_last[0].mT, 0)
  shared = lambda x: back(x).unflatten(1, (-1, group)).sum(2)
  return dict(y=y, last=last[None] / scale, d_q=d_q, d_k=shared(d_k), d_v=shared(d_v), d_initial=d_initial[None])


def computed(d, scale, dy, d_last):
  leaves = {k: d[k].detach().requires_grad_(True) for k in ('q', 'k', 'v', 'initial')}
  y, last = bpl.decay_attention(leaves['q'], leaves['k'], leaves['v'], d['log_decay'], scale=scale, initial_state=leaves['initial'],
                                return_state=True)
  g = torch.autograd.grad([y, last], list(leaves.values()), [dy, d_last])
  return dict(y=y, last=last, **{'d_' + k: v for k, v in zip(leaves, g)})


def norm(x):
  return float(torch.linalg.vector_norm(x.detach().double()))


@pytest.mark.parametrize('log_decay', [0.0, -1e-5])
@pytest.mark.parametrize('mean', [0.0, 0.5])
def test_a_state_that_lasts_is_as_good_as_one_of_32_bits(cuda, log_decay, mean):
  """8192 tokens of 80 heads are 128 chunks of one segment.  Each addition to a state rounds to half a step of 2^-23, one way or the other:
  sqrt(128) 2^-24 of its norm.  What a chunk brings passes twelve additions of accumulators that cut off up to a step, half of one on
  average, of less than the chunk's: 12 * 2^-24, and V in terms and the powers of the decays 4 * 2^-24 more.  The decay of a chunk is
  rounded once and multiplied in 128 times, always the same way: 128 * 2^-25 at most."""
  d = inputs(8192, 80, 80, 64, 64, BF16, decays=[log_decay] * 80, seed=21)
  d = {k: (v + mean if k in 'qkv' else v).to(cuda) for k, v in d.items()}
  g = torch.Generator().manual_seed(22)
  dy = (torch.randn(d['q'].shape, generator=g) + mean).to(BF16).to(cuda)
  d_last = torch.randn(d['initial'].shape, generator=g).to(cuda)
  got, want = computed(d, 0.125, dy, d_last), exactly(d, 0.125, dy.double(), d_last.double())
  most = (128 ** 0.5 + 16) * ref.U + (128 * ref.U / 2 if log_decay else 0)
  for name in ('last', 'd_initial'):
    assert norm(got[name] - want[name]) <= most * norm(want[name]), (name, norm(got[name] - want[name]) / norm(want[name]))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('tokens,heads,kv_heads,key,value', [(2500, 16, 16, 128, 128), (700, 8, 4, 64, 128), (600, 2, 2, 256, 256), (900, 3, 1, 192, 72),
                                                             (1000, 148, 148, 64, 64)])
def test_results_are_rounded_once(cuda, tokens, heads, kv_heads, key, value, dtype):
  """In the norm.  Results in 16 bits are off by what rounding the exact ones is off by, once.  On the way the products of tokens and the
  state that a chunk reads lose 2^-16 of themselves at most (two numbers of 16 bits each) and sums 2^-18 (64 roundings to 32 bits): 2^-15 +
  2^-18, a fiftieth of the 0.0017 of one rounding, which makes 1 + 1 / 5000 of the norm; 1.001 is asked for.  In 32 bits roundings add
  up like the square root of their number: two for each token that a state lasts (256 here), and the accumulators' and the heads' 8.
  What a call returns beside y changes none of its bits."""
  g = torch.Generator().manual_seed(tokens)
  d = {k: v.to(cuda) for k, v in inputs(tokens, heads, kv_heads, key, value, dtype, seed=tokens).items()}
  dy = torch.randn(tokens, heads, value, generator=g).to(dtype).to(cuda)
  d_last = torch.randn(d['initial'].shape, generator=g).to(cuda)
  got, want = computed(d, key ** -0.5, dy, d_last), exactly(d, key ** -0.5, dy.double(), d_last.double())
  for name, v in got.items():
    if v.dtype == F32:
      assert norm(v - want[name]) <= 32 * ref.U * norm(want[name]), name
    else:
      once = norm(want[name].to(dtype).double() - want[name])
      assert norm(v.double() - want[name]) <= 1.001 * once, (name, norm(v.double() - want[name]) / once)
  y = bpl.decay_attention(d['q'], d['k'], d['v'], d['log_decay'], scale=key ** -0.5, initial_state=d['initial'])
  assert torch.equal(y, got['y'])


def test_an_infinite_state_that_lasts_stays_infinite_on_tensor_cores(cuda):
  """(where the powers of its decay do not vanish)"""
  d = inputs(150, 1, 1, 64, 64, BF16, decays=[-0.01], seed=2)
  (y, last), _, _ = call(d, cuda)
  d['initial'][0, 0, 5, 7] = float('inf')
  (z, z_last), _, _ = call(d, cuda)
  keep = [i for i in range(64) if i != 7]
  assert torch.equal(z[..., keep], y[..., keep]) and torch.equal(z_last[..., keep], last[..., keep])
  assert float(z_last[0, 0, 5, 7]) == float('inf') and torch.equal(z_last[0, 0, 6:, 7], last[0, 0, 6:, 7])
  assert torch.equal(z[:, 0, 7].cpu(), torch.where(d['q'][:, 0, 5] > 0, float('inf'), -float('inf')).to(BF16))


# ---- the C targets -----------------------------------------------------------------------------------------------------
def opaque(d, scale, sequences=1):
  (tokens, heads, key), (_, kv_heads, value) = d['q'].shape, d['v'].shape
  strides = [s for n in 'qkv' for s in (d[n].stride(0), d[n].stride(1))]
  return struct.pack('<8IfI6q', tokens, sequences, tokens // sequences, heads, kv_heads, key, value, {F32: 0, F16: 1, BF16: 2}[d['q'].dtype], scale, 0,
                     *strides)


def workspace(name, packed, cuda):
  return torch.empty(_lib.workspace_bytes(name, packed) or 1, dtype=torch.uint8, device=cuda)


def shifted(shape, dtype, elements, cuda):
  """A result that does not lie at 16 bytes."""
  return torch.empty(math.prod(shape) + 8, dtype=dtype, device=cuda)[elements:elements + math.prod(shape)].view(shape)


@pytest.mark.parametrize('elements', [1, 4])
@pytest.mark.parametrize('kv_heads,key,value', [(2, 64, 64), (1, 128, 72), (2, 256, 64)])
def test_results_at_any_address(cuda, kv_heads, key, value, elements):
  """bfloat16 operands at 16 bytes, results at other addresses: what the 32-bit walk gives, which takes any."""
  d = {k: v.to(cuda) for k, v in inputs(100, 2, kv_heads, key, value, BF16, seed=key).items()}
  dy = torch.randn(100, 2, value, device=cuda).to(BF16)
  packed = opaque(d, 0.3)
  odd = dict(d, **{n: shifted(d[n].shape, BF16, 1, cuda).copy_(d[n]) for n in 'qkv'})
  leaves = {n: odd[n].detach().requires_grad_(True) for n in 'qkv'}
  want = bpl.decay_attention(*leaves.values(), d['log_decay'], scale=0.3, initial_state=d['initial'])
  want_grads = torch.autograd.grad(want, list(leaves.values()), dy)
  y = shifted(want.shape, BF16, elements, cuda)
  _lib.call('decay_attention', [d['q'], d['k'], d['v'], d['log_decay'], None, d['initial'], y, None, workspace('decay_attention', packed, cuda)], packed)
  assert torch.equal(y, want)
  for which in range(3):
    grads = [shifted(d[n].shape, BF16, elements if i == which else 0, cuda) for i, n in enumerate('qkv')]
    _lib.call('decay_attention_backward', [d['q'], d['k'], d['v'], d['log_decay'], None, d['initial'], dy, None, *grads, torch.empty_like(d['initial']),
                                           workspace('decay_attention_backward', packed, cuda)], packed)
    for i, (a, b) in enumerate(zip(grads, want_grads)):
      # (dk and dv are made of the same states, so that one's address decides for both; elsewhere tensor cores: a step of 16 bits)
      if i == which or (which > 0 and i > 0):
        assert torch.equal(a, b)
      else:
        assert (a.float() - b.float()).abs().max() <= 2 * ref.half_step(BF16) * b.float().abs().max()


# ---- plans -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('heads,kv_heads,batch,length', [(8, 8, 40, 70), (16, 4, 20, 129), (75, 75, 5, 64)])
def test_batches_of_many_sequences(cuda, heads, kv_heads, batch, length, dtype):
  """At least as many sequences as pieces that fill the card: cut between sequences, several to a segment, the last one with fewer.  Rounded
  once, as in test_results_are_rounded_once."""
  d = {k: v.to(cuda) for k, v in inputs(batch * length, heads, kv_heads, 64, 72, dtype, sequences=batch, seed=batch).items()}
  g = torch.Generator().manual_seed(1)
  dy = torch.randn(batch * length, heads, 72, generator=g).to(dtype).to(cuda)
  d_last = torch.randn(d['initial'].shape, generator=g).to(cuda)
  leaves = {k: (d[k] if k == 'initial' else d[k].unflatten(0, (batch, length))).detach().requires_grad_(True) for k in ('q', 'k', 'v', 'initial')}
  y, last = bpl.decay_attention(leaves['q'], leaves['k'], leaves['v'], d['log_decay'], scale=0.125, initial_state=leaves['initial'], return_state=True)
  grads = torch.autograd.grad([y, last], list(leaves.values()), [dy.unflatten(0, (batch, length)), d_last])
  got = dict(y=y, last=last, **{'d_' + k: v for k, v in zip(leaves, grads)})
  want = {k: [] for k in got}
  for i in range(batch):
    rows = slice(i * length, (i + 1) * length)
    one = {k: v[i:i + 1] if k == 'initial' else v if k == 'log_decay' else v[rows] for k, v in d.items()}
    for k, v in exactly(one, 0.125, dy[rows].double(), d_last[i:i + 1].double()).items():
      want[k].append(v)
  for name, v in got.items():
    w = torch.cat(want[name])
    assert v.isfinite().all()
    if v.dtype == F32:
      assert norm(v.reshape(w.shape) - w) <= 32 * ref.U * norm(w), name
    else:
      assert norm(v.reshape(w.shape).double() - w) <= 1.001 * norm(w.to(dtype).double() - w), name


def test_numbers_that_are_not_finite_in_many_chunks_of_a_block(cuda):
  """80 heads are one segment, so that a block walks 18 chunks and its tables of such numbers come round twice, forwards and backwards."""
  heads, tokens = 80, 1140
  d = {k: v.to(cuda) for k, v in inputs(tokens, heads, heads, 64, 64, BF16, seed=31).items()}
  dy = torch.randn(tokens, heads, 64, device=cuda).to(BF16)
  d_last = torch.zeros_like(d['initial'])
  clean = computed(d, 0.125, dy, d_last)
  bad = [(3, 0, 1, float('inf')), (64, 1, 0, float('nan')), (7 * 64 + 63, 2, 63, -float('inf')), (8 * 64, 3, 7, float('nan')), (12 * 64 + 5, 0, 40, float('inf')),
         (15 * 64 + 30, 4, 5, float('inf')), (17 * 64 + 51, 5, 6, float('nan'))]

  def spoilt(name, column_only, from_the_end, got):
    """Of heads 0 to 5: no numbers from the tokens on (to them, from the end) in those columns, or in all; all else to the last bit."""
    v, w = got[name], clean[name]
    spoil = torch.zeros_like(w, dtype=torch.bool)
    for t, h, c, _ in bad:
      spoil[(slice(0, t + 1) if from_the_end else slice(t, None)), h, (c if column_only else slice(None))] = True
    assert torch.equal(v[~spoil], w[~spoil]), name
    assert not torch.isfinite(v[spoil]).any() if column_only else not torch.isfinite(v[spoil]).all(), name

  e = dict(d, v=d['v'].clone())
  for t, h, c, x in bad:
    e['v'][t, h, c] = x
  got = computed(e, 0.125, dy, d_last)
  spoilt('y', True, False, got)
  spoil = torch.zeros(heads, 64, 64, dtype=torch.bool, device=cuda)
  for _, h, c, _ in bad:
    spoil[h, :, c] = True
  assert torch.equal(got['last'][0][~spoil], clean['last'][0][~spoil]) and not torch.isfinite(got['last'][0][spoil]).any()
  e = dict(d, q=d['q'].clone())
  for t, h, c, x in bad:
    e['q'][t, h, c] = x
  got = computed(e, 0.125, dy, d_last)
  spoilt('d_k', True, True, got)
  other = dy.clone()
  for t, h, c, x in bad:
    other[t, h, c] = x
  got = computed(d, 0.125, other, d_last)
  spoilt('d_v', True, True, got)
  spoilt('d_k', False, True, got)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_large_products_of_tokens_with_a_small_scale(cuda, dtype):
  """Products of tokens of 2^103, which the scale brings back, with decays from e^-1.3 to 1.  (Not above: at e^1.2 a state of 40 tokens is 2^67
  times as large, and its product with a token 2^165, which 32 bits do not hold whatever is done first.)"""
  d = inputs(40, 3, 3, 64, 64, dtype, decays=[-1.3, -0.2, 0.0], seed=13)
  for name in ('q', 'k'):
    d[name] = (d[name].double() * 2.0 ** 48).to(dtype)
  check(d, cuda, scale=2.0 ** -40)
