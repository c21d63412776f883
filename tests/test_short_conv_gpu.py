"""``short_conv`` and ``short_conv_step`` against the plain statement in 64 bits: widths, types, runs of tokens that end inside
sequences, sequences shorter than the taps, rows without alignment."""
import pytest
import torch

import brainpylib_b200 as bpl
import sequence_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inputs(tokens, channels, width, dtype=F32, *, sequences=1, bias=True, initial=True, wide=False, seed=0):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
  weight_type = F32 if wide else dtype
  return dict(x=r(tokens, channels).to(dtype), weight=r(channels, width).to(weight_type),
              bias=r(channels).to(weight_type) if bias else None,
              initial=r(sequences, channels, width - 1).to(dtype) if initial else None)


def to_gpu(d, cuda, leaf=False):
  return {k: v.to(cuda).requires_grad_(leaf) if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def call(g, silu, indptr=None):
  p = None if indptr is None else torch.tensor(indptr, dtype=torch.int32, device=g['x'].device)
  return bpl.short_conv(g['x'], g['weight'], g['bias'], activation='silu' if silu else None, indptr=p,
                        initial_state=g['initial'], return_state=True)


def reference(d, bounds, silu, **kw):
  w = {k: v.double() if v is not None else None for k, v in d.items()}
  args = (w['x'], w['weight'], w['bias'], bounds, w['initial'], silu)
  return ref.conv(*args, **kw), ref.conv(*args, **kw, absolute=True)


def check(d, cuda, bounds, silu):
  """A value is a sum of at most 9 products, times a sigmoid (16 roundings); its gradients sum up to 8 of them once more, those
  of the parameters over all tokens.  Last inputs are copies."""
  pairs = list(zip(bounds[:-1], bounds[1:]))
  g = torch.Generator().manual_seed(7)
  dy = torch.randn(d['x'].shape, generator=g, dtype=torch.float64).to(d['x'].dtype)
  d_last = torch.randn(len(pairs), d['x'].shape[1], d['weight'].shape[1] - 1, generator=g, dtype=torch.float64).to(d['x'].dtype)
  want, most = reference(d, pairs, silu, dy=dy.double(), d_last=d_last.double())
  plain = call(to_gpu(d, cuda), silu, bounds)
  ref.check(plain[0], want['y'], most['y'], 32, 'y')
  assert torch.equal(plain[1].double().cpu(), want['last'])
  leaf = to_gpu(d, cuda, True)
  names = [n for n in ('x', 'weight', 'bias', 'initial') if leaf[n] is not None]
  y, last = call(leaf, silu, bounds)
  assert torch.equal(y, plain[0]) and torch.equal(last, plain[1])
  got = torch.autograd.grad([y, last], [leaf[n] for n in names], [dy.to(cuda), d_last.to(cuda)])
  for n, v in zip(names, got):
    ref.check(v, want['d_' + n], most['d_' + n], 64 + (d['x'].shape[0] if n in ('weight', 'bias') else 0), 'd_' + n)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('width', range(1, 9))
def test_widths_types_and_alignments(cuda, width, dtype):
  for tokens, channels, silu, wide in ((1, 8, True, False), (70, 33, False, False), (37, 64, True, True), (130, 9, True, False)):
    check(inputs(tokens, channels, width, dtype, wide=wide, seed=tokens), cuda, [0, tokens], silu)


@pytest.mark.parametrize('bounds', [[0, 1, 2, 3, 4, 5, 40], [0, 0, 16, 32, 32, 32, 33, 80, 80], [3, 19, 35, 50], [0, 64, 128], [7, 7, 7],
                                    [5, 70, 71, 90], [0, 2, 4, 6, 9, 12], [0], [40]], ids=str)
def test_packed_sequences(cuda, bounds):
  """Sequences shorter than the taps, empty ones, bounds inside and at the ends of runs; rows outside are not read."""
  for initial, channels in ((True, 24), (False, 13)):
    d = inputs(bounds[-1] + 21, channels, 4, F32, sequences=len(bounds) - 1, initial=initial, seed=bounds[-1])
    d['x'][:bounds[0]] = float('nan')
    d['x'][bounds[-1]:] = float('inf')
    y, last = call(to_gpu(d, cuda), True, bounds)
    assert not y[:bounds[0]].any() and not y[bounds[-1]:].any()
    leaf = to_gpu(d, cuda, True)
    dy = torch.full_like(y, float('nan'))
    dy[bounds[0]:bounds[-1]] = 1
    for v in torch.autograd.grad(call(leaf, True, bounds)[0], [v for v in leaf.values() if v is not None], dy):
      assert torch.isfinite(v).all()
    d['x'][:bounds[0]] = 0
    d['x'][bounds[-1]:] = 0
    check(d, cuda, bounds, True)


def test_without_bias_and_without_initial_inputs(cuda):
  check(inputs(50, 40, 4, BF16, bias=False, initial=False), cuda, [0, 50], True)
  check(inputs(50, 40, 3, F32, bias=False, initial=True), cuda, [0, 50], False)


def test_many_tokens(cuda):
  """More runs than blocks of the first kernel hold, so that parts of sums are added up over many runs."""
  check(inputs(5003, 12, 4, F32, sequences=3), cuda, [0, 1000, 1001, 5003], True)


def test_batches_and_strided_rows_are_the_packed_call(cuda):
  b, length, c = 3, 29, 48
  d = to_gpu(inputs(b * length, c, 4, BF16, sequences=b, seed=6), cuda)
  y, last = call(d, True, [i * length for i in range(b + 1)])
  x = d['x'].reshape(b, length, c)
  kw = dict(activation='silu', initial_state=d['initial'], return_state=True)
  for shift in (0, 1, 8):
    wide = torch.zeros(b, length, 2 * c + 16, dtype=BF16, device=cuda)
    part = wide[:, :, shift:shift + c].copy_(x)
    y2, last2 = bpl.short_conv(part, d['weight'], d['bias'], **kw)
    assert torch.equal(y2.reshape(-1, c), y) and torch.equal(last2, last)
  apart = torch.zeros(b, length + 3, c, dtype=BF16, device=cuda)[:, 1:-2].copy_(x)
  y3, _ = bpl.short_conv(apart, d['weight'], d['bias'], **kw)
  assert torch.equal(y3.reshape(-1, c), y)
  across = x.transpose(1, 2).contiguous().transpose(1, 2)          # channels apart, tokens next to one another
  y4, _ = bpl.short_conv(across, d['weight'], d['bias'], **kw)
  assert torch.equal(y4.reshape(-1, c), y)


def test_no_rows(cuda):
  d = inputs(0, 8, 4, F32, sequences=2)
  y, last = call(to_gpu(d, cuda), True, [0, 0, 0])
  assert y.shape == (0, 8) and torch.equal(last.cpu(), d['initial'])
  check(d, cuda, [0, 0, 0], True)


def test_a_prompt_in_parts_and_token_by_token(cuda):
  d = inputs(40, 72, 4, BF16, initial=False, seed=8)
  g = to_gpu(d, cuda)
  y, last = call(g, True)
  head, tail = dict(g, x=g['x'][:27]), dict(g, x=g['x'][27:])
  y1, s1 = call(head, True)
  y2, s2 = call(dict(tail, initial=s1), True)
  assert torch.equal(torch.cat([y1, y2]), y) and torch.equal(s2, last)
  pool = torch.full((4, 72, 3), 7.0, dtype=BF16, device=cuda)
  pool[2] = s1[0]
  slots = torch.tensor([2], dtype=torch.int32, device=cuda)
  for t in range(27, 40):
    yt = bpl.short_conv_step(g['x'][t:t + 1], pool, g['weight'], g['bias'], activation='silu', slots=slots)
    assert torch.equal(yt[0], y[t])
  assert torch.equal(pool[2], last[0]) and (pool[[0, 1, 3]] == 7).all()


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,channels,width', [(1, 64, 4), (5, 33, 1), (9, 300, 2), (40, 260, 5), (3, 16, 8)])
def test_single_steps_on_a_pool(cuda, rows, channels, width, dtype):
  for wide, silu in ((False, True), (True, False)):
    d = inputs(rows, channels, width, dtype, initial=False, wide=wide, seed=rows)
    pool = torch.randn(rows + 3, channels, width - 1, generator=torch.Generator().manual_seed(1)).to(dtype)
    slots = torch.randperm(rows + 3, generator=torch.Generator().manual_seed(2))[:rows].to(torch.int32)
    slots[1::4] = -1 - slots[1::4]
    d['initial'] = pool[slots.clamp(min=0).long()]
    want, most = reference(d, [(i, i + 1) for i in range(rows)], silu)
    g, state = to_gpu(d, cuda), pool.to(cuda)
    y = bpl.short_conv_step(g['x'], state, g['weight'], g['bias'], activation='silu' if silu else None, slots=slots.to(cuda))
    live = slots >= 0
    ref.check(y[live.to(cuda)], want['y'][live], most['y'][live], 32)
    assert not y[(~live).to(cuda)].any()
    after = pool.double().clone()
    after[slots[live].long()] = want['last'][live]
    assert torch.equal(state.double().cpu(), after)


def test_steps_with_slots_that_are_taken_or_beyond_the_pool(cuda):
  d = to_gpu(inputs(300, 40, 4, F32, initial=False, seed=9), cuda)
  slots = torch.arange(300, dtype=torch.int32)
  slots[[7, 150, 299]] = 3
  slots[9] = 300
  slots[10] = 2 ** 31 - 1
  bad = torch.zeros(300, dtype=torch.bool)
  bad[[7, 9, 10, 150, 299]] = True
  good = torch.nonzero(~bad)[:, 0].to(cuda)
  pool = torch.randn(300, 40, 3, device=cuda, generator=torch.Generator(cuda).manual_seed(3))
  alone = pool.clone()
  want = bpl.short_conv_step(d['x'][good], alone, d['weight'], d['bias'], slots=slots[~bad].to(cuda))
  y = bpl.short_conv_step(d['x'], pool, d['weight'], d['bias'], slots=slots.to(cuda))
  assert torch.equal(y[good], want) and torch.isnan(y[bad.to(cuda)]).all() and torch.equal(pool, alone)


def test_bounds_that_are_no_bounds_touch_nothing_outside(cuda):
  for bounds in ([-5, 10, 3, 50, 2000000000, 7], [40, 30, 20, 10, 5, 0], [-2 ** 31, 2 ** 31 - 1, 0, 40, -1, 40]):
    g = to_gpu(inputs(40, 30, 4, F32, sequences=5, seed=10), cuda, True)
    y, last = call(g, True, bounds)
    assert y.shape == (40, 30) and last.shape == (5, 30, 3)
    torch.autograd.grad(y.sum() + last.sum(), [g['x'], g['initial']])
  torch.cuda.synchronize()
