"""The operators over whole sequences where there is nothing, or nothing finite, to compute with."""
import struct

import pytest
import torch

import brainpylib_b200 as bpl
import sequence_reference as ref
from brainpylib_b200._lib import workspace_bytes

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------------------------------------
# no channels
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('batched', [False, True])
def test_no_channels(cuda, batched, dtype):
  """The gradients of B and C are sums over no channels: zeros, whatever stood in the memory that they got."""
  lead, n = ((3, 40) if batched else (120,)), 16
  r = lambda *s: torch.randn(*s, device=cuda, generator=torch.Generator(cuda).manual_seed(0)).to(dtype).requires_grad_(True)
  x, delta, A = r(*lead, 0), r(*lead, 0), torch.zeros(0, n, device=cuda, requires_grad=True)
  B, C = r(*lead, 2, n), r(*lead, 2, n)
  y, last = bpl.state_scan(x, delta, A, B, C, return_state=True)
  assert y.shape == (*lead, 0) and last.shape == (3 if batched else 1, 0, n)
  rubbish = [torch.full_like(B, float('nan')) for _ in range(16)]
  torch.cuda.synchronize()
  del rubbish
  for g, of in zip(torch.autograd.grad([y, last], [x, delta, A, B, C], [torch.zeros_like(y), torch.zeros_like(last)]), (x, delta, A, B, C)):
    assert g.shape == of.shape and g.dtype == of.dtype and not g.any()


# ---------------------------------------------------------------------------------------------------------
# no rows
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_batches_of_sequences_without_a_token(cuda, dtype):
  """They leave the state that they came with, and hand its gradient on; as packed sequences without a token do."""
  b, c, n, w = 3, 40, 16, 4
  r = lambda *s, t=dtype: torch.randn(*s, device=cuda).to(t).requires_grad_(True)
  x, delta, z = r(b, 0, c), r(b, 0, c), r(b, 0, c)
  B, C = r(b, 0, 2, n), r(b, 0, 2, n)
  A, D, initial = r(c, n, t=F32), r(c, t=F32), r(b, c, n, t=F32)
  y, last = bpl.state_scan(x, delta, A, B, C, D, z=z, initial_state=initial, return_state=True)
  assert y.shape == (b, 0, c) and torch.equal(last, initial)
  cotangent = torch.randn_like(last)
  got = torch.autograd.grad([y, last], [x, delta, z, B, C, A, D, initial], [torch.zeros_like(y), cotangent])
  assert [g.shape for g in got[:5]] == [x.shape, x.shape, x.shape, B.shape, B.shape]
  assert not got[5].any() and not got[6].any() and torch.equal(got[7], cotangent)
  weight, bias, inputs = r(c, w), r(c), r(b, c, w - 1)
  y, last = bpl.short_conv(x, weight, bias, activation='silu', initial_state=inputs, return_state=True)
  assert y.shape == (b, 0, c) and torch.equal(last, inputs)
  cotangent = torch.randn_like(last)
  got = torch.autograd.grad([y, last], [x, weight, bias, inputs], [torch.zeros_like(y), cotangent])
  assert got[0].shape == x.shape and not got[1].any() and not got[2].any() and torch.equal(got[3], cotangent)


def test_no_rows_of_any_strides(cuda):
  """A tensor without rows is contiguous whatever its strides say, and has nothing to be copied."""
  x = torch.zeros(0, 32, device=cuda)[:, ::2]
  B = torch.zeros(0, 8, 4, device=cuda).transpose(1, 2)
  A = -torch.ones(16, 8, device=cuda)
  assert bpl.state_scan(x, x, A, B, B, z=x).shape == (0, 16)
  assert bpl.short_conv(x, torch.ones(16, 4, device=cuda)).shape == (0, 16)
  assert bpl.state_scan_step(x, x, A, B, B, torch.zeros(0, 16, 8, device=cuda), z=x).shape == (0, 16)
  assert bpl.short_conv_step(x, torch.zeros(0, 16, 3, device=cuda), torch.ones(16, 4, device=cuda)).shape == (0, 16)


# ---------------------------------------------------------------------------------------------------------
# infinities: what the definition makes of them, whether the states fill the lanes and the channels the blocks or not
# ---------------------------------------------------------------------------------------------------------
def positive(tokens, channels, state, groups=1, *, seed=0, delta=0.1, scale=1.0, dtype=F32):
  """Inputs of one sign, so that sums with infinite terms are infinite and no difference of infinities."""
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: (0.5 + torch.rand(*s, generator=g, dtype=torch.float64)).to(dtype)
  return dict(x=r(tokens, channels), delta=delta * r(tokens, channels), A=-scale * r(channels, state).to(F32), B=r(tokens, groups, state),
              C=r(tokens, groups, state), D=r(channels).to(F32), z=r(tokens, channels), delta_bias=None, softplus=False, initial=None)


def agree(got, want, most, operations, what):
  """As ``ref.check`` where the definition is finite; the same infinity where it is infinite; no claim where it is no number."""
  g = got.detach().double().cpu()
  far = torch.isinf(want)
  assert torch.equal(g[far], want[far]), f'{what}: {int((g[far] != want[far]).sum())} of {int(far.sum())} infinities lost'
  near = torch.isfinite(want)
  tol = ref.half_step(got.dtype) * want[near].abs() + operations * ref.U * most[near]
  assert ((g[near] - want[near]).abs() <= tol * (1 + 1e-9)).all(), what


def definition(d, bounds, **kw):
  w = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
  args = (w['x'], w['delta'], w['A'], w['B'], w['C'], w['D'], w['z'], w['delta_bias'], w['softplus'], bounds, w['initial'])
  return ref.scan(*args, **kw), ref.scan(*args, **kw, absolute=True)


def scan(d, cuda, bounds, leaf=False, return_state=True):
  g = {k: v.to(cuda).requires_grad_(leaf) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
  p = torch.tensor(bounds, dtype=torch.int32, device=cuda)
  return g, bpl.state_scan(g['x'], g['delta'], g['A'], g['B'], g['C'], g['D'], z=g['z'], delta_bias=g['delta_bias'],
                           delta_softplus=g['softplus'], indptr=p, initial_state=g['initial'], return_state=return_state)


STATES = [1, 2, 3, 4, 5, 10, 16, 17, 31, 50, 100, 128]


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('what', ['x', 'delta', 'initial'])
@pytest.mark.parametrize('state', STATES)
def test_an_infinite_input_is_infinite_to_the_end_of_its_sequence(cuda, state, what, dtype):
  bounds = [0, 9, 70, 90]
  pairs = list(zip(bounds[:-1], bounds[1:]))
  d = positive(95, 5, state, dtype=dtype, seed=state)
  if what == 'initial':
    d['initial'] = torch.rand(3, 5, state)
    d['initial'][1, 2] = float('inf')
  else:
    d[what][20, 2] = float('inf')
  want, most = definition(d, pairs)
  ops = 8 * 61 + state + 64
  y, last = scan(d, cuda, bounds)[1]
  assert torch.isinf(want['y'][30, 2]) and torch.isinf(want['last'][1, 2]).all()
  agree(y, want['y'], most['y'], ops, 'y')
  agree(last, want['last'], most['last'], ops, 'last')


@pytest.mark.parametrize('state', [1, 10, 16])
def test_an_infinite_time_passes_chunks(cuda, state):
  d = positive(3000, 5, state, scale=0.01, seed=state)
  d['delta'][20, 2] = float('inf')
  want, most = definition(d, [(0, 3000)])
  y, last = scan(d, cuda, [0, 3000])[1]
  assert torch.isinf(want['y'][20:, 2]).all()
  agree(y, want['y'], most['y'], 8 * 3000 + state + 64, 'y')
  agree(last, want['last'], most['last'], 8 * 3000 + state + 64, 'last')


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('what', ['x', 'delta', 'state'])
@pytest.mark.parametrize('rows,channels', [(5, 7), (120, 330)])
@pytest.mark.parametrize('state', STATES)
def test_a_step_with_an_infinite_input(cuda, state, rows, channels, what, dtype):
  d = positive(rows, channels, state, dtype=dtype, seed=state)
  d['initial'] = torch.rand(rows, channels, state)
  if what == 'state':
    d['initial'][3, 2] = float('inf')
  else:
    d[what][3, 2] = float('inf')
  want, most = definition(d, [(i, i + 1) for i in range(rows)])
  assert torch.isinf(want['y'][3, 2])
  g = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
  pool = g['initial'].clone()
  y = bpl.state_scan_step(g['x'], g['delta'], g['A'], g['B'], g['C'], pool, g['D'], z=g['z'])
  agree(y, want['y'], most['y'], state + 72, 'y')
  agree(pool, want['last'], most['last'], state + 72, 'state')


def gradients(d, cuda, bounds, dy, d_last):
  g, out = scan(d, cuda, bounds, True)
  names = [n for n in ('x', 'delta', 'A', 'B', 'C', 'D', 'z', 'delta_bias', 'initial') if g[n] is not None]
  return dict(zip(names, torch.autograd.grad(list(out), [g[n] for n in names], [dy.to(cuda), d_last.to(cuda)])))


def check_gradients(d, cuda, bounds, dy, d_last):
  pairs = list(zip(bounds[:-1], bounds[1:]))
  want, _ = definition(d, pairs, dy=dy.double(), d_last=d_last.double())
  # (the decay over an infinite time is 0 without an error, its majorant e^-t (1 + t) as well: taken at 10^4 here, where it is 0 in 64 bits)
  _, most = definition(dict(d, delta=d['delta'].double().clamp(max=1e4)), pairs, dy=dy.double(), d_last=d_last.double())
  tokens, channels = d['x'].shape
  ops = 16 * max(b - a for a, b in pairs) + 2 * d['A'].shape[1] + 128 + tokens + channels
  got = gradients(d, cuda, bounds, dy, d_last)
  for n, v in got.items():
    agree(v, want['d_' + n], most['d_' + n], ops, 'd_' + n)
  return got, want


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('what', ['x', 'delta', 'dy', 'B', 'C', 'initial', 'd_last'])
@pytest.mark.parametrize('state', STATES)
def test_gradients_beside_an_infinity(cuda, state, what, dtype):
  """Seven channels: the blocks are not full, and what stands beside them must not reach a sum over channels."""
  bounds = [0, 9, 70, 90]
  d = positive(95, 7, state, dtype=dtype, seed=state)
  if state % 2:
    d['D'] = d['z'] = None
  g = torch.Generator().manual_seed(1)
  dy = (0.5 + torch.rand(95, 7, generator=g, dtype=torch.float64)).to(dtype)
  d_last = 0.5 + torch.rand(3, 7, state, generator=g)
  d['initial'] = torch.rand(3, 7, state, generator=g)
  if what in ('initial', 'd_last'):
    (d['initial'] if what == 'initial' else d_last)[1, 2] = float('inf')
  elif what in ('B', 'C'):
    d[what][20, 0, 0] = float('inf')
  else:
    (dy if what == 'dy' else d[what])[20, 2] = float('inf')
  _, want = check_gradients(d, cuda, bounds, dy, d_last)
  assert any(torch.isinf(v).any() for k, v in want.items() if k.startswith('d_'))


def test_what_stands_behind_an_infinite_state_does_not_reach_the_rates(cuda):
  """The last token of the last sequence is infinite: no product of the sequence's gradient is, but what it multiplies."""
  for tokens, end in ((60, 20), (100, 32), (500, 17)):
    d = positive(tokens, 7, 16, seed=end)
    d['D'] = d['z'] = None
    d['x'][end - 1, 2] = float('inf')
    got, want = check_gradients(d, cuda, [0, end], torch.ones(tokens, 7), torch.zeros(1, 7, 16))
    assert torch.isfinite(want['d_A']).all() and torch.isfinite(got['A']).all()


def test_the_gradient_of_an_infinite_cotangent_without_a_skip(cuda):
  d = positive(40, 8, 16)
  d['D'] = d['z'] = None
  dy = torch.ones(40, 8)
  dy[20, 3] = float('inf')
  got, want = check_gradients(d, cuda, [0, 40], dy, torch.zeros(1, 8, 16))
  assert torch.isinf(got['x'][20, 3]) and torch.isinf(want['d_x'][20, 3])


# ---------------------------------------------------------------------------------------------------------
# states and gradients handed on through chunks of tokens
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('state', [1, 4, 10, 16])
def test_chunks_hand_on_what_single_tokens_would(cuda, state):
  """Few channels and thousands of tokens: a state passes chunks in one step.  Growth that would overflow over a chunk where there is
  nothing to grow, decays below the least number of 32 bits of a large state, infinite states."""
  tokens, channels = 3000, 8
  d = positive(tokens, channels, state, delta=1.0, scale=0.05, seed=state)
  d['D'] = d['z'] = None
  d['A'][0] = 2.0                                     # grows by e^2 to e^3 a token, for 20 tokens
  d['x'][:2980, 0] = 0
  d['A'][1] = -0.9                                    # from 1e37 to 1e-36 over about 190 tokens
  d['x'][:, 1] = 0
  d['x'][5, 1] = 1e37
  d['A'][2] = -3.0                                    # stays infinite
  d['x'][100, 2] = float('inf')
  d['A'][4], d['delta'][:, 4] = -1.6, 1.0             # 1e37 in front of a chunk whose decay is 2^-148
  d['x'][:, 4] = 0
  d['x'][63, 4] = 1e37
  want, most = definition(d, [(0, tokens)])
  y, last = scan(d, cuda, [0, tokens])[1]
  # (an exponent is rounded relative to its size: 200 tokens of exponents of 1 sum up to no more than the terms' bound)
  near = want['y'].abs() > 1e-30
  for c in range(channels):
    m = near[:, c]
    agree(y[:, c][m.to(cuda)], want['y'][:, c][m], most['y'][:, c][m], 8 * tokens + state + 64, f'y of channel {c}')
  assert torch.isposinf(y[100:, 2]).all() and torch.isposinf(last[0, 2]).all()
  assert torch.isfinite(y[:, 0]).all() and float(y[2999, 0]) > 1e10
  # (exponents of 102 in all from sums of 20 roundings: 102 * 20 * 2^-24 relative, and as much again for the tokens themselves)
  for t in (64, 127, 128):
    assert abs(float(y[t, 4]) / float(want['y'][t, 4]) - 1) <= 1e-3


@pytest.mark.parametrize('state', [4, 10, 16])
def test_chunks_hand_gradients_back_as_single_tokens_would(cuda, state):
  tokens, channels = 3000, 8
  d = positive(tokens, channels, state, delta=1.0, scale=0.05, seed=state)
  d['D'] = d['z'] = None
  d['A'][0] = 2.0                                     # the way back grows as well: only the first 20 tokens have a cotangent
  d['x'][:, 0] = 0
  dy = torch.ones(tokens, channels)
  dy[20:, 0] = 0
  d['A'][2] = -3.0
  dy[2900, 2] = float('inf')
  want, most = definition(d, [(0, tokens)], dy=dy.double(), d_last=torch.zeros(1, channels, state, dtype=torch.float64))
  got = gradients(d, cuda, [0, tokens], dy, torch.zeros(1, channels, state))
  for c in (0, 1, 3):
    agree(got['x'][:, c], want['d_x'][:, c], most['d_x'][:, c], 16 * tokens + 64, f'd_x of channel {c}')
  assert torch.isposinf(got['x'][:2901, 2]).all() and torch.isfinite(got['x'][2901:, 2]).all()


# ---------------------------------------------------------------------------------------------------------
# more blocks of channels than one launch of the gradient holds
# ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('tokens,channels,state,groups,dtype', [(2100, 6000, 100, 1, F32), (4444, 8000, 64, 1, BF16), (1500, 6000, 128, 2, BF16)])
def test_gradients_in_several_launches(cuda, tokens, channels, state, groups, dtype):
  g = torch.Generator().manual_seed(tokens)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
  d = dict(x=r(tokens, channels).to(dtype), delta=(0.1 * r(tokens, channels).abs()).to(dtype), A=-torch.exp(r(channels, state)).to(F32),
           B=r(tokens, groups, state).to(dtype), C=r(tokens, groups, state).to(dtype), D=r(channels).to(F32), z=r(tokens, channels).to(dtype),
           delta_bias=(0.05 * r(channels).abs()).to(F32), softplus=False, initial=None)
  dy, d_last = r(tokens, channels).to(dtype), torch.zeros(2, channels, state)
  bounds = [0, tokens // 3, tokens]
  one = 8 * tokens * groups * state
  lanes = 16 if state <= 64 else 32
  blocks = -(-channels // groups // (128 // lanes))
  scratch = workspace_bytes('state_scan_backward', struct.pack('<8I7q', tokens, 2, tokens, channels, groups, state,
                                                               {F32: 0, F16: 1, BF16: 2}[dtype], 0, *([channels] * 7)))
  assert scratch < blocks * one, 'all in one launch'
  got = gradients(d, cuda, bounds, dy, d_last)
  on_gpu = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
  want, most = definition(on_gpu, list(zip(bounds[:-1], bounds[1:])), dy=dy.double().to(cuda), d_last=d_last.double().to(cuda))
  operations = 16 * (tokens - tokens // 3) + 2 * state + 128
  for n, v in got.items():
    more = {'B': channels, 'C': channels, 'A': tokens, 'D': tokens, 'delta_bias': tokens}.get(n, 0)
    ref.check(v, want['d_' + n].cpu(), most['d_' + n].cpu(), operations + more, 'd_' + n)
  again = gradients(d, cuda, bounds, dy, d_last)
  assert all(torch.equal(got[n], again[n]) for n in got)
