"""``state_scan`` and ``state_scan_step`` against the plain statement in 64 bits, at sizes and bounds where a kernel that works
in tiles of tokens, lanes of states and chunks of long runs can go wrong."""
import pytest
import torch

import brainpylib_b200 as bpl
import sequence_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# roundings of a term: 8 for every token of its sequence (state), the time step (softplus: 16), products, the sum over up to
# 128 states, skip, gate (16)
def operations(bounds, state):
  return 8 * max([e - b for b, e in bounds] + [0]) + state + 64


def inputs(tokens, channels, state, groups=1, dtype=F32, *, sequences=1, gate=True, extras=True, initial=True, softplus=True,
           seed=0, scale=1.0):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
  d = dict(x=r(tokens, channels).to(dtype), delta=(0.5 * r(tokens, channels) - (2 if softplus else 0)).to(dtype),
           A=(-torch.exp(r(channels, state)) * scale).to(F32), B=r(tokens, groups, state).to(dtype),
           C=r(tokens, groups, state).to(dtype), D=None, z=None, delta_bias=None, initial=None, softplus=softplus)
  if not softplus:
    d['delta'] = d['delta'].abs() * 0.1
  if gate:
    d['z'] = r(tokens, channels).to(dtype)
  if extras:
    d['D'], d['delta_bias'] = r(channels).to(F32), (0.3 * r(channels) - 1).to(F32)
    if not softplus:
      d['delta_bias'] = d['delta_bias'].abs() * 0.05
  if initial:
    d['initial'] = r(sequences, channels, state).to(F32)
  return d


def wide(d):
  return {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def reference(d, bounds, **kw):
  w = wide(d)
  args = (w['x'], w['delta'], w['A'], w['B'], w['C'], w['D'], w['z'], w['delta_bias'], w['softplus'], bounds, w['initial'])
  return ref.scan(*args, **kw), ref.scan(*args, **kw, absolute=True)


def run(d, cuda, indptr=None, **kw):
  g = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
  p = None if indptr is None else torch.tensor(indptr, dtype=torch.int32, device=cuda)
  return bpl.state_scan(g['x'], g['delta'], g['A'], g['B'], g['C'], g['D'], z=g['z'], delta_bias=g['delta_bias'],
                        delta_softplus=g['softplus'], indptr=p, initial_state=g['initial'], return_state=True, **kw)


def check_forward(d, bounds, got):
  want, most = reference(d, bounds)
  ops = operations(bounds, d['A'].shape[1])
  ref.check(got[0].reshape(want['y'].shape), want['y'], most['y'], ops, 'y')
  ref.check(got[1], want['last'], most['last'], ops, 'last')


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('channels,state,groups', [(1, 1, 1), (33, 4, 1), (64, 16, 2), (75, 10, 3), (40, 16, 40), (130, 17, 1),
                                                   (24, 64, 2), (9, 128, 3), (300, 3, 1)])
def test_one_sequence_of_odd_sizes(cuda, channels, state, groups, dtype):
  for tokens in (1, 2, 15, 16, 17, 47):
    d = inputs(tokens, channels, state, groups, dtype, seed=tokens)
    check_forward(d, [(0, tokens)], run(d, cuda))


@pytest.mark.parametrize('softplus,gate,extras,initial', [(True, False, True, False), (False, True, False, True),
                                                          (False, False, False, False)])
def test_operands_left_out(cuda, softplus, gate, extras, initial):
  d = inputs(37, 50, 16, 1, BF16, gate=gate, extras=extras, initial=initial, softplus=softplus)
  check_forward(d, [(0, 37)], run(d, cuda))


BOUNDS = [[0, 1, 2, 3, 4, 5, 40], [0, 0, 16, 32, 32, 32, 33, 80, 80], [3, 19, 35, 50], [0, 64, 128], [7, 7, 7], [5, 70, 71, 90],
          [0, 200, 205, 300], [0], [40]]


@pytest.mark.parametrize('bounds', BOUNDS, ids=str)
def test_packed_sequences(cuda, bounds):
  """Empty sequences, sequences of one token, bounds on and beside those of tiles; rows in front of the first and behind the
  last one hold NaN and are left out."""
  tokens = bounds[-1] + 21
  pairs = list(zip(bounds[:-1], bounds[1:]))
  for initial in (True, False):
    d = inputs(tokens, 70, 16, 2, F32, sequences=len(pairs), initial=initial, seed=bounds[-1])
    for k in ('x', 'delta', 'B', 'C', 'z'):
      d[k][:bounds[0]] = float('nan')
      d[k][bounds[-1]:] = float('nan')
    got = run(d, cuda, bounds)
    for k in ('x', 'delta', 'B', 'C', 'z'):
      d[k][:bounds[0]] = 0
      d[k][bounds[-1]:] = 0
    check_forward(d, pairs, got)
    assert not got[0][bounds[-1]:].any() and not got[0][:bounds[0]].any()


@pytest.mark.parametrize('tokens,channels,state', [(3000, 8, 16), (2500, 16, 4), (1111, 5, 100)])
def test_long_runs_shared_out_in_chunks(cuda, tokens, channels, state):
  """Few channels: the tokens are cut into chunks, and states handed on through all of them; slow decays keep the first ones."""
  d = inputs(tokens, channels, state, 1, F32, scale=0.01, seed=3)
  check_forward(d, [(0, tokens)], run(d, cuda))
  bounds = [0, tokens // 3, tokens // 3 + 1, tokens // 3 + 1, tokens - 5]
  d = inputs(tokens, channels, state, 1, F32, sequences=4, scale=0.01, seed=4)
  check_forward(d, list(zip(bounds[:-1], bounds[1:])), run(d, cuda, bounds))


def test_an_infinite_state_stays_in_its_sequence(cuda):
  d = inputs(60, 40, 16, 1, F32, sequences=3, seed=5)
  d['x'][20:25] = float('inf')
  y, last = run(d, cuda, [0, 16, 30, 60])
  want, most = reference(d, [(0, 16), (16, 30), (30, 60)])
  ops = operations([(0, 30)], 16)
  for rows in (slice(0, 16), slice(30, 60)):
    ref.check(y[rows], want['y'][rows], most['y'][rows], ops)
  ref.check(last[0::2], want['last'][0::2], most['last'][0::2], ops)
  assert not torch.isfinite(y[20:30]).any()


def test_batches_and_strided_rows_are_the_packed_call(cuda):
  """A batch of equal sequences, rows that are parts of a wider projection, a batch whose rows have no single distance."""
  b, length, c, n = 3, 29, 48, 16
  d = inputs(b * length, c, n, 2, BF16, sequences=b, seed=6)
  bounds = [i * length for i in range(b + 1)]
  y, last = run(d, cuda, bounds)
  g = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
  fold = lambda t: t.reshape(b, length, *t.shape[1:])
  wide_rows = torch.cat([fold(g['x']), fold(g['z']), fold(g['delta']), fold(g['B']).flatten(2), fold(g['C']).flatten(2)], 2)
  parts = wide_rows.split([c, c, c, 2 * n, 2 * n], 2)
  kw = dict(delta_bias=g['delta_bias'], delta_softplus=True, initial_state=g['initial'], return_state=True)
  B, C = (p.unflatten(2, (2, n)) for p in parts[3:])
  y2, last2 = bpl.state_scan(parts[0], parts[2], g['A'], B, C, g['D'], z=parts[1], **kw)
  assert torch.equal(y2.reshape(-1, c), y) and torch.equal(last2, last)
  odd = torch.zeros(b, length + 2, c + 1, dtype=BF16, device=cuda)[:, 1:-1, 1:]
  odd.copy_(fold(g['x']))
  y3, last3 = bpl.state_scan(odd, fold(g['delta']), g['A'], fold(g['B']), fold(g['C']), g['D'], z=fold(g['z']).transpose(0, 1)
                             .contiguous().transpose(0, 1), **kw)
  assert torch.equal(y3.reshape(-1, c), y) and torch.equal(last3, last)


def test_no_rows_and_no_sequences(cuda):
  d = inputs(0, 8, 4, 1, F32, sequences=2)
  y, last = run(d, cuda, [0, 0, 0])
  assert y.shape == (0, 8) and torch.equal(last.cpu(), d['initial'])
  d = inputs(5, 8, 4, 1, F32, sequences=0)
  y, last = run(d, cuda, [0])
  assert not y.any() and last.shape == (0, 8, 4)


def test_a_prompt_in_one_call_in_parts_and_token_by_token(cuda):
  """The last state of a part continues it; single steps on a pool continue a prompt."""
  d = inputs(50, 72, 16, 1, F32, initial=False, seed=8)
  y, last = run(d, cuda)
  head = {k: v[:31] if k in ('x', 'delta', 'B', 'C', 'z') else v for k, v in d.items()}
  tail = {k: v[31:] if k in ('x', 'delta', 'B', 'C', 'z') else v for k, v in d.items()}
  y1, s1 = run(head, cuda)
  tail['initial'] = s1.cpu()
  y2, s2 = run(tail, cuda)
  assert torch.equal(torch.cat([y1, y2]), y) and torch.equal(s2, last)
  pool = torch.full((4, 72, 16), 7.0, device=cuda)
  pool[2] = s1[0]
  slots = torch.tensor([2], dtype=torch.int32, device=cuda)
  g = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
  want, most = reference(d, [(0, 50)])
  for t in range(31, 50):
    yt = bpl.state_scan_step(g['x'][t:t + 1], g['delta'][t:t + 1], g['A'], g['B'][t:t + 1], g['C'][t:t + 1], pool, g['D'],
                             z=g['z'][t:t + 1], delta_bias=g['delta_bias'], delta_softplus=True, slots=slots)
    ref.check(yt[0], want['y'][t], most['y'][t], operations([(0, 50)], 16))
  ref.check(pool[2], want['last'][0], most['last'][0], operations([(0, 50)], 16))
  assert (pool[[0, 1, 3]] == 7).all()


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,channels,state,groups', [(1, 64, 16, 1), (5, 33, 1, 1), (9, 70, 23, 2), (3, 20, 128, 4), (40, 260, 8, 1),
                                                      (301, 130, 16, 1), (95, 402, 7, 3), (150, 258, 33, 2)])
def test_single_steps_on_a_pool(cuda, rows, channels, state, groups, dtype):
  """Rows in any order of the pool, padding rows in between; the rest of the pool stays as it is."""
  for gate, extras in ((True, True), (False, False)):
    d = inputs(rows, channels, state, groups, dtype, gate=gate, extras=extras, initial=False, seed=rows)
    pool = torch.randn(rows + 3, channels, state, generator=torch.Generator().manual_seed(1))
    slots = torch.randperm(rows + 3, generator=torch.Generator().manual_seed(2))[:rows].to(torch.int32)
    slots[1::4] = -1 - slots[1::4]
    bounds = [(i, i + 1) for i in range(rows)]
    d['initial'] = pool[slots.clamp(min=0).long()]
    want, most = reference(d, bounds)
    g = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    state_gpu = pool.to(cuda)
    B, C = (g['B'], g['C']) if groups > 1 else (g['B'][:, 0], g['C'][:, 0])
    y = bpl.state_scan_step(g['x'], g['delta'], g['A'], B, C, state_gpu, g['D'], z=g['z'], delta_bias=g['delta_bias'],
                            delta_softplus=True, slots=slots.to(cuda))
    live = slots >= 0
    ops = operations([(0, 1)], state)
    ref.check(y[live.to(cuda)], want['y'][live], most['y'][live], ops, 'y')
    assert not y[(~live).to(cuda)].any()
    after = pool.double().clone()
    after[slots[live].long()] = want['last'][live]
    major = torch.zeros_like(after)
    major[slots[live].long()] = most['last'][live]
    ref.check(state_gpu, after, major, ops, 'state')


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows,channels,state,groups', [(200, 190, 20, 1), (100, 380, 128, 2), (95, 402, 61, 3), (38, 1000, 64, 4)])
def test_single_steps_of_many_rows_and_states(cuda, rows, channels, state, groups, dtype):
  test_single_steps_on_a_pool(cuda, rows, channels, state, groups, dtype)


def test_steps_with_slots_that_are_taken_or_beyond_the_pool(cuda):
  """The first row of a slot goes through; later ones, and slots beyond the pool, get NaN and change nothing."""
  for channels in (40, 200):
    taken_or_beyond(cuda, channels)


def test_steps_of_many_rows_and_states_that_are_taken(cuda):
  """The same where lanes hold eight states each."""
  for state in (20, 40, 100):
    taken_or_beyond(cuda, 130, state)


def taken_or_beyond(cuda, channels, state=16):
  d = inputs(300, channels, state, 1, F32, initial=False, seed=9)
  g = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
  slots = torch.arange(300, dtype=torch.int32)
  slots[[7, 150, 299]] = 3
  slots[9] = 300
  slots[10] = 2 ** 31 - 1
  bad = torch.zeros(300, dtype=torch.bool)
  bad[[7, 9, 10, 150, 299]] = True
  pool = torch.randn(300, channels, state, device=cuda, generator=torch.Generator(cuda).manual_seed(3))
  args = lambda i: (g['x'][i], g['delta'][i], g['A'], g['B'][i], g['C'][i])
  kw = lambda i: dict(z=g['z'][i], delta_bias=g['delta_bias'], delta_softplus=True)
  good = torch.nonzero(~bad)[:, 0].to(cuda)
  alone = pool.clone()
  want = bpl.state_scan_step(*args(good), alone, g['D'], slots=slots[~bad].to(cuda), **kw(good))
  every = torch.arange(300, device=cuda)
  y = bpl.state_scan_step(*args(every), pool, g['D'], slots=slots.to(cuda), **kw(every))
  assert torch.equal(y[good], want) and torch.isnan(y[bad.to(cuda)]).all() and torch.equal(pool, alone)


def test_bounds_that_are_no_bounds_touch_nothing_outside(cuda):
  """Bounds below zero, beyond the rows and out of order: whatever comes out, the call stays inside its operands."""
  d = inputs(40, 30, 16, 1, F32, sequences=5, seed=10)
  for bounds in ([-5, 10, 3, 50, 2000000000, 7], [40, 30, 20, 10, 5, 0], [-2 ** 31, 2 ** 31 - 1, 0, 40, -1, 40]):
    y, last = run(d, cuda, bounds)
    assert y.shape == (40, 30) and last.shape == (5, 30, 16)
  torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------------------------
# gradients
# ---------------------------------------------------------------------------------------------------------
def leaves(d, cuda):
  return {k: v.to(cuda).requires_grad_(True) if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def call(g, cuda, bounds=None, return_state=True):
  p = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=cuda)
  return bpl.state_scan(g['x'], g['delta'], g['A'], g['B'], g['C'], g['D'], z=g['z'], delta_bias=g['delta_bias'],
                        delta_softplus=g['softplus'], indptr=p, initial_state=g['initial'], return_state=return_state)


def cotangents(d, sequences, seed=11):
  g = torch.Generator().manual_seed(seed)
  dy = torch.randn(d['x'].shape, generator=g, dtype=torch.float64).to(d['x'].dtype)
  return dy, torch.randn(sequences, *d['A'].shape, generator=g, dtype=torch.float64).to(F32)


NAMES = ('x', 'delta', 'A', 'B', 'C', 'D', 'z', 'delta_bias', 'initial')


def check_gradients(d, cuda, bounds, dy, d_last):
  """A term passes forwards and backwards through its sequence (16 roundings a token), and sums over the channels of a group or
  over all tokens."""
  pairs = list(zip(bounds[:-1], bounds[1:]))
  g = leaves(d, cuda)
  y, last = call(g, cuda, bounds)
  names = [n for n in NAMES if g[n] is not None]
  got = torch.autograd.grad([y, last], [g[n] for n in names], [dy.to(cuda), d_last.to(cuda)])
  want, most = reference(d, pairs, dy=dy.double(), d_last=d_last.double())
  tokens, channels = d['x'].shape
  for n, v in zip(names, got):
    summed = {'B': channels, 'C': channels, 'A': tokens, 'D': tokens, 'delta_bias': tokens}.get(n, 0)
    ref.check(v, want['d_' + n], most['d_' + n], 2 * operations(pairs, d['A'].shape[1]) + summed, 'd_' + n)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('channels,state,groups', [(1, 1, 1), (33, 4, 1), (64, 16, 2), (75, 10, 3), (12, 16, 12), (130, 17, 1),
                                                   (24, 64, 2), (9, 128, 3), (200, 2, 1)])
def test_gradients_of_odd_sizes(cuda, channels, state, groups, dtype):
  for tokens in (1, 16, 17, 45):
    d = inputs(tokens, channels, state, groups, dtype, seed=tokens)
    check_gradients(d, cuda, [0, tokens], *cotangents(d, 1))


@pytest.mark.parametrize('bounds', BOUNDS, ids=str)
def test_gradients_of_packed_sequences(cuda, bounds):
  d = inputs(bounds[-1] + 21, 70, 16, 2, F32, sequences=len(bounds) - 1, seed=bounds[-1])
  dy, d_last = cotangents(d, len(bounds) - 1)
  for k in ('x', 'delta', 'B', 'C', 'z'):
    d[k][:bounds[0]] = 0
    d[k][bounds[-1]:] = 0
  check_gradients(d, cuda, bounds, dy, d_last)
  # what stands in rows outside does not reach a gradient
  g = leaves(d, cuda)
  want = torch.autograd.grad(call(g, cuda, bounds, False), [g[n] for n in NAMES], dy.to(cuda))
  for k in ('x', 'delta', 'B', 'C', 'z'):
    d[k][:bounds[0]] = float('nan')
    d[k][bounds[-1]:] = float('inf')
  dy[:bounds[0]] = float('nan')
  dy[bounds[-1]:] = float('nan')
  g = leaves(d, cuda)
  for a, b in zip(torch.autograd.grad(call(g, cuda, bounds, False), [g[n] for n in NAMES], dy.to(cuda)), want):
    assert torch.equal(a, b)


@pytest.mark.parametrize('tokens,channels,state', [(1500, 8, 16), (1111, 5, 100)])
def test_gradients_of_long_runs(cuda, tokens, channels, state):
  d = inputs(tokens, channels, state, 1, F32, scale=0.01, seed=3)
  check_gradients(d, cuda, [0, tokens], *cotangents(d, 1))
  bounds = [0, tokens // 3, tokens // 3 + 1, tokens // 3 + 1, tokens - 5]
  d = inputs(tokens, channels, state, 1, F32, sequences=4, scale=0.01, seed=4)
  check_gradients(d, cuda, bounds, *cotangents(d, 4))


@pytest.mark.parametrize('softplus,gate,extras,initial', [(True, False, True, False), (False, True, False, True),
                                                          (False, False, False, False)])
def test_gradients_with_operands_left_out(cuda, softplus, gate, extras, initial):
  d = inputs(37, 50, 16, 1, F32, gate=gate, extras=extras, initial=initial, softplus=softplus)
  check_gradients(d, cuda, [0, 37], *cotangents(d, 1))


def test_gradient_against_differences(cuda):
  """The gradient along a direction against the central difference of the definition: with steps of 2^-10 along a direction of
  size 1 the difference itself is off by the third derivative times 2^-20 / 6, here below 1e-4 of the result (checked by halving
  the step: the two differences agree to 4 times that)."""
  d = inputs(40, 24, 8, 2, F32, sequences=2, seed=21)
  bounds = [0, 23, 40]
  pairs = [(0, 23), (23, 40)]
  dy, d_last = cotangents(d, 2)
  g = leaves(d, cuda)
  got = torch.autograd.grad(call(g, cuda, bounds), [g[n] for n in NAMES], [dy.to(cuda), d_last.to(cuda)])
  w = wide(d)
  gen = torch.Generator().manual_seed(5)

  def loss(name, at):
    v = dict(w, **{name: at})
    r = ref.scan(v['x'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], True, pairs, v['initial'])
    return float((r['y'] * dy.double()).sum() + (r['last'] * d_last.double()).sum())

  for n, v in zip(NAMES, got):
    way = torch.randn(w[n].shape, generator=gen, dtype=torch.float64)
    way /= way.norm()
    slope = [(loss(n, w[n] + h * way) - loss(n, w[n] - h * way)) / (2 * h) for h in (2.0 ** -10, 2.0 ** -11)]
    scale = float(v.double().norm())
    assert abs(slope[0] - slope[1]) <= 4e-4 * scale, n
    assert abs(float((v.double().cpu() * way).sum()) - slope[1]) <= 2e-4 * scale, n


def test_gradients_of_inputs_that_were_broadcast(cuda):
  """Expanded operands: their gradients come back summed."""
  d = inputs(30, 40, 16, 1, F32, gate=False, initial=False, seed=12)
  g = leaves(d, cuda)
  step = torch.full((1, 40), -1.5, device=cuda, requires_grad=True)
  wide_step = step.expand(30, 40)
  y = bpl.state_scan(g['x'], wide_step, g['A'], g['B'], g['C'], delta_softplus=True)
  dy = torch.randn(30, 40, device=cuda, generator=torch.Generator(cuda).manual_seed(1))
  a, = torch.autograd.grad(y, step, dy, retain_graph=True)
  full = wide_step.detach().clone().requires_grad_(True)
  b, = torch.autograd.grad(bpl.state_scan(g['x'], full, g['A'], g['B'], g['C'], delta_softplus=True), full, dy)
  assert torch.equal(a, b.sum(0, keepdim=True))


def test_the_same_call_gives_the_same_bits_and_only_once_differentiable(cuda):
  d = inputs(700, 90, 16, 3, BF16, seed=13)
  dy, d_last = cotangents(d, 1)
  g = leaves(d, cuda)
  names = [n for n in NAMES]
  runs = [torch.autograd.grad(call(g, cuda), [g[n] for n in names], [dy.to(cuda), d_last.to(cuda)]) for _ in range(3)]
  for other in runs[1:]:
    assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
  first, = torch.autograd.grad(call(g, cuda, return_state=False), g['x'], dy.to(cuda), create_graph=True)
  with pytest.raises(RuntimeError):
    first.float().sum().backward()


def test_only_the_last_state_has_a_gradient(cuda):
  d = inputs(20, 16, 8, 1, F32, seed=14)
  _, d_last = cotangents(d, 1)
  g = leaves(d, cuda)
  _, last = call(g, cuda)
  got, = torch.autograd.grad(last, g['x'], d_last.to(cuda))
  want, most = reference(d, [(0, 20)], dy=torch.zeros(20, 16, dtype=torch.float64), d_last=d_last.double())
  ref.check(got, want['d_x'], most['d_x'], 2 * operations([(0, 20)], 8))
