"""The operators over whole sequences on operands as programs have them: parts of a wider projection, batches, long prompts in 16 bits;
and on operands of which every byte around is watched."""
import ctypes
import struct

import pytest
import torch

import brainpylib_b200 as bpl
import sequence_reference as ref
import test_short_conv_gpu as convs
import test_state_scan_gpu as scans
from brainpylib_b200 import _lib

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gradients_of_scan(d, bounds, dy, d_last):
  pairs = list(zip(bounds[:-1], bounds[1:]))
  want, most = scans.reference(d, pairs, dy=dy.double(), d_last=d_last.double())
  return want, most, 2 * scans.operations(pairs, d['A'].shape[1])


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('state,groups,shift', [(16, 2, 0), (10, 3, 1), (33, 1, 3)])
def test_gradients_through_parts_of_a_projection(cuda, state, groups, shift, dtype):
  """x, z, delta, B and C are columns of one projection of a batch, which begins at any element."""
  b, length, c = 3, 37, 48
  d = scans.inputs(b * length, c, state, groups, dtype, sequences=b, seed=state)
  bounds = [i * length for i in range(b + 1)]
  dy, d_last = scans.cotangents(d, b)
  sizes = [shift, c, c, c, groups * state, groups * state, 2]
  r = lambda n: torch.zeros(b * length, n, dtype=dtype)
  wide = torch.cat([r(shift), d['x'], d['z'], d['delta'], d['B'].flatten(1), d['C'].flatten(1), r(2)], 1).reshape(b, length, -1)
  wide = wide.to(cuda).requires_grad_(True)
  g = {k: v.to(cuda).requires_grad_(True) for k, v in d.items() if k in ('A', 'D', 'delta_bias', 'initial')}
  _, x, z, delta, B, C, _ = wide.split(sizes, 2)
  B, C = (t.unflatten(2, (groups, state)) for t in (B, C))
  out = bpl.state_scan(x, delta, g['A'], B, C, g['D'], z=z, delta_bias=g['delta_bias'], delta_softplus=True, initial_state=g['initial'],
                       return_state=True)
  got = torch.autograd.grad(list(out), [wide, *g.values()], [dy.to(cuda).reshape(b, length, c), d_last.to(cuda)])
  want, most, ops = gradients_of_scan(d, bounds, dy, d_last)
  parts = dict(zip(['_', 'x', 'z', 'delta', 'B', 'C', '__'], got[0].reshape(b * length, -1).split(sizes, 1)))
  assert not parts['_'].any() and not parts['__'].any()
  for n in ('x', 'z', 'delta', 'B', 'C'):
    ref.check(parts[n].reshape(want['d_' + n].shape), want['d_' + n], most['d_' + n], ops + (c if n in 'BC' else 0), 'd_' + n)
  for n, v in zip(g, got[1:]):
    ref.check(v, want['d_' + n], most['d_' + n], ops + b * length, 'd_' + n)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('width,shift', [(4, 0), (3, 1), (2, 4)])
def test_gradients_of_the_convolution_through_parts_of_a_projection(cuda, width, shift, dtype):
  b, length, c = 3, 37, 48
  d = convs.inputs(b * length, c, width, dtype, sequences=b, seed=width)
  bounds = [(i * length, (i + 1) * length) for i in range(b)]
  g = torch.Generator().manual_seed(7)
  dy = torch.randn(b * length, c, generator=g, dtype=torch.float64).to(dtype)
  d_last = torch.randn(b, c, width - 1, generator=g, dtype=torch.float64).to(dtype)
  wide = torch.cat([torch.zeros(b * length, shift, dtype=dtype), d['x'], torch.zeros(b * length, 5, dtype=dtype)], 1)
  wide = wide.reshape(b, length, -1).to(cuda).requires_grad_(True)
  p = {k: v.to(cuda).requires_grad_(True) for k, v in d.items() if k != 'x'}
  out = bpl.short_conv(wide[:, :, shift:shift + c], p['weight'], p['bias'], activation='silu', initial_state=p['initial'], return_state=True)
  got = torch.autograd.grad(list(out), [wide, *p.values()], [dy.to(cuda).reshape(b, length, c), d_last.to(cuda)])
  want, most = convs.reference(d, bounds, True, dy=dy.double(), d_last=d_last.double())
  ref.check(got[0].reshape(b * length, -1)[:, shift:shift + c], want['d_x'], most['d_x'], 64, 'd_x')
  for n, v in zip(p, got[1:]):
    ref.check(v, want['d_' + n], most['d_' + n], 64 + b * length, 'd_' + n)


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('state', [10, 16])
def test_long_prompts_in_16_bits(cuda, state, dtype):
  """Few channels: states and gradients pass chunks of tokens."""
  for tokens, bounds in ((2500, [0, 2500]), (1300, [0, 433, 434, 434, 1295])):
    pairs = list(zip(bounds[:-1], bounds[1:]))
    d = scans.inputs(tokens, 24, state, 2, dtype, sequences=len(pairs), scale=0.05, seed=state)
    scans.check_forward(d, pairs, scans.run(d, cuda, bounds))
    scans.check_gradients(d, cuda, bounds, *scans.cotangents(d, len(pairs)))


# ---------------------------------------------------------------------------------------------------------
# every byte around the operands
# ---------------------------------------------------------------------------------------------------------
class Arena:
  """Operands cut out of one buffer.  Around those that are read lie numbers that are none, which must not reach a result; around those that
  are written, and in the scratch memory, a pattern, which must be as it was around them."""
  GUARD, PATTERN = 8192, 0x3c                 # (as numbers: 0.0115 in 32 bits and in bfloat16)

  def __init__(self, cuda):
    self.read = torch.full((1 << 22,), 0xff, dtype=torch.uint8, device=cuda)
    self.written = torch.full((1 << 26,), self.PATTERN, dtype=torch.uint8, device=cuda)
    self.at, self.out, self.given = [self.GUARD, self.GUARD], [], []

  def _cut(self, which, nbytes):
    start = self.at[which]
    self.at[which] += -(-nbytes // 256) * 256 + self.GUARD
    buffer = (self.read, self.written)[which]
    assert self.at[which] <= buffer.numel()
    return start, buffer[start:start + nbytes]

  def operand(self, t):
    if t is None:
      return None
    _, place = self._cut(0, t.numel() * t.element_size())
    view = place.view(t.dtype).reshape(t.shape)
    self.given.append((view, t.clone()))
    return view.copy_(t)

  def result(self, shape, dtype):
    nbytes = torch.empty(shape, dtype=dtype, device='meta').numel() * dtype.itemsize
    start, place = self._cut(1, nbytes)
    self.out.append((start, nbytes))
    return place.view(dtype).reshape(shape)

  def check(self):
    torch.cuda.synchronize()
    for view, t in self.given:
      assert torch.equal(view, t.to(view.device)), 'an operand was written'
    rest = torch.ones(self.written.numel(), dtype=torch.bool, device=self.written.device)
    for start, nbytes in self.out:
      rest[start:start + nbytes] = False
    assert (self.written[rest] == self.PATTERN).all(), 'bytes beside the results were written'


def call(name, opaque, buffers):
  _lib.lib().bpl_clear_status()
  pointers = (ctypes.c_void_p * len(buffers))(*[None if t is None or t.numel() == 0 else t.data_ptr() for t in buffers])
  _lib.target(name)(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), pointers, opaque, len(opaque))
  message = ctypes.create_string_buffer(256)
  assert _lib.lib().bpl_last_status(message, 256) == 0, message.value


BOUNDS = [[0, 40], [3, 17, 17, 31], [-5, 10, 3, 50, 2000000000, 7], [40, 30, 20, 10, 5, 0], [-2 ** 31, 2 ** 31 - 1, 0, 40, -1, 40], [9]]


@pytest.mark.parametrize('dtype,code', [(F32, 0), (BF16, 2)])
@pytest.mark.parametrize('channels,state,groups', [(30, 16, 1), (33, 10, 3), (7, 3, 1), (20, 128, 2)])
@pytest.mark.parametrize('tokens', [40, 700])
def test_the_scan_and_its_gradient_stay_inside_their_operands(cuda, tokens, channels, state, groups, dtype, code):
  """Bounds below zero, beyond the rows and out of order among them: whatever comes out of those, nothing else is read or written."""
  for bounds in BOUNDS:
    if tokens != 40:
      bounds = [v * 17 if 0 < v <= 50 else v for v in bounds]
    n = len(bounds) - 1
    d = scans.inputs(tokens, channels, state, groups, dtype, sequences=n, seed=tokens)
    dy, d_last = scans.cotangents(d, n)
    a = Arena(cuda)
    x, delta, A, B, C, D, z, bias, initial = (a.operand(d[k]) for k in ('x', 'delta', 'A', 'B', 'C', 'D', 'z', 'delta_bias', 'initial'))
    indptr = a.operand(torch.tensor(bounds, dtype=torch.int32))
    y, last = a.result((tokens, channels), dtype), a.result((n, channels, state), F32)
    saved = a.result((-(-tokens // 16), channels, state), F32)
    opaque = struct.pack('<8I7q', tokens, n, 0, channels, groups, state, code, 1, channels, channels, channels, groups * state, state,
                         groups * state, state)
    scratch = a.result((_lib.workspace_bytes('state_scan', opaque),), torch.uint8)
    operands = [x, delta, A, B, C, D, z, bias, indptr, initial]
    call('state_scan', opaque, operands + [y, last, saved, scratch])
    a.check()
    grown = [a.operand(dy), a.operand(d_last)]
    results = [a.result(t.shape, t.dtype) for t in (x, delta, A, B, C, D, z, bias, initial)]
    scratch = a.result((_lib.workspace_bytes('state_scan_backward', opaque),), torch.uint8)
    call('state_scan_backward', opaque, operands + [saved] + grown + results + [scratch])
    a.check()
    for t in [y, last] + results:
      assert not torch.isnan(t).any()


@pytest.mark.parametrize('dtype,code', [(F32, 0), (BF16, 2)])
@pytest.mark.parametrize('channels,width', [(30, 4), (33, 3), (64, 8), (5, 1)])
@pytest.mark.parametrize('tokens', [40, 700])
def test_the_convolution_and_its_gradient_stay_inside_their_operands(cuda, tokens, channels, width, dtype, code):
  for bounds in BOUNDS:
    if tokens != 40:
      bounds = [v * 17 if 0 < v <= 50 else v for v in bounds]
    n = len(bounds) - 1
    d = convs.inputs(tokens, channels, width, dtype, sequences=n, seed=tokens)
    g = torch.Generator().manual_seed(7)
    a = Arena(cuda)
    x, weight, bias, initial = (a.operand(d[k]) for k in ('x', 'weight', 'bias', 'initial'))
    indptr = a.operand(torch.tensor(bounds, dtype=torch.int32))
    y, last = a.result((tokens, channels), dtype), a.result((n, channels, width - 1), dtype)
    opaque = struct.pack('<8Iq', tokens, n, 0, channels, width, code, code, 1, channels)
    operands = [x, weight, bias, indptr, initial]
    call('short_conv', opaque, operands + [y, last])
    a.check()
    grown = [a.operand(torch.randn(tokens, channels, generator=g).to(dtype)), a.operand(torch.randn(n, channels, width - 1, generator=g).to(dtype))]
    results = [a.result(t.shape, t.dtype) for t in (x, weight, bias, initial)]
    scratch = a.result((_lib.workspace_bytes('short_conv_backward', opaque),), torch.uint8)
    call('short_conv_backward', opaque, operands + grown + results + [scratch])
    a.check()
    for t in [y, last] + results:
      assert not torch.isnan(t).any()


@pytest.mark.parametrize('dtype,code', [(F32, 0), (BF16, 2)])
@pytest.mark.parametrize('rows,channels,state', [(5, 33, 10), (200, 260, 16), (200, 260, 33)])
def test_the_single_steps_stay_inside_their_operands(cuda, rows, channels, state, dtype, code):
  """Slots beyond the pool, taken ones and padding."""
  d = scans.inputs(rows, channels, state, 1, dtype, initial=False, seed=rows)
  c = convs.inputs(rows, channels, 4, dtype, initial=False, seed=rows)
  slots = torch.arange(rows, dtype=torch.int32)
  slots[1:5] = torch.tensor([0, -1, 2 ** 31 - 1, rows], dtype=torch.int32)
  a = Arena(cuda)
  operands = [a.operand(d[k]) for k in ('x', 'delta', 'A', 'B', 'C', 'D', 'z', 'delta_bias')] + [a.operand(slots)]
  pool, y = a.result((rows, channels, state), F32).fill_(1), a.result((rows, channels), dtype)
  opaque = struct.pack('<8I7q', rows, rows, 0, channels, 1, state, code, 1, channels, channels, channels, state, 0, state, 0)
  call('state_scan_step', opaque, operands + [pool, y])
  a.check()
  bad = torch.tensor([1, 3, 4], device=cuda)
  good = torch.ones(rows, dtype=torch.bool, device=cuda)
  good[bad] = False
  assert torch.isnan(y[bad]).all() and not torch.isnan(y[good]).any() and not y[2].any() and (pool[1:5] == 1).all()
  operands = [a.operand(c[k]) for k in ('x', 'weight', 'bias')] + [operands[-1]]
  pool, y = a.result((rows, channels, 3), dtype).fill_(1), a.result((rows, channels), dtype)
  call('short_conv_step', struct.pack('<8Iq', rows, rows, 0, channels, 4, code, code, 1, channels), operands + [pool, y])
  a.check()
  assert torch.isnan(y[bad]).all() and not torch.isnan(y[good]).any() and not y[2].any() and (pool[1:5] == 1).all()
