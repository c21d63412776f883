"""Waits of the walk of ``decay_attention`` on tensor cores that run out: what such a block was to write is NaN, the program goes on, and the
time of the kernels in front does not count.  In processes of their own, so that the count of such blocks is theirs."""
import subprocess
import sys
import textwrap

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

START = '''
  import ctypes
  import torch
  import brainpylib_b200 as bpl
  from brainpylib_b200 import _lib
  lib = _lib.lib()
  lib.bpl_tensor_walk_patience_for_tests.argtypes = [ctypes.c_int64]
  lib.bpl_tensor_walk_patience_for_tests.restype = None
  cuda = torch.device('cuda', 0)

  def rows(*size, dtype=torch.bfloat16):
    return torch.randn(*size, device=cuda, dtype=torch.float32).to(dtype).requires_grad_(True)

  def call(q, k, v, log_decay, initial=None, **kw):
    y, last = bpl.decay_attention(q, k, v, log_decay, initial_state=initial, return_state=True, **kw)
    leaves = [t for t in (q, k, v, initial) if t is not None]
    return [y, last] + list(torch.autograd.grad([y, last], leaves, [torch.ones_like(y), torch.ones_like(last)]))
'''


def run(code):
  r = subprocess.run([sys.executable, '-c', textwrap.dedent(START) + textwrap.dedent(code)], cwd=ROOT, capture_output=True, text=True, timeout=300)
  assert r.returncode == 0 and 'done' in r.stdout, r.stdout + r.stderr[-2000:]


@pytest.mark.parametrize('heads,kv_heads,key,value', [(2, 2, 64, 64), (4, 2, 128, 128), (1, 1, 256, 72)])
def test_a_block_that_gives_up_leaves_no_numbers(heads, kv_heads, key, value):
  """Nothing is copied, so that every block waits in vain: results, last states and gradients have no numbers, but for the
  rows and the states without tokens.  Afterwards the same calls give what they gave before."""
  run(f'''
  tokens, bounds = 2500, [3, 700, 700, 2400]
  args = [rows(tokens, {heads}, {key}), rows(tokens, {kv_heads}, {key}), rows(tokens, {kv_heads}, {value}),
          -torch.rand({heads}, device=cuda), rows(3, {heads}, {key}, {value}, dtype=torch.float32)]
  kw = dict(indptr=torch.tensor(bounds, dtype=torch.int32, device=cuda))
  want = call(*args, **kw)
  assert lib.bpl_tensor_walk_failures() == 0 and all(torch.isfinite(t).all() for t in want)
  lib.bpl_tensor_walk_patience_for_tests(0)
  y, last, dq, dk, dv, d_initial = call(*args, **kw)
  torch.cuda.synchronize()
  lib.bpl_tensor_walk_patience_for_tests(-1)
  assert lib.bpl_tensor_walk_failures() > 0
  for t in (y, dq, dk, dv):
    assert torch.isnan(t[3:2400]).all() and not t[:3].any() and not t[2400:].any()
  for t, w in ((last, args[4]), (d_initial, torch.ones_like(last))):
    assert torch.isnan(t[[0, 2]]).all() and torch.equal(t[1], w[1])
  again = call(*args, **kw)
  assert all(torch.equal(a, b) for a, b in zip(again, want))
  print('done')
  ''')


def test_time_of_the_kernels_in_front_does_not_count():
  """Three segments of 43,700 tokens of 40 heads: the pass over the states takes a millisecond on 80 SMs, while blocks of the walk behind
  it wait on others already.  Waits of a million clocks, half a millisecond, are enough for them."""
  run('''
  tokens, heads = 131_072, 40
  args = [rows(tokens, heads, 8), rows(tokens, heads, 8), rows(tokens, heads, 8), torch.full((heads,), -0.01, device=cuda)]
  with torch.no_grad():
    go = lambda: bpl.decay_attention(*args, return_state=True)
    want = go()
    lib.bpl_tensor_walk_patience_for_tests(1_000_000)
    got = go()
    torch.cuda.synchronize()
  assert lib.bpl_tensor_walk_failures() == 0
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  print('done')
  ''')
