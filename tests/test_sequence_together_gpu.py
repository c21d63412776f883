"""The operators over whole sequences as a layer uses them: convolution, scan, gradients and clipping in a training step; a prompt
and the tokens after it on a pool of states; captured into CUDA graphs, on other streams, beside the operators of a network."""
import subprocess
import sys
import textwrap

import pytest
import torch

import brainpylib_b200 as bpl
import sequence_reference as ref
from conftest import ROOT

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
BOUNDS = [0, 13, 13, 60, 77]


def layer(cuda, tokens, channels=48, state=16, groups=2, dtype=F32, seed=0):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
  d = dict(x=r(tokens, channels).to(dtype), weight=r(channels, 4).to(dtype) / 2, bias=r(channels).to(dtype),
           delta=r(tokens, channels).to(dtype), A=-torch.exp(r(channels, state)).to(F32), B=r(tokens, groups, state).to(dtype),
           C=r(tokens, groups, state).to(dtype), D=r(channels).to(F32), z=r(tokens, channels).to(dtype),
           delta_bias=(r(channels) - 2).to(F32))
  return {k: v.to(cuda) for k, v in d.items()}


def forward(p, indptr, **kw):
  u = bpl.short_conv(p['x'], p['weight'], p['bias'], activation='silu', indptr=indptr)
  return bpl.state_scan(u, p['delta'], p['A'], p['B'], p['C'], p['D'], z=p['z'], delta_bias=p['delta_bias'],
                        delta_softplus=True, indptr=indptr, **kw)


def test_a_training_step(cuda):
  """Forward, backward and clipping of the layer against the same in 64 bits; the gradient of the convolution's output is the
  scan's gradient by its input."""
  p = layer(cuda, BOUNDS[-1])
  indptr = torch.tensor(BOUNDS, dtype=torch.int32, device=cuda)
  leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
  dy = torch.randn(p['x'].shape, generator=torch.Generator().manual_seed(1))
  y = forward(leaves, indptr)
  y.backward(dy.to(cuda))
  w = {k: v.double().cpu() for k, v in p.items()}
  pairs = list(zip(BOUNDS[:-1], BOUNDS[1:]))
  u = ref.conv(w['x'], w['weight'], w['bias'], pairs, None, True)['y']
  scan = lambda **kw: ref.scan(u, w['delta'], w['A'], w['B'], w['C'], w['D'], w['z'], w['delta_bias'], True, pairs, None,
                               dy=dy.double(), **kw)
  s = scan()
  c = ref.conv(w['x'], w['weight'], w['bias'], pairs, None, True, dy=s['d_x'])
  want = dict(s, **{k: c[k] for k in ('d_x', 'd_weight', 'd_bias')})
  # 47 tokens, 16 states: 1000 roundings of terms whose sizes add up to less than 50 times the largest value
  for name, v in leaves.items():
    scale = want['d_' + name].abs().max()
    assert (v.grad.double().cpu() - want['d_' + name]).abs().max() <= 50_000 * ref.U * scale, name
  assert (y.detach().double().cpu() - s['y']).abs().max() <= 50_000 * ref.U * s['y'].abs().max()
  grads = [leaves[k].grad for k in ('weight', 'bias', 'A', 'D', 'delta_bias')]
  total = sum(float((want['d_' + k] ** 2).sum()) for k in ('weight', 'bias', 'A', 'D', 'delta_bias')) ** 0.5
  before = [g.clone() for g in grads]
  norm = bpl.clip_gradients(grads, total / 2)
  assert abs(float(norm) - total) <= 50_000 * ref.U * total
  for g, b in zip(grads, before):
    assert torch.allclose(g, b * (total / 2 / (float(norm) + 1e-6)), rtol=4 * ref.U, atol=0)


def prompts_then_tokens(p, indptr, n_prompt, pools, slots):
  """Prompts of the first rows into the pools, then one token after the other for every sequence."""
  head = {k: v[:n_prompt] if v.shape[0] == p['x'].shape[0] else v for k, v in p.items()}
  u, last_inputs = bpl.short_conv(head['x'], p['weight'], p['bias'], activation='silu', indptr=indptr, return_state=True)
  y, last = bpl.state_scan(u, head['delta'], p['A'], head['B'], head['C'], p['D'], z=head['z'], delta_bias=p['delta_bias'],
                           delta_softplus=True, indptr=indptr, return_state=True)
  pools[0].index_copy_(0, slots.long(), last_inputs)
  pools[1].index_copy_(0, slots.long(), last)
  out = [y]
  n = slots.shape[0]
  for at in range(n_prompt, p['x'].shape[0], n):
    rows = slice(at, at + n)
    u = bpl.short_conv_step(p['x'][rows], pools[0], p['weight'], p['bias'], activation='silu', slots=slots)
    out.append(bpl.state_scan_step(u, p['delta'][rows], p['A'], p['B'][rows], p['C'][rows], pools[1], p['D'], z=p['z'][rows],
                                   delta_bias=p['delta_bias'], delta_softplus=True, slots=slots))
  return torch.cat(out)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_prompts_and_the_tokens_after_them_eager_and_captured(cuda, dtype):
  """A captured run replayed on other inputs gives the eager run's bits; two graphs replayed in turn do not disturb one another."""
  indptr = torch.tensor([0, 9, 40], dtype=torch.int32, device=cuda)
  slots = torch.tensor([4, 1], dtype=torch.int32, device=cuda)
  new_pools = lambda: [torch.zeros(6, 48, 3, dtype=dtype, device=cuda), torch.zeros(6, 48, 16, device=cuda)]
  runs = []
  for seed in (1, 2):
    p, pools = layer(cuda, 40 + 2 * 7, dtype=dtype, seed=seed), new_pools()
    prompts_then_tokens(p, indptr, 40, pools, slots)        # (loads the kernels)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      out = prompts_then_tokens(p, indptr, 40, pools, slots)
    runs.append((p, pools, graph, out))
  for round_ in range(3):
    fresh = [layer(cuda, 40 + 2 * 7, dtype=dtype, seed=10 * round_ + k) for k in range(2)]
    for (p, pools, graph, out), new in zip(runs, fresh):
      for k, v in new.items():
        p[k].copy_(v)
    runs[0][2].replay()
    runs[1][2].replay()
    for (p, pools, graph, out), new in zip(runs, fresh):
      other = new_pools()
      assert torch.equal(out, prompts_then_tokens(new, indptr, 40, other, slots))
      assert all(torch.equal(a, b) for a, b in zip(pools, other))


def test_a_captured_training_step_is_the_eager_one(cuda):
  indptr = torch.tensor(BOUNDS, dtype=torch.int32, device=cuda)
  leaves = {k: v.requires_grad_(True) for k, v in layer(cuda, BOUNDS[-1], dtype=BF16).items()}
  dy = torch.randn(BOUNDS[-1], 48, device=cuda).to(BF16)

  def step():
    grads = torch.autograd.grad(forward(leaves, indptr), list(leaves.values()), dy)
    return bpl.clip_gradients(list(grads), 0.5), grads

  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    step()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    norm, grads = step()
  new = layer(cuda, BOUNDS[-1], dtype=BF16, seed=5)
  with torch.no_grad():
    for k, v in leaves.items():
      v.copy_(new[k])
  graph.replay()
  want_norm, want = step()
  assert torch.equal(norm, want_norm) and all(torch.equal(a, b) for a, b in zip(grads, want))


def test_a_backward_pass_captured_beside_a_living_eager_graph_does_not_end_the_process():
  """Whatever the capture makes of it, the program goes on and can use the operators afterwards."""
  code = textwrap.dedent('''
    import sys
    sys.path[:0] = ['tests', '.']
    import torch
    import test_sequence_together_gpu as t
    cuda = torch.device('cuda', 0)
    indptr = torch.tensor(t.BOUNDS, dtype=torch.int32, device=cuda)
    leaves = {k: v.requires_grad_(True) for k, v in t.layer(cuda, t.BOUNDS[-1]).items()}
    alive = t.forward(leaves, indptr)
    alive.sum().backward(retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
      with torch.cuda.graph(graph):
        t.forward(leaves, indptr).sum().backward()
      graph.replay()
      print('captured')
    except RuntimeError as e:
      print('refused', str(e)[:80])
    torch.cuda.synchronize()
    del graph
    alive.sum().backward()
    assert torch.isfinite(leaves['A'].grad).all()
    torch.cuda.synchronize()
    print('went on')
  ''')
  r = subprocess.run([sys.executable, '-c', code], cwd=ROOT, capture_output=True, text=True, timeout=300)
  assert r.returncode == 0 and 'went on' in r.stdout, r.stdout + r.stderr[-2000:]


def test_on_another_stream_than_the_default(cuda):
  p = layer(cuda, 3000, channels=24, groups=1)
  want = forward(p, None, return_state=True)
  torch.cuda.synchronize()
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    q = {k: v * 2 / 2 for k, v in p.items()}                # written on this stream just before
    got = forward(q, None, return_state=True)
    leaves = {k: v.detach().requires_grad_(True) for k, v in q.items()}
    grads = torch.autograd.grad(forward(leaves, None), list(leaves.values()), torch.ones_like(got[0]))
    norm = bpl.clip_gradients(list(grads), 1.0)
  side.synchronize()
  assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.isfinite(norm)


def test_two_threads_at_once(cuda):
  import threading
  p = [layer(cuda, 2000, channels=24, groups=1, seed=s) for s in range(2)]
  want = [forward(q, None) for q in p]
  got = [None, None]

  def work(k):
    with torch.cuda.stream(torch.cuda.Stream()):
      for _ in range(20):
        got[k] = forward(p[k], None)
      torch.cuda.current_stream().synchronize()

  torch.cuda.synchronize()
  threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
  [t.start() for t in threads]
  [t.join() for t in threads]
  assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_behind_a_projection_of_spikes(cuda):
  """Spikes of a population through a stored matrix, one time step after the other, then leaky units over the whole run."""
  g = torch.Generator(cuda).manual_seed(2)
  n_pre, n_post, steps = 300, 64, 20
  indices = torch.randint(0, n_post, (n_pre * 10,), dtype=torch.int32, device=cuda, generator=g)
  indptr = torch.arange(0, n_pre * 10 + 1, 10, dtype=torch.int32, device=cuda)
  data = torch.rand(n_pre * 10, device=cuda, generator=g).requires_grad_(True)
  spikes = (torch.rand(steps, n_pre, device=cuda, generator=g) < 0.1).float()
  rows = torch.stack([bpl.event_csr_matvec(data, indices, indptr, s, shape=(n_pre, n_post), transpose=True) for s in spikes])
  rate = torch.full((n_post, 1), -1.0, device=cuda).requires_grad_(True)
  ones = torch.ones(steps, 1, device=cuda)
  y = bpl.state_scan(rows, torch.full((steps, n_post), 0.1, device=cuda), rate, ones, ones)
  y.square().sum().backward()
  dense = torch.zeros(n_pre, n_post, dtype=torch.float64, device=cuda)
  dense.index_put_((torch.arange(n_pre, device=cuda).repeat_interleave(10), indices.long()), data.detach().double(), accumulate=True)
  h, want = torch.zeros(n_post, dtype=torch.float64, device=cuda), []
  for s in spikes.double():
    h = h * torch.exp(torch.tensor(-0.1, dtype=torch.float64)) + 0.1 * (s @ dense)
    want.append(h)
  assert torch.allclose(y.double(), torch.stack(want), rtol=1e-5, atol=1e-6)
  assert torch.isfinite(data.grad).all() and float(bpl.gradient_norm([data.grad, rate.grad])) > 0


def test_what_the_operators_refuse_on_the_gpu(cuda):
  p = layer(cuda, 5)
  state = torch.zeros(5, 48, 16, device=cuda)
  args = lambda q: (q['x'], q['delta'], q['A'], q['B'], q['C'])
  grown = dict(p, A=p['A'].clone().requires_grad_(True))
  with pytest.raises(ValueError, match='no gradient'):
    bpl.state_scan_step(*args(grown), state)
  with torch.no_grad():
    bpl.state_scan_step(*args(grown), state)
  with pytest.raises(ValueError, match='no gradient'):
    bpl.short_conv_step(p['x'], torch.zeros(5, 48, 3, device=cuda), p['weight'].requires_grad_(True))
  with pytest.raises(RuntimeError):
    torch.func.vmap(lambda x: bpl.state_scan(x, p['delta'], *args(p)[2:]))(p['x'].expand(2, 5, 48))
  with pytest.raises(bpl.GPUOperatorNotFound):
    bpl.state_scan(p['x'].cpu(), *args(p)[1:])
  with pytest.raises(ValueError, match='requires|place'):
    bpl.clip_gradients([grown['A']], 1.0)


def test_flags_of_other_types_than_bool(cuda):
  p = layer(cuda, 20)
  args = (p['x'], p['delta'], p['A'], p['B'], p['C'])
  for flag in (True, False):
    want = bpl.state_scan(*args, delta_softplus=flag, return_state=True)
    got = bpl.state_scan(*args, delta_softplus=int(flag), return_state=1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pools = [torch.ones(20, 48, 16, device=cuda) for _ in range(2)]
    assert torch.equal(bpl.state_scan_step(*args, pools[0], delta_softplus=flag), bpl.state_scan_step(*args, pools[1], delta_softplus=int(flag)))
    assert torch.equal(*pools)


def test_a_state_written_by_a_step_counts_as_changed(cuda):
  p = layer(cuda, 5)
  state = torch.zeros(5, 48, 16, device=cuda)
  w = torch.ones(5, 48, 16, device=cuda, requires_grad=True)
  product = (w * state).sum()
  bpl.state_scan_step(p['x'], p['delta'], p['A'], p['B'], p['C'], state)
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):
    product.backward()
