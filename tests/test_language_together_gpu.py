"""The layers of language models as a model uses them: rows of a table, normed and rotated heads, attention and clipping in a training
step; prompts and the tokens after them on a pool of states; captured into CUDA graphs, on other streams, in two threads."""
import subprocess
import sys
import textwrap
import threading

import pytest
import torch

import brainpylib_b200 as bpl
import language_reference as ref
from conftest import ROOT

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
BOUNDS = [0, 13, 13, 100, 177]
HEADS, KV, SIZE = 4, 2, 64


def model(cuda, dtype=F32, seed=0, vocabulary=50):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
  width = (HEADS + 2 * KV) * SIZE
  d = dict(table=r(vocabulary, width).to(dtype), q_weight=r(SIZE).to(F32), k_weight=r(SIZE).to(F32))
  return {k: v.to(cuda) for k, v in d.items()}


def text(cuda, tokens, seed=1, vocabulary=50):
  return torch.randint(0, vocabulary, (tokens,), generator=torch.Generator().manual_seed(seed)).to(cuda)


def constants(cuda):
  return (10_000.0 ** -(torch.arange(0, SIZE, 2, device=cuda) / SIZE)), -torch.exp2(-torch.arange(1, HEADS + 1, device=cuda).float())


def heads(p, ids, positions, frequencies):
  rows = bpl.embedding(ids, p['table'], scale=0.5)
  q, k, v = (t.unflatten(-1, (-1, SIZE)) for t in rows.split([HEADS * SIZE, KV * SIZE, KV * SIZE], -1))
  q, k = bpl.norm_rotate(q, k, positions, frequencies, p['q_weight'], p['k_weight'])
  return q, k, v


def forward(p, ids, indptr, positions, frequencies, log_decay, **kw):
  return bpl.decay_attention(*heads(p, ids, positions, frequencies), log_decay, indptr=indptr, **kw)


def places(bounds, cuda):
  return torch.cat([torch.arange(e - b) for b, e in zip(bounds[:-1], bounds[1:])]).to(torch.int32).to(cuda)


def test_a_training_step(cuda):
  """Forward, backward and clipping against the same in 64 bits: 87 tokens, sums over 64 elements and 177 tokens and a chain of four
  operators leave a few thousand roundings of terms whose sizes add up to less than 100 times the largest value."""
  p, ids, positions = model(cuda), text(cuda, BOUNDS[-1]), places(BOUNDS, cuda)
  frequencies, log_decay = constants(cuda)
  indptr = torch.tensor(BOUNDS, dtype=torch.int32, device=cuda)
  leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
  dy = torch.randn(BOUNDS[-1], HEADS, SIZE, generator=torch.Generator().manual_seed(2))
  y = forward(leaves, ids, indptr, positions, frequencies, log_decay)
  y.backward(dy.to(cuda))
  w = {k: v.double().cpu().requires_grad_(True) for k, v in p.items()}
  rows = ref.embedding(ids.cpu(), w['table'], 0.5)
  q, k, v = (t.unflatten(-1, (-1, SIZE)) for t in rows.split([HEADS * SIZE, KV * SIZE, KV * SIZE], -1))
  angle = ref.angles(positions.cpu(), frequencies.cpu())
  q, k = ref.rotation(q, angle, w['q_weight'], 1e-6, False), ref.rotation(k, angle, w['k_weight'], 1e-6, False)
  pairs = list(zip(BOUNDS[:-1], BOUNDS[1:]))
  a = ref.attention(q.detach(), k.detach(), v.detach(), log_decay.double().cpu(), SIZE ** -0.5, pairs, None, dy.double())
  want = torch.autograd.grad([q, k, v], list(w.values()), [a['d_q'], a['d_k'], a['d_v']])
  close = lambda got, want: (got.detach().double().cpu() - want).abs().max() <= 500_000 * ref.U * want.abs().max()
  assert close(y, a['y'])
  for name, g in zip(w, want):
    assert close(leaves[name].grad, g), name
  grads = [v.grad for v in leaves.values()]
  total = sum(float((g ** 2).sum()) for g in want) ** 0.5
  before = [g.clone() for g in grads]
  norm = bpl.clip_gradients(grads, total / 2)
  assert abs(float(norm) - total) <= 500_000 * ref.U * total
  for g, b in zip(grads, before):
    assert torch.allclose(g, b * (total / 2 / (float(norm) + 1e-6)), rtol=4 * ref.U, atol=0)


def prompts_then_tokens(p, ids, indptr, n_prompt, at, pool, slots, frequencies, log_decay, first):
  """Prompts into the pool, then one token after the other for every sequence."""
  y, last = forward(p, ids[:n_prompt], indptr, at[:n_prompt], frequencies, log_decay, return_state=True)
  pool.index_copy_(0, slots.long(), last)
  out, n = [y], slots.shape[0]
  for i, start in enumerate(range(n_prompt, ids.shape[0], n)):
    q, k, v = heads(p, ids[start:start + n], first + i, frequencies)
    out.append(bpl.decay_attention_step(q, k, v, log_decay, pool, slots=slots))
  return torch.cat(out)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_prompts_and_the_tokens_after_them_eager_and_captured(cuda, dtype):
  """What the steps give is what the whole sequences give; a captured run replayed on other tokens gives the eager run's bits, and two
  graphs replayed in turn do not disturb one another."""
  bounds = [0, 70, 100]
  indptr = torch.tensor(bounds, dtype=torch.int32, device=cuda)
  slots = torch.tensor([4, 1], dtype=torch.int32, device=cuda)
  first = torch.tensor([70, 30], dtype=torch.int32, device=cuda)
  frequencies, log_decay = constants(cuda)
  at = places(bounds, cuda)
  new_pool = lambda: torch.zeros(6, HEADS, SIZE, SIZE, device=cuda)
  go = lambda p, ids, pool: prompts_then_tokens(p, ids, indptr, 100, at, pool, slots, frequencies, log_decay, first)
  p = model(cuda, dtype)
  ids = text(cuda, 100 + 2 * 9)
  got = go(p, ids, new_pool())
  for s, (b, e) in enumerate(zip(bounds[:-1], bounds[1:])):
    whole = torch.cat([ids[b:e], ids[100 + s::2]])
    n = whole.shape[0]
    y = forward(p, whole, None, torch.arange(n, device=cuda), frequencies, log_decay)
    steps = torch.cat([got[b:e], got[100 + s::2]])
    # both are within the same bounds of the exact result: sums of at most 79 products of 64 normed elements each
    tolerance = (79 * 64 * 2.0 ** -20 if dtype == F32 else 3 * 2.0 ** -8) * float(y.float().abs().max()) * (1 if dtype == F32 else 4)
    assert (y.float() - steps.float()).abs().max() <= tolerance
  runs = []
  for seed in (1, 2):
    ids, pool = text(cuda, 100 + 2 * 9, seed), new_pool()
    go(p, ids, pool)                                        # (loads the kernels)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      out = go(p, ids, pool)
    runs.append((ids, pool, graph, out))
  for round_ in range(3):
    for i, (ids, pool, _, _) in enumerate(runs):
      ids.copy_(text(cuda, 118, 10 * round_ + i))
      pool.zero_()
    runs[0][2].replay()
    runs[1][2].replay()
    for i, (ids, pool, _, out) in enumerate(runs):
      other = new_pool()
      assert torch.equal(out, go(p, ids, other)) and torch.equal(pool, other)


def gradients(p, ids, indptr, positions, frequencies, log_decay, dy):
  return list(torch.autograd.grad(forward(p, ids, indptr, positions, frequencies, log_decay), list(p.values()), dy))


def test_a_captured_training_step_is_the_eager_one(cuda):
  frequencies, log_decay = constants(cuda)
  indptr, positions = torch.tensor(BOUNDS, dtype=torch.int32, device=cuda), places(BOUNDS, cuda)
  leaves = {k: v.requires_grad_(True) for k, v in model(cuda, BF16).items()}
  ids, dy = text(cuda, BOUNDS[-1]), torch.randn(BOUNDS[-1], HEADS, SIZE, device=cuda).to(BF16)

  def step():
    grads = gradients(leaves, ids, indptr, positions, frequencies, log_decay, dy)
    return bpl.clip_gradients(grads, 0.5), grads

  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    step()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    norm, grads = step()
  new = model(cuda, BF16, seed=5)
  with torch.no_grad():
    for k, v in leaves.items():
      v.copy_(new[k])
  ids.copy_(text(cuda, BOUNDS[-1], 9))
  graph.replay()
  want_norm, want = step()
  assert torch.equal(norm, want_norm) and all(torch.equal(a, b) for a, b in zip(grads, want))


def test_a_backward_pass_captured_beside_a_living_eager_graph_does_not_end_the_process():
  """Whatever the capture makes of it, the program goes on and can use the operators afterwards."""
  code = textwrap.dedent('''
    import sys
    sys.path[:0] = ['tests', '.']
    import torch
    import test_language_together_gpu as t
    cuda = torch.device('cuda', 0)
    frequencies, log_decay = t.constants(cuda)
    args = (t.text(cuda, t.BOUNDS[-1]), torch.tensor(t.BOUNDS, dtype=torch.int32, device=cuda), t.places(t.BOUNDS, cuda), frequencies, log_decay)
    leaves = {k: v.requires_grad_(True) for k, v in t.model(cuda).items()}
    alive = t.forward(leaves, *args)
    alive.sum().backward(retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
      with torch.cuda.graph(graph):
        t.forward(leaves, *args).sum().backward()
      graph.replay()
      print('captured')
    except RuntimeError as e:
      print('refused', str(e)[:80])
    torch.cuda.synchronize()
    del graph
    alive.sum().backward()
    assert torch.isfinite(leaves['table'].grad).all()
    torch.cuda.synchronize()
    print('went on')
  ''')
  r = subprocess.run([sys.executable, '-c', code], cwd=ROOT, capture_output=True, text=True, timeout=300)
  assert r.returncode == 0 and 'went on' in r.stdout, r.stdout + r.stderr[-2000:]


def test_on_another_stream_than_the_default(cuda):
  frequencies, log_decay = constants(cuda)
  p, ids = model(cuda, BF16), text(cuda, 3000)
  positions = torch.arange(3000, device=cuda)
  want = forward(p, ids, None, positions, frequencies, log_decay, return_state=True)
  dy = torch.ones_like(want[0])
  want_grads = gradients({k: v.clone().requires_grad_(True) for k, v in p.items()}, ids, None, positions, frequencies, log_decay, dy)
  torch.cuda.synchronize()
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    q = {k: v * 2 / 2 for k, v in p.items()}                # written on this stream just before
    got = forward(q, ids, None, positions, frequencies, log_decay, return_state=True)
    grads = gradients({k: v.requires_grad_(True) for k, v in q.items()}, ids, None, positions, frequencies, log_decay, dy)
  side.synchronize()
  assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))


def test_two_threads_at_once(cuda):
  frequencies, log_decay = constants(cuda)
  p = [{k: v.requires_grad_(True) for k, v in model(cuda, BF16, seed=s).items()} for s in range(2)]
  ids, positions = text(cuda, 2000), torch.arange(2000, device=cuda)
  dy = torch.randn(2000, HEADS, SIZE, device=cuda).to(BF16)
  want = [gradients(q, ids, None, positions, frequencies, log_decay, dy) for q in p]
  got = [None, None]

  def work(k):
    with torch.cuda.stream(torch.cuda.Stream()):
      for _ in range(10):
        got[k] = gradients(p[k], ids, None, positions, frequencies, log_decay, dy)
      torch.cuda.current_stream().synchronize()

  torch.cuda.synchronize()
  threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
  [t.start() for t in threads]
  [t.join() for t in threads]
  assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))


def test_attention_behind_a_short_convolution(cuda):
  """Values that pass the taps of a convolution first, gradients through both."""
  g = torch.Generator(cuda).manual_seed(3)
  r = lambda *s: torch.randn(*s, device=cuda, generator=g, requires_grad=True)
  q, k, v, taps = r(90, 2, 32), r(90, 2, 32), r(90, 2 * 32), r(64, 4)
  log_decay = torch.tensor([-0.1, -0.01], device=cuda)
  u = bpl.short_conv(v, taps, activation='silu')
  y = bpl.decay_attention(q, k, u.unflatten(-1, (2, 32)), log_decay)
  got = torch.autograd.grad(y.square().sum(), [q, v, taps])
  p = [t.detach().double().requires_grad_(True) for t in (q, k, v, taps)]
  windows = torch.cat([torch.zeros(3, 64, device=cuda, dtype=torch.float64), p[2]]).unfold(0, 4, 1)
  w = torch.nn.functional.silu((windows * p[3]).sum(-1)).unflatten(-1, (2, 32))
  n = torch.arange(90, device=cuda)
  counts = torch.exp(log_decay.double()[:, None, None] * (n[:, None] - n).clamp(min=0)).tril() * 32 ** -0.5
  z = torch.einsum('ihk,jhk,hij,jhv->ihv', p[0], p[1], counts, w)
  want = torch.autograd.grad(z.square().sum(), [p[0], p[2], p[3]])
  for a, b in zip(got, want):        # (a chain of four sums of at most 90 * 32 terms: 2^14 roundings at most)
    assert (a.double() - b).abs().max() <= 2.0 ** -10 * b.abs().max()


def test_what_the_operators_refuse_on_the_gpu(cuda):
  frequencies, log_decay = constants(cuda)
  p, ids = model(cuda), text(cuda, 5)
  q, k, v = heads(p, ids, torch.arange(5, device=cuda), frequencies)
  state = torch.zeros(5, HEADS, SIZE, SIZE, device=cuda)
  grown = q.detach().clone().requires_grad_(True)
  with pytest.raises(ValueError, match='no gradient'):
    bpl.decay_attention_step(grown, k, v, log_decay, state)
  with torch.no_grad():
    bpl.decay_attention_step(grown, k, v, log_decay, state)
  with pytest.raises(ValueError, match='constants'):
    bpl.decay_attention(q, k, v, log_decay.clone().requires_grad_(True))
  with pytest.raises(ValueError, match='frequencies'):
    bpl.norm_rotate(q, k, torch.arange(5, device=cuda), frequencies.clone().requires_grad_(True))
  with pytest.raises(RuntimeError):
    torch.func.vmap(lambda t: bpl.decay_attention(t, k, v, log_decay))(q.expand(2, *q.shape))
  with pytest.raises(RuntimeError):
    torch.func.vmap(lambda t: bpl.embedding(t, p['table']))(ids.expand(2, 5))
  with pytest.raises(bpl.GPUOperatorNotFound):
    bpl.decay_attention(q.cpu(), k, v, log_decay)
  with pytest.raises(bpl.GPUOperatorNotFound):
    bpl.embedding(ids.cpu(), p['table'])
  leaf = p['table'].clone().requires_grad_(True)
  first, = torch.autograd.grad(bpl.embedding(ids, leaf).sum(), leaf, create_graph=True)
  with pytest.raises(RuntimeError, match='differentiable once'):
    first.sum().backward()
  y = bpl.decay_attention(grown, k, v, log_decay)
  first, = torch.autograd.grad(y.sum(), grown, create_graph=True)
  with pytest.raises(RuntimeError, match='differentiable once'):
    first.sum().backward()


def test_a_state_written_by_a_step_counts_as_changed(cuda):
  frequencies, log_decay = constants(cuda)
  q, k, v = heads(model(cuda), text(cuda, 5), torch.arange(5, device=cuda), frequencies)
  state = torch.zeros(5, HEADS, SIZE, SIZE, device=cuda)
  w = torch.ones_like(state, requires_grad=True)
  product = (w * state).sum()
  bpl.decay_attention_step(q, k, v, log_decay, state)
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):
    product.backward()


def test_scales_that_are_no_numbers_are_refused_on_the_gpu(cuda):
  frequencies, log_decay = constants(cuda)
  p, ids = model(cuda), text(cuda, 5)
  at = torch.arange(5, device=cuda)
  q, k, v = heads(p, ids, at, frequencies)
  nan = float('nan')
  with pytest.raises(ValueError, match='scale must be a number'):
    bpl.embedding(ids, p['table'], scale=nan)
  with pytest.raises(ValueError, match='eps must be a number'):
    bpl.norm_rotate(q, k, at, frequencies, eps=nan)
  with pytest.raises(ValueError, match='scale must be a number'):
    bpl.decay_attention(q, k, v, log_decay, scale=nan)
  with pytest.raises(ValueError, match='scale must be a number'):
    bpl.decay_attention_step(q, k, v, log_decay, torch.zeros(5, HEADS, SIZE, SIZE, device=cuda), scale=nan)
