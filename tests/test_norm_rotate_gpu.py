"""``norm_rotate`` and its gradients against the plain statement in 64 bits: sizes, types, parts of heads that are not rotated, far
positions, strides."""
import pytest
import torch

import brainpylib_b200 as bpl
import language_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inputs(tokens, heads, k_heads, size, rotated, dtype, *, weights='wide', far=100, seed=0):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
  w = dict(wide=F32, same=dtype, none=None)[weights]
  d = dict(q=r(tokens, heads, size).to(dtype), k=(3 * r(tokens, k_heads, size)).to(dtype),
           positions=torch.randint(-far, far + 1, (tokens,), generator=g),
           frequencies=(10_000.0 ** -(torch.arange(rotated // 2, dtype=torch.float64) * 2 / max(rotated, 1))).to(F32),
           q_weight=None if w is None else r(size).to(w), k_weight=None if w is None else r(size).to(w))
  return d, r(tokens, heads, size).to(dtype), r(tokens, k_heads, size).to(dtype)


def call(d, cuda, leaf=False, **kw):
  g = {k: v if v is None else v.to(cuda) for k, v in d.items()}
  leaves = [k for k in ('q', 'k', 'q_weight', 'k_weight') if leaf and g[k] is not None]
  for k in leaves:
    g[k].requires_grad_(True)
  return bpl.norm_rotate(*g.values(), **kw), [g[k] for k in leaves], ['d_' + k for k in leaves]


def check(d, gq, gk, cuda, interleaved=False, eps=1e-6):
  """A value: the norm (a sum of squares and a root: size + 4 roundings), two products, a rotation of two terms (cosine and sine off by
  2^-23 at most: 6 roundings of the two terms).  A gradient goes through the same, and through a mean of products; those of weights add
  up all rows (in parts: fewer than rows + 64 additions)."""
  (q, k), leaves, names = call(d, cuda, True, interleaved=interleaved, eps=eps)
  with torch.no_grad():
    plain, _, _ = call(d, cuda, interleaved=interleaved, eps=eps)
  assert torch.equal(plain[0], q) and torch.equal(plain[1], k)
  got = dict(zip(names, torch.autograd.grad([q, k], leaves, [gq.to(cuda), gk.to(cuda)])))
  size, rows = d['q'].shape[2], d['q'].shape[0]
  angle = ref.angles(d['positions'], d['frequencies'])
  for name, out, g in (('q', q, gq), ('k', k, gk)):
    x = d[name].double().requires_grad_(True)
    w = None if d[name + '_weight'] is None else d[name + '_weight'].double().requires_grad_(True)
    want = ref.rotation(x, angle, w, eps, interleaved)
    r = (x.detach().square().mean(-1, keepdim=True) + eps).rsqrt()
    n = (x.detach() * r).abs()
    aw = torch.ones(size, dtype=torch.float64) if w is None else w.detach().abs()
    # both terms of a rotation at their full size
    most = lambda t: t + ref.turn(t.abs(), torch.full_like(angle, torch.pi / 2), interleaved).abs()
    ref.check(out, want.detach(), most(n * aw), size + 16, name)
    wanted = torch.autograd.grad(want, [x] if w is None else [x, w], g.double())
    dz = most(g.double().abs())
    dn = dz * aw
    ref.check(got['d_' + name], wanted[0], r * (dn + n * (dn * n).mean(-1, keepdim=True)), 3 * size + 48, 'd_' + name)
    if w is not None:
      ref.check(got[f'd_{name}_weight'], wanted[1], (dz * n).sum((0, 1)), rows * x.shape[1] + size + 64, f'd_{name}_weight')


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('size,rotated', [(2, 2), (6, 4), (16, 16), (64, 64), (80, 80), (96, 32), (100, 50), (128, 128), (128, 64), (156, 156),
                                          (250, 250), (256, 256), (256, 6), (64, 0)])
def test_sizes_and_types(cuda, size, rotated, dtype):
  for interleaved in (False, True):
    d, gq, gk = inputs(5, 4, 2, size, rotated, dtype, weights='wide' if interleaved else 'same', seed=size)
    check(d, gq, gk, cuda, interleaved)


@pytest.mark.parametrize('tokens,heads,k_heads', [(1, 1, 1), (1, 64, 8), (3, 5, 5), (700, 3, 1), (2500, 2, 2)])
def test_rows_and_heads(cuda, tokens, heads, k_heads):
  check(*inputs(tokens, heads, k_heads, 32, 32, BF16, seed=tokens), cuda)
  check(*inputs(tokens, heads, k_heads, 32, 32, F32, weights='none', seed=tokens), cuda, True)


def test_far_positions(cuda):
  """Angles of any number of turns keep 32 bits of their fraction."""
  for far in (10 ** 6, 2 ** 31 - 1, 2 ** 45):
    d, gq, gk = inputs(9, 2, 2, 64, 64, F32, far=far)
    check(d, gq, gk, cuda)
  d, gq, gk = inputs(9, 2, 2, 64, 64, F32, far=2 ** 31 - 1)
  short = dict(d, positions=d['positions'].to(torch.int32))
  assert all(torch.equal(a, b) for a, b in zip(call(d, cuda)[0], call(short, cuda)[0]))


def test_one_weight_only_and_one_cotangent_only(cuda):
  d, gq, gk = inputs(6, 2, 3, 64, 64, F32)
  (q, k), _, _ = call(dict(d, k_weight=None), cuda)
  whole, _, _ = call(d, cuda)
  assert torch.equal(q, whole[0]) and not torch.equal(k, whole[1])
  (q, k), leaves, _ = call(d, cuda, True)
  both = torch.autograd.grad([q, k], leaves, [gq.to(cuda), torch.zeros_like(k)])
  (q, k), leaves, _ = call(d, cuda, True)
  one = torch.autograd.grad(q, leaves, gq.to(cuda), allow_unused=True)
  assert all(torch.equal(a, b) for a, b in zip(both, one))
  assert not one[1].any() and not one[3].any()


def test_strides_and_batches_are_the_packed_call(cuda):
  d, gq, gk = inputs(24, 4, 2, 64, 64, BF16)
  want, _, _ = call(d, cuda)
  rest = [d[n].to(cuda) for n in ('positions', 'frequencies', 'q_weight', 'k_weight')]
  for shift in (0, 1, 8):
    rows = torch.zeros(24, 8 * 64 + 16, dtype=BF16, device=cuda)
    q = rows[:, shift:shift + 256].unflatten(1, (4, 64)).copy_(d['q'])
    k = rows[:, shift + 256:shift + 384].unflatten(1, (2, 64)).copy_(d['k'])
    got = bpl.norm_rotate(q, k, *rest)
    # without alignment the squares of a head are added in another order: off by less than 64 * 2^-23 before rounding, which can then
    # go to the neighbouring number, a step of 2^-7 of the smaller one at most (and around zero a few times 2^-18 of the other term)
    assert all(torch.equal(a, b) if shift != 1 else torch.allclose(a.float(), b.float(), rtol=1.01 * 2 ** -7, atol=2 ** -15)
               for a, b in zip(got, want))
  q, k = d['q'].to(cuda).transpose(0, 1).contiguous().transpose(0, 1), d['k'].to(cuda)[:, :1].expand(24, 2, 64)
  got = bpl.norm_rotate(q, k, *rest)
  assert torch.equal(got[0], want[0]) and torch.equal(got[1][:, 1], want[1][:, 0])
  batched = [d[n].to(cuda).unflatten(0, (3, 8)) for n in ('q', 'k', 'positions')]
  got = bpl.norm_rotate(*batched, *rest[1:])
  assert all(torch.equal(a.flatten(0, 1), b) for a, b in zip(got, want))
  q = d['q'].to(cuda).unflatten(0, (3, 8)).transpose(1, 2).contiguous().transpose(1, 2)       # (batch, heads, length, size) in memory
  assert torch.equal(bpl.norm_rotate(q, *batched[1:], *rest[1:])[0].flatten(0, 1), want[0])


def test_nothing_to_do(cuda):
  d, _, _ = inputs(0, 4, 2, 64, 64, BF16)
  (q, k), leaves, _ = call(d, cuda, True)
  assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
  grads = torch.autograd.grad([q.sum() + k.sum()], leaves)
  assert not grads[2].any() and not grads[3].any()


def test_rows_stay_apart(cuda):
  """A row of zeros is zero; rows of NaN and infinities leave the others alone."""
  d, gq, gk = inputs(6, 2, 2, 64, 64, F32)
  want, _, _ = call(d, cuda)
  d['q'][2, 1], d['k'][4, 0, 3], d['q'][0, 0] = float('nan'), float('inf'), 0
  got, _, _ = call(d, cuda)
  for w, g, bad in ((want[0], got[0], [(2, 1), (0, 0)]), (want[1], got[1], [(4, 0)])):
    keep = torch.ones(6, 2, dtype=torch.bool)
    for at in bad:
      keep[at] = False
    assert torch.equal(w[keep], g[keep])
  assert torch.isnan(got[0][2, 1]).all() and not got[0][0, 0].any()


def test_against_differences(cuda):
  """Gradients against central differences of the 64-bit statement at the operator's own inputs, and the operator's own values along
  them: a step of 2^-8 leaves h^2 / 6 of the third derivative (below 50 here) and 2^-24 / h of the values."""
  d, gq, gk = inputs(3, 2, 1, 16, 16, F32, far=10)
  (q, k), leaves, names = call(d, cuda, True)
  got = dict(zip(names, torch.autograd.grad([q, k], leaves, [gq.to(cuda), gk.to(cuda)])))
  h = 2.0 ** -8

  def loss(e):
    (a, b), _, _ = call(e, cuda)
    return float((a.double().cpu() * gq.double()).sum() + (b.double().cpu() * gk.double()).sum())

  for name in ('q', 'k', 'q_weight', 'k_weight'):
    way = torch.randn(d[name].shape, generator=torch.Generator().manual_seed(5))
    up, down = dict(d, **{name: d[name] + h * way}), dict(d, **{name: d[name] - h * way})
    slope = (loss(up) - loss(down)) / (2 * h)
    size = float((got[name_of(name)].cpu().double() * way.double()).abs().sum())
    assert abs(slope - float((got[name_of(name)].cpu().double() * way.double()).sum())) < 5e-3 * (1 + size), name


def name_of(leaf):
  return 'd_' + leaf
