"""``embedding`` and the gradient of its table against the plain statement in 64 bits: types, widths without alignment, ids that name
nothing, frequent tokens over many runs, sorts of one block and of many."""
import struct

import pytest
import torch

import brainpylib_b200 as bpl
import language_reference as ref
from brainpylib_b200 import _lib

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inputs(tokens, vocabulary, width, dtype, *, seed=0, spread=1.0):
  g = torch.Generator().manual_seed(seed)
  ids = (torch.rand(tokens, generator=g, dtype=torch.float64) ** spread * vocabulary).long().clamp(max=vocabulary - 1)
  weight = torch.randn(vocabulary, width, generator=g, dtype=torch.float64).to(dtype)
  return ids, weight, torch.randn(tokens, width, generator=g, dtype=torch.float64).to(dtype)


def check(cuda, ids, weight, dy, scale=1.5, wide=True):
  """A value is one product; a gradient a sum over at most as many tokens as there are, times the scale."""
  i = ids.to(cuda) if wide else ids.to(torch.int32).to(cuda)
  w = weight.to(cuda).requires_grad_(True)
  y = bpl.embedding(i, w, scale=scale)
  with torch.no_grad():
    assert torch.equal(torch.nan_to_num(bpl.embedding(i, w, scale=scale), nan=-7.0), torch.nan_to_num(y, nan=-7.0))
  want = ref.embedding(ids, weight.double(), scale)
  assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want))
  ref.check(torch.nan_to_num(y), torch.nan_to_num(want), torch.nan_to_num(want).abs(), 2, 'y')
  got, = torch.autograd.grad(y, w, dy.to(cuda))
  args = (ids, dy.double(), weight.shape[0], scale)
  most = int(torch.bincount(ids[(ids >= 0) & (ids < weight.shape[0])].reshape(-1)).max()) if ids.numel() else 0
  ref.check(got, ref.embedding_gradient(*args), ref.embedding_gradient(*args, absolute=True), most + 2, 'd_weight')
  again, = torch.autograd.grad(bpl.embedding(i, w, scale=scale), w, dy.to(cuda))
  assert torch.equal(got, again)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('tokens,vocabulary,width', [(1, 1, 1), (1, 300, 64), (3, 7, 5), (17, 1, 33), (64, 2047, 40), (65, 2048, 8),
                                                     (300, 5000, 136), (2000, 50, 24), (33, 100_000, 3)])
def test_types_and_sizes(cuda, tokens, vocabulary, width, dtype):
  check(cuda, *inputs(tokens, vocabulary, width, dtype, seed=tokens), wide=tokens % 2 == 0)


@pytest.mark.parametrize('tokens', [2047, 2048, 2049, 4097, 20_000])
@pytest.mark.parametrize('vocabulary,spread', [(3, 1.0), (700, 6.0), (5000, 1.0), (70_001, 3.0)])
def test_many_tokens(cuda, tokens, vocabulary, spread):
  """One block sorts up to 2048 tokens, several more; rows whose tokens fill many runs."""
  check(cuda, *inputs(tokens, vocabulary, 12, F32, seed=tokens, spread=spread))


def test_a_sort_of_several_tiles_per_block(cuda):
  ids, weight, dy = inputs(1_100_000, 5_000_000, 1, F32, spread=2.0)
  check(cuda, ids, weight, dy)


def test_all_tokens_the_same(cuda):
  ids, weight, dy = inputs(9000, 20, 16, F32)
  check(cuda, torch.full_like(ids, 19), weight, dy)
  check(cuda, torch.zeros_like(ids), weight, dy)


def test_wide_rows(cuda):
  check(cuda, *inputs(50, 40, 2056, BF16))
  check(cuda, *inputs(50, 40, 2057, F16))


def test_ids_that_name_nothing(cuda):
  """Padding is zero, ids beyond the table are NaN, and neither has a gradient, not even of NaN."""
  for tokens in (40, 6000):
    ids, weight, dy = inputs(tokens, 30, 24, BF16)
    ids[::3], ids[1::7] = -1, 30
    ids[2::11], ids[5] = -2 ** 40, 2 ** 40
    dy[(ids < 0) | (ids >= 30)] = float('nan')
    i, w = ids.to(cuda), weight.to(cuda).requires_grad_(True)
    y = bpl.embedding(i, w)
    assert not y[i < 0].any() and torch.isnan(y[i >= 30]).all()
    got, = torch.autograd.grad(y, w, dy.to(cuda))
    clean = torch.nan_to_num(dy.double())
    ref.check(got, ref.embedding_gradient(ids, clean, 30, 1.0), ref.embedding_gradient(ids, clean, 30, 1.0, absolute=True), tokens, 'd_weight')
  none = torch.full((5,), -1, device=cuda)
  w = torch.ones(4, 8, device=cuda, requires_grad=True)
  got, = torch.autograd.grad(bpl.embedding(none, w), w, torch.ones(5, 8, device=cuda))
  assert not got.any()


def test_no_tokens_and_no_table(cuda):
  w = torch.ones(4, 8, device=cuda, requires_grad=True)
  y = bpl.embedding(torch.zeros(2, 0, dtype=torch.int64, device=cuda), w)
  assert y.shape == (2, 0, 8)
  got, = torch.autograd.grad(y.sum(), w)
  assert not got.any()
  empty = torch.ones(0, 8, device=cuda)
  assert torch.isnan(bpl.embedding(torch.zeros(3, dtype=torch.int32, device=cuda), empty)).all()
  assert bpl.embedding(torch.zeros(3, dtype=torch.int32, device=cuda), torch.ones(5, 0, device=cuda)).shape == (3, 0)


def test_shapes_and_strides(cuda):
  """Ids of any shape and order, tables that are part of a wider one, cotangents that are not dense."""
  ids, weight, dy = inputs(60, 25, 16, BF16)
  want = bpl.embedding(ids.to(cuda), weight.to(cuda), scale=2)
  assert torch.equal(bpl.embedding(ids.reshape(3, 4, 5).to(cuda), weight.to(cuda), scale=2).reshape(60, 16), want)
  across = ids.reshape(4, 15).t().contiguous().t().to(cuda)
  assert torch.equal(bpl.embedding(across, weight.to(cuda), scale=2).reshape(60, 16), want)
  for shift in (0, 1, 8):
    wide = torch.zeros(25, 40, dtype=BF16, device=cuda)
    part = wide[:, shift:shift + 16].copy_(weight)
    assert torch.equal(bpl.embedding(ids.to(cuda), part, scale=2), want)
    leaf = wide.clone().requires_grad_(True)
    got, = torch.autograd.grad(bpl.embedding(ids.to(cuda), leaf[:, shift:shift + 16]), leaf, dy.to(cuda))
    dense = ref.embedding_gradient(ids, dy.double(), 25, 1.0)
    ref.check(got[:, shift:shift + 16], dense, ref.embedding_gradient(ids, dy.double(), 25, 1.0, absolute=True), 60, 'd_weight')
    assert not got[:, :shift].any() and not got[:, shift + 16:].any()
  w = weight.to(cuda).requires_grad_(True)
  got, = torch.autograd.grad(bpl.embedding(ids.to(cuda), w), w, dy.to(cuda).t().contiguous().t())
  assert torch.equal(got, torch.autograd.grad(bpl.embedding(ids.to(cuda), w), w, dy.to(cuda))[0])


def test_against_differences(cuda):
  """The table's gradient against what a small change of an element changes: the operator is linear, so differences are exact but for
  roundings (of at most 2^-24 of the sums)."""
  ids, weight, dy = inputs(50, 9, 4, F32, seed=3)
  w = weight.to(cuda).requires_grad_(True)
  loss = lambda t: float((bpl.embedding(ids.to(cuda), t, scale=0.5).double() * dy.to(cuda).double()).sum())
  got, = torch.autograd.grad(bpl.embedding(ids.to(cuda), w, scale=0.5), w, dy.to(cuda))
  with torch.no_grad():
    for row, column in ((0, 0), (4, 3), (8, 1)):
      up, down = w.clone(), w.clone()
      up[row, column] += 1
      down[row, column] -= 1
      assert abs((loss(up) - loss(down)) / 2 - float(got[row, column])) < 60 * 10 * 2.0 ** -24


def test_scratch_memory_at_any_word(cuda):
  """Frequent tokens over many runs, whose parts of sums lie in the scratch memory: the same bits wherever that is."""
  ids, weight, dy = (t.to(cuda) for t in inputs(3000, 3, 64, F32))
  w = weight.requires_grad_(True)
  want, = torch.autograd.grad(bpl.embedding(ids, w), w, dy)
  opaque = struct.pack('<5Ifq', 3000, 3, 64, 0, 1, 1.0, 64)
  memory = torch.empty(_lib.workspace_bytes('embedding_backward', opaque) + 16, dtype=torch.uint8, device=cuda)
  for shift in (0, 4, 8):
    got = torch.empty_like(want)
    _lib.call('embedding_backward', [ids, dy, got, memory[shift:]], opaque)
    assert torch.equal(got, want)
