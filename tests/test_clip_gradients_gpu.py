"""``gradient_norm`` and ``clip_gradients`` against the formula in 64 bits: types, sizes beside packets and chunks, many tensors,
strides, values whose squares leave 32 bits, and calls that are refused."""
import math

import pytest
import torch

import brainpylib_b200 as bpl
import sequence_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64


def make(cuda, sizes, dtypes, seed=0, scale=1.0):
  g = torch.Generator(cuda).manual_seed(seed)
  return [(torch.randn(n, device=cuda, generator=g, dtype=F64) * scale).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def norm_of(ts, p=2.0):
  parts = [t.double().abs().flatten() for t in ts]
  if p == 2.0:
    return math.sqrt(sum(float((t * t).sum()) for t in parts))
  return max([float(t.max()) for t in parts if t.numel()] + [0.0])


def check(cuda, ts, max_norm, p=2.0):
  """The norm is a sum of squares, each rounded in 32 bits and added up to 8 at a time there: 10 roundings relative (all terms have
  one sign), half a step for the result.  A product is rounded once, its factor once: one step and a half a step of the type."""
  want = norm_of(ts, p)
  tol = (12 * ref.U if p == 2.0 else ref.U) * want
  before = [t.clone() for t in ts]
  out = [torch.full_like(t, 7) for t in ts]
  norm = bpl.gradient_norm(ts, norm_type=p)
  assert norm.shape == () and norm.dtype == (F64 if any(t.dtype == F64 for t in ts) else F32)
  assert abs(float(norm) - want) <= tol
  assert torch.equal(bpl.clip_gradients(ts, max_norm, norm_type=p, out=out), norm)
  assert all(torch.equal(a, b) for a, b in zip(ts, before))
  assert torch.equal(bpl.clip_gradients(ts, max_norm, norm_type=p), norm)
  factor = min(1.0, max_norm / (want + 1e-6))
  for a, b, o in zip(before, ts, out):
    assert torch.equal(b, o)
    exact = a.double() * factor
    if factor == 1.0:
      assert torch.equal(b, a)
    else:
      small = 2.0 ** -25 if a.dtype == F16 else 0.0
      assert ((b.double() - exact).abs() <= exact.abs() * (ref.half_step(a.dtype) + 16 * ref.U) + small).all()


@pytest.mark.parametrize('p', [2.0, math.inf])
@pytest.mark.parametrize('dtypes', [[F32], [F16], [BF16], [F64], [F32, BF16, F64, F16]], ids=str)
def test_types_and_sizes(cuda, dtypes, p):
  sizes = [1, 3, 0, 4, 5, 8, 9, 1023, 4096, 4097, 8191, 8192, 8193, 70_001]
  for max_norm in (0.5, 1e9, 0.0):
    check(cuda, make(cuda, sizes, dtypes), max_norm, p)


@pytest.mark.parametrize('count', [1, 24, 25, 160, 161, 1000, 1001, 2300])
def test_many_tensors(cuda, count):
  check(cuda, make(cuda, [i % 37 for i in range(count)], [F32, BF16], seed=count), 1.0)


def test_views_of_a_bucket_at_any_address(cuda):
  for dtype in (F32, BF16):
    bucket = make(cuda, [300_000], [dtype])[0]
    sizes = [1, 7, 100_001, 2, 5000, 190_000]
    check(cuda, list(bucket.split(sizes + [300_000 - sum(sizes)])), 0.25)
    # results at other addresses modulo 16 bytes than their gradients
    grads = list(bucket[1:].split([10_000, 289_999]))
    other = torch.zeros(300_004, dtype=dtype, device=cuda)
    out = [other[2:10_002], other[10_002:300_001]]
    bpl.clip_gradients(grads, 0.1, out=out)
    factor = 0.1 / (norm_of(grads) + 1e-6)
    for g, o in zip(grads, out):
      assert ((o.double() - g.double() * factor).abs() <= g.double().abs() * factor * (ref.half_step(dtype) + 16 * ref.U)).all()
    assert not other[:2].any() and not other[300_001:].any()


def test_a_large_tensor(cuda):
  check(cuda, make(cuda, [30_000_001], [BF16]) + make(cuda, [5], [F32]), 3.0)


def test_other_memory_orders_gaps_and_broadcast_gradients(cuda):
  base = make(cuda, [60 * 50], [F32])[0].reshape(60, 50)
  dense = base.t()
  gaps = make(cuda, [60 * 50], [F32], seed=1)[0].reshape(60, 50)[::2, 5:20]
  row = make(cuda, [50], [F32], seed=2)[0].expand(3, 50)
  want = norm_of([dense, gaps, row])
  assert abs(float(bpl.gradient_norm([dense, gaps, row])) - want) <= 12 * ref.U * want
  with pytest.raises(ValueError):
    bpl.clip_gradients([dense, row], 1.0)
  kept = [dense.clone(), gaps.clone()]
  want = norm_of(kept)
  bpl.clip_gradients([dense, None, gaps], 1.0)
  for t, k in zip((dense, gaps), kept):
    assert ((t - k.double() / (want + 1e-6)).abs() <= k.abs() * 4 * ref.U).all()
  out = [torch.zeros(50, 60, device=cuda), torch.zeros(30, 15, device=cuda)]
  bpl.clip_gradients([dense, gaps], 0.5, out=out)
  factor = 0.5 / (norm_of([dense, gaps]) + 1e-6)
  for t, o in zip((dense, gaps), out):
    assert ((o - t.double() * factor).abs() <= t.abs() * 8 * ref.U).all()


def test_squares_beyond_the_range_of_32_bits(cuda):
  for value in (1e30, 3e38, 1e-30, 1e-40):
    t = torch.full((1000,), value, device=cuda)
    want = float(t[0].double()) * math.sqrt(1000)
    got = float(bpl.gradient_norm([t]))
    assert got == math.inf if want > 3.4e38 else abs(got - want) <= 2 * ref.U * want + 2.0 ** -150
  t = torch.full((1000,), 1e30, device=cuda)
  bpl.clip_gradients([t], 1.0)
  assert abs(float(t[0]) * math.sqrt(1000) - 1) < 8 * ref.U
  mixed = torch.zeros(4096, device=cuda)
  mixed[::64] = 1e25
  assert abs(float(bpl.gradient_norm([mixed])) / 8e25 - 1) < 4 * ref.U


def test_norms_that_are_no_finite_number(cuda):
  for p in (2.0, math.inf):
    t = torch.ones(5000, device=cuda)
    t[777] = math.inf
    assert float(bpl.clip_gradients([t], 1.0, norm_type=p)) == math.inf
    assert torch.isnan(t[777]) and not t[:777].any() and not t[778:].any()
    t = torch.ones(5000, device=cuda)
    t[4999] = math.nan
    assert math.isnan(float(bpl.clip_gradients([t], 1.0, norm_type=p))) and torch.isnan(t).all()


def test_nothing_to_clip(cuda):
  assert float(bpl.clip_gradients([], 1.0)) == 0.0 and float(bpl.gradient_norm([None])) == 0.0
  empty = torch.zeros(0, device=cuda)
  assert float(bpl.clip_gradients([empty], 1.0)) == 0.0
  zeros = torch.zeros(100, device=cuda)
  assert float(bpl.clip_gradients(zeros, 1.0)) == 0.0 and not zeros.any()


def test_results_that_share_memory_are_refused(cuda):
  t = torch.randn(100, device=cuda)
  kept = t.clone()
  for grads, out in (([t, t], None), ([t, t[50:]], None), ([t[:60], t[40:]], None), ([t[:50], t[50:]], [t[1:51], t[51:]][:1] + [t[50:]]),
                     ([t], [t[:]])):
    if out is not None and len(grads) == 1:
      bpl.clip_gradients(grads, 1e9, out=out)             # its own gradient is in place
      continue
    with pytest.raises(ValueError):
      bpl.clip_gradients(grads, 1.0, out=out)
  assert torch.equal(t, kept)


def test_the_same_bits_every_time_and_a_changed_version(cuda):
  ts = make(cuda, [100_000, 50_001, 7], [BF16, F32])
  norms = {float(bpl.gradient_norm(ts)) for _ in range(5)}
  assert len(norms) == 1
  w = torch.randn(10, device=cuda, requires_grad=True)
  t = torch.randn(10, device=cuda)
  y = (w * t).sum()
  bpl.clip_gradients([t], 0.1)
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):
    y.backward()


def test_gradients_of_this_library(cuda):
  """The weight gradients of a CSR product and of the operators over sequences, clipped together."""
  g = torch.Generator(cuda).manual_seed(1)
  r = lambda *s: torch.randn(*s, device=cuda, generator=g)
  indptr = torch.arange(0, 401, 4, dtype=torch.int32, device=cuda)
  indices = torch.randint(0, 50, (400,), dtype=torch.int32, device=cuda, generator=g)
  data = r(400).requires_grad_(True)
  weight, A = r(100, 4).requires_grad_(True), (-r(100, 8).abs()).requires_grad_(True)
  rows = torch.stack([bpl.csr_matvec(data, indices, indptr, r(50), shape=(100, 50)) for _ in range(6)])
  y = bpl.state_scan(bpl.short_conv(rows, weight, activation='silu'), r(6, 100), A, r(6, 8), r(6, 8), delta_softplus=True)
  y.square().sum().backward()
  grads = [p.grad for p in (data, weight, A)]
  want = norm_of(grads)
  assert want > 0.01
  norm = bpl.clip_gradients(grads, 0.01)
  assert abs(float(norm) - want) <= 12 * ref.U * want
  assert abs(norm_of(grads) - 0.01 * want / (want + 1e-6)) <= 0.01 * 16 * ref.U
