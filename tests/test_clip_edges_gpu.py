"""``gradient_norm`` and ``clip_gradients`` at the ends of their ranges."""
import math

import pytest
import torch

import brainpylib_b200 as bpl
import sequence_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('value,max_norm', [(3e38, 1.0), (3e38, 1e-5), (1e37, 1e-9), (1e30, 1e-12), (1e-30, 1e-37)])
def test_a_factor_below_the_normal_numbers_of_32_bits(cuda, value, max_norm, dtype):
  """The factor is a quotient in 64 bits, a result its product with an element rounded once (and once more from 32 to 16 bits)."""
  g = torch.Generator().manual_seed(0)
  t = ((0.5 + 0.5 * torch.rand(5003, generator=g, dtype=F64)) * value).to(dtype)
  wide = t.double()
  factor = max_norm / (math.sqrt(float((wide * wide).sum())) + 1e-6)
  want = wide * min(1.0, factor)
  got, out = t.to(cuda), torch.zeros(5003, dtype=dtype, device=cuda)
  bpl.clip_gradients([got.clone()], max_norm, out=[out])            # (results at other places: by elements or packets alike)
  bpl.clip_gradients([got], max_norm)
  for r in (got, out):
    # the norm: 12 roundings, the factor's one in 32 bits, the product's one; half the least subnormal number
    assert ((r.double().cpu() - want).abs() <= want * (ref.half_step(dtype) + 16 * ref.U) + 2.0 ** -150).all()


def test_operands_that_require_a_gradient(cuda):
  """A norm that a loss could contain would have no gradient: refused, as the single steps refuse it, unless no gradients are recorded."""
  leaf = torch.nn.Parameter(torch.randn(10, device=cuda))
  grown = torch.randn(10, device=cuda, requires_grad=True) * 2
  plain = torch.randn(10, device=cuda)
  for t in (leaf, grown):
    for grads in ([t], [plain, t], t, (plain, None, t)):
      for call in (bpl.gradient_norm, lambda g: bpl.clip_gradients(g, 1.0)):
        with pytest.raises(ValueError, match='no gradient'):
          call(grads)
    for out in ([torch.zeros(10, device=cuda)], (torch.zeros(10, device=cuda),)):
      with pytest.raises(ValueError, match='no gradient'):
        bpl.clip_gradients([t], 1.0, out=out)
      with pytest.raises(ValueError, match='no gradient'):
        bpl.clip_gradients([plain], 1.0, out=[t])
    with torch.no_grad():
      want = float(t.double().norm())
      assert abs(float(bpl.gradient_norm([t])) - want) <= 12 * ref.U * want
      assert abs(float(bpl.clip_gradients([t], 1e9, out=out)) - want) <= 12 * ref.U * want and torch.equal(out[0], t)


def test_norms_of_64_bits(cuda):
  """Squares and sums of float64 have 53 bits throughout: a thread adds up to 400 of them, 8 warps and 1200 blocks in at most 20 steps."""
  for sizes in ([1], [100_003], [7, 2_000_000, 33]):
    ts = [torch.randn(n, dtype=F64, device=cuda, generator=torch.Generator(cuda).manual_seed(n)) for n in sizes]
    want = math.sqrt(math.fsum(float(v) for t in ts for v in [(t * t).cpu().sum()]))
    got = bpl.gradient_norm(ts)
    assert got.dtype == F64 and abs(float(got) - want) <= 500 * 2.0 ** -53 * want
    bpl.clip_gradients(ts, want / 2)
    assert abs(float(bpl.gradient_norm(ts)) - want / 2) <= 500 * 2.0 ** -53 * want + 1e-6


def test_a_list_that_another_thread_changes_meanwhile(cuda):
  """The call holds the tensors that it has found; which it finds is the threads' affair."""
  import threading
  tensors = [torch.ones(1000, device=cuda) for _ in range(200)]
  grads, done = list(tensors), threading.Event()

  def change():
    while not done.is_set():
      grads.clear()
      grads.extend(torch.ones(1000, device=cuda) for _ in range(3))

  other = threading.Thread(target=change)
  other.start()
  try:
    for _ in range(2000):
      norm = bpl.clip_gradients(grads, 1e9)
  finally:
    done.set()
    other.join()
  assert torch.isfinite(norm)
