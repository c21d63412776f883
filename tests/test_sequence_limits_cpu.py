"""Refusals of the operators over whole sequences and of clipping at the ends of their ranges, without a GPU."""
import pytest
import torch

import brainpylib_b200 as bpl
from brainpylib_b200._lib import workspace_bytes
from test_sequence_checks_cpu import call, scan_descriptor

ADDRESSES = [4096 * (i + 1) for i in range(24)]           # (that no check reads)


def without(*missing):
  return [None if i in missing else a for i, a in enumerate(ADDRESSES)]


def test_the_gradient_without_channels_still_writes_those_of_B_and_C():
  for missing in (16, 17):
    code, text = call('state_scan_backward', scan_descriptor(channels=0), without(missing))
    assert code == 3 and 'null buffer' in text


def test_the_gradient_s_scratch_grows_with_what_the_card_runs_at_once_not_with_the_channels():
  """Parts of dB and dC: 8 bytes a token, group and state for every block of channels, of which a launch holds two rounds over the card
  at most (or 2 GiB); one more is the sum so far."""
  for tokens, channels, state in ((16_384, 4096, 128), (16_384, 8192, 128), (16_384, 16_384, 64), (100_000, 4096, 100)):
    one = 8 * tokens * state
    for dtype in (0, 1, 2):
      size = workspace_bytes('state_scan_backward', scan_descriptor(tokens=tokens, length=tokens, channels=channels, state=state, dtype=dtype))
      chunks = 16 * 4 * channels * (2 * state + 3)
      assert one <= size <= max(2 ** 31, 2 * 148 * one) + one + chunks, (tokens, channels, state, dtype, size)


@pytest.mark.parametrize('call', [bpl.gradient_norm, lambda g: bpl.clip_gradients(g, 1.0),
                                  lambda g: bpl.clip_gradients(g, 1.0, out=[torch.zeros(3)])])
def test_norms_have_no_gradient(call):
  for t in (torch.ones(3, requires_grad=True), torch.nn.Parameter(torch.ones(3)), torch.ones(3, requires_grad=True) * 2):
    with pytest.raises(ValueError, match='no gradient'):
      call([t])
    with torch.no_grad(), pytest.raises(bpl.GPUOperatorNotFound):
      call([t])


def test_more_tokens_or_sequences_than_31_bits_count():
  """Tensors of no channels, no rows, or one element seen many times: their sizes are counted, not their bytes."""
  many, state = 2 ** 31, 4
  A = torch.zeros(0, state)
  with pytest.raises(ValueError, match='2\\^31 tokens'):
    x, B = torch.zeros(many, 0), torch.zeros(1, state).expand(many, state)
    bpl.state_scan(x, x, A, B, B)
  with pytest.raises(ValueError, match='2\\^31 tokens'):
    bpl.short_conv(torch.zeros(2, many // 2, 0), torch.zeros(0, 4))
  bounds = torch.zeros(1, dtype=torch.int32).expand(many + 1)
  x, B = torch.zeros(3, 8), torch.zeros(3, state)
  with pytest.raises(ValueError, match='2\\^31 sequences'):
    bpl.state_scan(x, x, torch.zeros(8, state), B, B, indptr=bounds)
  with pytest.raises(ValueError, match='2\\^31 sequences'):
    bpl.short_conv(x, torch.zeros(8, 4), indptr=bounds)
  with pytest.raises(ValueError, match='2\\^31 sequences'):
    bpl.short_conv(torch.zeros(many, 0, 8), torch.zeros(8, 4))
  with pytest.raises(bpl.GPUOperatorNotFound):
    bpl.short_conv(x, torch.zeros(8, 4), indptr=bounds[:many])
