"""Refusals of the operators over whole sequences and of clipping at the ends of their ranges, without a GPU."""
import pytest
import torch

import brainpylib_b200 as bpl
from brainpylib_b200._lib import workspace_bytes
from test_sequence_checks_cpu import call, conv_descriptor, scan_descriptor

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


@pytest.mark.parametrize('name,descriptor,indptr', [('state_scan', scan_descriptor, 8), ('state_scan_backward', scan_descriptor, 8),
                                                    ('short_conv', conv_descriptor, 3), ('short_conv_backward', conv_descriptor, 3)])
def test_descriptors_whose_sequences_are_not_their_tokens(name, descriptor, indptr):
  """Without bounds, sequences of one length fill the tokens: a kernel goes by all three.  No GPU is reached."""
  for bad in (dict(sequences=2, length=4), dict(sequences=1, length=5), dict(sequences=3, length=1), dict(sequences=0, length=4),
              dict(sequences=2 ** 31 - 1, length=2), dict(tokens=0, sequences=1, length=4)):
    code, text = call(name, descriptor(**bad), without(indptr))
    assert code == 3 and 'sequences' in text, bad
  assert call(name, descriptor(sequences=2 ** 31), ADDRESSES)[0] == 3


def test_the_rates_are_needed_without_tokens_as_well():
  """Sequences without a token still come with states, and threads that read their rates."""
  code, text = call('state_scan', scan_descriptor(tokens=0, sequences=1, length=0), without(2))
  assert code == 3 and 'null buffer' in text
