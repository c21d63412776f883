"""Refusals of the operators over whole sequences and of clipping at the ends of their ranges, without a GPU."""
from test_sequence_checks_cpu import call, scan_descriptor

ADDRESSES = [4096 * (i + 1) for i in range(24)]           # (that no check reads)


def without(*missing):
  return [None if i in missing else a for i, a in enumerate(ADDRESSES)]


def test_the_gradient_without_channels_still_writes_those_of_B_and_C():
  for missing in (16, 17):
    code, text = call('state_scan_backward', scan_descriptor(channels=0), without(missing))
    assert code == 3 and 'null buffer' in text
