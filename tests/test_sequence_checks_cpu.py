"""Refusals of the operators over whole sequences and of clipping, without a GPU: what raises before any launch, and what the C
targets report through the status channel."""
import ctypes
import struct

import pytest
import torch

import brainpylib_b200 as bpl
from brainpylib_b200 import _lib

F32, BF16 = torch.float32, torch.bfloat16


def scan_args(tokens=6, channels=8, state=4, groups=2, dtype=F32):
  z = torch.zeros
  return dict(x=z(tokens, channels, dtype=dtype), delta=z(tokens, channels, dtype=dtype), A=z(channels, state),
              B=z(tokens, groups, state, dtype=dtype), C=z(tokens, groups, state, dtype=dtype))


def scan(**changes):
  a = scan_args()
  kw = {k: v for k, v in changes.items() if k not in a}
  a.update({k: v for k, v in changes.items() if k in a})
  return bpl.state_scan(a['x'], a['delta'], a['A'], a['B'], a['C'], **kw)


def step(state=None, **changes):
  a = scan_args()
  kw = {k: v for k, v in changes.items() if k not in a}
  a.update({k: v for k, v in changes.items() if k in a})
  return bpl.state_scan_step(a['x'], a['delta'], a['A'], a['B'], a['C'], torch.zeros(6, 8, 4) if state is None else state, **kw)


@pytest.mark.parametrize('error,changes', [
  (TypeError, dict(x=[1.0])),
  (TypeError, dict(x=torch.zeros(6, 8, dtype=torch.float64))),
  (ValueError, dict(x=torch.zeros(8))),
  (ValueError, dict(x=torch.zeros(1, 1, 6, 8))),
  (ValueError, dict(delta=torch.zeros(6, 7))),
  (TypeError, dict(delta=torch.zeros(6, 8, dtype=BF16))),
  (ValueError, dict(A=torch.zeros(7, 4))),
  (ValueError, dict(A=torch.zeros(8, 129))),
  (ValueError, dict(A=torch.zeros(8, 0))),
  (TypeError, dict(A=torch.zeros(8, 4, dtype=BF16))),
  (ValueError, dict(B=torch.zeros(5, 2, 4))),
  (ValueError, dict(B=torch.zeros(6, 2, 3))),
  (ValueError, dict(B=torch.zeros(6, 3, 4), C=torch.zeros(6, 3, 4))),
  (ValueError, dict(B=torch.zeros(6, 0, 4), C=torch.zeros(6, 0, 4))),
  (ValueError, dict(C=torch.zeros(6, 4))),
  (ValueError, dict(D=torch.zeros(7))),
  (TypeError, dict(D=torch.zeros(8, dtype=torch.float64))),
  (ValueError, dict(z=torch.zeros(6, 9))),
  (TypeError, dict(z=torch.zeros(6, 8, dtype=BF16))),
  (ValueError, dict(delta_bias=torch.zeros(1))),
])
def test_operands_of_the_scan_and_its_step(error, changes):
  with pytest.raises(error):
    scan(**changes)
  with pytest.raises(error):
    step(**changes)


@pytest.mark.parametrize('error,changes', [
  (TypeError, dict(indptr=torch.tensor([0, 6]))),
  (ValueError, dict(indptr=torch.zeros(0, dtype=torch.int32))),
  (ValueError, dict(indptr=torch.zeros(1, 2, dtype=torch.int32))),
  (ValueError, dict(initial_state=torch.zeros(2, 8, 4))),
  (TypeError, dict(initial_state=torch.zeros(1, 8, 4, dtype=BF16))),
  (ValueError, dict(indptr=torch.tensor([0, 2, 6], dtype=torch.int32), initial_state=torch.zeros(1, 8, 4))),
])
def test_sequences_of_the_scan(error, changes):
  with pytest.raises(error):
    scan(**changes)


def test_packed_bounds_do_not_go_with_batches():
  a = {k: v[None] if k != 'A' else v for k, v in scan_args().items()}
  with pytest.raises(ValueError, match='indptr'):
    bpl.state_scan(a['x'], a['delta'], a['A'], a['B'], a['C'], indptr=torch.tensor([0, 6], dtype=torch.int32))
  with pytest.raises(ValueError, match='indptr'):
    bpl.short_conv(torch.zeros(1, 6, 8), torch.zeros(8, 4), indptr=torch.tensor([0, 6], dtype=torch.int32))


@pytest.mark.parametrize('error,changes', [
  (ValueError, dict(state=torch.zeros(5, 8, 4))),
  (ValueError, dict(state=torch.zeros(6, 8, 5))),
  (ValueError, dict(state=torch.zeros(6, 32))),
  (ValueError, dict(state=torch.zeros(6, 4, 8).transpose(1, 2))),
  (TypeError, dict(state=torch.zeros(6, 8, 4, dtype=BF16))),
  (TypeError, dict(slots=torch.zeros(6, dtype=torch.int64))),
  (ValueError, dict(slots=torch.zeros(5, dtype=torch.int32))),
  (ValueError, dict(x=torch.zeros(70_000, 8), slots=torch.zeros(70_000, dtype=torch.int32))),
])
def test_states_and_slots_of_the_single_steps(error, changes):
  with pytest.raises(error):
    step(**changes)
  changes = dict(changes)
  state = changes.pop('state', torch.zeros(6, 8, 4))
  with pytest.raises(error):
    bpl.short_conv_step(changes.pop('x', torch.zeros(6, 8)), state, torch.zeros(8, 5), **changes)


@pytest.mark.parametrize('error,args,kw', [
  (ValueError, (torch.zeros(6, 8), torch.zeros(8, 9)), {}),
  (ValueError, (torch.zeros(6, 8), torch.zeros(8, 0)), {}),
  (ValueError, (torch.zeros(6, 8), torch.zeros(7, 4)), {}),
  (TypeError, (torch.zeros(6, 8), torch.zeros(8, 4, dtype=BF16)), {}),
  (TypeError, (torch.zeros(6, 8, dtype=BF16), torch.zeros(8, 4, dtype=torch.float16)), {}),
  (TypeError, (torch.zeros(6, 8, dtype=BF16), torch.zeros(8, 4), torch.zeros(8, dtype=BF16)), {}),
  (ValueError, (torch.zeros(6, 8), torch.zeros(8, 4), torch.zeros(7)), {}),
  (ValueError, (torch.zeros(6, 8), torch.zeros(8, 4)), dict(activation='relu')),
  (ValueError, (torch.zeros(6, 8), torch.zeros(8, 4)), dict(initial_state=torch.zeros(1, 8, 4))),
  (TypeError, (torch.zeros(6, 8, dtype=torch.int32), torch.zeros(8, 4)), {}),
])
def test_operands_of_the_convolution(error, args, kw):
  with pytest.raises(error):
    bpl.short_conv(*args, **kw)


@pytest.mark.parametrize('call', [
  lambda: scan(), lambda: step(), lambda: bpl.short_conv(torch.zeros(6, 8), torch.zeros(8, 4)),
  lambda: bpl.short_conv_step(torch.zeros(6, 8), torch.zeros(6, 8, 3), torch.zeros(8, 4)),
  lambda: bpl.gradient_norm([torch.zeros(3)]), lambda: bpl.clip_gradients([torch.zeros(3)], 1.0)])
def test_operands_on_the_cpu_are_refused(call):
  with pytest.raises(bpl.GPUOperatorNotFound):
    call()


@pytest.mark.parametrize('error,args,kw', [
  (ValueError, ([torch.zeros(3)], -1.0), {}),
  (ValueError, ([torch.zeros(3)], float('nan')), {}),
  (ValueError, ([torch.zeros(3)], 1.0), dict(norm_type=1.0)),
  (ValueError, ([torch.zeros(3)], 1.0), dict(out=[])),
  (ValueError, ([torch.zeros(3), None], 1.0), dict(out=[None, torch.zeros(3)])),
  (TypeError, ([1.0], 1.0), {}),
  (TypeError, ([torch.zeros(3, dtype=torch.int32)], 1.0), {}),
  (TypeError, ([torch.zeros(3, 3).to_sparse()], 1.0), {}),
])
def test_arguments_of_clipping(error, args, kw):
  with pytest.raises(error):
    bpl.clip_gradients(*args, **kw)


# ---- the C targets ------------------------------------------------------------------------------------------------------
def status():
  message = ctypes.create_string_buffer(256)
  code = _lib.lib().bpl_last_status(message, 256)
  _lib.lib().bpl_clear_status()
  return code, message.value.decode()


def scan_descriptor(tokens=4, sequences=1, length=4, channels=8, groups=1, state=4, dtype=0, flags=0):
  return struct.pack('<8I7q', tokens, sequences, length, channels, groups, state, dtype, flags, *([8] * 7))


def conv_descriptor(tokens=4, sequences=1, length=4, channels=8, width=4, dtype=0, weight_dtype=0, flags=0):
  return struct.pack('<8Iq', tokens, sequences, length, channels, width, dtype, weight_dtype, flags, 8)


def clip_descriptor(elements, dtype=0, norm_type=2, norm_dtype=0, flags=1, max_norm=1.0):
  return struct.pack('<4Id', len(elements), norm_type, norm_dtype, flags, max_norm) + b''.join(
    struct.pack('<QII', n, dtype, 0) for n in elements)


def call(name, opaque, buffers):
  _lib.lib().bpl_clear_status()
  _lib.target(name)(None, (ctypes.c_void_p * len(buffers))(*buffers), opaque, len(opaque))
  return status()


@pytest.mark.parametrize('name', ['state_scan', 'state_scan_backward', 'state_scan_step', 'short_conv', 'short_conv_backward',
                                  'short_conv_step', 'clip_gradients'])
def test_targets_refuse_descriptors_of_another_size_and_missing_buffers(name):
  none = [None] * 24
  assert call(name, b'12345', none) == (1, 'Invalid opaque object size')
  good = scan_descriptor() if 'scan' in name else conv_descriptor() if 'conv' in name else clip_descriptor([5])
  code, text = call(name, good, none)
  assert code == 3 and name in text
  assert name not in bpl.gpu_ops.target_names()          # (the registry lists the reference's names)


def test_targets_refuse_sizes_they_cannot_take():
  none = [None] * 24
  for name in ('state_scan', 'state_scan_backward', 'state_scan_step'):
    for bad in (dict(state=0), dict(state=129), dict(groups=0), dict(groups=3), dict(dtype=3), dict(tokens=2 ** 31)):
      assert call(name, scan_descriptor(**bad), none)[0] == 3, (name, bad)
  for name in ('short_conv', 'short_conv_backward', 'short_conv_step'):
    for bad in (dict(width=0), dict(width=9), dict(dtype=3), dict(dtype=1, weight_dtype=2), dict(tokens=2 ** 31)):
      assert call(name, conv_descriptor(**bad), none)[0] == 3, (name, bad)
  some = [4096 * (i + 1) for i in range(24)]                # (addresses that no check reads)
  assert 'rows' in call('state_scan_step', scan_descriptor(tokens=65_536, sequences=65_536), some)[1]
  assert 'state for every row' in call('state_scan_step', scan_descriptor(tokens=5, sequences=4), some[:8] + [None] + some[9:])[1]
  assert 'state for every row' in call('short_conv_step', conv_descriptor(tokens=5, sequences=4), some[:3] + [None] + some[4:])[1]
  assert 'null buffer' in call('state_scan_step', scan_descriptor(), some[:9] + [None] + some[10:])[1]        # (no states)
  assert 'null buffer' in call('short_conv_step', conv_descriptor(), some[:4] + [None] + some[5:])[1]
  for bad in (dict(dtype=4), dict(norm_type=1), dict(norm_dtype=1), dict(max_norm=-1.0), dict(max_norm=float('nan'))):
    assert call('clip_gradients', clip_descriptor([5, 5], **bad), some)[0] == 3, bad
  assert call('clip_gradients', clip_descriptor([2 ** 40, 5]), some)[0] == 3
  # two gradients of 2048 floats whose results overlap; a result over another gradient
  grads, parts = [1 << 20, 2 << 20], [8 << 20, 9 << 20]
  for out in ([3 << 20, (3 << 20) + 8188], [3 << 20, (1 << 20) + 4]):
    code, text = call('clip_gradients', clip_descriptor([2048, 2048]), grads + out + parts)
    assert code == 3 and 'share memory' in text


def test_workspaces():
  w = _lib.workspace_bytes
  assert w('state_scan', scan_descriptor(tokens=16)) == 0                      # one chunk hands nothing on
  long = w('state_scan', scan_descriptor(tokens=100_000))
  assert long > 0 and long % (8 * 5 * 4) == 0
  assert w('state_scan_backward', scan_descriptor(tokens=100)) >= 100 * 2 * 4 * 4
  assert w('short_conv_backward', conv_descriptor(tokens=100)) >= 8 * 5 * 4
  assert w('clip_gradients', clip_descriptor([5])) > 0
  assert w('state_scan_step', scan_descriptor()) == w('short_conv', conv_descriptor()) == 0
  for name in ('state_scan', 'state_scan_backward', 'short_conv_backward', 'clip_gradients'):
    assert w(name, b'123') == 0
