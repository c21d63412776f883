"""Refusals of the layers of language models, without a GPU: what raises before any launch, and what the C targets report through the
status channel."""
import ctypes
import struct

import pytest
import torch

import brainpylib_b200 as bpl
from brainpylib_b200 import _lib

F32, F16, BF16, I32 = torch.float32, torch.float16, torch.bfloat16, torch.int32
z = torch.zeros


# ---- embedding -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('error,ids,weight,kw', [
  (TypeError, [1, 2], z(4, 3), {}),
  (TypeError, z(3), z(4, 3), {}),
  (TypeError, z(3, dtype=torch.int16), z(4, 3), {}),
  (TypeError, z(3, dtype=I32), z(4, 3, dtype=torch.float64), {}),
  (TypeError, z(3, dtype=I32), None, {}),
  (ValueError, z(3, dtype=I32), z(4), {}),
  (ValueError, z(3, dtype=I32), z(4, 3, 2), {}),
  (ValueError, z(3, dtype=I32), z(4, 3), dict(scale=float('nan'))),
  (ValueError, z(3, dtype=I32), z(1, 1).expand(2 ** 31, 1), {}),
  (ValueError, z(1, dtype=I32).expand(2 ** 31), z(4, 3), {}),
  (ValueError, z(3, dtype=I32), z(1, 1).expand(1, 2 ** 28), {}),
  (bpl.GPUOperatorNotFound, z(3, dtype=I32), z(4, 3), {}),
])
def test_embedding(error, ids, weight, kw):
  with pytest.raises(error):
    bpl.embedding(ids, weight, **kw)


# ---- norm_rotate -----------------------------------------------------------------------------------------------------------
def rotate(**changes):
  a = dict(q=z(6, 4, 8), k=z(6, 2, 8), positions=z(6, dtype=I32), frequencies=z(4), q_weight=z(8), k_weight=z(8))
  kw = {k: v for k, v in changes.items() if k not in a}
  a.update({k: v for k, v in changes.items() if k in a})
  return bpl.norm_rotate(*a.values(), **kw)


@pytest.mark.parametrize('error,changes', [
  (TypeError, dict(q=3)),
  (TypeError, dict(q=z(6, 4, 8, dtype=torch.float64))),
  (TypeError, dict(k=z(6, 2, 8, dtype=BF16))),
  (ValueError, dict(q=z(6, 8))),
  (ValueError, dict(q=z(5, 4, 8))),
  (ValueError, dict(q=z(6, 4, 10))),
  (ValueError, dict(q=z(6, 4, 7), k=z(6, 2, 7), q_weight=None, k_weight=None)),
  (ValueError, dict(q=z(6, 4, 258), k=z(6, 2, 258), q_weight=None, k_weight=None)),
  (ValueError, dict(q=z(6, 4, 0), k=z(6, 2, 0), q_weight=None, k_weight=None)),
  (ValueError, dict(q=z(2, 3, 4, 8))),
  (ValueError, dict(q=z(1, 65536, 8).expand(6, 65536, 8))),
  (ValueError, dict(positions=z(5, dtype=I32))),
  (ValueError, dict(positions=z(6, 1, dtype=I32))),
  (TypeError, dict(positions=z(6))),
  (ValueError, dict(frequencies=z(5))),
  (ValueError, dict(frequencies=z(2, 2))),
  (TypeError, dict(frequencies=z(4, dtype=torch.float64))),
  (ValueError, dict(frequencies=z(4, requires_grad=True))),
  (ValueError, dict(q_weight=z(7))),
  (TypeError, dict(q_weight=z(8, dtype=BF16))),
  (TypeError, dict(q=z(6, 4, 8, dtype=BF16), k=z(6, 2, 8, dtype=BF16), k_weight=z(8, dtype=BF16))),
  (ValueError, dict(eps=float('nan'))),
  (bpl.GPUOperatorNotFound, dict()),
])
def test_norm_rotate(error, changes):
  with pytest.raises(error):
    rotate(**changes)


# ---- decay_attention ---------------------------------------------------------------------------------------------------------
def attend(**changes):
  a = dict(q=z(6, 4, 8), k=z(6, 2, 8), v=z(6, 2, 5), log_decay=z(4))
  kw = {k: v for k, v in changes.items() if k not in a}
  a.update({k: v for k, v in changes.items() if k in a})
  return bpl.decay_attention(*a.values(), **kw)


def step(**changes):
  a = dict(q=z(6, 4, 8), k=z(6, 2, 8), v=z(6, 2, 5), log_decay=z(4), state=z(6, 4, 8, 5))
  kw = {k: v for k, v in changes.items() if k not in a}
  a.update({k: v for k, v in changes.items() if k in a})
  return bpl.decay_attention_step(*a.values(), **kw)


@pytest.mark.parametrize('error,changes', [
  (TypeError, dict(q=None)),
  (TypeError, dict(q=z(6, 4, 8, dtype=torch.float64))),
  (TypeError, dict(k=z(6, 2, 8, dtype=BF16))),
  (TypeError, dict(v=z(6, 2, 5, dtype=F16))),
  (ValueError, dict(q=z(6, 8))),
  (ValueError, dict(k=z(5, 2, 8))),
  (ValueError, dict(v=z(7, 2, 5))),
  (ValueError, dict(k=z(6, 2, 7))),
  (ValueError, dict(v=z(6, 1, 5))),
  (ValueError, dict(k=z(6, 3, 8), v=z(6, 3, 5))),
  (ValueError, dict(k=z(6, 0, 8), v=z(6, 0, 5))),
  (ValueError, dict(q=z(6, 0, 8), log_decay=z(0))),
  (ValueError, dict(q=z(6, 4, 257), k=z(6, 2, 257))),
  (ValueError, dict(q=z(6, 4, 0), k=z(6, 2, 0))),
  (ValueError, dict(v=z(6, 2, 257))),
  (ValueError, dict(v=z(6, 2, 0))),
  (ValueError, dict(log_decay=z(2))),
  (TypeError, dict(log_decay=z(4, dtype=BF16))),
  (ValueError, dict(log_decay=z(4, requires_grad=True))),
  (ValueError, dict(scale=float('nan'))),
  (bpl.GPUOperatorNotFound, dict()),
])
def test_operands_of_the_attention_and_its_step(error, changes):
  with pytest.raises(error):
    attend(**changes)
  with pytest.raises(error):
    step(**changes)


@pytest.mark.parametrize('error,changes', [
  (TypeError, dict(indptr=torch.tensor([0, 6]))),
  (ValueError, dict(indptr=z(0, dtype=I32))),
  (ValueError, dict(indptr=z(1, 2, dtype=I32))),
  (ValueError, dict(initial_state=z(2, 4, 8, 5))),
  (TypeError, dict(initial_state=z(1, 4, 8, 5, dtype=BF16))),
  (ValueError, dict(indptr=torch.tensor([0, 2, 6], dtype=I32), initial_state=z(1, 4, 8, 5))),
  (ValueError, dict(q=z(2, 3, 4, 8), k=z(2, 3, 2, 8), v=z(2, 3, 2, 5), indptr=torch.tensor([0, 6], dtype=I32))),
])
def test_sequences_of_the_attention(error, changes):
  with pytest.raises(error):
    attend(**changes)


@pytest.mark.parametrize('error,changes', [
  (ValueError, dict(q=z(1, 6, 4, 8), k=z(1, 6, 2, 8), v=z(1, 6, 2, 5))),
  (ValueError, dict(state=z(5, 4, 8, 5))),
  (ValueError, dict(state=z(6, 4, 5, 8))),
  (ValueError, dict(state=z(6, 4, 8))),
  (ValueError, dict(state=z(6, 4, 5, 8).transpose(2, 3))),
  (TypeError, dict(state=z(6, 4, 8, 5, dtype=BF16))),
  (ValueError, dict(slots=z(5, dtype=I32))),
  (TypeError, dict(slots=z(6, dtype=torch.int64))),
  (ValueError, dict(q=z(1, 4, 8).expand(65536, 4, 8), k=z(1, 2, 8).expand(65536, 2, 8), v=z(1, 2, 5).expand(65536, 2, 5))),
])
def test_states_of_the_step(error, changes):
  with pytest.raises(error):
    step(**changes)


# ---- the C targets -----------------------------------------------------------------------------------------------------------
def refuse(name, opaque, n_buffers, what, given=()):
  """Runs a target whose call has to be refused before any launch: no buffer is a real one."""
  lib = _lib.lib()
  lib.bpl_clear_status()
  buffers = (ctypes.c_void_p * n_buffers)(*[256 if i in given else None for i in range(n_buffers)])
  _lib.target(name)(None, buffers, opaque, len(opaque))
  message = ctypes.create_string_buffer(256)
  code = lib.bpl_last_status(message, 256)
  lib.bpl_clear_status()
  assert code in (1, 3) and what in message.value.decode(), (code, message.value)


def embedding_opaque(tokens=4, vocabulary=5, width=6, dtype=0, wide=0, scale=1.0, stride=6):
  return struct.pack('<5Ifq', tokens, vocabulary, width, dtype, wide, scale, stride)


def rotate_opaque(tokens=4, q_heads=2, k_heads=1, size=8, rotated=8, dtype=0, weight_dtype=0, flags=0):
  return struct.pack('<8IfI4q', tokens, q_heads, k_heads, size, rotated, dtype, weight_dtype, flags, 1e-6, 0, 16, 8, 8, 8)


def attend_opaque(tokens=4, sequences=1, length=4, heads=2, kv_heads=1, key=8, value=8, dtype=0):
  return struct.pack('<8IfI6q', tokens, sequences, length, heads, kv_heads, key, value, dtype, 1.0, 0, 16, 8, 8, 8, 8, 8)


def test_descriptor_sizes():
  for name, n in (('embedding', 3), ('embedding_backward', 4), ('norm_rotate', 8), ('norm_rotate_backward', 13), ('decay_attention', 9),
                  ('decay_attention_backward', 13), ('decay_attention_step', 7)):
    refuse(name, b'short', n, 'Invalid opaque')


def test_targets_refuse_missing_buffers_and_sizes_out_of_range():
  for name, n in (('embedding', 3), ('embedding_backward', 4)):
    refuse(name, embedding_opaque(), n, 'null buffer')
    refuse(name, embedding_opaque(tokens=2 ** 31), n, 'fewer than')
    refuse(name, embedding_opaque(vocabulary=2 ** 31), n, 'fewer than')
    refuse(name, embedding_opaque(dtype=3), n, 'fewer than')
  for name, n in (('norm_rotate', 8), ('norm_rotate_backward', 13)):
    refuse(name, rotate_opaque(), n, 'null buffer')
    for bad in (dict(size=7), dict(size=258), dict(size=0), dict(rotated=10), dict(rotated=3), dict(dtype=3), dict(weight_dtype=1),
                dict(tokens=2 ** 31), dict(q_heads=65536)):
      refuse(name, rotate_opaque(**bad), n, 'heads of 2')
  for name, n in (('decay_attention', 9), ('decay_attention_backward', 13), ('decay_attention_step', 7)):
    refuse(name, attend_opaque() if n > 7 else attend_opaque(sequences=4), n, 'null buffer')
    for bad in (dict(key=0), dict(key=257), dict(value=257), dict(kv_heads=0), dict(heads=0), dict(heads=3, kv_heads=2), dict(dtype=3), dict(heads=65536)):
      refuse(name, attend_opaque(**bad), n, 'heads of 1')
  for name, n in (('decay_attention', 9), ('decay_attention_backward', 13)):
    refuse(name, attend_opaque(sequences=2), n, 'are not the tokens', given=[i for i in range(n) if i != 4])
    refuse(name, attend_opaque(sequences=2 ** 31), n, '2^31 sequences', given=[i for i in range(n) if i != 4])
  refuse('decay_attention_step', attend_opaque(tokens=5), 7, 'a state for every row', given=(0, 1, 2, 3, 5, 6))
  refuse('decay_attention_step', attend_opaque(tokens=65536, sequences=65536), 7, '65535 rows', given=(0, 1, 2, 3, 5, 6))


def test_nothing_to_do_needs_no_buffers():
  lib = _lib.lib()
  for name, opaque, n in (('embedding', embedding_opaque(tokens=0), 3), ('embedding', embedding_opaque(width=0), 3),
                          ('norm_rotate', rotate_opaque(tokens=0), 8),
                          ('decay_attention_step', attend_opaque(tokens=0), 7)):
    lib.bpl_clear_status()
    _lib.target(name)(None, (ctypes.c_void_p * n)(), opaque, len(opaque))
    assert lib.bpl_last_status(None, 0) == 0, name


def test_workspaces_of_descriptors_out_of_range():
  for name, size in (('embedding_backward', 32), ('norm_rotate_backward', 72), ('decay_attention', 88), ('decay_attention_backward', 88)):
    assert _lib.lib().bpl_workspace_bytes(name.encode(), b'x', 1) == 0
    _lib.lib().bpl_workspace_bytes(name.encode(), b'\xff' * size, size)
    _lib.lib().bpl_workspace_bytes(name.encode(), b'\x00' * size, size)
