"""The device-side step over an 8-bit cache, without a GPU: the references' own rules, the layout, and what the Python classes and the
C ABI refuse before anything reaches a device."""
import ctypes

import numpy as np
import pytest
import torch

from kv8_helpers import decode, encode, pitch_of, plan_reference, sample_reference, write_reference
from paged_infer_b200 import _lib, api


class NoContext:
    """Stands for a context on device 0 where no device is: every check ahead of the library's call."""
    device, handle = 0, None


def refused(status):
    return pytest.raises(api.PiError, match=f"error {status}")


def test_every_entry_refuses_a_null_context():
    L = _lib.lib()
    assert L.pi_step_plan(None, None, None, None, 1, None, 0) == _lib.PI_ERR_INVALID_ARG
    assert L.pi_kv8_pool_create(None, None, _lib.PI_INT8, None, None, ctypes.byref(ctypes.c_void_p())) == _lib.PI_ERR_INVALID_ARG
    assert L.pi_kv8_copy_block(None, None, 0, 1) == _lib.PI_ERR_INVALID_ARG
    assert L.pi_kv8_read_token(None, None, 0, 0, 0, None, None) == _lib.PI_ERR_INVALID_ARG
    assert L.pi_kv8_write(None, None, 0, _lib.PI_F32, None, 0, None, 0, None, 0) == _lib.PI_ERR_INVALID_ARG
    assert L.pi_kv8_attention(None, None, 0, 1, _lib.PI_F32, None, 0, None, 0, None, 0, 0, 1, 1, 0, 1.0) == _lib.PI_ERR_INVALID_ARG
    assert L.pi_sample(None, None, _lib.PI_F32, 0, 0, 1, None, None, None, None, None, None, None) == _lib.PI_ERR_INVALID_ARG
    assert L.pi_kv8_pool_bytes(None) == 0 and L.pi_kv8_pool_pitch(None) == 0
    L.pi_kv8_pool_destroy(None)


def test_tensors_elsewhere_or_of_another_form_are_refused():
    c = NoContext()
    i = torch.zeros(4, dtype=torch.int32)
    for t in (i, i.float(), i[::2]):
        with refused(_lib.PI_ERR_INVALID_ARG):
            api.StepPlan(c, 16, t.view(2, -1) if t.is_contiguous() else t[None])
    with refused(_lib.PI_ERR_INVALID_ARG):
        api.StepPlan(c, 16, i)
    layout = api.KvLayout(1, 2, 16, 1, 64)
    codes, scales = torch.zeros(1, 2, 1, 2, 16, 64, dtype=torch.int8), torch.zeros(1, 2, 1, 2)
    for a, b in ((codes, scales), (codes, None), (codes.float(), scales), (codes[:, :1], scales)):
        with refused(_lib.PI_ERR_INVALID_ARG):
            api.KvCache8(c, layout, codes=a, scales=b)
    f = torch.zeros(2)
    with refused(_lib.PI_ERR_INVALID_ARG):
        api.sample(c, torch.zeros(2, 8), f, i[:2], f, f, f, i[:2])


def test_pitch_holds_the_head_dim():
    for d in range(1, 257):
        assert api.KvCache8.pitch_of(d) == pitch_of(d) >= d
    with refused(_lib.PI_ERR_INVALID_ARG):
        api.KvCache8.pitch_of(257)


def test_step_arrays_match_the_header():
    assert ctypes.sizeof(_lib.StepArraysC) == 4 * 4 + 7 * 8
    assert _lib.StepArraysC.tables.offset == 16 and _lib.StepArraysC.slots.offset == 16 + 5 * 8


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_codes_are_within_half_a_step(kind):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((64, 64)).astype(np.float32)
    s = np.float32(np.abs(x).max() * (np.float32(1) / np.float32(127 if kind == "int8" else 448)))
    y = decode(encode(x, s, kind), kind) * s
    step = s / 2 if kind == "int8" else np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10)   # e4m3: half a step of the value, or of the subnormals
    assert (np.abs(y - x) <= step * (1 + 1e-6)).all()


def test_references_follow_their_rules():
    # a block whose scale does not grow keeps its codes; one that grows keeps its values up to half a new step
    rng = np.random.default_rng(2)
    for grow in (0.5, 3.0):
        codes, scales = np.zeros((2, 1, 2, 4, 32), np.uint8), np.zeros((2, 1, 2), np.float32)
        k, v = rng.standard_normal((2, 3, 1, 32)).astype(np.float32)
        codes, scales = write_reference(codes, scales, k, v, [4, 5, 6], "int8", 4)
        after, s2 = write_reference(codes, scales, k[:1] * grow * 4, v[:1] * 0.01, [7], "int8", 4)
        assert (after[1, 0, 1, :3] == codes[1, 0, 1, :3]).all() and s2[1, 0, 1] == scales[1, 0, 1]
        kept = decode(after[1, 0, 0, :3], "int8") * s2[1, 0, 0]
        assert (np.abs(kept - k[:, 0]) <= (s2[1, 0, 0] + scales[1, 0, 0]) / 2 * 1.001).all()
    tables, lens, cu, seq, pos, slots, counts = plan_reference([3, 0], [2, 4], [7, 5], np.array([[9, -1], [-1, -1]], np.int32), 4, 8)
    assert tables.tolist() == [[9, 7], [5, -1]] and lens.tolist() == [2, 1] and counts.tolist() == [6, 2, 0]
    assert slots.tolist() == [39, 28, 20, 21, 22, 23, -1, -1] and cu.tolist() == [0, 2, 6]
    assert sample_reference(np.array([1.0, 3.0, 3.0, 2.0]), 0, 0, 1, 0, 0.9) == (1, 1.0)
    assert sample_reference(np.array([1.0, 3.0, 3.0, 2.0]), 1.0, 2, 1, 0, 0.6) == (2, 0.5)
    assert sample_reference(np.zeros(4), 1.0, 0, 0.5, 0, 0.5) == (1, 0.5)
