"""The token-model operators without a GPU: refusals that come before any CUDA
call, workspace and tape sizes, zero-trip calls, and the 64-bit reference's own
properties."""
import ctypes as C

import numpy as np
import pytest
import torch

import stadeb200 as sb
import token_ref as R
from stadeb200 import _lib
from stadeb200 import token_ops as T

F32, F64, BF16 = _lib.STADE_F32, _lib.STADE_F64, _lib.STADE_BF16
N = None


def _call(name, *args):
    o = _lib.make_opts()
    return getattr(_lib.lib(), name)(*args, C.byref(o))


@pytest.mark.parametrize("name,args", [
    ("stade_embed", (7, N, N, N, 1.0, 0, 4, 4, 4)),
    ("stade_embed", (F32, N, N, N, 1.0, 0, -1, 4, 4)),
    ("stade_embed", (F32, N, N, N, 1.0, 0, 4, 4, 4)),
    ("stade_embed", (F32, N, N, N, 1.0, 0, 1 << 31, 4, 4)),
    ("stade_embed_b", (-1, N, N, N, 1.0, 0, 4, 4, 4)),
    ("stade_embed_b", (F32, N, N, N, 1.0, 0, 4, -4, 4)),
    ("stade_embed_b", (F32, N, N, N, 1.0, 0, 4, 4, 4)),
    ("stade_layer_norm", (F32, N, N, N, N, N, N, 1e-5, 4, 4)),
    ("stade_layer_norm", (F32, N, N, N, N, N, N, -1.0, 4, 4)),
    ("stade_layer_norm", (F32, N, N, N, N, N, N, float("nan"), 4, 4)),
    ("stade_layer_norm", (9, N, N, N, N, N, N, 1e-5, 4, 4)),
    ("stade_layer_norm_b", (F32, N, N, N, N, N, N, N, N, 4, 4)),
    ("stade_layer_norm_b", (F32, N, N, N, N, N, N, N, N, 4, -4)),
    ("stade_tape8_push", (F32, N, N, N, 4, 4)),
    ("stade_tape8_pop", (F32, N, N, N, 4, -1)),
    ("stade_act_tape8", (F32, 0, N, N, N, N, 4, 4)),
    ("stade_act_tape8", (F32, 5, N, N, N, N, 4, 4)),
    ("stade_act_tape8_b", (F32, 1, N, N, N, N, 4, 4)),
    ("stade_expert_mm", (F32, N, N, N, N, 4, 2, 4, 4)),
    ("stade_expert_mm", (F32, N, N, N, N, 4, 1 << 16, 4, 4)),
    ("stade_expert_mm", (F32, N, N, N, N, 4, 2, 1 << 21, 4)),
    ("stade_expert_mm_b", (F32, N, N, N, N, N, N, 4, 2, 4, 4)),
    ("stade_expert_mm_b", (F32, N, N, N, N, N, N, 4, 2, -4, 4)),
])
def test_invalid_arguments(name, args):
    assert _call(name, *args) == _lib.STADE_EINVAL
    assert _lib.lib().stade_last_error()


@pytest.mark.parametrize("name,args", [
    ("stade_tape8_push", (F64, N, N, N, 4, 4)),
    ("stade_act_tape8_b", (F64, 1, N, N, N, N, 4, 4)),
])
def test_unsupported_types(name, args):
    assert _call(name, *args) == _lib.STADE_ENOTSUP


@pytest.mark.parametrize("name,args", [
    ("stade_embed", (F32, N, N, N, 1.0, 0, 0, 4, 4)),
    ("stade_embed", (F32, N, N, N, 1.0, 0, 4, 4, 0)),
    ("stade_embed_b", (F32, N, N, N, 1.0, 0, 0, 4, 4)),
    ("stade_layer_norm", (F32, N, N, N, N, N, N, 1e-5, 0, 4)),
    ("stade_layer_norm_b", (F32, N, N, N, N, N, N, N, N, 0, 4)),
    ("stade_tape8_push", (F32, N, N, N, 0, 4)),
    ("stade_act_tape8", (F32, 2, N, N, N, N, 4, 0)),
    ("stade_expert_mm", (F32, N, N, N, N, 0, 2, 4, 4)),
    ("stade_expert_mm_b", (F32, N, N, N, N, N, N, 0, 2, 4, 4)),
])
def test_nothing_to_do(name, args):
    if name == "stade_embed_b":
        o = _lib.make_opts()
        args = (F32, C.c_void_p(256), N, N, 1.0, 0, 0, 4, 4)   # an address that nothing touches
        assert _lib.lib().stade_embed_b(*args, C.byref(o)) == _lib.STADE_OK
        return
    assert _call(name, *args) == _lib.STADE_OK


def test_sizes_of_tapes_and_workspaces():
    L = _lib.lib()
    assert L.stade_initstacks_tape8(5, 64) == 10 and L.stade_initstacks_tape8(5, 65) == 15
    assert L.stade_initstacks_tape8(0, 64) == 0
    assert T.embed_b_workspace(1000, 50, 8) >= 2 * 2 * 4 * 1000
    assert T.embed_b_workspace(0, 50, 8) == 0
    assert T.layer_norm_b_workspace(torch.float64, 100, 64) >= T.layer_norm_b_workspace(torch.float32, 100, 64) > 0
    assert T.expert_mm_workspace(torch.bfloat16, 100, 4, 8, 8) > 0
    assert T.expert_mm_b_workspace(torch.bfloat16, 0, 4, 8, 8) == 0


def test_python_refusals():
    t = torch.zeros(4, 4)
    with pytest.raises(ValueError):          # not on a GPU
        sb.layer_norm_cuda(t, None, None, t, t, t, 1e-5, 4, 4)
    with pytest.raises(TypeError):
        sb.layer_norm_cuda(t.int(), None, None, t, t, t, 1e-5, 4, 4)
    with pytest.raises(TypeError):
        sb.embed_cuda(t, t, [1], 1.0, 4, 4, 4)
    with pytest.raises(ValueError):
        sb.embed_cuda(t, t, t, 1.0, -1, 4, 4)
    with pytest.raises(ValueError):
        sb.act_tape8_cuda("swish", t, t, t, t, 4, 4)
    with pytest.raises(ValueError):
        sb.expert_mm_cuda(t, t, t, t, 4, -2, 4, 4)


def test_reference_tape_is_within_half_a_step():
    rng = np.random.RandomState(0)
    x = (rng.randn(3, 70) * np.exp2(rng.randint(-9, 9, (3, 70)))).astype(np.float32).astype(np.float64)
    q, e = R.tape8(x)
    v = R.tape8_values(q, e)
    step = np.repeat(np.exp2(e.astype(float) - 127), 32, axis=1)[:, :70]
    clipped = np.abs(q) == 127
    assert np.all(np.abs(v - x)[~clipped] <= step[~clipped] / 2)
    assert np.all(np.abs(v - x) < step)


@pytest.mark.parametrize("act", list(T.ACTIVATIONS))
def test_reference_slopes_against_differences(act):
    x, h = np.linspace(-4, 4, 81) + 0.013, 1e-6
    fd = (R.act(act, x + h) - R.act(act, x - h)) / (2 * h)
    assert np.abs(fd - R.act_slope(act, x)).max() < 1e-8
