"""Host side of the token-model operators: embed, layer_norm, the 8-bit tape
and expert_mm, each with its reverse sweep (`_b`).

Arrays are contiguous CUDA tensors of one device, the current one; the element
type (Float32, Float64, bfloat16, float16; not Float64 on the 8-bit tape) is
that of the activation array. layer_norm's parameters and statistics and every
parameter adjoint are Float32 for Float32 and the 16-bit types and Float64 for
Float64.

The reverse sweeps add to their adjoint outputs and set the consumed seed yb
to zero, as the generated sweeps do; `accumulate=False` stores instead of
adding and `consume=False` leaves yb as it is. The calls are asynchronous on
`stream` (default: torch's current stream); a `workspace` tensor of at least
the queried bytes replaces the library's cached one. That one is shared: calls
on streams with no order between them, or from several host threads, need a
workspace each.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import (STADE_ADJ_STORE, STADE_BF16, STADE_F16, STADE_F32, STADE_F64, STADE_OK,
                   STADE_SEED_KEEP, check, lib, stade_opts)
from . import kernels

_DTYPES = {torch.float32: STADE_F32, torch.float64: STADE_F64, torch.bfloat16: STADE_BF16,
           torch.float16: STADE_F16}
ACTIVATIONS = {"relu": 1, "tanh": 2, "silu": 3, "gelu": 4}


_TYPES = {t: (code, t, torch.float64 if t == torch.float64 else torch.float32)
          for t, code in _DTYPES.items()}


def _dtype(t, name: str):
    """(dtype code, element type, parameter type, current device) by an
    activation array."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a CUDA tensor, got {type(t).__name__}")
    types = _TYPES.get(t.dtype)
    if types is None:
        raise TypeError(f"{name}: unsupported dtype {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name}: tensor must live on a CUDA device")
    return *types, torch.cuda.current_device()


def _arr(d: int, t, dtype, n: int, name: str) -> int:
    """Address of an array after its checks: CUDA, type, contiguity, length,
    and the current device d, on which the call runs."""
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_contiguous() and t.numel() >= n
            and t.get_device() == d):
        return t.data_ptr()
    kernels._arr(t, dtype, n, name)
    raise ValueError(f"{name}: tensor lives on {t.device}, the current device is cuda:{d}")


# The current stream's handle without building a Stream object, which costs as
# much as the launch of a kernel.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _run(fn, *args, stream=None, workspace=None, flags=0) -> None:
    if stream is not None:
        handle = stream.cuda_stream
    elif _raw_stream is not None:
        handle = _raw_stream(torch.cuda.current_device())
    else:
        handle = torch.cuda.current_stream().cuda_stream
    if workspace is None:
        o = stade_opts(handle, None, 0, flags)
    else:
        o = stade_opts(handle, *kernels._workspace(workspace), flags)
    code = fn(*args, C.byref(o))
    if code != STADE_OK:
        check(code)


def _opt(d, t, dtype, n, name):
    return None if t is None else _arr(d, t, dtype, n, name)


def _flags(accumulate: bool, consume: bool) -> int:
    return (0 if accumulate else STADE_ADJ_STORE) | (0 if consume else STADE_SEED_KEEP)


def _sizes(*sizes) -> None:
    if min(sizes) < 0:
        raise ValueError(f"negative size in {sizes}")


def _act(act: str) -> int:
    if act not in ACTIVATIONS:
        raise ValueError(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[act]


# ---------------------------------------------------------------------------
def embed_cuda(w, ids, y, scale, n_s, n_v, n_d, *, base=0, stream=None):
    """y[s] = scale w[ids[s] - base]; ids below base are padding (zero rows).
    ids: int64. Gathers rows of any n_v x n_d array by an index list."""
    _sizes(n_s, n_v, n_d)
    code, T, _, d = _dtype(y, "y")
    _run(lib().stade_embed, code, _arr(d, w, T, n_v * n_d, "w"),
         _arr(d, ids, torch.int64, n_s, "ids"), _arr(d, y, T, n_s * n_d, "y"), float(scale), base,
         n_s, n_v, n_d, stream=stream)


def embed_b_cuda(wb, ids, yb, scale, n_s, n_v, n_d, *, base=0, accumulate=True, consume=True,
                 stream=None, workspace=None):
    """wb[v] += scale * sum of yb[s] over the positions s that hold id v, in
    increasing s (bit-identical from call to call)."""
    _sizes(n_s, n_v, n_d)
    code, T, P, d = _dtype(yb, "yb")
    _run(lib().stade_embed_b, code, _arr(d, wb, P, n_v * n_d, "wb"),
         _arr(d, ids, torch.int64, n_s, "ids"), _arr(d, yb, T, n_s * n_d, "yb"), float(scale),
         base, n_s, n_v, n_d, stream=stream, workspace=workspace,
         flags=_flags(accumulate, consume))


def embed_b_workspace(n_s, n_v, n_d) -> int:
    return lib().stade_embed_b_workspace(n_s, n_v, n_d)


# ---------------------------------------------------------------------------
def layer_norm_cuda(x, w, b, y, m_stack, r_stack, eps, n_s, n_d, *, stream=None):
    """y = (x - mean) rstd w + b over rows of n_d; w and b may be None. The
    tape m_stack, r_stack (n_s each) receives mean and rstd."""
    _sizes(n_s, n_d)
    code, T, P, d = _dtype(x, "x")
    _run(lib().stade_layer_norm, code, _arr(d, x, T, n_s * n_d, "x"), _opt(d, w, P, n_d, "w"),
         _opt(d, b, P, n_d, "b"), _arr(d, y, T, n_s * n_d, "y"),
         _arr(d, m_stack, P, n_s, "m_stack"), _arr(d, r_stack, P, n_s, "r_stack"), float(eps), n_s,
         n_d, stream=stream)


def layer_norm_b_cuda(x, xb, w, wb, bb, yb, m_stack, r_stack, n_s, n_d, *, accumulate=True,
                      consume=True, stream=None, workspace=None):
    """Reverse sweep of layer_norm from x and the tape; xb, wb and bb may be
    None (not wanted)."""
    _sizes(n_s, n_d)
    code, T, P, d = _dtype(x, "x")
    _run(lib().stade_layer_norm_b, code, _arr(d, x, T, n_s * n_d, "x"),
         _opt(d, xb, T, n_s * n_d, "xb"), _opt(d, w, P, n_d, "w"), _opt(d, wb, P, n_d, "wb"),
         _opt(d, bb, P, n_d, "bb"), _arr(d, yb, T, n_s * n_d, "yb"),
         _arr(d, m_stack, P, n_s, "m_stack"), _arr(d, r_stack, P, n_s, "r_stack"), n_s, n_d,
         stream=stream, workspace=workspace, flags=_flags(accumulate, consume))


def layer_norm_b_workspace(dtype, n_s, n_d) -> int:
    return lib().stade_layer_norm_b_workspace(_DTYPES[dtype], n_s, n_d)


# ---------------------------------------------------------------------------
def initstacks_tape8_cuda(n_s, n_d, device=None):
    """The 8-bit tape of an n_s x n_d array: (q_stack, e_stack), 33/32 bytes
    per value and a few more where a row ends inside a scale group."""
    d = device or "cuda"
    q = torch.empty(max(n_s * n_d, 1), dtype=torch.int8, device=d)
    e = torch.empty(max(lib().stade_initstacks_tape8(n_s, n_d), 1), dtype=torch.uint8, device=d)
    return q, e


def _tape(d, q, e, n_s, n_d):
    return (_arr(d, q, torch.int8, n_s * n_d, "q_stack"),
            _arr(d, e, torch.uint8, lib().stade_initstacks_tape8(n_s, n_d), "e_stack"))


def tape8_push_cuda(x, q_stack, e_stack, n_s, n_d, *, stream=None):
    """Writes x to the 8-bit tape."""
    _sizes(n_s, n_d)
    code, T, _, d = _dtype(x, "x")
    _run(lib().stade_tape8_push, code, _arr(d, x, T, n_s * n_d, "x"),
         *_tape(d, q_stack, e_stack, n_s, n_d), n_s, n_d, stream=stream)


def tape8_pop_cuda(x, q_stack, e_stack, n_s, n_d, *, stream=None):
    """Restores x from the 8-bit tape (overwrites x)."""
    _sizes(n_s, n_d)
    code, T, _, d = _dtype(x, "x")
    _run(lib().stade_tape8_pop, code, _arr(d, x, T, n_s * n_d, "x"),
         *_tape(d, q_stack, e_stack, n_s, n_d), n_s, n_d, stream=stream)


def act_tape8_cuda(act, x, y, q_stack, e_stack, n_s, n_d, *, stream=None):
    """y = f(x), f one of relu, tanh, silu, gelu (erf form); x goes to the
    8-bit tape for act_tape8_b."""
    _sizes(n_s, n_d)
    code, T, _, d = _dtype(x, "x")
    _run(lib().stade_act_tape8, code, _act(act), _arr(d, x, T, n_s * n_d, "x"),
         _arr(d, y, T, n_s * n_d, "y"), *_tape(d, q_stack, e_stack, n_s, n_d), n_s, n_d,
         stream=stream)


def act_tape8_b_cuda(act, xb, yb, q_stack, e_stack, n_s, n_d, *, accumulate=True, consume=True,
                     stream=None):
    """xb += yb f'(x^), x^ the input as the 8-bit tape holds it."""
    _sizes(n_s, n_d)
    code, T, _, d = _dtype(yb, "yb")
    _run(lib().stade_act_tape8_b, code, _act(act), _arr(d, xb, T, n_s * n_d, "xb"),
         _arr(d, yb, T, n_s * n_d, "yb"), *_tape(d, q_stack, e_stack, n_s, n_d), n_s, n_d,
         stream=stream, flags=_flags(accumulate, consume))


# ---------------------------------------------------------------------------
def expert_mm_cuda(x, w, y, off, n_s, n_e, n_i, n_o, *, stream=None, workspace=None):
    """y[s] = x[s] w[e] for the rows off[e] .. off[e + 1] - 1 of expert e; w:
    n_e x n_i x n_o, off: n_e + 1 rising bounds (int64, on the device). Rows in
    no group get y = 0."""
    _sizes(n_s, n_e, n_i, n_o)
    code, T, _, d = _dtype(x, "x")
    _run(lib().stade_expert_mm, code, _arr(d, x, T, n_s * n_i, "x"),
         _arr(d, w, T, n_e * n_i * n_o, "w"), _arr(d, y, T, n_s * n_o, "y"),
         _arr(d, off, torch.int64, n_e + 1, "off"), n_s, n_e, n_i, n_o, stream=stream,
         workspace=workspace)


def expert_mm_workspace(dtype, n_s, n_e, n_i, n_o) -> int:
    return lib().stade_expert_mm_workspace(_DTYPES[dtype], n_s, n_e, n_i, n_o)


def expert_mm_b_cuda(x, xb, w, wb, yb, off, n_s, n_e, n_i, n_o, *, accumulate=True, consume=True,
                     stream=None, workspace=None):
    """xb[s] += yb[s] w[e]^T and wb[e] += x^T yb over the rows of expert e; xb
    or wb may be None (not wanted)."""
    _sizes(n_s, n_e, n_i, n_o)
    code, T, P, d = _dtype(yb, "yb")
    _run(lib().stade_expert_mm_b, code, _opt(d, x, T, n_s * n_i, "x"),
         _opt(d, xb, T, n_s * n_i, "xb"), _opt(d, w, T, n_e * n_i * n_o, "w"),
         _opt(d, wb, P, n_e * n_i * n_o, "wb"), _arr(d, yb, T, n_s * n_o, "yb"),
         _arr(d, off, torch.int64, n_e + 1, "off"), n_s, n_e, n_i, n_o, stream=stream,
         workspace=workspace, flags=_flags(accumulate, consume))


def expert_mm_b_workspace(dtype, n_s, n_e, n_i, n_o) -> int:
    return lib().stade_expert_mm_b_workspace(_DTYPES[dtype], n_s, n_e, n_i, n_o)
