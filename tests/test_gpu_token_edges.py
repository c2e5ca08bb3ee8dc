"""The token-model operators where their values and their callers leave the
ordinary range."""
import ctypes as C
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import stadeb200 as sb
import token_ref as R
from stadeb200 import _lib
from stadeb200 import token_ops as T

pytestmark = pytest.mark.gpu

NO64 = ["f32", "bf16", "f16"]
NEW = dict(accumulate=False, consume=False)


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.float64) * scale


# ---- activations -------------------------------------------------------------------
# widths of the kernels for whole eights, for pairs and for single values
WIDTHS = [32, 30, 31]


def _act_both(act, x, yb):
    """y, and xb for the seed yb, through the tape."""
    n_s, n_d = x.shape
    y, xb = torch.full_like(x, math.nan), torch.full_like(x, math.nan)
    q, e = sb.initstacks_tape8_cuda(n_s, n_d)
    sb.act_tape8_cuda(act, x, y, q, e, n_s, n_d)
    sb.act_tape8_b_cuda(act, xb, yb, q, e, n_s, n_d, **NEW)
    return y, xb


@pytest.mark.parametrize("dt", NO64)
@pytest.mark.parametrize("act", list(T.ACTIVATIONS))
@pytest.mark.parametrize("n_d", WIDTHS)
def test_act_tape8_far_out(n_d, act, dt):
    """From 60 on every activation is 0 (tanh: -1) to the left with slope 0
    and x (tanh: 1) to the right with slope 1 (tanh: 0), to the type's largest
    value: sigmoid(-60) and the tails of tanh and Phi there are below 1e-25."""
    dt = R.DTYPES[dt]
    far = [60.0, 96.0, 150.0, 1000.0, 6e4] + ([1e15, 1e30, 1e36] if dt != torch.float16 else [])
    far.append(torch.finfo(dt).max)
    x = torch.tensor([-v for v in far] + far, dtype=torch.float64).to(dt)
    n = len(far)
    x = x[:, None].expand(2 * n, n_d).contiguous().cuda()       # a group of one value each
    yb = _rand(1, 2 * n, n_d).to(dt).cuda()
    y, xb = (R.f64(t) for t in _act_both(act, x, yb))
    X, seed = R.f64(x), R.f64(yb)
    left, right, slope = (-1.0, 1.0, 0.0) if act == "tanh" else (0.0, X[n:], 1.0)
    assert np.abs(y[:n] - left).max() < 1e-20 and np.all(y[n:] == right)
    assert np.abs(xb[:n]).max() < 1e-20 and np.abs(xb[n:] - slope * seed[n:]).max() < 1e-20


@pytest.mark.parametrize("dt", NO64)
@pytest.mark.parametrize("act", list(T.ACTIVATIONS))
@pytest.mark.parametrize("n_d", WIDTHS)
def test_act_tape8_infinities(n_d, act, dt):
    """Infinities and NaN give what the formulas in 64 bits give, in every type:
    x / (1 + exp(-x)) and x (1 + erf) / 2 are NaN at -infinity. Their groups
    come back as NaN."""
    dt = R.DTYPES[dt]
    x = _rand(2, 3, n_d).to(dt)
    x[0, 3], x[1, 7], x[2, 0] = math.inf, -math.inf, math.nan
    with np.errstate(all="ignore"):
        ref = R.act(act, R.f64(x))
    y, xb = _act_both(act, x.cuda(), torch.ones(3, n_d, dtype=dt, device="cuda"))
    got = R.f64(y)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[np.isinf(ref)], ref[np.isinf(ref)])
    assert np.isfinite(got).sum() >= 3 * n_d - 3
    assert torch.isnan(xb).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("act", list(T.ACTIVATIONS))
@pytest.mark.parametrize("n_d", WIDTHS)
def test_act_tape8_tails(n_d, act, dt):
    """The tails of the 16-bit forms, where values and slopes fall off as
    exp(-x) or exp(-x^2 / 2), keep the type's relative precision: a quarter
    of a rounding beside the one of the result."""
    dt = R.DTYPES[dt]
    at = torch.linspace(2.0, 12.0 if dt == torch.bfloat16 else 5.0, 41).to(dt)
    x = torch.cat([-at, at])[:, None].expand(82, n_d).contiguous().cuda()
    yb = torch.ones_like(x)
    y, xb = _act_both(act, x, yb)
    X = R.f64(x)
    V = R.tape8_values(*R.tape8(X))
    for name, out, ref in (("y", y, _act64(act, X)), ("slope", xb, _slope64(act, V))):
        tol = 1.25 * R.UNIT[dt] * np.abs(ref) + R.TINY[dt]
        err = np.abs(R.f64(out) - ref)
        assert np.all(err <= tol), f"{name}: {(err / tol).max():.2f} x bound at x = {X.flat[(err / tol).argmax()]}"


_erfc = np.vectorize(math.erfc)


def _act64(act, x):
    return 0.5 * x * _erfc(-x / math.sqrt(2)) if act == "gelu" else R.act(act, x)


def _slope64(act, x):
    if act == "gelu":
        return 0.5 * _erfc(-x / math.sqrt(2)) + x * np.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    return R.act_slope(act, x)


# ---- expert_mm ---------------------------------------------------------------------
def _same(out, ref, scale, k, name):
    """Infinities and NaN in the same places, the rest within the bound."""
    o = R.f64(out).reshape(ref.shape)
    inf = np.isinf(ref)
    assert np.array_equal(np.isnan(o), np.isnan(ref)), f"{name}: NaN in other places"
    assert np.array_equal(np.isinf(o), inf) and np.array_equal(o[inf], ref[inf]), name
    ok = np.isfinite(ref)
    tol = (R.UNIT[out.dtype] * 1.001 * np.abs(ref) + R.TINY[out.dtype] + k * R.UNIT[R.par(out.dtype)] * scale)
    assert np.all(np.abs(o - ref)[ok] <= tol[ok]), name


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("off", [[0, 3, 3, 9], [0, 130, 131, 400]])
def test_expert_mm_infinities(off, whole, dt):
    """An infinity in x, w or yb reaches every result its row or column has a
    part in, as in a plain product; whatever the number of rows. whole: values
    of few bits, whose lower planes are 0."""
    dt = R.DTYPES[dt]
    n_s, n_e, n_i, n_o = off[-1], 3, 72, 136
    x, w, yb = _rand(1, n_s, n_i), _rand(2, n_e, n_i, n_o), _rand(3, n_s, n_o)
    if whole:
        x, w, yb = (torch.sign(t) * torch.ceil(t.abs()) for t in (x, w, yb))
    x, w, yb = (t.to(dt).cuda() for t in (x, w, yb))
    x[1, 5], x[off[2] + 2, 71] = math.inf, -math.inf
    w[2, 70, 9] = math.inf
    yb[2, 0], yb[off[2] + 1, 130] = -math.inf, math.inf
    o = torch.tensor(off).cuda()
    X, W, Y = R.f64(x), R.f64(w), R.f64(yb)
    with np.errstate(all="ignore"):
        ref, mag = R.expert_mm(X, W, off)
        xr, wr, mx, mw = R.expert_mm_b(X, W, Y, off)
    y, xb = torch.zeros(n_s, n_o, dtype=dt, device="cuda"), torch.zeros(n_s, n_i, dtype=dt, device="cuda")
    wb = torch.zeros(n_e, n_i, n_o, device="cuda")
    sb.expert_mm_cuda(x, w, y, o, n_s, n_e, n_i, n_o)
    sb.expert_mm_b_cuda(x, xb, w, wb, yb, o, n_s, n_e, n_i, n_o, **NEW)
    _same(y, ref, mag, 2 * n_i + 8, "y")
    _same(xb, xr, mx, 2 * n_o + 8, "xb")
    _same(wb, wr, mw, 2 * n_s + 8, "wb")


@pytest.mark.parametrize("n_s,n_e,n_i,n_o", [(512, 64, 64, 136), (1024, 2000, 72, 40), (4096, 512, 64, 72), (3001, 400, 40, 33)])
def test_expert_mm_f32_one_expert_takes_all(n_s, n_e, n_i, n_o):
    """Few rows a group on average, all of them in one group. One chain of n
    Float32 additions loses about sqrt(n / 6) u in the 2-norm, 1.6e-6 for
    4,096; sums in pieces stay below 5e-7, the tensor cores' at 2.3e-7."""
    off = [0] * 6 + [n_s] * (n_e - 5)
    x, w, yb = (t.float().cuda() for t in (_rand(1, n_s, n_i), _rand(2, n_e, n_i, n_o), _rand(3, n_s, n_o)))
    o = torch.tensor(off).cuda()
    y, xb = torch.empty(n_s, n_o, device="cuda"), torch.empty(n_s, n_i, device="cuda")
    wb = torch.full((n_e, n_i, n_o), math.nan, device="cuda")
    sb.expert_mm_cuda(x, w, y, o, n_s, n_e, n_i, n_o)
    sb.expert_mm_b_cuda(x, xb, w, wb, yb, o, n_s, n_e, n_i, n_o, **NEW)
    X, W, Y = x.double(), w[5].double(), yb.double()
    for name, out, ref in (("y", y, X @ W), ("xb", xb, Y @ W.T), ("wb", wb[5], X.T @ Y)):
        err = ((out.double() - ref).norm() / ref.norm()).item()
        assert err < 5e-7, f"{name}: {err:.2e}"
    wb[5] = 0
    assert not wb.any()


# ---- ids -----------------------------------------------------------------------
def test_embed_smallest_id_is_padding():
    """Ids down to the type's smallest value are padding, not past the table."""
    L = _lib.lib()
    L.stade_device_error()
    w = _rand(1, 10, 8).float().cuda()
    ids = torch.tensor([1, -2 ** 63, 10, -2 ** 63 + 5, 0]).cuda()
    y = torch.full((5, 8), math.nan, device="cuda")
    sb.embed_cuda(w, ids, y, 1.0, 5, 10, 8, base=1)
    wb = torch.zeros(10, 8, device="cuda")
    sb.embed_b_cuda(wb, ids, torch.ones(5, 8, device="cuda"), 1.0, 5, 10, 8, base=1)
    assert L.stade_device_error() == 0
    assert torch.equal(y[0], w[0]) and torch.equal(y[2], w[9]) and not y[1].any() and not y[3:].any()
    assert (wb[0] == 1).all() and (wb[9] == 1).all() and not wb[1:9].any()


# ---- threads, streams, workspaces ----------------------------------------------------
@pytest.mark.parametrize("op", ["fwd", "bwd", "sort", "cluster"])
def test_host_threads(op):
    """Calls that share a kernel but want different amounts of shared memory, from
    four threads on streams of their own: none takes another's limit for its
    launch. Two sizes of each kernel, 98 KB and 26 KB in reverse for instance."""
    L, failed = _lib.lib(), []

    def calls(k, s):
        """(C function, arguments, a check of the results)"""
        o = _lib.make_opts(s.cuda_stream, None, 0, _lib.STADE_ADJ_STORE | _lib.STADE_SEED_KEEP)
        if op in ("sort", "cluster"):
            n_s, n_v, n_d = (100, 400 if k else 12, 4) if op == "sort" else (65536 if k else 5000, 500 if k else 12, 1)
            ids = torch.arange(n_s, device="cuda") % n_v
            yb, wb = torch.ones(n_s, n_d, device="cuda"), torch.zeros(n_v, n_d, device="cuda")
            ws = torch.empty(T.embed_b_workspace(n_s, n_v, n_d), dtype=torch.uint8, device="cuda")
            o.workspace, o.workspace_bytes = ws.data_ptr(), ws.numel()
            args = (_lib.STADE_F32, wb.data_ptr(), ids.data_ptr(), yb.data_ptr(), 1.0, 0, n_s, n_v, n_d)
            want = torch.bincount(ids, minlength=n_v).float()[:, None].expand(n_v, n_d)
            return L.stade_embed_b, args, o, lambda: torch.equal(wb, want), (ids, yb, ws)
        n_s, n_d = 64, 2048 if k else (1100 if op == "fwd" else 400)
        x = _rand(k, n_s, n_d).float().cuda()
        y, m, r = torch.empty_like(x), torch.empty(n_s, device="cuda"), torch.empty(n_s, device="cuda")
        ref = torch.from_numpy(R.layer_norm(R.f64(x), None, None, 1e-5)[0])
        if op == "fwd":
            args = (_lib.STADE_F32, x.data_ptr(), None, None, y.data_ptr(), m.data_ptr(), r.data_ptr(), 1e-5, n_s, n_d)
            return L.stade_layer_norm, args, o, lambda: (y.cpu() - ref).abs().max() < 1e-5, (x, m, r)
        T.layer_norm_cuda(x, None, None, y, m, r, 1e-5, n_s, n_d)
        torch.cuda.synchronize()
        bb = torch.zeros(n_d, device="cuda")
        ws = torch.empty(T.layer_norm_b_workspace(torch.float32, n_s, n_d), dtype=torch.uint8, device="cuda")
        o.workspace, o.workspace_bytes = ws.data_ptr(), ws.numel()
        args = (_lib.STADE_F32, x.data_ptr(), None, None, None, bb.data_ptr(), y.data_ptr(), m.data_ptr(), r.data_ptr(), n_s, n_d)
        return L.stade_layer_norm_b, args, o, lambda: (bb.cpu() - ref.sum(0)).abs().max() < 1e-4, (x, y, m, r, ws)

    def work(k):
        torch.cuda.set_device(0)
        s = torch.cuda.Stream()
        fn, args, o, good, _keep = calls(k, s)
        torch.cuda.synchronize()
        ready.wait()
        codes = {fn(*args, C.byref(o)) for _ in range(4000 if op != "cluster" else 1000)}
        s.synchronize()
        if codes != {_lib.STADE_OK} or not good():
            failed.append((k, codes, L.stade_last_error()))

    ready = threading.Barrier(4)
    threads = [threading.Thread(target=work, args=(k % 2,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_device_error_waits_for_other_streams():
    """The error word of a call that is still queued on another stream."""
    L = _lib.lib()
    L.stade_device_error()
    w, ids, y = torch.ones(4, 8, device="cuda"), torch.tensor([9]).cuda(), torch.empty(1, 8, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)
        sb.embed_cuda(w, ids, y, 1.0, 1, 4, 8)
    assert L.stade_device_error() != 0
    assert L.stade_device_error() == 0


def test_workspace_refusals():
    """Host memory, gaps between elements and an empty tensor are no workspace."""
    n_s, n_v, n_d = 64, 10, 8
    ids, yb, wb = torch.arange(n_s).cuda() % n_v, torch.ones(n_s, n_d, device="cuda"), torch.zeros(n_v, n_d, device="cuda")
    need = T.embed_b_workspace(n_s, n_v, n_d)
    for bad in (torch.empty(need, dtype=torch.uint8), torch.empty(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="workspace"):
            T.embed_b_cuda(wb, ids, yb, 1.0, n_s, n_v, n_d, workspace=bad)
    with pytest.raises(sb.StadeError, match="workspace"):
        T.embed_b_cuda(wb, ids, yb, 1.0, n_s, n_v, n_d, workspace=torch.empty(0, device="cuda"))
    assert not wb.any() and (yb == 1).all()


_GROWN = r"""
import sys
sys.path[:0] = [{pkg!r}]
import torch
import stadeb200 as sb
from stadeb200 import _lib
cached = _lib.lib().stade_workspace_cached_bytes
n_s, n_v, n_d = 3000, 500, 64
ids = torch.arange(n_s).cuda() * 7 % n_v
yb = torch.randn(n_s, n_d, generator=torch.Generator().manual_seed(1)).cuda()
wb, want = torch.empty(n_v, n_d, device="cuda"), torch.empty(n_v, n_d, device="cuda")
new = dict(accumulate=False, consume=False)
sb.embed_b_cuda(want, ids, yb, 1.0, n_s, n_v, n_d, **new)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    sb.embed_b_cuda(wb, ids, yb, 1.0, n_s, n_v, n_d, **new)
before = cached()
big = 200000
sb.embed_b_cuda(torch.empty(n_v, 8, device="cuda"), torch.arange(big).cuda() % n_v, torch.ones(big, 8, device="cuda"),
                1.0, big, n_v, 8, **new)
assert cached() > before, "the second call has to want more"
# what has been freed is handed out again, and filled
fill = [torch.full((before // 4,), 7, dtype=torch.int32, device="cuda") for _ in range(8)]
g.replay()
torch.cuda.synchronize()
assert torch.equal(wb, want)
assert all((t == 7).all() for t in fill)
sb.embed_b_cuda(wb, ids, yb, 1.0, n_s, n_v, n_d, **new)
assert torch.equal(wb, want)
print("ok")
"""


def test_graph_outlives_the_growth_of_the_cached_workspace():
    """A graph whose call used the library's workspace is replayed after a larger
    call has made the cache grow. In a process of its own, whose cache starts
    empty."""
    pkg = os.path.dirname(os.path.dirname(os.path.abspath(sb.__file__)))
    r = subprocess.run([sys.executable, "-c", _GROWN.format(pkg=pkg)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-2000:]
