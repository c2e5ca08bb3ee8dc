"""The token-model operators on the GPU against plain implementations in 64
bits (token_ref.py), at the sizes, alignments and values where they can go
wrong: single rows, odd widths, unaligned arrays, empty and one-sided groups,
padding ids, long runs of one id, infinities and NaN, streams, workspaces."""
import math

import numpy as np
import pytest
import torch

import stadeb200 as sb
import token_ref as R
from stadeb200 import _lib
from stadeb200 import token_ops as T

pytestmark = pytest.mark.gpu

ALL = ["f32", "f64", "bf16", "f16"]
NO64 = ["f32", "bf16", "f16"]


def _rand(seed, *shape, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.float64) * scale + shift


def _dev(t, dt, offset=0):
    """A contiguous CUDA copy, `offset` elements past an aligned address."""
    buf = torch.zeros(t.numel() + offset, dtype=dt, device="cuda")
    v = buf[offset:offset + t.numel()].view(t.shape)
    v.copy_(t.to(dt))
    return v


# ---- layer_norm --------------------------------------------------------------------
NORM_SIZES = [(1, 1, 0), (1, 512, 0), (3, 7, 0), (5, 33, 1), (37, 96, 0), (2, 1000, 0), (9, 1024, 1),
              (4, 784, 0), (3, 2500, 0), (2, 4096, 0), (3, 5000, 3), (2, 8191, 0), (1, 16384, 0),
              (2, 20000, 0), (300, 64, 0), (2, 40001, 0),
              # enough rows for several a turn and turns beyond a block's first, row
              # counts that end inside one; widths with every remainder class
              (1300, 1024, 0), (2501, 800, 0), (1500, 1023, 0), (2400, 771, 0), (700, 4096, 0),
              (650, 5000, 0), (630, 5001, 0), (320, 8192, 0), (310, 8187, 0), (160, 9000, 0),
              (40, 12282, 0)]


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n_s,n_d,off", NORM_SIZES)
def test_layer_norm(n_s, n_d, off, dt):
    dt = R.DTYPES[dt]
    P = R.par(dt)
    x = _dev(_rand(1, n_s, n_d, scale=1.5, shift=0.7), dt, off)
    w, b = _dev(_rand(2, n_d, shift=1.0), P, off), _dev(_rand(3, n_d), P)
    y = _dev(torch.zeros(n_s, n_d), dt, off)
    m, r = torch.empty(n_s, dtype=P, device="cuda"), torch.empty(n_s, dtype=P, device="cuda")
    sb.layer_norm_cuda(x, w, b, y, m, r, 1e-5, n_s, n_d)
    X = R.f64(x)
    ref, mean, rstd, mag = R.layer_norm(X, R.f64(w), R.f64(b), 1e-5)
    R.assert_close(y, ref, mag, 2 * n_d + 16, "y")
    R.assert_close(m, mean, np.abs(X).mean(1), n_d + 4, "mean")
    R.assert_close(r, rstd, rstd * (1 + np.abs(X).mean(1) * rstd), 2 * n_d + 16, "rstd")


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n_s,n_d,off", NORM_SIZES)
def test_layer_norm_b(n_s, n_d, off, dt):
    dt = R.DTYPES[dt]
    P = R.par(dt)
    x = _dev(_rand(1, n_s, n_d, scale=1.5, shift=0.7), dt, off)
    w, yb = _dev(_rand(2, n_d, shift=1.0), P, off), _dev(_rand(4, n_s, n_d), dt, off)
    X, W, YB = R.f64(x), R.f64(w), R.f64(yb)
    _, mean, rstd, _ = R.layer_norm(X, W, None, 1e-5)
    m, r = torch.tensor(mean).to(P).cuda(), torch.tensor(rstd).to(P).cuda()
    (xb, wb, bb), (mx, mw, mb) = R.layer_norm_b(X, W, YB, R.f64(m), R.f64(r))
    # stored, the seed kept
    o = [torch.full((n_s, n_d), math.nan, dtype=dt, device="cuda"),
         torch.full((n_d,), math.nan, dtype=P, device="cuda"),
         torch.full((n_d,), math.nan, dtype=P, device="cuda")]
    sb.layer_norm_b_cuda(x, o[0], w, o[1], o[2], yb, m, r, n_s, n_d, accumulate=False, consume=False)
    assert np.array_equal(R.f64(yb), YB)
    R.assert_close(o[0], xb, mx, 3 * n_d + 32, "xb")
    R.assert_close(o[1], wb, mw, n_s + 8, "wb")
    R.assert_close(o[2], bb, mb, n_s + 8, "bb")
    # added, the seed consumed
    first = _rand(5, n_s, n_d), _rand(6, n_d), _rand(7, n_d)
    a = [_dev(first[0], dt, off), _dev(first[1], P), _dev(first[2], P)]
    F = [R.f64(t) for t in a]
    sb.layer_norm_b_cuda(x, a[0], w, a[1], a[2], yb, m, r, n_s, n_d)
    assert not yb.any()
    R.assert_close(a[0], F[0] + xb, mx + np.abs(F[0]), 3 * n_d + 32, "xb +=")
    R.assert_close(a[1], F[1] + wb, mw + np.abs(F[1]), n_s + 8, "wb +=")
    R.assert_close(a[2], F[2] + bb, mb + np.abs(F[2]), n_s + 8, "bb +=")


@pytest.mark.parametrize("n_s,n_d", [(40, 96), (3, 9000), (700, 40)])
@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (0, 0, 0)])
def test_layer_norm_b_parts(want, n_s, n_d):
    """Any of xb, wb, bb may be left out; w None counts as ones; the seed is
    consumed whatever is asked for."""
    x, yb = _dev(_rand(1, n_s, n_d), torch.float32), _dev(_rand(2, n_s, n_d), torch.float32)
    X, YB = R.f64(x), R.f64(yb)
    y = torch.empty_like(x)
    m, r = torch.empty(n_s, device="cuda"), torch.empty(n_s, device="cuda")
    sb.layer_norm_cuda(x, None, None, y, m, r, 1e-5, n_s, n_d)
    R.assert_close(y, *[R.layer_norm(X, None, None, 1e-5)[i] for i in (0, 3)], 2 * n_d + 16)
    ref, mag = R.layer_norm_b(X, None, YB, R.f64(m), R.f64(r))
    out = [torch.zeros(s, device="cuda") if k else None
           for k, s in zip(want, ((n_s, n_d), (n_d,), (n_d,)))]
    sb.layer_norm_b_cuda(x, out[0], None, out[1], out[2], yb, m, r, n_s, n_d)
    for o, v, g, k in zip(out, ref, mag, (3 * n_d + 32, n_s + 8, n_s + 8)):
        if o is not None:
            R.assert_close(o, v, g, k)
    assert not yb.any()


def test_layer_norm_constant_and_nonfinite_rows():
    """A constant row has variance 0: y = b and rstd = 1 / sqrt(eps). A row
    with a NaN or an infinity is NaN throughout and leaves the others alone."""
    n_d = 300
    x = _rand(1, 4, n_d).float()
    x[1] = 3.0
    x[2, 5] = math.inf
    x[3, 299] = math.nan
    x = x.cuda()
    b = _rand(2, n_d).float().cuda()
    y, m, r = torch.empty_like(x), torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    sb.layer_norm_cuda(x, None, b, y, m, r, 1e-5, 4, n_d)
    assert torch.equal(y[1], b)
    assert abs(r[1].item() * math.sqrt(1e-5) - 1) < 1e-6
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all() and torch.isfinite(y[0]).all()


def test_layer_norm_mean_far_from_zero():
    """The centred second pass keeps the variance where a one-pass sum of
    squares would lose it: mean 1000, spread 0.01."""
    n_d = 768
    x = (_rand(1, 3, n_d, scale=0.01) + 1000.0).float()
    y, m, r = torch.empty(3, n_d, device="cuda"), torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    sb.layer_norm_cuda(x.cuda(), None, None, y, m, r, 0.0, 3, n_d)
    ref, _, rstd, _ = R.layer_norm(x.double().numpy(), None, None, 0.0)
    # the mean's rounding, 1000 * 2^-24 of a spread of 0.01, is all that is lost
    assert np.abs(R.f64(y) - ref).max() < 4 * 1000 * 2.0 ** -24 / 0.01
    assert np.abs(R.f64(r) / rstd - 1).max() < 1e-4


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n_s,n_d,off", [(1300, 1, 0), (300, 64, 0), (37, 96, 0), (40, 1000, 0), (9, 1024, 1),
                                         (700, 4096, 0), (40, 5001, 0), (3, 20000, 0)])
def test_layer_norm_b_rows_at_their_mean(n_s, n_d, off, dt):
    """Where every x is its row's mean, h is 0 whatever rstd is: wb is exactly
    0 and xb is rstd (g - mean(g))."""
    dt = R.DTYPES[dt]
    P = R.par(dt)
    at = (torch.arange(n_s, dtype=torch.float64) * 37 % 255 - 127)
    x = _dev(at[:, None].expand(n_s, n_d), dt, off)
    yb = _dev(_rand(1, n_s, n_d), dt, off)
    m, r = at.to(P).cuda(), torch.full((n_s,), 1e-5 ** -0.5, dtype=P, device="cuda")
    xb = torch.full((n_s, n_d), math.nan, dtype=dt, device="cuda")
    wb, bb = torch.full((n_d,), math.nan, dtype=P, device="cuda"), torch.zeros(n_d, dtype=P, device="cuda")
    (want, _, _), (mag, _, _) = R.layer_norm_b(R.f64(x), None, R.f64(yb), R.f64(m), R.f64(r))
    sb.layer_norm_b_cuda(x, xb, None, wb, bb, yb, m, r, n_s, n_d, accumulate=False, consume=False)
    assert torch.equal(wb, torch.zeros_like(wb))
    R.assert_close(xb, want, mag, 3 * n_d + 32, "xb")


def test_layer_norm_b_against_differences():
    n_s, n_d, h = 5, 41, 1e-6
    x, w, b, yb = _rand(1, n_s, n_d), _rand(2, n_d), _rand(3, n_d), _rand(4, n_s, n_d)
    dx, dw, db = _rand(5, n_s, n_d), _rand(6, n_d), _rand(7, n_d)

    def value(t):
        a = [v.cuda() for v in (x + t * dx, w + t * dw, b + t * db)]
        y = torch.empty_like(a[0])
        m, r = torch.empty(n_s, dtype=torch.float64, device="cuda"), torch.empty(n_s, dtype=torch.float64, device="cuda")
        sb.layer_norm_cuda(*a, y, m, r, 1e-5, n_s, n_d)
        return (y.cpu() * yb).sum().item(), a, m, r

    fd = (value(h)[0] - value(-h)[0]) / (2 * h)
    _, a, m, r = value(0.0)
    xb, wb, bb = torch.zeros_like(a[0]), torch.zeros_like(a[1]), torch.zeros_like(a[2])
    sb.layer_norm_b_cuda(a[0], xb, a[1], wb, bb, yb.cuda(), m, r, n_s, n_d)
    dot = (xb.cpu() * dx).sum() + (wb.cpu() * dw).sum() + (bb.cpu() * db).sum()
    # central difference: h^2 truncation and 2^-53 / h rounding of a value of order 100
    assert abs(dot.item() - fd) < 1e-6 * max(1.0, abs(fd))


# ---- embed ------------------------------------------------------------------------
EMBED_SIZES = [(1, 1, 1, 0), (1, 1000, 784, 0), (5, 3, 32, 0), (96, 1000, 784, 0), (257, 50, 33, 1),
               (3000, 7, 64, 0), (2048, 512, 40, 0), (2049, 511, 100, 3), (5000, 100000, 24, 0),
               (9000, 3000, 17, 0), (300, 20, 4100, 0), (4096, 70000, 8, 0), (4097, 300, 24, 0),
               (140000, 600, 3, 0), (20000, 20, 260, 0),
               (65536, 70000, 5, 0), (65537, 3000, 4, 1), (8193, 2 ** 18, 2, 0)]


def _ids(seed, n_s, n_v, base):
    rng = np.random.RandomState(seed)
    ids = (n_v ** rng.rand(n_s)).astype(np.int64) % n_v + base    # small ids far more often
    ids[3::11] = base - 1
    ids[7::29] = -5
    return ids


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("base", [0, 1])
@pytest.mark.parametrize("n_s,n_v,n_d,off", EMBED_SIZES)
def test_embed(n_s, n_v, n_d, off, base, dt):
    dt = R.DTYPES[dt]
    w = _dev(_rand(1, n_v, n_d), dt, off)
    ids = _ids(2, n_s, n_v, base)
    y = _dev(torch.full((n_s, n_d), math.nan), dt, off)
    sb.embed_cuda(w, torch.from_numpy(ids).cuda(), y, 1.7, n_s, n_v, n_d, base=base)
    ref = R.embed(R.f64(w), ids, 1.7, base)
    R.assert_close(y, ref, np.abs(ref), 2)
    assert _lib.lib().stade_device_error() == 0


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n_s,n_v,n_d,off", EMBED_SIZES)
def test_embed_b(n_s, n_v, n_d, off, dt):
    dt = R.DTYPES[dt]
    P = R.par(dt)
    yb = _dev(_rand(3, n_s, n_d), dt, off)
    ids = _ids(4, n_s, n_v, 0)
    dev = torch.from_numpy(ids).cuda()
    ref, mag, cnt = R.embed_b(R.f64(yb), ids, 1.7, n_v)
    wb = _dev(torch.full((n_v, n_d), math.nan), P, off)
    sb.embed_b_cuda(wb, dev, yb, 1.7, n_s, n_v, n_d, accumulate=False, consume=False)
    R.assert_close(wb, ref, mag, cnt.max() + 4, "wb")
    again = torch.full_like(wb, math.nan)
    sb.embed_b_cuda(again, dev, yb, 1.7, n_s, n_v, n_d, accumulate=False, consume=False)
    assert torch.equal(wb, again)
    old = _dev(_rand(5, n_v, n_d), P, off)
    O = R.f64(old)
    sb.embed_b_cuda(old, dev, yb, 1.7, n_s, n_v, n_d)
    R.assert_close(old, O + ref, mag + np.abs(O), cnt.max() + 4, "wb +=")
    assert not yb.any()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n_d", [8, 129])
def test_embed_b_one_id_takes_all(n_d, dt):
    """70,001 positions of one id, one of another, in a table of 40,000."""
    dt = R.DTYPES[dt]
    n_s, n_v = 70001, 40000
    yb = _dev(_rand(3, n_s, n_d), dt)
    ids = torch.full((n_s,), 31234, dtype=torch.int64)
    ids[777] = 39999
    wb = torch.full((n_v, n_d), math.nan, device="cuda")
    sb.embed_b_cuda(wb, ids.cuda(), yb, 0.5, n_s, n_v, n_d, accumulate=False, consume=False)
    Y = R.f64(yb)
    ref, mag = np.zeros((n_v, n_d)), np.zeros((n_v, n_d))
    ref[39999], mag[39999] = 0.5 * Y[777], 0.5 * np.abs(Y[777])
    ref[31234] = 0.5 * (Y.sum(0) - Y[777])
    mag[31234] = 0.5 * np.abs(Y).sum(0)
    R.assert_close(wb, ref, mag, n_s)


def test_embed_ids_out_of_range_set_the_error_word():
    L = _lib.lib()
    L.stade_device_error()
    w = _rand(1, 10, 8).float().cuda()
    ids = torch.tensor([3, 10, 2 ** 40, -2 ** 40, 9]).cuda()
    y = torch.full((5, 8), math.nan, device="cuda")
    sb.embed_cuda(w, ids, y, 1.0, 5, 10, 8)
    assert L.stade_device_error() != 0 and L.stade_device_error() == 0
    assert not y[1:4].any() and torch.equal(y[0], w[3]) and torch.equal(y[4], w[9])
    wb = torch.zeros(10, 8, device="cuda")
    sb.embed_b_cuda(wb, ids, torch.ones(5, 8, device="cuda"), 1.0, 5, 10, 8)
    assert L.stade_device_error() != 0
    want = torch.zeros(10, 8)
    want[3] = want[9] = 1
    assert torch.equal(wb.cpu(), want)


def test_embed_table_past_32_bits():
    """A table of more than 2^32 elements: rows at its end."""
    n_v, n_d = 70000, 65536
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    w = torch.zeros(n_v, n_d, dtype=torch.bfloat16, device="cuda")
    w[69999] = 2.0
    w[65537, 5] = 3.0
    ids = torch.tensor([69999, 65537, 0]).cuda()
    y = torch.empty(3, n_d, dtype=torch.bfloat16, device="cuda")
    sb.embed_cuda(w, ids, y, 1.0, 3, n_v, n_d)
    assert (y[0] == 2).all() and y[1, 5] == 3 and y[1].sum() == 3 and not y[2].any()


# ---- 8-bit tape ---------------------------------------------------------------------
TAPE_SIZES = [(1, 1, 0), (1, 32, 0), (3, 31, 0), (2, 33, 1), (5, 1990, 0), (4, 4096, 0), (7, 100, 2),
              (130, 64, 0), (2, 8200, 0), (9, 40, 0), (3, 4097, 0), (6, 48, 4), (1000, 5, 0)]


def _spread(seed, n_s, n_d, dt):
    """Values over many binades, whole groups of zeros, exact halves of a step."""
    x = _rand(seed, n_s, n_d)
    g = torch.Generator().manual_seed(seed + 1)
    lim = 4 if dt == torch.float16 else 30
    x = x * torch.exp2(torch.randint(-lim, lim, (n_s, n_d), generator=g).double())
    x.view(-1)[::7] = 0.0
    if n_d >= 64:
        x[0, 32:64] = 0.0
        x[-1, :32] = torch.arange(32, dtype=torch.float64) + 0.5
        x[-1, 0] = 127.75
    return x.to(dt)


@pytest.mark.parametrize("dt", NO64)
@pytest.mark.parametrize("n_s,n_d,off", TAPE_SIZES)
def test_tape8_push_pop(n_s, n_d, off, dt):
    dt = R.DTYPES[dt]
    x = _dev(_spread(1, n_s, n_d, dt), dt, off)
    q, e = sb.initstacks_tape8_cuda(n_s, n_d)
    sb.tape8_push_cuda(x, q, e, n_s, n_d)
    Q, E = R.tape8(R.f64(x))
    assert np.array_equal(e.cpu().numpy().reshape(E.shape), E)
    assert np.array_equal(q.cpu().numpy().reshape(Q.shape), Q)
    back = _dev(torch.full((n_s, n_d), math.nan), dt, off)
    sb.tape8_pop_cuda(back, q, e, n_s, n_d)
    V = R.tape8_values(Q, E)
    assert np.array_equal(R.f64(back), V)
    step = np.repeat(np.exp2(E.astype(float) - 127), 32, axis=1)[:, :n_d]
    assert np.all(np.abs(V - R.f64(x)) < step)


@pytest.mark.parametrize("dt", NO64)
def test_tape8_limits(dt):
    """The largest and the smallest values of the type, signed zeros,
    infinities and NaN."""
    dt = R.DTYPES[dt]
    big, small = torch.finfo(dt).max, torch.finfo(dt).smallest_normal
    x = torch.zeros(6, 64, dtype=dt)
    x[0, :] = torch.linspace(-1, 1, 64).to(dt) * big
    x[1, :] = torch.linspace(-4, 4, 64).to(dt) * small
    x[2, 1] = torch.tensor(small, dtype=dt) / 4
    x[3, 3], x[3, 40] = math.inf, 1.0
    x[4, 63], x[4, 0] = math.nan, 2.0
    x[5, 9] = -0.0
    q, e = sb.initstacks_tape8_cuda(6, 64)
    sb.tape8_push_cuda(x.cuda(), q, e, 6, 64)
    Q, E = R.tape8(R.f64(x))
    assert np.array_equal(e.cpu().numpy().reshape(E.shape), E)
    assert np.array_equal(q.cpu().numpy().reshape(Q.shape), Q)
    back = torch.empty(6, 64, dtype=dt, device="cuda")
    sb.tape8_pop_cuda(back, q, e, 6, 64)
    assert np.array_equal(R.f64(back), R.tape8_values(Q, E), equal_nan=True)


@pytest.mark.parametrize("dt", NO64)
@pytest.mark.parametrize("act", list(T.ACTIVATIONS))
@pytest.mark.parametrize("n_s,n_d,off", [(1, 1, 0), (3, 33, 1), (4, 1990, 0), (5, 256, 0), (2, 8192, 0)])
def test_act_tape8(n_s, n_d, off, act, dt):
    dt = R.DTYPES[dt]
    x = _dev(_rand(1, n_s, n_d, scale=2.5), dt, off)
    if n_d >= 256:
        x[0, 0], x[0, 1], x[0, 2] = 0.0, 30.0, -30.0
    y = _dev(torch.full((n_s, n_d), math.nan), dt, off)
    q, e = sb.initstacks_tape8_cuda(n_s, n_d)
    sb.act_tape8_cuda(act, x, y, q, e, n_s, n_d)
    X = R.f64(x)
    R.assert_close(y, R.act(act, X), 1 + np.abs(X), 64, "y")
    Q, E = R.tape8(X)
    assert np.array_equal(q.cpu().numpy().reshape(Q.shape), Q)
    V = R.tape8_values(Q, E)
    yb = _dev(_rand(2, n_s, n_d), dt, off)
    YB = R.f64(yb)
    ref = YB * R.act_slope(act, V)
    scale = np.abs(YB) * (1 + np.abs(V))
    xb = _dev(torch.full((n_s, n_d), math.nan), dt, off)
    sb.act_tape8_b_cuda(act, xb, yb, q, e, n_s, n_d, accumulate=False, consume=False)
    assert np.array_equal(R.f64(yb), YB)
    R.assert_close(xb, ref, scale, 64, "xb")
    old = _dev(_rand(3, n_s, n_d), dt, off)
    O = R.f64(old)
    sb.act_tape8_b_cuda(act, old, yb, q, e, n_s, n_d)
    R.assert_close(old, O + ref, scale + np.abs(O), 64, "xb +=")
    assert not yb.any()


@pytest.mark.parametrize("dt", NO64)
@pytest.mark.parametrize("n_d", [64, 61])
def test_act_tape8_b_in_place(n_d, dt):
    """xb and yb may be one array when adjoints are stored and the seed kept."""
    dt = R.DTYPES[dt]
    x, yb = _dev(_rand(1, 9, n_d), dt), _dev(_rand(2, 9, n_d), dt)
    q, e = sb.initstacks_tape8_cuda(9, n_d)
    sb.act_tape8_cuda("gelu", x, torch.empty_like(x), q, e, 9, n_d)
    xb = torch.empty_like(x)
    new = dict(accumulate=False, consume=False)
    sb.act_tape8_b_cuda("gelu", xb, yb, q, e, 9, n_d, **new)
    sb.act_tape8_b_cuda("gelu", yb, yb, q, e, 9, n_d, **new)
    assert torch.equal(xb, yb)


@pytest.mark.parametrize("act", list(T.ACTIVATIONS))
def test_act_tape8_slope_against_differences(act):
    """Where the tape holds x exactly (whole sixty-fourths below one), the
    reverse sweep is the derivative of the forward: central differences of the
    plain 64-bit function."""
    x = torch.arange(-64, 64).float().view(4, 32) / 64
    x[0, 31] = 1.0
    X = x.double().numpy()
    q, e = sb.initstacks_tape8_cuda(4, 32)
    y = torch.empty(4, 32, device="cuda")
    sb.act_tape8_cuda(act, x.cuda(), y, q, e, 4, 32)
    xb, yb = torch.zeros(4, 32, device="cuda"), torch.ones(4, 32, device="cuda")
    sb.act_tape8_b_cuda(act, xb, yb, q, e, 4, 32)
    h = 1e-5
    fd = (R.act(act, X + h) - R.act(act, X - h)) / (2 * h)
    assert np.abs(R.f64(xb) - fd).max() < 1e-5


def test_act_tape8_nonfinite():
    """A NaN or an infinity in x passes through y at its place and comes back
    as NaN in the whole group's gradient."""
    x = _rand(1, 2, 64).float()
    x[0, 3], x[1, 40] = math.nan, math.inf
    for act in T.ACTIVATIONS:
        y, xb = torch.empty(2, 64, device="cuda"), torch.zeros(2, 64, device="cuda")
        q, e = sb.initstacks_tape8_cuda(2, 64)
        sb.act_tape8_cuda(act, x.cuda(), y, q, e, 2, 64)
        assert torch.isnan(y).sum() == 1 and torch.isnan(y[0, 3])
        sb.act_tape8_b_cuda(act, xb, torch.ones(2, 64, device="cuda"), q, e, 2, 64)
        nan = torch.isnan(xb).cpu()
        assert nan[0, :32].all() and nan[1, 32:].all() and nan.sum() == 64


# ---- expert_mm --------------------------------------------------------------------
EXPERT_SIZES = [  # off, n_i, n_o
    ([0, 1], 1, 1), ([0, 1], 64, 64), ([0, 0, 3, 3, 8], 16, 24), ([0, 5, 5, 133], 72, 200),
    ([0, 300, 301, 700], 264, 136), ([0, 1, 2, 3, 4, 5, 6, 7, 8], 128, 512), ([0, 0, 0], 32, 32),
    ([0, 130, 260], 33, 47), ([0, 257, 1000], 784, 512), ([0, 64, 128, 640], 520, 264),
    ([0, 17, 17, 80], 200, 10), ([0, 24], 1024, 8), ([0, 2000], 64, 96), ([0, 31, 500], 40, 1030),
    # few rows a group over wide weights
    ([0, 3, 3, 9, 10], 1100, 72), ([0, 5], 1500, 33), ([0, 1, 16], 515, 2100), ([0, 8, 16], 2049, 130)]


def _expert_case(off, n_i, n_o, dt, shift=0, n_s=None):
    n_s, n_e = n_s or max(off[-1], 1), len(off) - 1
    x = _dev(_rand(1, n_s, n_i), dt, shift)
    w = _dev(_rand(2, n_e, n_i, n_o, scale=1 / math.sqrt(n_i)), dt, shift)
    yb = _dev(_rand(3, n_s, n_o, scale=0.5), dt, shift)
    return x, w, yb, torch.tensor(off).cuda(), (n_s, n_e, n_i, n_o)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("off,n_i,n_o", EXPERT_SIZES)
def test_expert_mm(off, n_i, n_o, dt):
    dt = R.DTYPES[dt]
    x, w, _, o, n = _expert_case(off, n_i, n_o, dt)
    y = torch.full((n[0], n_o), math.nan, dtype=dt, device="cuda")
    sb.expert_mm_cuda(x, w, y, o, *n)
    ref, mag = R.expert_mm(R.f64(x), R.f64(w), off)
    R.assert_close(y, ref, mag, 2 * n_i + 8)
    assert _lib.lib().stade_device_error() == 0


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("off,n_i,n_o", EXPERT_SIZES)
def test_expert_mm_b(off, n_i, n_o, dt):
    dt = R.DTYPES[dt]
    P = R.par(dt)
    x, w, yb, o, n = _expert_case(off, n_i, n_o, dt)
    YB = R.f64(yb)
    xr, wr, mx, mw = R.expert_mm_b(R.f64(x), R.f64(w), YB, off)
    xb = torch.full((n[0], n_i), math.nan, dtype=dt, device="cuda")
    wb = torch.full((n[1], n_i, n_o), math.nan, dtype=P, device="cuda")
    sb.expert_mm_b_cuda(x, xb, w, wb, yb, o, *n, accumulate=False, consume=False)
    R.assert_close(xb, xr, mx, 2 * n_o + 8, "xb")
    R.assert_close(wb, wr, mw, 2 * n[0] + 8, "wb")
    assert np.array_equal(R.f64(yb), YB)
    again = torch.full_like(wb, math.nan)
    sb.expert_mm_b_cuda(x, None, None, again, yb, o, *n, accumulate=False, consume=False)
    assert torch.equal(wb, again)
    a, b = _dev(_rand(5, n[0], n_i), dt), _dev(_rand(6, n[1], n_i, n_o), P)
    A, B = R.f64(a), R.f64(b)
    sb.expert_mm_b_cuda(x, a, w, b, yb, o, *n)
    R.assert_close(a, A + xr, mx + np.abs(A), 2 * n_o + 8, "xb +=")
    R.assert_close(b, B + wr, mw + np.abs(B), 2 * n[0] + 8, "wb +=")
    assert not yb.any()
    assert _lib.lib().stade_device_error() == 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("off", [[0, 70, 200], [0, 3, 11]])
def test_expert_mm_unaligned(off, shift, dt):
    dt = R.DTYPES[dt]
    n_i, n_o = 72, 136
    x, w, yb, o, n = _expert_case(off, n_i, n_o, dt, shift)
    y, xb = _dev(torch.zeros(n[0], n_o), dt, shift), _dev(torch.zeros(n[0], n_i), dt, shift)
    wb = _dev(torch.zeros(2, n_i, n_o), R.par(dt), shift)
    sb.expert_mm_cuda(x, w, y, o, *n)
    ref, mag = R.expert_mm(R.f64(x), R.f64(w), off)
    R.assert_close(y, ref, mag, 2 * n_i + 8)
    sb.expert_mm_b_cuda(x, xb, w, wb, yb, o, *n, consume=False)
    xr, wr, mx, mw = R.expert_mm_b(R.f64(x), R.f64(w), R.f64(yb), off)
    R.assert_close(xb, xr, mx, 2 * n_o + 8)
    R.assert_close(wb, wr, mw, 2 * n[0] + 8)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_expert_mm_groups_do_not_touch_one_another(dt):
    """NaN in one expert's rows and weights stays in that expert's results,
    also where its rows share a tile with the neighbours'."""
    dt = R.DTYPES[dt]
    off, n_i, n_o = [0, 50, 83, 200], 72, 136
    x, w, yb, o, n = _expert_case(off, n_i, n_o, dt)
    x[50:83], w[1], yb[50:83] = math.nan, math.nan, math.nan
    y, xb = torch.zeros(200, n_o, dtype=dt, device="cuda"), torch.zeros(200, n_i, dtype=dt, device="cuda")
    wb = torch.zeros(3, n_i, n_o, device="cuda")
    sb.expert_mm_cuda(x, w, y, o, *n)
    sb.expert_mm_b_cuda(x, xb, w, wb, yb, o, *n, consume=False)
    ref, mag = R.expert_mm(R.f64(x), R.f64(w), off)
    xr, wr, mx, mw = R.expert_mm_b(R.f64(x), R.f64(w), R.f64(yb), off)
    R.assert_close(y, ref, np.nan_to_num(mag), 2 * n_i + 8)
    R.assert_close(xb, xr, np.nan_to_num(mx), 2 * n_o + 8)
    R.assert_close(wb, wr, np.nan_to_num(mw), 2 * n[0] + 8)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_expert_mm_rows_of_no_group(dt):
    """Rows before the first and after the last bound: y and xb are zero there,
    wb gets nothing from them."""
    dt = R.DTYPES[dt]
    off, n_i, n_o = [7, 20, 90], 64, 72
    x, w, yb, o, n = _expert_case(off, n_i, n_o, dt, n_s=300)
    y = torch.full((300, n_o), math.nan, dtype=dt, device="cuda")
    xb = torch.full((300, n_i), math.nan, dtype=dt, device="cuda")
    wb = torch.full((2, n_i, n_o), math.nan, device="cuda")
    x[:7], x[90:], yb[:7], yb[90:] = math.nan, math.nan, math.nan, math.nan
    sb.expert_mm_cuda(x, w, y, o, *n)
    sb.expert_mm_b_cuda(x, xb, w, wb, yb, o, *n, accumulate=False, consume=False)
    assert not y[:7].any() and not y[90:].any() and not xb[:7].any() and not xb[90:].any()
    ref, mag = R.expert_mm(R.f64(x), R.f64(w), off)
    _, wr, _, mw = R.expert_mm_b(np.nan_to_num(R.f64(x)), R.f64(w), np.nan_to_num(R.f64(yb)), off)
    R.assert_close(y, ref, np.nan_to_num(mag), 2 * n_i + 8)
    R.assert_close(wb, wr, mw, 2 * 300 + 8)
    assert _lib.lib().stade_device_error() == 0


@pytest.mark.parametrize("bad,same", [([0, 40, 30, 100], [0, 40, 40, 100]),
                                      ([-5, 40, 50, 100], [0, 40, 50, 100]),
                                      ([0, 40, 50, 2 ** 40], [0, 40, 50, 100])])
def test_expert_mm_bad_bounds_are_clamped(bad, same):
    L = _lib.lib()
    L.stade_device_error()
    x, w, yb, o, n = _expert_case(same, 64, 64, torch.bfloat16)
    y = torch.empty(100, 64, dtype=torch.bfloat16, device="cuda")
    sb.expert_mm_cuda(x, w, y, torch.tensor(bad).cuda(), *n)
    assert L.stade_device_error() != 0
    ref, mag = R.expert_mm(R.f64(x), R.f64(w), same)
    R.assert_close(y, ref, mag, 2 * 64 + 8)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_expert_mm_many_experts(dt):
    """2,500 experts, most of them empty."""
    dt = R.DTYPES[dt]
    rng = np.random.RandomState(3)
    cnt = (rng.rand(2500) < 0.2) * rng.randint(1, 4, 2500)
    off = [0] + np.cumsum(cnt).tolist()
    x, w, yb, o, n = _expert_case(off, 16, 24, dt)
    y, wb = torch.empty(n[0], 24, dtype=dt, device="cuda"), torch.empty(2500, 16, 24, device="cuda")
    sb.expert_mm_cuda(x, w, y, o, *n)
    ref, mag = R.expert_mm(R.f64(x), R.f64(w), off)
    R.assert_close(y, ref, mag, 2 * 16 + 8)
    sb.expert_mm_b_cuda(x, None, w, wb, yb, o, *n, accumulate=False, consume=False)
    _, wr, _, mw = R.expert_mm_b(R.f64(x), R.f64(w), R.f64(yb), off)
    R.assert_close(wb, wr, mw, 2 * n[0] + 8)


def test_expert_mm_b_against_differences():
    off, n_i, n_o, h = [0, 4, 4, 9], 7, 5, 1e-6
    n = (9, 3, n_i, n_o)
    x, w, yb = _rand(1, 9, n_i), _rand(2, 3, n_i, n_o), _rand(3, 9, n_o)
    dx, dw = _rand(4, 9, n_i), _rand(5, 3, n_i, n_o)
    o = torch.tensor(off).cuda()

    def value(t):
        y = torch.empty(9, n_o, dtype=torch.float64, device="cuda")
        sb.expert_mm_cuda((x + t * dx).cuda(), (w + t * dw).cuda(), y, o, *n)
        return (y.cpu() * yb).sum().item()

    fd = (value(h) - value(-h)) / (2 * h)
    xb = torch.zeros(9, n_i, dtype=torch.float64, device="cuda")
    wb = torch.zeros(3, n_i, n_o, dtype=torch.float64, device="cuda")
    sb.expert_mm_b_cuda(x.cuda(), xb, w.cuda(), wb, yb.cuda(), o, *n)
    dot = ((xb.cpu() * dx).sum() + (wb.cpu() * dw).sum()).item()
    assert abs(dot - fd) < 1e-7 * max(1.0, abs(fd))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_expert_mm_at_length(dt):
    """Long sums: 3,000 rows a group, widths 1,024 and 1,536, relative 2-norm
    against 64 bits. A sum of n products of either sign loses about
    sqrt(n) u rather than the bound's n u."""
    dt = R.DTYPES[dt]
    off, n_i, n_o = [0, 2900, 6000], 1024, 1536
    x, w, yb, o, n = _expert_case(off, n_i, n_o, dt)
    y, xb = torch.empty(6000, n_o, dtype=dt, device="cuda"), torch.empty(6000, n_i, dtype=dt, device="cuda")
    wb = torch.empty(2, n_i, n_o, device="cuda")
    sb.expert_mm_cuda(x, w, y, o, *n)
    sb.expert_mm_b_cuda(x, xb, w, wb, yb, o, *n, accumulate=False, consume=False)
    X, W, Y = x.double(), w.double(), yb.double()
    for e in range(2):
        r = slice(off[e], off[e + 1])
        for out, ref in ((y[r], X[r] @ W[e]), (xb[r], Y[r] @ W[e].T), (wb[e], X[r].T @ Y[r])):
            err = ((out.double() - ref).norm() / ref.norm()).item()
            assert err < R.UNIT[out.dtype] + 64 * 2.0 ** -24


# ---- streams, workspaces, launches ------------------------------------------------------
def test_other_streams_and_own_workspaces():
    """Calls on a stream of their own, with the caller's workspace, after work
    queued there: they see that work's results and leave the cache alone."""
    n_s, n_d, n_v = 300, 136, 50
    s = torch.cuda.Stream()
    ids = torch.randint(0, n_v, (n_s,), generator=torch.Generator().manual_seed(1)).cuda()
    src = _rand(1, n_s, n_d).float().cuda()
    w = _rand(2, 1, n_d, n_d).float().cuda()
    off = torch.tensor([0, n_s]).cuda()
    torch.cuda.synchronize()
    ref, _, _ = R.embed_b(R.f64(src), ids.cpu().numpy(), 1.0, n_v)
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        yb = src * 1.0
        wb = torch.empty(n_v, n_d, device="cuda")
        ws = torch.empty(T.embed_b_workspace(n_s, n_v, n_d), dtype=torch.uint8, device="cuda")
        T.embed_b_cuda(wb, ids, yb, 1.0, n_s, n_v, n_d, accumulate=False, consume=False, stream=s,
                       workspace=ws)
        y = torch.empty(n_s, n_d, device="cuda")
        ws2 = torch.empty(T.expert_mm_workspace(torch.float32, n_s, 1, n_d, n_d), dtype=torch.uint8,
                          device="cuda")
        T.expert_mm_cuda(src, w, y, off, n_s, 1, n_d, n_d, stream=s, workspace=ws2)
    s.synchronize()
    assert np.abs(R.f64(wb) - ref).max() < 1e-4
    assert (y.double() - src.double() @ w[0].double()).abs().max() < 1e-4
    small = torch.empty(256, dtype=torch.uint8, device="cuda")
    with pytest.raises(sb.StadeError):
        T.embed_b_cuda(wb, ids, yb, 1.0, n_s, n_v, n_d, workspace=small)


def test_calls_inside_a_captured_graph():
    """Every operator replays from a CUDA graph with new inputs in place."""
    n_s, n_d, n_v = 200, 128, 40
    x = _rand(1, n_s, n_d).bfloat16().cuda()
    ids = (torch.arange(n_s) * 7 % n_v).cuda()
    off = torch.tensor([0, 90, 200]).cuda()
    w = _rand(2, 2, n_d, n_d, scale=0.1).bfloat16().cuda()
    y, z = torch.empty_like(x), torch.empty_like(x)
    m, r = torch.empty(n_s, device="cuda"), torch.empty(n_s, device="cuda")
    q, e = sb.initstacks_tape8_cuda(n_s, n_d)
    xb, wb = torch.empty_like(x), torch.empty(2, n_d, n_d, device="cuda")
    tb = torch.empty(n_v, n_d, device="cuda")

    def step():
        sb.layer_norm_cuda(x, None, None, y, m, r, 1e-5, n_s, n_d)
        sb.expert_mm_cuda(y, w, z, off, n_s, 2, n_d, n_d)
        sb.act_tape8_cuda("gelu", z, y, q, e, n_s, n_d)
        sb.expert_mm_b_cuda(x, xb, w, wb, y, off, n_s, 2, n_d, n_d, accumulate=False, consume=False)
        sb.embed_b_cuda(tb, ids, xb, 1.0, n_s, n_v, n_d, accumulate=False, consume=False)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    x.copy_(_rand(9, n_s, n_d).bfloat16())
    g.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (y, q, xb, wb, tb)]
    step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, (y, q, xb, wb, tb)))


def test_embed_b_of_a_long_batch_in_a_graph():
    """The sort that runs in a cluster, and what overlaps it, replayed."""
    n_s, n_v, n_d = 9000, 3000, 36
    yb = _rand(1, n_s, n_d).bfloat16().cuda()
    ids = torch.from_numpy(_ids(2, n_s, n_v, 0)).cuda()
    wb, again = torch.empty(n_v, n_d, device="cuda"), torch.empty(n_v, n_d, device="cuda")
    args = (1.5, n_s, n_v, n_d)
    sb.embed_b_cuda(again, ids, yb, *args, accumulate=False, consume=False)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sb.embed_b_cuda(wb, ids, yb, *args, accumulate=False, consume=False)
    ids.copy_(torch.from_numpy(_ids(7, n_s, n_v, 0)))
    for _ in range(3):
        wb.fill_(math.nan)
        g.replay()
    sb.embed_b_cuda(again, ids, yb, *args, accumulate=False, consume=False)
    assert torch.equal(wb, again)


def test_zero_sizes():
    e = torch.empty(0, device="cuda")
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    sb.layer_norm_cuda(e, None, None, e, e, e, 1e-5, 0, 64)
    wb = torch.ones(64, device="cuda")
    sb.layer_norm_b_cuda(e, e, None, wb, None, e, e, e, 0, 64)
    assert (wb == 1).all()
    sb.layer_norm_b_cuda(e, e, None, wb, None, e, e, e, 0, 64, accumulate=False)
    assert not wb.any()
    tb = torch.ones(3, 4, device="cuda")
    sb.embed_b_cuda(tb, ids, e, 1.0, 0, 3, 4)
    assert (tb == 1).all()
    sb.embed_b_cuda(tb, ids, e, 1.0, 0, 3, 4, accumulate=False)
    assert not tb.any()
    y = torch.ones(2, 4, device="cuda")
    sb.expert_mm_cuda(torch.ones(2, 3, device="cuda"), e, y,
                      torch.zeros(1, dtype=torch.int64, device="cuda"), 2, 0, 3, 4)
    assert not y.any()
    gw = torch.ones(2, 3, 4, device="cuda")
    sb.expert_mm_b_cuda(e, e, torch.ones(2, 3, 4, device="cuda"), gw, e,
                        torch.zeros(3, dtype=torch.int64, device="cuda"), 0, 2, 3, 4, accumulate=False)
    assert not gw.any()
