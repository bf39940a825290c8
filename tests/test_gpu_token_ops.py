"""Layer norm and token embedding with their gradients, against the formulas in 64 bits.

Tolerances.  u = 2^-24 is a 32-bit rounding, half = finfo(type).eps / 2 the rounding of the output.  A 32-bit sum of n
terms in any order is off by at most n u sum|terms| (first order); the kernels' lanes add at most LANE(n) = n / 64 + 16
terms in a row along a row of n columns (one wave a row is the least parallel form), and at most rows + 16 down the rows.
Every bound below adds these to a few u for the products and is evaluated in 64 bits from the test's own inputs.
"""
import math

import pytest
import torch

from hfuse_amd import launcher as H
from hfuse_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


def floor(t):
    """Half the distance of the smallest numbers of the type (flushing them to zero is allowed a whole one)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(shape, seed, type=torch.float32, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen(seed)) * scale + mean).to(type)


def check(got, want, tol, what):
    got, want, tol = got.double().cpu(), want.cpu(), torch.as_tensor(tol, dtype=torch.float64).cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs().max()), torch.nonzero(bad)[:4].tolist())


# ------------------------------------------------------------------ layer norm
def norm64(x, w, b, eps):
    """-> (y, mean, rstd) and their bounds without the output's rounding."""
    n = x.shape[1]
    x = x.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(n, dtype=torch.float64) if b is None else b.double()
    y = d * rstd * w + b
    lane = (n / 64 + 16) * U
    tmean = lane * x.abs().mean(1, keepdim=True) + U * mean.abs()
    # the squares see every difference off by the mean's error and one rounding: the variance is off by
    # lane * var + 2 |d| (u |d| + 0) + tmean^2 (the first-order term of tmean sums to zero up to lane)
    tvar = (lane + 4 * U) * var + tmean ** 2 + 2 * tmean * lane * d.abs().mean(1, keepdim=True)
    trstd = rstd * (0.5 * tvar / (var + eps) + 4 * U)
    ty = w.abs() * (rstd * (tmean + U * d.abs()) + d.abs() * trstd) + 4 * U * ((d * rstd * w).abs() + b.abs())
    return y, mean, rstd, ty, tmean, trstd


def run_norm(x, w, b, eps, cuda, put=lambda t: t):
    dev = lambda t: None if t is None else t.to(cuda)
    y, mean, rstd = ops.run(ops.layer_norm(put(dev(x)), x.shape[-1], dev(w), dev(b), eps))
    torch.cuda.synchronize()
    return y, mean, rstd


def check_norm(x, w, b, eps, got, what):
    y, mean, rstd = got
    wy, wm, wr, ty, tm, tr = norm64(x, w, b, eps)
    check(mean, wm, tm, (what, "mean"))
    check(rstd, wr, tr, (what, "rstd"))
    check(y, wy, ty + half(x.dtype) * (wy.abs() + ty) + floor(x.dtype), (what, "y"))


COLS = [1, 2, 7, 8, 63, 64, 65, 100, 257, 512, 1000, 1024, 1155, 2048, 2056, 4096, 5001, 8192, 8200, 16392, 33000]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_over_row_lengths(cuda, type, cols):
    t = TYPES[type]
    for rows, params in ((1, t), (5, torch.float32), (67, t), (300, torch.float32), (301, t)):
        x = rand((rows, cols), cols + rows, t, 2.0, 0.5)
        w, b = rand((cols,), 1, params, 0.2, 1.0), rand((cols,), 2, params)
        check_norm(x, w, b, 1e-5, run_norm(x, w, b, 1e-5, cuda), (type, cols, rows))


@pytest.mark.parametrize("rows", [1, 2, 3, 255, 256, 257, 1025, 5000, 20011])
def test_layer_norm_over_row_counts(cuda, rows):
    for cols, t in ((96, torch.bfloat16), (513, torch.float32)):
        x, w, b = rand((rows, cols), rows, t), rand((cols,), 3, t), rand((cols,), 4, t)
        check_norm(x, w, b, 1e-6, run_norm(x, w, b, 1e-6, cuda), (rows, cols))


@pytest.mark.parametrize("type", TYPES)
def test_layer_norm_optional_parameters_and_shapes(cuda, type):
    t = TYPES[type]
    x, w, b = rand((6, 264), 5, t), rand((264,), 6, t), rand((264,), 7, t)
    for weight, bias in ((None, None), (w, None), (None, b), (w, b)):
        check_norm(x, weight, bias, 1e-5, run_norm(x, weight, bias, 1e-5, cuda), (type, weight is None, bias is None))
    # two normalised dimensions, a batch in front, statistics of torch's shape
    y, mean, rstd = ops.run(ops.layer_norm(x.view(2, 3, 11, 24).to(cuda), (11, 24), w.view(11, 24).to(cuda)))
    assert y.shape == (2, 3, 11, 24) and mean.shape == rstd.shape == (2, 3, 1, 1) and mean.dtype == torch.float32
    check_norm(x, w, None, 1e-5, (y.view(6, 264), mean.view(6, 1), rstd.view(6, 1)), type)
    y, mean, rstd = ops.run(ops.layer_norm(x[0].to(cuda), 264))                      # one row without a batch
    assert y.shape == (264,) and mean.shape == (1,)
    check_norm(x[:1], None, None, 1e-5, (y[None], mean[None], rstd[None]), type)


@pytest.mark.parametrize("cols", [8, 65, 520, 2049, 4104])
def test_layer_norm_strided_rows(cuda, cols):
    """Rows cut out of wider ones (at an odd element), every other row, one row repeated, and columns that are not adjacent."""
    for t in TYPES.values():
        x, w, b = rand((10, cols), 8, t), rand((cols,), 9, t), rand((cols,), 10, t)

        def wide(v):
            buf = torch.full((10, cols + 5), float("nan"), device=v.device, dtype=t)
            buf[:, 3:3 + cols] = v
            return buf[:, 3:3 + cols]
        check_norm(x, w, b, 1e-5, run_norm(x, w, b, 1e-5, cuda, wide), ("wide", cols, t))
        check_norm(x, w, b, 1e-5, run_norm(x, w, b, 1e-5, cuda, lambda v: v.repeat_interleave(2, 0)[::2]), ("every other", cols, t))
        check_norm(x, w, b, 1e-5, run_norm(x, w, b, 1e-5, cuda, lambda v: v.t().contiguous().t()), ("transposed", cols, t))
        one = x[:1].expand(10, cols)
        check_norm(one, w, b, 1e-5, run_norm(x, w, b, 1e-5, cuda, lambda v: v[:1].expand(10, cols)), ("repeated", cols, t))


def test_layer_norm_hard_rows(cuda):
    """Constant rows, a large mean, tiny and huge values; a row of infinities or NaN leaves the other rows alone."""
    cols = 1000
    x = rand((8, cols), 11)
    x[1], x[2] = 3.25, 0.0
    x[3] += 4096.0
    x[4] *= 1e-18
    x[5] *= 1e15
    w, b = rand((cols,), 12), rand((cols,), 13)
    got = run_norm(x, w, b, 1e-5, cuda)
    check_norm(x, w, b, 1e-5, got, "hard")
    many = run_norm(x.repeat(40, 1), w, b, 1e-5, cuda)                                # the same rows among more of them
    check_norm(x, w, b, 1e-5, [v[160:168] for v in many], "hard, many")
    assert torch.equal(got[0][2].cpu(), b)                                            # 0 * w + b
    bad = x.clone()
    bad[6, 17], bad[7, 999] = float("nan"), float("inf")
    y, mean, rstd = run_norm(bad, w, b, 1e-5, cuda)
    assert torch.equal(y[:6], got[0][:6]) and torch.isnan(y[6:]).all() and torch.isnan(rstd[6:]).all()
    y, _, rstd = run_norm(torch.zeros(1, 64), None, None, 0.0, cuda)                  # 0 * (1 / 0)
    assert torch.isinf(rstd).all() and torch.isnan(y).all()


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", [5, 100, 1000, 1155, 1920, 5001, 6656, 12290, 14336, 20001, 33000])
def test_layer_norm_of_constant_rows_is_the_bias(cuda, type, cols):
    """Rows of one number come out as the bias, bit for bit, and with that number as their mean.

    Whole numbers up to 2^24 / cols have exact sums (multiples of 1 below 2^24), so sum / cols is the number itself, and so it
    is for any bf16 number up to 2^16 columns and any f16 number up to 2^13 (8 and 11 bits).  Of any other number c the rounded
    mean is k steps of c's last place off, k <= cols / 64 + 16 or, where a row is shared by more lanes, fewer; all
    differences are then the same k steps, cols * k < 2^24 of them add up exactly, and the mean of the differences takes them
    back to zero."""
    t = TYPES[type]
    b, w = rand((cols,), 1, t), rand((cols,), 2, t)
    top = min((1 << 24) // cols, 1024 if t != torch.bfloat16 else 256)
    whole = torch.arange(1, top + 1, dtype=torch.float32)
    for rows in (whole, whole[-200:], -whole[:301]):
        x = rows[:, None].to(t).expand(len(rows), cols).contiguous()
        assert torch.equal(x[:, 0].float(), rows)
        y, mean, rstd = run_norm(x, w, b, 1e-5, cuda)
        assert torch.equal(mean.cpu()[:, 0], rows) and torch.equal(y.cpu(), b.expand_as(y)), (type, cols, len(rows))
        check(rstd, torch.full((len(rows), 1), (1e-5) ** -0.5, dtype=torch.float64), 8 * U * (1e-5) ** -0.5, "rstd")
    any_number = torch.exp(torch.rand((300,), generator=gen(cols)) * 11).to(t)               # up to 6e4
    x = any_number[:, None].expand(300, cols).contiguous()
    y, mean, _ = run_norm(x, w, b, 1e-5, cuda)
    assert torch.equal(mean.cpu()[:, 0], any_number.float()) and torch.equal(y.cpu(), b.expand_as(y)), (type, cols)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", [100, 1000, 1155, 5001, 12290, 20001])
def test_layer_norm_of_rows_with_a_large_mean(cuda, type, cols):
    """The rounding of the row's sum, 32-bit steps of the mean, does not reach y: only those of the differences do.

    The sums of the 16-bit rows are exact up to 2^13 columns (all values in [64, 128), 2^11 steps of which 2^13 are below 2^24),
    so their mean is off by its own rounding, U |mean|, which may stay.  Else
    near, the rounded mean, is off by tm at most (norm64).  The differences x - near are off by U each, their mean by
    ts = (lane + 3 U)(mean|d| + tm), so a difference from the mean by td = 2 U |d| + U tm + ts.  The mean of their squares is
    var + (near - mean)^2 with a relative (lane + 6 U), and the square taken off again is off by 2 tm ts."""
    t, eps = TYPES[type], 1e-5
    w, b = rand((cols,), 1, torch.float32), rand((cols,), 2, torch.float32)
    for rows in (3, 300):
        x = rand((rows, cols), cols + rows, t, 1.0, 2e4 if t == torch.float32 else 100.0)
        y, mean, rstd = run_norm(x, w, b, eps, cuda)
        wy, wm, wr, _, tm, _ = norm64(x, w, b, eps)
        d = x.double() - wm
        var, size, lane = (d * d).mean(1, keepdim=True), d.abs().mean(1, keepdim=True), (cols / 64 + 16) * U
        ts = (lane + 3 * U) * (size + tm)
        td = 2 * U * d.abs() + U * tm + ts + (0 if t == torch.float32 else U * wm.abs())
        trstd = wr * (0.5 * ((lane + 6 * U) * (var + tm ** 2) + 2 * tm * ts) / (var + eps) + 4 * U)
        ty = w.double().abs() * (wr * td + d.abs() * trstd) + 4 * U * ((d * wr * w).abs() + b.double().abs())
        check(mean, wm, ts + U * (wm.abs() + ts), (type, cols, rows, "mean"))
        check(rstd, wr, trstd, (type, cols, rows, "rstd"))
        check(y, wy, ty + half(t) * (wy.abs() + ty) + floor(t), (type, cols, rows, "y"))


@pytest.mark.parametrize("cols", [100, 1155, 4096, 8200, 20001])
def test_layer_norm_mean_is_as_exact_as_one_sum(cuda, cols):
    """A mean that is small beside the spread is the sum's, not corrected by the mean of the differences: those of one binade
    are all rounded by the same last bits of the mean, up to U / 2 each, which does not average out.

    Root mean square of the sum's own error: a partial sum of m terms of size 1 is about sqrt(m) and is rounded by a uniform
    error of U sqrt(m / 3) at most, there are cols / m of them at each of the log2(cols) levels of a tree, which gives
    U sqrt(cols / 3) a level, and the k terms a lane adds one after another count as k / 2 levels; with 2 levels for the quotient.
    Half as much again for what is not independent, and the mean's rounding."""
    x = rand((2000, cols), cols, torch.float32, 1.0, 0.02)
    _, mean, _ = run_norm(x, None, None, 1e-5, cuda)
    want = x.double().mean(1, keepdim=True)
    rms = lambda e: float((e * e).mean().sqrt())
    k = max(16, cols / 1024 + 4)
    assert rms(mean.cpu().double() - want) <= 1.5 * U * math.sqrt((math.log2(cols) + k / 2 + 2) / (3 * cols)) + U * rms(want), cols


def grad64(dy, x, mean, rstd, w):
    n, rows = x.shape[1], x.shape[0]
    dy, x, mean, rstd = dy.double(), x.double(), mean.double().view(-1, 1), rstd.double().view(-1, 1)
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double()
    h, g = (x - mean) * rstd, dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rstd * (g - c1 - h * c2)
    lane = (n / 64 + 16) * U
    t = rstd.abs() * (8 * U * (g.abs() + c1.abs() + (h * c2).abs()) + lane * g.abs().mean(1, keepdim=True)
                      + h.abs() * (lane + 6 * U) * (g * h).abs().mean(1, keepdim=True))
    down = (rows + 16) * U
    return (dx, t), ((dy * h).sum(0), (down + 4 * U) * (dy * h).abs().sum(0)), (dy.sum(0), down * dy.abs().sum(0))


def stats(x, eps=1e-5):
    x = x.double()
    mean = x.mean(1)
    return mean.float(), (1 / torch.sqrt(x.var(1, unbiased=False) + eps)).float()


def check_grad(dy, x, mean, rstd, w, got, what):
    for (want, tol), g, name in zip(grad64(dy, x, mean, rstd, w), got, ("dx", "dweight", "dbias")):
        if g is not None:
            check(g.view(want.shape), want, tol + half(g.dtype) * (want.abs() + tol) + floor(g.dtype), (what, name))


def run_grad(dy, x, mean, rstd, w, cuda, mask=None, put=lambda t: t):
    got = ops.run(ops.layer_norm_backward(put(dy.to(cuda)), put(x.to(cuda)), x.shape[-1], mean.to(cuda), rstd.to(cuda),
                                          None if w is None else w.to(cuda), mask))
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_backward_over_row_lengths(cuda, type, cols):
    t = TYPES[type]
    for rows, params in ((1, t), (5, torch.float32), (67, t), (300, torch.float32), (301, t)):
        x, dy = rand((rows, cols), cols + rows, t, 2.0, 0.5), rand((rows, cols), cols, t, 0.1)
        w, (mean, rstd) = rand((cols,), 1, params, 0.2, 1.0), stats(x)
        got = run_grad(dy, x, mean, rstd, w, cuda)
        assert got[1].dtype == got[2].dtype == params
        check_grad(dy, x, mean, rstd, w, got, (type, cols, rows))


@pytest.mark.parametrize("rows", [1, 2, 3, 255, 256, 257, 511, 513, 1025, 5000, 20011])
def test_layer_norm_backward_over_row_counts(cuda, rows):
    for cols, t in ((96, torch.bfloat16), (513, torch.float32), (2048, torch.float16)):
        x, dy, w = rand((rows, cols), rows, t), rand((rows, cols), rows + 1, t), rand((cols,), 3, t)
        mean, rstd = stats(x)
        check_grad(dy, x, mean, rstd, w, run_grad(dy, x, mean, rstd, w, cuda), (rows, cols))


def test_layer_norm_backward_wanted_outputs(cuda):
    for cols in (100, 2056):
        x, dy, w = rand((37, cols), 14, torch.bfloat16), rand((37, cols), 15, torch.bfloat16), rand((cols,), 16)
        mean, rstd = stats(x)
        for mask in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1), (1, 1, 1)):
            got = run_grad(dy, x, mean, rstd, w, cuda, mask)
            assert [g is not None for g in got] == [bool(m) for m in mask]
            check_grad(dy, x, mean, rstd, w, got, (cols, mask))
        got = run_grad(dy, x, mean, rstd, None, cuda)
        assert got[1] is None and got[2] is None
        check_grad(dy, x, mean, rstd, None, got, (cols, "no weight"))
        check_grad(dy, x, mean, rstd, None, run_grad(dy, x, mean, rstd, None, cuda, (1, 1, 1)), (cols, "no weight, all"))


@pytest.mark.parametrize("cols", [8, 65, 520, 2049, 4104])
def test_layer_norm_backward_strided_rows(cuda, cols):
    for t in TYPES.values():
        x, dy, w = rand((10, cols), 17, t), rand((10, cols), 18, t), rand((cols,), 19, t)
        mean, rstd = stats(x)

        def wide(v):
            buf = torch.full((10, cols + 3), float("nan"), device=v.device, dtype=t)
            buf[:, 1:1 + cols] = v
            return buf[:, 1:1 + cols]
        check_grad(dy, x, mean, rstd, w, run_grad(dy, x, mean, rstd, w, cuda, put=wide), ("wide", cols, t))
        # the gradient of a sum: one number for all of dy
        got = ops.run(ops.layer_norm_backward(dy[:1, :1].to(cuda).expand(10, cols), x.to(cuda), cols, mean.to(cuda), rstd.to(cuda), w.to(cuda)))
        check_grad(dy[:1, :1].expand(10, cols), x, mean, rstd, w, got, ("broadcast", cols, t))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", [100, 1000, 1920, 6656, 12344, 14336, 20002])
def test_layer_norm_backward_of_a_sum(cuda, type, cols):
    """dy of ones without a weight: g - mean(g) is nothing.  Where the h come in pairs (h, -h) beside each other, so that every
    partial sum of g h is nothing as well, dx is zero to the bit: rstd - rstd."""
    t = TYPES[type]
    half_row = rand((300, cols // 2), cols, t, 2.0)
    x = torch.stack((half_row, -half_row), 2).view(300, cols)
    mean, rstd = torch.zeros(300), stats(x)[1]
    for rows in (300, 7):
        dx, _, db = run_grad(torch.ones(rows, cols, dtype=t), x[:rows], mean[:rows], rstd[:rows], None, cuda, (1, 0, 1))
        assert not dx.any(), (type, cols, rows, float(dx.abs().max()))
        assert (db == rows).all()      # (whole numbers up to 2^8, or 300 = 75 * 4: exact in every type)


def test_layer_norm_gradient_against_differences(cuda):
    """d/dx, d/dw and d/db of sum(y * c) by central differences of the forward formula in 64 bits (error about h^2 and 1e-16 / h,
    far below the 32-bit bounds of the kernel, which check_grad's tolerances also cover)."""
    rows, cols, h = 3, 37, 1e-5
    x, w, b, c = rand((rows, cols), 20), rand((cols,), 21), rand((cols,), 22), rand((rows, cols), 23)
    y, mean, rstd = ops.run(ops.layer_norm(x.to(cuda), cols, w.to(cuda), b.to(cuda)))
    dx, dw, db = ops.run(ops.layer_norm_backward(c.to(cuda), x.to(cuda), cols, mean, rstd, w.to(cuda)))
    f = lambda x, w, b: (norm64(x, w, b, 1e-5)[0] * c.double()).sum()
    for got, k in ((dx, 0), (dw, 1), (db, 2)):
        args = [x.double(), w.double(), b.double()]
        base = args[k].clone()
        want = torch.zeros_like(base)
        for i in range(base.numel()):
            for sign in (1, -1):
                moved = base.clone()
                moved.view(-1)[i] += sign * h
                args[k] = moved
                want.view(-1)[i] += sign * f(*args) / (2 * h)
        check(got, want, 1e-5 * (1 + want.abs()), k)


def shifted(pad, at):
    """Rows cut out of wider ones: a row starts at element `at`, pad + cols elements behind the one before."""
    def put(v):
        buf = torch.full((v.shape[0], v.shape[1] + pad), float("nan"), device=v.device, dtype=v.dtype)
        buf[:, at:at + v.shape[1]] = v
        return buf[:, at:at + v.shape[1]]
    return put


# Every way rows of several waves are cut: two, three and four slots a lane, whole workgroups, rows that are read again, each
# with a last slot that repeats elements and one that does not.
WIDE_COLS = [4104, 4605, 7176, 7677, 9001, 12289, 12296, 14337, 16383, 16384, 16389, 24577, 30003, 32765, 32768, 32771, 40007]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", WIDE_COLS)
def test_layer_norm_of_wide_rows(cuda, type, cols):
    t = TYPES[type]
    for rows, params, put in ((300 if cols < 8192 else 5, t, lambda v: v), (259 if cols < 8192 else 4, torch.float32, shifted(5, 3))):
        x = rand((rows, cols), cols + rows, t, 2.0, 0.5)
        w, b = rand((cols,), 1, params, 0.2, 1.0), rand((cols,), 2, params)
        check_norm(x, w, b, 1e-5, run_norm(x, w, b, 1e-5, cuda, put), (type, cols, rows))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", WIDE_COLS)
def test_layer_norm_backward_of_wide_rows(cuda, type, cols):
    """Over more rows than there are workgroups where a workgroup takes several in turn."""
    t = TYPES[type]
    for rows, params, put in ((300 if cols <= 16384 else 131, t, lambda v: v), (5, torch.float32, shifted(3, 1))):
        x, dy = rand((rows, cols), cols + rows, t, 2.0, 0.5), rand((rows, cols), cols, t, 0.1)
        w, (mean, rstd) = rand((cols,), 1, params, 0.2, 1.0), stats(x)
        check_grad(dy, x, mean, rstd, w, run_grad(dy, x, mean, rstd, w, cuda, put=put), (type, cols, rows))


@pytest.mark.parametrize("rows, cols, type, params", [(8203, 1155, "f32", "f32"), (8200, 2056, "bf16", "bf16"), (9001, 4104, "f16", "f16"),
                                                      (16411, 8192, "bf16", "f32"), (8300, 8200, "f32", "f32")])
def test_layer_norm_over_several_rows_a_workgroup(cuda, rows, cols, type, params):
    """Rows of several waves, each workgroup with several in turn; the last two are more than 256 MiB and read past the caches.
    Bounds in 64 bits on the GPU, over the first, the last and every seventh row."""
    t, p = TYPES[type], TYPES[params]
    g = torch.Generator(device=cuda).manual_seed(rows)
    x = (torch.randn((rows, cols), generator=g, device=cuda) * 2 + torch.randn((rows, 1), generator=g, device=cuda)).to(t)
    w, b = (torch.randn((cols,), generator=g, device=cuda).to(p) for _ in range(2))
    got = ops.run(ops.layer_norm(x, cols, w, b))
    for part in (slice(0, 600), slice(rows - 600, rows), slice(0, rows, 7)):
        check_norm(x[part], w, b, 1e-5, [v[part] for v in got], (rows, cols, part))


def test_layer_norm_backward_past_the_caches(cuda):
    """x and dy of more than 256 MiB; 64 bits on the GPU."""
    rows, cols, t = 9001, 8192, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(9)
    x, dy = (torch.randn((rows, cols), generator=g, device=cuda).to(t) for _ in range(2))
    w = torch.randn((cols,), generator=g, device=cuda)
    mean, rstd = stats(x)
    got = ops.run(ops.layer_norm_backward(dy, x, cols, mean, rstd, w))
    check_grad(dy, x, mean, rstd, w, got, "past the caches")


# ------------------------------------------------------------------ embedding
def ids(n, vocab, seed, bad=True):
    t = torch.randint(0, vocab, (n,), generator=gen(seed))
    if bad and n > 4:
        t[1], t[3], t[-1] = -1, vocab, -(1 << 31)
    return t


def lookup64(tokens, w, scale):
    used = (tokens >= 0) & (tokens < w.shape[0])
    return torch.where(used[:, None], w.double()[tokens.clamp(0, w.shape[0] - 1)] * scale, torch.zeros((), dtype=torch.float64))


def lookup_tol(want, t):
    return (4 * U + half(t)) * want.abs() + floor(t)      # scale to 32 bits, the product, the output


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", [1, 3, 8, 63, 64, 130, 255, 1000, 1024, 2056, 4096, 9001])
def test_embedding(cuda, type, cols):
    t = TYPES[type]
    w = rand((53, cols), cols, t)
    for n, it in ((1, torch.int64), (2, torch.int32), (70, torch.int32), (301, torch.int64)):
        tok = ids(n, 53, n)
        for scale in (1.0, -0.37, math.sqrt(cols)):
            (out,) = ops.run(ops.embedding(tok.to(it).to(cuda), w.to(cuda), scale))
            want = lookup64(tok, w, scale)
            check(out, want, lookup_tol(want, t), (type, cols, n, scale))


def test_embedding_copies_bits_and_keeps_shapes(cuda):
    for t, it in ((torch.float32, torch.int32), (torch.bfloat16, torch.int16), (torch.float16, torch.int16)):
        w = torch.randint(-30000, 30000, (20, 24), generator=gen(24)).to(it).view(t) if t != torch.float32 else \
            torch.randint(-(1 << 31), 1 << 31, (20, 24), generator=gen(24)).to(torch.int32).view(t)
        tok = torch.randint(0, 20, (3, 5), generator=gen(25))
        (out,) = ops.run(ops.embedding(tok.to(cuda), w.to(cuda)))
        assert out.shape == (3, 5, 24)
        same = (out.cpu().view(it) == w[tok].view(it)) | torch.isnan(w[tok])      # NaN stay NaN
        assert same.all() and torch.equal(torch.isnan(out.cpu()), torch.isnan(w[tok]))
        (out,) = ops.run(ops.embedding(tok[0, 0].to(cuda), w.to(cuda)))           # a token without dimensions
        assert out.shape == (24,)
        wide = torch.zeros((20, 31), dtype=t)
        wide[:, 2:26] = w
        (out,) = ops.run(ops.embedding(tok.t().to(cuda), wide.to(cuda)[:, 2:26]))  # strided tokens and table
        assert torch.equal(torch.nan_to_num(out.cpu()), torch.nan_to_num(w[tok.t()]))


def table_grad64(dy, tokens, vocab, scale, pad):
    used = (tokens >= 0) & (tokens < vocab)
    if pad is not None:
        used &= tokens != pad
    rows = torch.nonzero(used)[:, 0]
    want = torch.zeros((vocab, dy.shape[1]), dtype=torch.float64).index_add_(0, tokens[rows], dy[rows].double())
    size = torch.zeros_like(want).index_add_(0, tokens[rows], dy[rows].double().abs())
    count = torch.bincount(tokens[rows], minlength=vocab).double()[:, None]
    return want * scale, (count + 4) * U * size * abs(scale)


def check_table_grad(dy, tokens, vocab, cuda, scale=1.0, pad=None, dtype=None, what=None):
    (got,) = ops.run(ops.embedding_backward(dy.to(cuda), tokens.to(cuda), vocab, scale, pad, dtype))
    torch.cuda.synchronize()
    assert got.dtype == (dtype or dy.dtype) and got.shape == (vocab, dy.shape[-1])
    want, tol = table_grad64(dy.reshape(-1, dy.shape[-1]), tokens.long().reshape(-1), vocab, scale, pad)
    check(got, want, tol + half(got.dtype) * (want.abs() + tol) + floor(got.dtype), what)
    return got


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", [1, 3, 8, 63, 64, 130, 255, 1000, 1024, 2056, 4096, 9001])
def test_embedding_backward_over_row_lengths(cuda, type, cols):
    t = TYPES[type]
    for n, vocab, it in ((1, 5, torch.int64), (40, 1, torch.int32), (301, 77, torch.int64)):
        dy = rand((n, cols), cols + n, t)
        check_table_grad(dy, ids(n, vocab, n).to(it), vocab, cuda, 1.7, None, None, (type, cols, n))
        check_table_grad(dy, ids(n, vocab, n).to(it), vocab, cuda, -0.3, vocab // 2, torch.float32, (type, cols, n, "pad"))


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 1024, 1025, 4097, 16384, 40001])
@pytest.mark.parametrize("vocab", [1, 2, 300, 1000, 50000])
def test_embedding_backward_over_sizes(cuda, n, vocab):
    dy = rand((n, 24), n, torch.bfloat16)
    check_table_grad(dy, ids(n, vocab, n + vocab), vocab, cuda, 1.0, None, torch.float32, (n, vocab))
    skewed = (vocab ** torch.rand((n,), generator=gen(n))).long().clamp(0, vocab) - 1     # low ids most of the time, some -1
    check_table_grad(dy, skewed, vocab, cuda, 0.5, 0, None, (n, vocab, "skewed"))


@pytest.mark.parametrize("n", [900, 1030, 131073, 300007])
@pytest.mark.parametrize("vocab", [512, 513, 400000, (1 << 27) + 5])
def test_embedding_backward_long_lists_and_large_vocabularies(cuda, n, vocab):
    """Sorts of one to four digits, of one workgroup's tokens to several steps a workgroup; compared on the rows named and
    by the sum of all others."""
    cols = 5 if vocab < 1 << 20 else 1
    tok = (torch.rand((n,), generator=gen(n), dtype=torch.float64) ** 3 * vocab).long()
    tok[::11], tok[n // 2:n // 2 + 200], tok[-1] = -1, 7, vocab - 1
    dy = rand((n, cols), vocab % 1000)
    (got,) = ops.run(ops.embedding_backward(dy.to(cuda), tok.to(cuda), vocab, 0.5))
    got = got.cpu()
    named, at = torch.unique(tok[tok >= 0], return_inverse=True)
    want, tol = table_grad64(dy[tok >= 0], at, len(named), 0.5, None)
    check(got[named], want, tol + half(torch.float32) * (want.abs() + tol) + floor(torch.float32), (n, vocab))
    got[named] = 0
    assert not got.any()


@pytest.mark.parametrize("shape", ["one", "two ends", "last", "runs", "sorted", "reversed", "none"])
def test_embedding_backward_token_patterns(cuda, shape):
    """All rows on one id, on the table's first and last, in runs longer and shorter than any tile, and no usable id at all."""
    n, vocab = 9973, 2000
    at = torch.arange(n)
    tok = {"one": torch.full((n,), 777), "two ends": (at % 2) * (vocab - 1), "last": torch.full((n,), vocab - 1), "runs": (at // 129) * 7,
           "sorted": at * vocab // n, "reversed": (n - 1 - at) * vocab // n, "none": torch.full((n,), -1)}[shape]
    for cols, t in ((40, torch.float32), (264, torch.bfloat16)):
        dy = rand((n, cols), 26, t)
        check_table_grad(dy, tok, vocab, cuda, 2.0, None, None, (shape, cols))
        check_table_grad(dy, tok, vocab, cuda, 2.0, int(tok[0]) if shape != "none" else 0, None, (shape, cols, "pad"))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cols", [1, 5, 24, 130, 257, 520, 1031])
def test_embedding_backward_few_tokens_of_few_ids(cuda, type, cols):
    """One launch's largest batch and its neighbour, an id with up to all of the rows, next to ids with one or none."""
    t = TYPES[type]
    for n, vocab in ((1024, 1), (1024, 3), (1025, 3), (999, 40)):
        tok = torch.where(torch.rand((n,), generator=gen(n)) < 0.6, vocab // 2, ids(n, vocab, n))
        for pad, dtype in ((None, None), (0, torch.float32)):
            a = check_table_grad(rand((n, cols), n, t), tok, vocab, cuda, 1.3, pad, dtype, (type, cols, n, vocab, pad))
            assert torch.equal(a, check_table_grad(rand((n, cols), n, t), tok, vocab, cuda, 1.3, pad, dtype))


def test_embedding_backward_leaves_unused_rows_unread(cuda):
    """NaN in the dy rows of padding and of ids outside the table reaches nothing; other ids keep theirs to themselves."""
    n, vocab, cols = 500, 60, 72
    tok = torch.randint(0, vocab, (n,), generator=gen(27))
    tok[::5], tok[1::7] = -1, 3
    dy = rand((n, cols), 28)
    clean = check_table_grad(dy, tok, vocab, cuda, 1.0, 3)
    dirty = dy.clone()
    dirty[(tok == -1) | (tok == 3)] = float("nan")
    (got,) = ops.run(ops.embedding_backward(dirty.to(cuda), tok.to(cuda), vocab, 1.0, 3))
    assert torch.equal(got, clean) and not got[3].any()
    dirty[tok == 9] = float("inf")
    (got,) = ops.run(ops.embedding_backward(dirty.to(cuda), tok.to(cuda), vocab, 1.0, 3))
    keep = torch.arange(vocab, device=cuda) != 9
    assert torch.equal(got[keep], clean[keep]) and torch.isinf(got[9]).all()


@pytest.mark.parametrize("n, vocab, cols", [(500, 60, 40), (3000, 200, 40), (3000, 50000, 400), (6000, 200, 40)])
def test_long_ids_are_no_short_ones(cuda, n, vocab, cols):
    """Ids whose low word alone would name a row: the lookup and the gradient's three ways to sort them leave them out."""
    tok = torch.randint(0, vocab, (n,), generator=gen(n))
    tok[::3] += 1 << 32
    tok[1::7] -= 1 << 32
    tok[5], tok[6] = (1 << 63) - 1, -(1 << 63)
    w, dy = rand((vocab, cols), 47), rand((n, cols), 48)
    (out,) = ops.run(ops.embedding(tok.to(cuda), w.to(cuda)))
    used = (tok >= 0) & (tok < vocab)
    assert torch.equal(out.cpu(), torch.where(used[:, None], w[tok.clamp(0, vocab - 1)], torch.zeros(())))
    check_table_grad(dy, tok, vocab, cuda, 1.0, None, None, (n, vocab))
    check_table_grad(dy, tok, vocab, cuda, 1.0, int(tok[used][0]), None, (n, vocab, "pad"))


def test_embedding_backward_strided_and_broadcast(cuda):
    n, vocab, cols = 130, 40, 56
    tok, dy = ids(n, vocab, 29), rand((n, cols), 30, torch.bfloat16)
    want, tol = table_grad64(dy, tok, vocab, 1.0, None)
    tol = tol + half(dy.dtype) * (want.abs() + tol) + floor(dy.dtype)
    wide = torch.full((n, cols + 9), float("nan"), device=cuda, dtype=dy.dtype)
    wide[:, 5:5 + cols] = dy.to(cuda)
    check(ops.run(ops.embedding_backward(wide[:, 5:5 + cols], tok.to(cuda), vocab))[0], want, tol, "wide")
    check(ops.run(ops.embedding_backward(dy.to(cuda).t().contiguous().t(), tok.to(cuda), vocab))[0], want, tol, "transposed")
    check_table_grad(dy.view(10, 13, cols), tok.view(10, 13), vocab, cuda, what="batch")
    ones = torch.ones((1, 1), device=cuda).expand(n, cols)                              # the gradient of a sum
    count = torch.bincount(tok[(tok >= 0) & (tok < vocab)], minlength=vocab).double()[:, None].expand(vocab, cols)
    assert torch.equal(ops.run(ops.embedding_backward(ones, tok.to(cuda), vocab))[0].double().cpu(), count)


def test_long_offsets(cuda):
    """Tables and batches of more than 2^31 elements: the last rows are found, counted and written."""
    vocab, cols = 70001, 32768
    w = torch.zeros((vocab, cols), device=cuda, dtype=torch.bfloat16)
    w[-1], w[-2] = 3.0, 5.0
    (out,) = ops.run(ops.embedding(torch.tensor([vocab - 1, 0, vocab - 2], device=cuda), w, 2.0))
    assert (out[0] == 6).all() and not out[1].any() and (out[2] == 10).all()
    last = torch.tensor([vocab - 1, -1, vocab - 2], device=cuda)
    (dw,) = ops.run(ops.embedding_backward(w[-3:], last, vocab))                      # a long table: rows 5, 3 go to its end
    assert not dw[-1].any() and (dw[-2] == 3).all() and not dw[:-2].any()
    del dw
    tok = torch.arange(vocab, device=cuda) % 3 - 1
    (dw,) = ops.run(ops.embedding_backward(w[:, :8], tok, 2))                         # a long batch: its last rows add up
    want = torch.zeros((2, 8), device=cuda)
    for row, value in ((vocab - 2, 5.0), (vocab - 1, 3.0)):
        if int(tok[row]) >= 0:
            want[int(tok[row])] += value
    assert torch.equal(dw.float(), want) and want.any()
    del dw
    w[-1, ::2] = 1.0
    y, mean, rstd = ops.run(ops.layer_norm(w, cols))
    assert float(mean[-1, 0]) == 2.0 and float(mean[-2, 0]) == 5.0 and (y[-1, ::2] == -1).all() and (y[-1, 1::2] == 1).all()
    assert not y[:-1].any()
    dx, dweight, dbias = ops.run(ops.layer_norm_backward(w, w, cols, mean, rstd, output_mask=(1, 1, 1)))
    assert (dbias[::2] == 6).all() and (dbias[1::2] == 8).all() and not dx[:-2].any()


def test_more_lanes_than_a_grid_has_threads(cuda):
    """Rows of five elements take eight lanes each: 2^29 tokens and some are more than 2^32 lanes."""
    n = (1 << 29) + 1000
    tok = torch.zeros(n, device=cuda, dtype=torch.int32)
    tok[-1], tok[-2], tok[1 << 29] = 2, -1, 1
    w = torch.arange(15, device=cuda).view(3, 5).to(torch.bfloat16) + 1
    (out,) = ops.run(ops.embedding(tok, w))
    assert torch.equal(out[-1], w[2]) and not out[-2].any() and torch.equal(out[1 << 29], w[1]) and torch.equal(out[-3], w[0])
    assert torch.equal(out[(1 << 29) - 1], w[0]) and torch.equal(out[5], w[0])


def test_more_rows_of_layer_norm_than_a_grid_has_threads(cuda):
    """Two rows of two elements a group of eight lanes: 2^30 rows and some are more than 2^32 lanes all the same."""
    n = (1 << 30) + 1000
    x = torch.zeros((n, 2), device=cuda, dtype=torch.bfloat16)
    rows = torch.tensor([0, 5, (1 << 29) + 3, (1 << 30) - 1, 1 << 30, n - 1], device=cuda)
    x[rows] = torch.tensor([3.0, 5.0], device=cuda, dtype=torch.bfloat16)
    y, mean, rstd = ops.run(ops.layer_norm(x, 2, eps=0.0))
    want = torch.tensor([-1.0, 1.0], device=cuda, dtype=torch.bfloat16).expand(len(rows), 2)
    assert torch.equal(y[rows], want) and (mean[rows] == 4).all() and (rstd[rows] == 1).all()
    assert int(torch.count_nonzero(mean)) == len(rows)
    del y, mean, rstd


def test_empty_batches(cuda):
    w = rand((9, 16), 31).to(cuda)
    none = torch.zeros((2, 0), dtype=torch.int64, device=cuda)
    assert ops.run(ops.embedding(none, w))[0].shape == (2, 0, 16)
    (dw,) = ops.run(ops.embedding_backward(torch.zeros((2, 0, 16), device=cuda), none, 9))
    assert dw.shape == (9, 16) and not dw.any()
    x = torch.zeros((0, 16), device=cuda)
    y, mean, rstd = ops.run(ops.layer_norm(x, 16, w[0]))
    assert y.shape == (0, 16) and mean.shape == (0, 1)
    dx, dweight, dbias = ops.run(ops.layer_norm_backward(x, x, 16, mean, rstd, w[0]))
    assert dx.shape == (0, 16) and not dweight.any() and not dbias.any() and dweight.shape == (16,)


# ------------------------------------------------------------------ the operators together, and how they are called
def embed_and_norm(tok, table, w, b, scale, pad, dy):
    """One training pass over the input end of a token model: forward, then back to the table."""
    (h,) = ops.run(ops.embedding(tok, table, scale))
    y, mean, rstd = ops.run(ops.layer_norm(h, h.shape[-1], w, b))
    dh, dw, db = ops.run(ops.layer_norm_backward(dy, h, h.shape[-1], mean, rstd, w))
    (dtable,) = ops.run(ops.embedding_backward(dh, tok, table.shape[0], scale, pad, torch.float32))
    return y, dw, db, dtable


@pytest.mark.parametrize("type", TYPES)
def test_input_end_of_a_token_model(cuda, type):
    """Embedding, layer norm and both gradients in a row against the same steps in 64 bits on the intermediate tensors as
    they were rounded (each step's own bound), and the whole against 64-bit autograd."""
    t = TYPES[type]
    vocab, cols, pad, scale = 97, 200, 0, math.sqrt(200)
    tok = torch.randint(0, vocab, (6, 50), generator=gen(32))
    for i, used in enumerate((50, 1, 0, 17, 33, 49)):
        tok[i, used:] = pad
    table, w, b = rand((vocab, cols), 33, t, 0.05), rand((cols,), 34, t, 0.1, 1.0), rand((cols,), 35, t)
    dy = rand((6, 50, cols), 36, t, 0.1)
    dev = [v.to(cuda) for v in (tok, table, w, b)]
    y, dw, db, dtable = embed_and_norm(*dev, scale, pad, dy.to(cuda))
    params = [v.double().requires_grad_() for v in (table, w, b)]
    h = params[0][tok] * scale
    want = torch.nn.functional.layer_norm(h, (cols,), params[1], params[2], 1e-5)
    grads = torch.autograd.grad(want, params, dy.double())
    grads = (grads[0].clone(), *grads[1:])
    grads[0][pad] = 0
    # the rounding of h (half a step, relative to each element) passes through a map whose gain per row is at most
    # rstd |w| sqrt(cols) in norm; four roundings of the type, with that gain below 3 sigma of the outputs' own scale
    k = half(t) * 16 + 1e-5
    for got, ref in ((y, want), (dw, grads[1]), (db, grads[2]), (dtable, grads[0])):
        scale_of = ref.detach().abs().amax()
        check(got.view(ref.shape), ref.detach(), k * scale_of, type)
    assert not dtable[pad].any()


def test_same_bits_every_time(cuda):
    """Nothing depends on the order in which workgroups finish."""
    same_bits(20000, 5000, 136, torch.bfloat16, cuda)
    same_bits(5000, 900, 1155, torch.float32, cuda)      # elements that two accesses of a row hold
    same_bits(3000, 900, 2049, torch.float16, cuda)


def same_bits(n, vocab, cols, t, cuda):
    tok = (vocab ** torch.rand((n,), generator=gen(37))).long() - 1
    args = [v.to(cuda) for v in (tok.clamp(0, vocab - 1), rand((vocab, cols), 38, t), rand((cols,), 39, t), rand((cols,), 40, t))]
    dy = rand((n, cols), 41, t).to(cuda)
    first = embed_and_norm(*args, 1.5, None, dy)
    for _ in range(5):
        for a, b in zip(first, embed_and_norm(*args, 1.5, None, dy)):
            assert torch.equal(a, b)


def test_graph_capture_and_replay(cuda):
    """The whole pass captured once and replayed on new inputs, with eager work between the replays."""
    n, vocab, cols = 3000, 700, 264
    tok = torch.randint(0, vocab, (n,), generator=gen(42)).to(cuda)
    table, w, b = (rand(s, 43 + i, torch.bfloat16).to(cuda) for i, s in enumerate(((vocab, cols), (cols,), (cols,))))
    dy = rand((n, cols), 46, torch.bfloat16).to(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        embed_and_norm(tok, table, w, b, 2.0, 5, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = embed_and_norm(tok, table, w, b, 2.0, 5, dy)
    for i in range(4):
        tok.copy_(torch.randint(-1, vocab, (n,), generator=gen(50 + i)) if i != 2 else torch.full((n,), 6))
        dy.copy_(rand((n, cols), 60 + i, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, embed_and_norm(tok, table, w, b, 2.0, 5, dy)):
            assert torch.equal(got, want), i
        torch.cuda.synchronize()


def test_kept_ops_captured_and_replayed(cuda):
    """Ops that a program keeps, built before the capture, run eagerly, captured twice and replayed: each run reads what its
    inputs hold then."""
    n, vocab, cols = 3000, 700, 264
    tok = torch.randint(0, vocab, (n,), generator=gen(92)).to(cuda)
    table, w, dy = rand((vocab, cols), 93).to(cuda), rand((cols,), 94).to(cuda), rand((n, cols), 95).to(cuda)
    look = ops.embedding(tok, table, 2.0)
    norm = ops.layer_norm(look.outputs[0], cols, w)
    norm_grad = ops.layer_norm_backward(dy, look.outputs[0], cols, *norm.outputs[1:], w)
    kept = (look, norm, norm_grad, ops.embedding_backward(norm_grad.outputs[0], tok, vocab, 2.0))

    def eager():
        for op in kept:
            ops.run(op)
        torch.cuda.synchronize()
        return [v.clone() for op in kept for v in op.outputs]
    eager()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            for op in kept:
                ops.run(op)
    for i in range(4):
        tok.copy_(torch.randint(-1, vocab, (n,), generator=gen(96 + i)))
        dy.copy_(rand((n, cols), 100 + i))
        for op in kept:
            for v in op.outputs:
                v.fill_(7)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = [v.clone() for op in kept for v in op.outputs]
        assert all(torch.equal(a, b) for a, b in zip(got, eager())), i


def test_two_graphs_and_a_side_stream(cuda):
    """Two captured gradients hold workspaces of their own; a launch on another stream keeps its tensors until it has run."""
    n, vocab, cols = 4000, 900, 72
    tok = [torch.randint(0, vocab, (n,), generator=gen(70 + i)).to(cuda) for i in range(2)]
    dy = [rand((n, cols), 72 + i).to(cuda) for i in range(2)]
    want = [ops.run(ops.embedding_backward(dy[i], tok[i], vocab))[0].clone() for i in range(2)]
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.run(ops.embedding_backward(dy[i], tok[i], vocab))[0])
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    s = streams[0]
    s.wait_stream(torch.cuda.current_stream())
    got = [ops.run(ops.embedding_backward(dy[0], tok[0], vocab), stream=0)[0]]             # the default stream by its handle
    s.wait_stream(torch.cuda.current_stream())
    got += [ops.run(ops.embedding_backward(dy[i % 2], tok[i % 2], vocab), stream=s)[0] for i in range(4)]
    got += [ops.run(ops.embedding_backward(dy[0], tok[0], vocab), stream=s.cuda_stream)[0]]
    filler = [torch.full((1 << 20,), 7.0, device=cuda) for _ in range(8)]                # would reuse freed workspaces
    s.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for g, i in zip(got, (0, 0, 1, 0, 1, 0))) and len(filler) == 8


def test_run_on_a_stream_that_is_late(cuda):
    """An op built on one stream and run where another is current: its workspace is not given away before that one is done."""
    n, vocab, cols = 30000, 3000, 256
    tok, dy = torch.randint(0, vocab, (n,), generator=gen(90)).to(cuda), rand((n, cols), 91).to(cuda)
    want = ops.run(ops.embedding_backward(dy, tok, vocab))[0].clone()
    busy = torch.randn((4096, 4096), device=cuda)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    op = ops.embedding_backward(dy, tok, vocab)
    size = op.keep[-1].numel()
    with torch.cuda.stream(s):
        for _ in range(20):
            busy = torch.tanh(busy @ busy)
        (got,) = ops.run(op)
    del op
    junk = [torch.full((size,), 255, device=cuda, dtype=torch.uint8) for _ in range(3)]    # runs at once, next to the busy stream
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all((j == 255).all() for j in junk)


def test_operators_refuse_what_does_not_fit(cuda):
    x, w = torch.zeros((4, 8), device=cuda), torch.ones(8, device=cuda)
    t = torch.zeros(4, dtype=torch.int64, device=cuda)
    m = torch.zeros(4, device=cuda)
    cases = [
        (TypeError, lambda: ops.layer_norm(x.double(), 8)), (ValueError, lambda: ops.layer_norm(x, 4)),
        (ValueError, lambda: ops.layer_norm(x, (2, 4, 8))), (ValueError, lambda: ops.layer_norm(x, ())),
        (ValueError, lambda: ops.layer_norm(x, 8, w[:4])), (TypeError, lambda: ops.layer_norm(x, 8, w.half())),
        (TypeError, lambda: ops.layer_norm(x.half(), 8, w.half(), w)), (TypeError, lambda: ops.layer_norm(x, 8, w.cpu())),
        (ValueError, lambda: ops.layer_norm(x, 8, w, None, -1.0)), (ValueError, lambda: ops.layer_norm(x, 8, w, None, float("nan"))),
        (ValueError, lambda: ops.layer_norm(x[:, :0], 0)),
        (ValueError, lambda: ops.layer_norm_backward(x[:2], x, 8, m, m)), (ValueError, lambda: ops.layer_norm_backward(x.half(), x, 8, m, m)),
        (ValueError, lambda: ops.layer_norm_backward(x, x, 8, m[:3], m)), (TypeError, lambda: ops.layer_norm_backward(x, x, 8, m.half(), m)),
        (ValueError, lambda: ops.layer_norm_backward(x, x, 8, m, m, w, (0, 0, 0))), (ValueError, lambda: ops.layer_norm_backward(x, x, 8, m, m, w, (1, 1))),
        (TypeError, lambda: ops.embedding(t.short(), x)), (TypeError, lambda: ops.embedding(t, x.int())), (TypeError, lambda: ops.embedding(t.cpu(), x)),
        (ValueError, lambda: ops.embedding(t, w)), (ValueError, lambda: ops.embedding(t, x, float("inf"))), (ValueError, lambda: ops.embedding(t, x[:0])),
        (ValueError, lambda: ops.embedding_backward(x, t[:3], 9)), (ValueError, lambda: ops.embedding_backward(x, t, 0)),
        (ValueError, lambda: ops.embedding_backward(x, t, 9, padding_idx=9)), (ValueError, lambda: ops.embedding_backward(x, t, 9, padding_idx=-1)),
        (TypeError, lambda: ops.embedding_backward(x, t, 9, dtype=torch.float16)), (ValueError, lambda: ops.embedding_backward(x, t, 9, float("nan"))),
    ]
    for error, make in cases:
        with pytest.raises(error):
            make()
    with pytest.raises(KeyError):       # no fusion list names them
        ops.run_fused(ops.layer_norm(x, 8), ops.embedding(t, x))


def test_c_interface_without_optional_outputs(cuda):
    """The statistics are optional for serving; the argument builders take [rows, cols] tensors."""
    x, w = rand((5, 72), 80, torch.bfloat16), rand((72,), 81)
    xd, y = x.to(cuda), torch.empty((5, 72), device=cuda, dtype=torch.bfloat16)
    H.launch_native("layer_norm_forward", H.layer_norm_args(xd, y, w.to(cuda), eps=1e-5))
    torch.cuda.synchronize()
    want, _, _, tol, _, _ = norm64(x, w, None, 1e-5)
    check(y, want, tol + half(y.dtype) * (want.abs() + tol) + floor(y.dtype), "y")
