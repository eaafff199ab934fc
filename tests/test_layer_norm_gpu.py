"""Layer norm, forward and backward, against its formulas in 64 bits.

Tolerances, with u = 2^-24 and h half a step of the result's type (2^-24 or 2^-8): a sum of n f32 values that are added in
runs of at most r and then as a tree is off by at most (r + 20) u sum|x|, and every other operation by u of its result.  r is
at most n / 32 for the kernels' 32 or more partial sums of a row, and rows / 8 + 8 for a column's.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import autograph_b200 as ag

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]
EPS = 1e-5


def _rand(shape, seed, scale=1.0, shift=0.0):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape) * scale + shift)


def _inputs(dev, rows, cols, dtype, seed=0, shift=0.3):
    """x, weight, bias, dy on the device in the type of the test."""
    return [t.to(dtype).to(dev.torch_device) for t in (
        _rand((rows, cols), seed, 1.5, shift), _rand(cols, seed + 1, 0.2, 1.0), _rand(cols, seed + 2, 0.3),
        _rand((rows, cols), seed + 3, 0.7))]


def _forward64(x, w, b, eps=EPS):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    hat = (x - mean) * rstd
    y = hat * (1 if w is None else w.double()) + (0 if b is None else b.double())
    return y, mean[:, 0], rstd[:, 0], hat


def _check_forward(x, w, b, y, mean, rstd, eps=EPS):
    n = x.shape[1]
    ey, emean, erstd, hat = _forward64(x, w, b, eps)
    size = x.double().abs().mean(1)
    off_mean = (n / 32 + 22) * U * size
    assert ((mean.double() - emean).abs() <= off_mean + 1e-45).all()
    # the variance: its own sum, and the mean's error squared
    rel_var = (n / 32 + 24) * U + (off_mean * erstd).square() + 2 * off_mean * erstd
    assert ((rstd.double() - erstd).abs() <= erstd * (rel_var + 4 * U)).all()
    aw = torch.ones(n, device=x.device).double() if w is None else w.double().abs()
    ab = torch.zeros(n, device=x.device).double() if b is None else b.double().abs()
    off = ((off_mean * erstd)[:, None] + U * (x.double() * erstd[:, None]).abs() + hat.abs() * (rel_var[:, None] + 8 * U)) * aw
    off += 2 * U * (ab + (hat * aw).abs()) + HALF[y.dtype] * ey.abs()
    assert ((y.double() - ey).abs() <= off * 1.01 + 1e-45).all()


def _backward64(x, w, mean, rstd, dy):
    x, dy, mean, rstd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    hat = (x - mean) * rstd
    d = dy if w is None else dy * w.double()
    dx = rstd * (d - d.mean(1, keepdim=True) - hat * (d * hat).mean(1, keepdim=True))
    return dx, (dy * hat).sum(0), dy.sum(0), hat, d


def _check_backward(x, w, mean, rstd, dy, dx, dw, db):
    rows, n = x.shape
    ex, ew, eb, hat, d = _backward64(x, w, mean, rstd, dy)
    r = rstd.double()[:, None]
    off_hat = U * ((x.double() * r).abs() + (mean.double()[:, None] * r).abs() + 2 * hat.abs())
    if dx is not None:
        run = (n / 32 + 24) * U
        off_along = run * d.abs().mean(1, keepdim=True)
        off_across = run * (d * hat).abs().mean(1, keepdim=True) + (d.abs() * off_hat).mean(1, keepdim=True)
        across = (d * hat).mean(1, keepdim=True).abs()
        off = r * (6 * U * (d.abs() + d.mean(1, keepdim=True).abs() + hat.abs() * across) + off_along + hat.abs() * off_across +
                   off_hat * across)
        assert ((dx.double() - ex).abs() <= off * 1.01 + HALF[dx.dtype] * ex.abs() + 1e-45).all()
    run = (rows / 8 + 40) * U
    if dw is not None:
        off = run * (dy.double() * hat).abs().sum(0) + (dy.double().abs() * off_hat).sum(0)
        assert ((dw.double() - ew).abs() <= off * 1.01 + HALF[dw.dtype] * ew.abs() + 1e-45).all()
    if db is not None:
        off = run * dy.double().abs().sum(0)
        assert ((db.double() - eb).abs() <= off * 1.01 + HALF[db.dtype] * eb.abs() + 1e-45).all()


SIZES = [(1, 1), (1, 2), (3, 1), (5, 3), (1, 84), (100, 84), (7, 31), (9, 33), (33, 64), (257, 129), (64, 255), (17, 256),
         (31, 257), (40, 512), (13, 1000), (300, 1021), (11, 1024), (5, 2011), (6, 4096), (3, 8200), (2, 16384), (150, 8192),
         (9, 25088), (1, 32768), (2, 40001), (1, 70001), (1, 300000), (2000, 10), (5000, 24), (4097, 128)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_both_directions(dev, rows, cols, dtype):
    x, w, b, dy = _inputs(dev, rows, cols, dtype, seed=rows * 7 + cols)
    y, mean, rstd = dev.layer_norm_keep(x, w, b, eps=EPS)
    _check_forward(x, w, b, y, mean, rstd)
    dx, dw, db = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
    _check_backward(x, w, mean, rstd, dy, dx, dw, db)
    assert torch.equal(y, dev.layer_norm(x, w, b, eps=EPS))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(20000, 1), (30001, 2), (8192, 3), (12345, 5), (60000, 8), (65536, 16)])
def test_many_short_rows(dev, rows, cols, dtype):
    """The column sums come from every thread block there is room for."""
    x, w, b, dy = _inputs(dev, rows, cols, dtype, seed=rows + cols)
    y, mean, rstd = dev.layer_norm_keep(x, w, b, eps=EPS)
    _check_forward(x, w, b, y, mean, rstd)
    grads = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
    _check_backward(x, w, mean, rstd, dy, *grads)
    again = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(100, 84), (65, 1021), (3, 25088)])
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(dev, rows, cols, dtype, has_w, has_b):
    x, w, b, dy = _inputs(dev, rows, cols, dtype, seed=5)
    w, b = w if has_w else None, b if has_b else None
    y, mean, rstd = dev.layer_norm_keep(x, w, b)
    _check_forward(x, w, b, y, mean, rstd)
    dx, dw, db = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=has_b)
    _check_backward(x, w, mean, rstd, dy, dx, dw, db)
    assert (dw is None) == (not has_w) and (db is None) == (not has_b)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [84, 1024, 25088])
def test_parts_of_the_backward_pass(dev, cols, dtype):
    """Each gradient alone has the bits that it has with the others."""
    x, w, b, dy = _inputs(dev, 50, cols, dtype, seed=11)
    _, mean, rstd = dev.layer_norm_keep(x, w, b)
    dx, dw, db = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
    assert torch.equal(dx, dev.layer_norm_backward(x, dy, mean, rstd, w)[0])
    none, dw2, db2 = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True, want_dx=False)
    assert none is None and torch.equal(dw, dw2) and torch.equal(db, db2)
    out = torch.empty_like(db)
    code = ag._capi.AG_F32 if dtype == torch.float32 else ag._capi.AG_BF16
    ag._capi.check(ag.lib().ag_layer_norm_backward(
        dev._h, code, x.data_ptr(), None, mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), 50, cols, None, 0.0, None,
        out.data_ptr()))
    assert torch.equal(out, db)
    ag._capi.check(ag.lib().ag_layer_norm_backward(
        dev._h, code, x.data_ptr(), None, mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), 50, cols, None, 0.0,
        out.data_ptr(), None))
    assert torch.equal(out, dw)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(7, 40), (130, 1024), (65, 1021), (4, 25088)])
def test_rows_off_sixteen_bytes(dev, rows, cols, dtype):
    """Operands that start one value behind an aligned address."""
    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)
    x, w, b, dy = [moved(t) for t in _inputs(dev, rows, cols, dtype, seed=21)]
    y, mean, rstd = dev.layer_norm_keep(x, w, b)
    _check_forward(x, w, b, y, mean, rstd)
    dx, dw, db = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
    _check_backward(x, w, mean, rstd, dy, dx, dw, db)
    # and one operand alone: which columns a thread takes, and so the order of a row's sums, goes by the alignment of all
    for operands in ((x.clone(), w, b), (x, w.clone(), b.clone()), (x.clone(), w.clone(), b.clone())):
        y, mean, rstd = dev.layer_norm_keep(*operands)
        _check_forward(*operands, y, mean, rstd)
    dx, dw, db = dev.layer_norm_backward(x.clone(), dy, mean, rstd, w, has_bias=True)
    _check_backward(x, w, mean, rstd, dy, dx, dw, db)


@gpu
def test_strided_and_shaped_operands(dev):
    x, w, b, dy = _inputs(dev, 24, 60, torch.float32, seed=31)
    want = dev.layer_norm(x.t().contiguous().t(), w, b)
    assert torch.equal(dev.layer_norm(x, w, b), want)
    cube = x.view(2, 12, 5, 12)
    y, mean, rstd = dev.layer_norm_keep(cube, w.view(5, 12), b.view(5, 12))
    assert y.shape == cube.shape and mean.shape == (2, 12) == rstd.shape
    assert torch.equal(y.view(24, 60), want)
    dx, dw, db = dev.layer_norm_backward(cube, dy.view(2, 12, 5, 12), mean, rstd, w.view(5, 12), has_bias=True)
    flat = dev.layer_norm_backward(x, dy, mean.reshape(-1), rstd.reshape(-1), w, has_bias=True)
    assert all(torch.equal(a.reshape(-1), c.reshape(-1)) for a, c in zip((dx, dw, db), flat))
    assert dw.shape == (5, 12) == db.shape
    assert torch.equal(dev.layer_norm(x), dev.layer_norm(x, shape=(60,)))
    assert dev.layer_norm(x.view(24, 5, 12), shape=(5, 12)).shape == (24, 5, 12)
    assert torch.equal(dev.layer_norm(x.view(24, 5, 12), shape=(5, 12)).view(24, 60), dev.layer_norm(x))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [100, 1024, 3000, 25088])
def test_no_rows(dev, cols, dtype):
    x = torch.empty((0, cols), dtype=dtype, device=dev.torch_device)
    w = torch.ones(cols, dtype=dtype, device=dev.torch_device)
    y, mean, rstd = dev.layer_norm_keep(x, w, w)
    assert y.shape == (0, cols) and mean.shape == (0,)
    dx, dw, db = dev.layer_norm_backward(x, x, mean, rstd, w, has_bias=True)
    assert dx.shape == (0, cols) and not dw.any() and not db.any()
    dw.fill_(3), db.fill_(-2)
    dev.layer_norm_backward(x, x, mean, rstd, w, has_bias=True, beta=0.5, dweight=dw, dbias=db)
    assert (dw == 1.5).all() and (db == -1).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(100, 84), (513, 1024), (40, 8200)])
def test_gradients_accumulate(dev, rows, cols, dtype):
    x, w, b, dy = _inputs(dev, rows, cols, dtype, seed=41)
    _, mean, rstd = dev.layer_norm_keep(x, w, b)
    _, dw, db = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
    old_w, old_b = _rand(cols, 1).to(dtype).to(x.device), _rand(cols, 2).to(dtype).to(x.device)
    got_w, got_b = old_w.clone(), old_b.clone()
    dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True, beta=1.0, dweight=got_w, dbias=got_b)
    _, ew, eb, hat, _ = _backward64(x, w, mean, rstd, dy)
    for got, old, e, size in ((got_w, old_w, ew, (dy.double() * hat).abs().sum(0)), (got_b, old_b, eb, dy.double().abs().sum(0))):
        want = e + old.double()
        # the f32 sum's own error, as in _check_backward, and the last addition's
        off = (rows / 8 + 60) * U * size + 2 * U * old.double().abs() + HALF[dtype] * want.abs()
        assert ((got.double() - want).abs() <= off * 1.01).all()
    # beta = 0 does not read what was there
    nan_w, nan_b = torch.full_like(dw, float("nan")), torch.full_like(db, float("nan"))
    dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True, dweight=nan_w, dbias=nan_b)
    assert torch.equal(nan_w, dw) and torch.equal(nan_b, db)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [84, 1024, 4100, 25088])
def test_values_that_are_not_finite_stay_in_their_row(dev, cols, dtype):
    rows = 37
    x, w, b, dy = _inputs(dev, rows, cols, dtype, seed=51)
    clean, cm, cr = dev.layer_norm_keep(x, w, b)
    x2 = x.clone()
    x2[3, cols // 2], x2[20, 0], x2[36, cols - 1] = float("nan"), float("inf"), -float("inf")
    y, mean, rstd = dev.layer_norm_keep(x2, w, b)
    keep = [r for r in range(rows) if r not in (3, 20, 36)]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(mean[keep], cm[keep]) and torch.equal(rstd[keep], cr[keep])
    assert y[[3, 20, 36]].isnan().all()
    dx, dw, db = dev.layer_norm_backward(x2, dy, mean, rstd, w, has_bias=True)
    dx0, _, db0 = dev.layer_norm_backward(x, dy, cm, cr, w, has_bias=True)
    assert torch.equal(dx[keep], dx0[keep]) and dx[3].isnan().all() and torch.equal(db, db0) and dw.isnan().all()
    # a gradient that is not finite: its row of dx, its column of the sums
    dy2 = dy.clone()
    dy2[5, 1 % cols] = float("inf")
    dx, dw, db = dev.layer_norm_backward(x, dy2, cm, cr, w, has_bias=True)
    others = [c for c in range(cols) if c != 1 % cols]
    _, dw0, _ = dev.layer_norm_backward(x, dy, cm, cr, w, has_bias=True)
    assert torch.equal(dw[others], dw0[others]) and torch.equal(db[others], db0[others]) and db[1 % cols] == float("inf")
    rest = [r for r in range(rows) if r != 5]
    assert torch.equal(dx[rest], dx0[rest]) and not dx[5].isfinite().any()


@gpu
@pytest.mark.parametrize("cols", [64, 1000, 4096, 25088])
def test_constant_rows_and_far_means(dev, cols):
    x = torch.full((4, cols), 3.25, device=dev.torch_device)
    y, mean, rstd = dev.layer_norm_keep(x)
    assert not y.any() and (mean == 3.25).all()
    assert ((rstd.double() - EPS ** -0.5).abs() <= 4 * U * EPS ** -0.5 + U * EPS ** -0.5).all()
    # a mean a thousand deviations away costs the rounding of the mean and no more: the variance is a sum of squared
    # differences, not a difference of sums
    far = _rand((5, cols), 3, 1.0, 1000.0).float().to(dev.torch_device)
    y, mean, rstd = dev.layer_norm_keep(far)
    _check_forward(far, None, None, y, mean, rstd)
    assert (rstd > 0.8).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [5, 84, 1000, 2011, 4096, 8190, 25088, 70001])
def test_rows_of_one_value(dev, cols, dtype):
    """Values of full mantissas, whose sums are rounded.  A first mean m is off by at most (cols / 32 + 22) u of c, so that
    c - m is exact; the mean of these equal differences is off by the same share of them, less than u / 4 of c, and added to
    m gives c.  The variance is then zero up to that share of (c - m)^2."""
    c = torch.cat([torch.tensor([1000.1, 1 / 3, 1234.567, -777.77, 1e-3, 3e7]),
                   500 + 1500 * torch.rand(58, generator=torch.Generator().manual_seed(cols))])
    x = c.to(dtype).to(dev.torch_device)[:, None].expand(64, cols).contiguous()
    _, w, b, _ = _inputs(dev, 1, cols, dtype, seed=91)
    y, mean, rstd = dev.layer_norm_keep(x, w, b)
    assert torch.equal(mean, x[:, 0].float()) and torch.equal(y, b.expand(64, cols))
    run = (cols / 32 + 24) * U
    var = 4 * run * (run * x[:, 0].double()).square()
    want = 1 / math.sqrt(EPS)
    assert ((rstd.double() - want).abs() <= want * (4 * U + var / EPS / 2)).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(9, 84), (9, 1000), (9, 2011), (5, 25088), (3, 70001)])
@pytest.mark.parametrize("shift", [0.0, 30.0, 1000.1])
def test_far_means_are_rounded_once(dev, rows, cols, dtype, shift):
    """The mean is off by its own rounding, that of the differences it is put right by (u of each) and that of their sum,
    (cols / 32 + 24) u of their size, however far it is.  A first mean m that is off by q = (cols / 32 + 22) u |mean| adds
    q to the differences."""
    x = _rand((rows, cols), 7, 1.0, shift).to(dtype).to(dev.torch_device)
    y, mean, rstd = dev.layer_norm_keep(x)
    _check_forward(x, None, None, y, mean, rstd)
    x = x.double()
    exact = x.mean(1)
    spread = (x - exact[:, None]).abs().mean(1) + (cols / 32 + 22) * U * x.abs().mean(1)
    assert ((mean.double() - exact).abs() <= U * exact.abs() + (cols / 32 + 25) * U * spread + 1e-45).all()


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12])
def test_small_and_large_values(dev, scale):
    x = (_rand((9, 500), 8) * scale).float().to(dev.torch_device)
    y, mean, rstd = dev.layer_norm_keep(x)
    _check_forward(x, None, None, y, mean, rstd)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(100, 84), (600, 1021), (5, 25088), (2, 70001)])
def test_in_place_and_again(dev, rows, cols, dtype):
    x, w, b, dy = _inputs(dev, rows, cols, dtype, seed=61)
    y, mean, rstd = dev.layer_norm_keep(x, w, b)
    first = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
    for _ in range(3):
        again = dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
        assert all(torch.equal(a, c) for a, c in zip(first, again))
    z = x.clone()
    code = ag._capi.AG_F32 if dtype == torch.float32 else ag._capi.AG_BF16
    ag._capi.check(ag.lib().ag_layer_norm_forward(dev._h, code, z.data_ptr(), w.data_ptr(), b.data_ptr(), rows, cols,
                                                  ctypes.c_float(EPS), z.data_ptr(), None, None))
    assert torch.equal(z, y)


@gpu
def test_gradients_are_the_differences_of_the_values(dev):
    """The loss sum(c * layer_norm(x)) moved along random directions, in 64 bits, against the kernel's f32 gradients."""
    x, w, b, c = _inputs(dev, 6, 50, torch.float32, seed=71)
    _, mean, rstd = dev.layer_norm_keep(x, w, b)
    grads = dev.layer_norm_backward(x, c, mean, rstd, w, has_bias=True)
    loss = lambda x, w, b: (_forward64(x, w, b)[0] * c.double()).sum()
    args = [x.double(), w.double(), b.double()]
    h = 1e-5
    for i, g in enumerate(grads):
        d = _rand(tuple(args[i].shape), 100 + i).to(x.device)
        up, down = [list(args), list(args)]
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        slope = (loss(*up) - loss(*down)) / (2 * h)
        got = (g.double() * d).sum()
        # f32 gradients (a few u of the terms) and differences good to about h^2
        assert abs(got - slope) <= 1e-5 * (g.double() * d).abs().sum() + 1e-7


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_another_stream_and_a_graph(dev, dtype):
    """Inputs made on another stream; a captured pass replayed on new values, next to eager calls that use the workspace."""
    dev.set_guards(False)
    side = torch.cuda.Stream()
    side.wait_stream(dev.stream)
    with torch.cuda.stream(side):
        x, w, b, dy = _inputs(dev, 700, 1024, dtype, seed=81)
        y, mean, rstd = dev.layer_norm_keep(x, w, b)
    torch.cuda.synchronize()
    _check_forward(x, w, b, y, mean, rstd)
    torch.cuda.set_stream(dev.stream)
    dev.layer_norm_backward(x, dy, mean, rstd, w, has_bias=True)
    dev.wait()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=dev.stream):
        gy, gm, gr = dev.layer_norm_keep(x, w, b)
        grads = dev.layer_norm_backward(x, dy, gm, gr, w, has_bias=True)
    big = _inputs(dev, 3000, 2048, dtype, seed=82)
    for seed in (83, 84):
        x.copy_(_inputs(dev, 700, 1024, dtype, seed=seed)[0])
        dev.layer_norm_backward(big[0], big[3], torch.zeros(3000, device=x.device), torch.ones(3000, device=x.device), big[1],
                                has_bias=True)
        graph.replay()
        dev.wait()
        _check_forward(x, w, b, gy, gm, gr)
        _check_backward(x, w, gm, gr, dy, *grads)
    del graph


@gpu
def test_many_rows(dev):
    """More values than 32 bits count (bf16): the last rows have the values of a call of their own."""
    rows, cols = (1 << 22) + 3, 520
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=dev.torch_device)
    x[:] = _rand((1, cols), 1).to(torch.bfloat16).to(x.device)
    x[-5:] = _rand((5, cols), 2).to(torch.bfloat16).to(x.device)
    dev.set_guards(False)
    y, mean, rstd = dev.layer_norm_keep(x)
    dx, _, _ = dev.layer_norm_backward(x, x, mean, rstd)
    y5, m5, r5 = dev.layer_norm_keep(x[-5:].clone())
    dx5, _, _ = dev.layer_norm_backward(x[-5:].clone(), x[-5:].clone(), m5, r5)
    assert torch.equal(y[-5:], y5) and torch.equal(mean[-5:], m5) and torch.equal(dx[-5:], dx5)
    assert torch.equal(y[0], y[rows - 6]) and torch.equal(dx[0], dx[rows - 6])


@gpu
def test_refusals(dev):
    x = torch.ones((4, 8), device=dev.torch_device)
    w = torch.ones(8, device=dev.torch_device)
    m = torch.ones(4, device=dev.torch_device)
    cases = [
        (ag._capi.AG_ERR_SHAPE, lambda: dev.layer_norm(x, w[:7])),
        (ag._capi.AG_ERR_SHAPE, lambda: dev.layer_norm(x, w, w[:7])),
        (ag._capi.AG_ERR_SHAPE, lambda: dev.layer_norm(x, shape=(4,))),
        (ag._capi.AG_ERR_SHAPE, lambda: dev.layer_norm(x, shape=())),
        (ag._capi.AG_ERR_SHAPE, lambda: dev.layer_norm(x[:, :0])),
        (ag._capi.AG_ERR_DTYPE, lambda: dev.layer_norm(x, w.bfloat16())),
        (ag._capi.AG_ERR_DTYPE, lambda: dev.layer_norm(x.half())),
        (ag._capi.AG_ERR_DTYPE, lambda: dev.layer_norm(x.double())),
        (ag._capi.AG_ERR_INVALID, lambda: dev.layer_norm(x, eps=0.0)),
        (ag._capi.AG_ERR_INVALID, lambda: dev.layer_norm(x, eps=-1e-5)),
        (ag._capi.AG_ERR_INVALID, lambda: dev.layer_norm(x, eps=float("nan"))),
        (ag._capi.AG_ERR_INVALID, lambda: dev.layer_norm(x, eps=float("inf"))),
        (ag._capi.AG_ERR_INVALID, lambda: dev.layer_norm(x.cpu())),
        (ag._capi.AG_ERR_INVALID, lambda: dev.layer_norm(x, w.cpu())),
        (ag._capi.AG_ERR_SHAPE, lambda: dev.layer_norm_backward(x, x[:2], m, m)),
        (ag._capi.AG_ERR_SHAPE, lambda: dev.layer_norm_backward(x, x, m[:3], m)),
        (ag._capi.AG_ERR_DTYPE, lambda: dev.layer_norm_backward(x, x, m.double(), m)),
        (ag._capi.AG_ERR_DTYPE, lambda: dev.layer_norm_backward(x, x.bfloat16(), m, m)),
        (ag._capi.AG_ERR_SHAPE, lambda: dev.layer_norm_backward(x, x, m, m, w, dweight=w[:7])),
        (ag._capi.AG_ERR_DTYPE, lambda: dev.layer_norm_backward(x, x, m, m, w, dweight=w.bfloat16())),
        (ag._capi.AG_ERR_INVALID, lambda: dev.layer_norm_backward(x, x, m, m, w, beta=1.0)),
        (ag._capi.AG_ERR_INVALID, lambda: dev.layer_norm_backward(x, x, m, m, w, dweight=torch.ones(16, device=x.device)[::2])),
    ]
    for status, call in cases:
        with pytest.raises(ag.AgError) as err:
            call()
        assert err.value.status == status
    # the C entries themselves: overlapping results, missing operands, bad sizes
    f, b, p = ag.lib().ag_layer_norm_forward, ag.lib().ag_layer_norm_backward, lambda t: t.data_ptr()
    inv, shape, dt = ag._capi.AG_ERR_INVALID, ag._capi.AG_ERR_SHAPE, ag._capi.AG_ERR_DTYPE
    flat = torch.ones(64, device=dev.torch_device)
    assert f(dev._h, 0, None, None, None, 4, 8, EPS, p(x), None, None) == inv
    assert f(dev._h, 0, p(x), None, None, 4, 8, EPS, None, None, None) == inv
    assert f(dev._h, 0, p(x), None, None, -1, 8, EPS, p(x), None, None) == shape
    assert f(dev._h, 0, p(x), None, None, 4, 0, EPS, p(x), None, None) == shape
    assert f(dev._h, 0, p(x), None, None, 1 << 40, 1 << 40, EPS, p(x), None, None) == shape
    assert f(dev._h, 2, p(x), None, None, 4, 8, EPS, p(x), None, None) == dt
    assert f(dev._h, 0, p(flat), None, None, 4, 8, EPS, p(flat) + 16, None, None) == inv
    assert b(dev._h, 0, p(x), None, None, p(m), p(x), 4, 8, p(flat), 0.0, None, None) == inv
    assert b(dev._h, 0, p(x), None, p(m), p(m), p(flat), 4, 8, p(flat), 0.0, None, None) == inv
    assert b(dev._h, 0, p(flat), None, p(m), p(m), p(x), 4, 8, p(flat) + 64, 0.0, None, None) == inv
    assert b(dev._h, 0, p(x), None, p(m), p(m), p(x), 4, 8, None, 0.0, p(flat), p(flat) + 16) == inv
    assert b(dev._h, 0, p(x), None, p(m), p(m), p(x), 4, 8, p(flat), 0.0, p(flat) + 64, None) == inv
    assert b(dev._h, 0, p(x), None, p(m), p(m), p(x), 4, 8, None, 0.0, None, None) == 0   # nothing asked for


@gpu
def test_results_that_overlap_operands_are_refused(dev):
    """Rows are written while the operands of others are still read.  Nothing is launched: the operands keep their values."""
    f, b, inv = ag.lib().ag_layer_norm_forward, ag.lib().ag_layer_norm_backward, ag._capi.AG_ERR_INVALID
    store = torch.ones(400, device=dev.torch_device)
    p = lambda i: store.data_ptr() + 4 * i
    # [4, 8] x at 0, y at 40, weight at 80, bias at 90, mean at 100, rstd at 110, apart from each other
    at = dict(x=0, y=40, weight=80, bias=90, mean=100, rstd=110)
    size = dict(x=32, y=32, weight=8, bias=8, mean=4, rstd=4)

    def forward(**moved):
        a = {**at, **moved}
        return f(dev._h, 0, p(a["x"]), p(a["weight"]), p(a["bias"]), 4, 8, EPS, p(a["y"]), p(a["mean"]), p(a["rstd"]))
    for result in ("y", "mean", "rstd"):
        for other in at:
            if other == result:
                continue
            # on its last value, and with the result's last value on its first
            places = [at[other] + size[other] - 1, at[other] - size[result] + 1]
            for place in places:
                if place >= 0:
                    assert forward(**{result: place}) == inv, (result, other, place)
    assert forward(y=1) == inv
    at = dict(x=0, dy=40, weight=80, mean=100, rstd=110, dx=120, dweight=160, dbias=170)
    size = dict(x=32, dy=32, weight=8, mean=4, rstd=4, dx=32, dweight=8, dbias=8)

    def backward(**moved):
        a = {**at, **moved}
        return b(dev._h, 0, p(a["x"]), p(a["weight"]), p(a["mean"]), p(a["rstd"]), p(a["dy"]), 4, 8, p(a["dx"]), 0.0,
                 p(a["dweight"]), p(a["dbias"]))
    for result in ("dx", "dweight", "dbias"):
        for other in at:
            if other == result:
                continue
            for place in (at[other] + size[other] - 1, at[other] - size[result] + 1):
                if place >= 0:
                    assert backward(**{result: place}) == inv, (result, other, place)
    dev.wait()
    assert (store == 1).all()
    # side by side is no overlap, and y may be x
    at = dict(x=0, y=32, weight=64, bias=72, mean=80, rstd=84)
    assert forward() == 0 and forward(y=0) == 0
    at = dict(x=0, dy=32, weight=64, mean=72, rstd=76, dx=80, dweight=112, dbias=120)
    assert backward() == 0
    dev.wait()


def test_refusals_without_a_device():
    f, b = ag.lib().ag_layer_norm_forward, ag.lib().ag_layer_norm_backward
    assert f(None, 0, None, None, None, 4, 8, EPS, None, None, None) == ag._capi.AG_ERR_INVALID
    assert b(None, 0, None, None, None, None, None, 4, 8, None, 0.0, None, None) == ag._capi.AG_ERR_INVALID
