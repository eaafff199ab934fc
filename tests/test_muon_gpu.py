"""Newton-Schulz orthogonalisation and Muon's update against their formulas in 64 bits.

Tolerances, as 2-norms relative to the result, with u = 2^-24.  A sum of m f32 products in one chain is off by at most m u of
its terms, and, the roundings being independent of each other, by about sqrt(m) u: a step x -> A x + (B a + C a a) x with
a = x x^T perturbs x by (8 + 2 sqrt(m)) u of its norm (the two sums whose errors reach x in first order, and 8 u for the
operations around them).  A perturbation grows by at most A = 3.4445 in every later step, so that five steps add up to
1 + A + ... + A^4 = 198 times that where the values themselves do not grow (a rank-deficient matrix, whose few singular values
are near one from the start).  Where they grow along, within a factor of some ten of each other, it is five times that and the
few units of their condition: 2e-5 is allowed at every size here.
A bf16 result is off by half a step, 2^-8, of its elements, and its computation by at most half of that again.
"""
import math

import numpy as np
import pytest
import torch

import autograph_b200 as ag

gpu = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315
F32, BF16 = torch.float32, torch.bfloat16
DTYPES, IDS = [F32, BF16], ["f32", "bf16"]
U = 2.0 ** -24


def _polar64(g, steps=5):
    x = g.double()
    norm = x.norm()
    x = x / norm if norm > 0 else x
    flip = g.shape[0] > g.shape[1]
    x = x.T if flip else x
    for _ in range(steps):
        a = x @ x.T
        x = A * x + (B * a + C * (a @ a)) @ x
    return x.T if flip else x


def _rand(shape, seed, scale=1.0):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape) * scale)


def _gradient(rows, cols, seed, batch=None):
    """Activations behind a Relu times output gradients: one singular value far above the others."""
    r = np.random.default_rng(seed)
    batch = batch or 3 * min(rows, cols) + 16
    x = np.maximum(r.standard_normal((batch, rows)), 0)
    return torch.from_numpy(x.T @ r.standard_normal((batch, cols)) / batch)


def _tol(dtype, full_rank=True, m=0):
    return (2e-5 if full_rank else 198 * (8 + 2 * math.sqrt(m)) * U) if dtype == F32 else 1.5 * 2.0 ** -8


def _close(got, want, dtype, full_rank=True):
    want = want.to(got.device)
    off = (got.double() - want).norm() / want.norm()
    assert off <= _tol(dtype, full_rank, max(got.shape)), f"{tuple(got.shape)}: {off:.2e}"


SIZES = [(1, 1), (1, 2), (2, 1), (1, 300), (777, 1), (2, 3), (5, 7), (6, 25), (16, 150), (150, 16), (84, 10), (128, 84),
         (256, 128), (64, 27), (128, 576), (127, 129), (128, 128), (129, 128), (130, 257), (255, 64), (256, 256), (257, 300),
         (63, 2000), (2000, 65), (384, 640), (512, 512), (300, 1100), (1100, 300), (513, 1025), (777, 1009), (1024, 768)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_one_matrix(dev, rows, cols, dtype):
    for g in (_rand((rows, cols), rows + cols), _gradient(rows, cols, rows * 3 + cols)):
        g = g.to(dtype).to(dev.torch_device)
        o, = dev.newton_schulz([g])
        assert o.shape == g.shape and o.dtype == dtype
        # square gaussians have singular values down to 1 / n of the largest
        _close(o, _polar64(g), dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols,seed", [(2048, 2048, 1), (1500, 4100, 2), (25088, 512, 3), (200, 30000, 4), (4096, 1024, 5)])
def test_large_matrices(dev, rows, cols, seed, dtype):
    gen = torch.Generator("cuda").manual_seed(seed)
    n = min(rows, cols)
    x = torch.randn((3 * n, rows), generator=gen, device=dev.torch_device, dtype=torch.float64).relu_()
    g = (x.T @ torch.randn((3 * n, cols), generator=gen, device=dev.torch_device, dtype=torch.float64)).to(dtype)
    del x
    o, = dev.newton_schulz([g])
    _close(o, _polar64(g), dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_list_of_matrices(dev, dtype):
    """Matrices of all sizes in one call.  How many thread blocks share a matrix goes by the whole call, and the order of its
    sums with it: the same call has the same bits again, a matrix alone has those of its own call."""
    gs = [_gradient(r, c, i).to(dtype).to(dev.torch_device) for i, (r, c) in enumerate(SIZES)]
    together = dev.newton_schulz(gs)
    for g, o, again in zip(gs, together, dev.newton_schulz(gs)):
        assert torch.equal(o, again)
        _close(o, _polar64(g), dtype)
    many = [_rand((3, 5), i).to(dtype).to(dev.torch_device) for i in range(100)]
    for g, o in zip(many, dev.newton_schulz(many)):
        _close(o, _polar64(g), dtype)
    assert dev.newton_schulz([]) == []


@gpu
def test_a_list_larger_than_one_workspace(dev):
    """Matrices whose planes together are beyond the 4 GiB that a launch takes go in several."""
    dev.set_guards(False)
    g = torch.randn((4096, 8192), device=dev.torch_device, generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    want, = dev.newton_schulz([g])
    outs = dev.newton_schulz([g] * 9 + [g[:100, :200].contiguous()])
    assert all(torch.equal(o, want) for o in outs[:8])
    _close(outs[9], _polar64(g[:100, :200]), BF16)
    _close(want[:, :64].contiguous(), _polar64(g)[:, :64], BF16)


@gpu
def test_a_list_without_memory_for_its_last_matrix_changes_nothing(dev):
    """33 matrices go in two launches, of which the second's workspace of 3 GB is not to be had: the first one's matrices keep
    their weights and momenta too."""
    dev.set_guards(False)
    sizes = [(3, 5)] * 32 + [(8192, 16384)]
    own = ag.Device(0)   # a device object whose workspace has not grown
    torch.cuda.set_stream(own.stream)
    w, g = [[torch.ones(s, device=own.torch_device, dtype=BF16) for s in sizes] for _ in range(2)]
    v = [torch.zeros(s, device=own.torch_device) for s in sizes]
    own.wait()
    hog = []
    try:
        hog.append(torch.empty(torch.cuda.mem_get_info()[0] - (2 << 30), dtype=torch.uint8, device=own.torch_device))
        with pytest.raises(ag.AgError) as err:
            own.muon_update(w, g, v, 0.1)
    finally:
        hog.clear()
        torch.cuda.empty_cache()
        torch.cuda.set_stream(dev.stream)
    own.wait()
    assert err.value.status == ag._capi.AG_ERR_OOM
    assert all((t == 1).all() for t in w) and not any(t.any() for t in v)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(40, 60), (300, 200), (200, 1500)])
@pytest.mark.parametrize("steps", [1, 2, 3, 7])
def test_steps(dev, rows, cols, dtype, steps):
    g = _gradient(rows, cols, steps).to(dtype).to(dev.torch_device)
    # each step beyond the fifth adds one more
    want = _polar64(g, steps)
    off = (dev.newton_schulz([g], steps=steps)[0].double() - want).norm() / want.norm()
    assert off <= _tol(dtype) * max(1.0, steps / 5)


def _beside_the_rounding(dev, g, steps):
    """The error of a bf16 result relative to that of the 64-bit result rounded to bf16.  Where the computation's error is
    independent of the rounding's and less than 0.32 of it, this is below 1.05."""
    want = _polar64(g, steps)
    off = (dev.newton_schulz([g], steps=steps)[0].double() - want).norm()
    return off / (want.bfloat16().double() - want).norm()


@gpu
@pytest.mark.parametrize("steps", [1, 5, 8, 10, 20])
@pytest.mark.parametrize("rows,cols,rank", [(128, 128, None), (256, 256, None), (300, 257, None), (1024, 1024, None),
                                            (300, 500, 5), (500, 300, 40)])
def test_bf16_results_are_as_good_as_their_rounding(dev, rows, cols, rank, steps):
    """Products of 22-bit values perturb x by about 1e-7 a step, and its map's slopes (A at zero, -1.6 to 4 around one)
    make that 1e-4 at most in twenty steps: far less than 0.32 of the rounding's 1.65e-3.  What bf16 left of a low rank's zeros
    are singular values of some 1e-4 of the largest, which grow as what rounds them off does."""
    g = _gradient(rows, cols, 7, batch=rank).bfloat16().to(dev.torch_device)
    assert _beside_the_rounding(dev, g, steps) <= 1.05


@gpu
@pytest.mark.parametrize("steps", [5, 9, 20])
@pytest.mark.parametrize("rows,cols,rank", [(1000, 2100, 5), (2000, 4100, 30), (2048, 2048, None)])
def test_long_sums_of_bf16_results(dev, rows, cols, rank, steps):
    """Sums over thousands of values, in pieces of 48 additions that are cut off by up to 2^-23 each: 3e-6 of x a step on
    average, which grows like the roundings to a few 1e-4 in twenty steps."""
    g = _gradient(rows, cols, 7, batch=rank).bfloat16().to(dev.torch_device)
    assert _beside_the_rounding(dev, g, steps) <= 1.05


@gpu
@pytest.mark.parametrize("steps", [3, 5, 6, 7, 8, 9])
@pytest.mark.parametrize("rows,cols,rank", [(500, 1300, 40), (1300, 500, 5), (256, 1300, 1), (512, 2048, 100)])
def test_low_ranks_of_long_matrices(dev, rows, cols, rank, steps):
    """Gradients of few examples in bf16, whose rounding leaves singular values of some 1e-4 of the largest.  f32: no further from
    64 bits than twice the same steps in f32 products, whose errors are of the same kind and size and may lie otherwise."""
    g = _gradient(rows, cols, 7, batch=rank).bfloat16().to(dev.torch_device)
    want = _polar64(g, steps)
    x = g.float().T if rows > cols else g.float()
    x = x / x.norm()
    for _ in range(steps):
        a = x @ x.T
        x = A * x + (B * a + C * (a @ a)) @ x
    plain = ((x.T if rows > cols else x).double() - want).norm()
    off = (dev.newton_schulz([g.float()], steps=steps)[0].double() - want).norm()
    assert off <= 2 * plain
    assert _beside_the_rounding(dev, g, steps) <= 1.05


@gpu
@pytest.mark.parametrize("rows,cols", [(96, 200), (300, 500), (500, 300), (256, 1300)])
@pytest.mark.parametrize("rank", [1, 2, 5, 40])
def test_rank_deficient(dev, rows, cols, rank):
    """Singular values of zero stay near zero: what rounding puts there grows by at most A a step."""
    g = _gradient(rows, cols, rank, batch=rank).float().to(dev.torch_device)
    o, = dev.newton_schulz([g])
    _close(o, _polar64(g), F32, full_rank=False)
    b = g.bfloat16()
    _close(dev.newton_schulz([b])[0], _polar64(b), BF16, full_rank=False)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("power", [0.5, 1.0])
def test_decaying_singular_values(dev, dtype, power):
    r = np.random.default_rng(5)
    u, v = np.linalg.qr(r.standard_normal((256, 256)))[0], np.linalg.qr(r.standard_normal((600, 256)))[0]
    g = torch.from_numpy((u * np.arange(1, 257.0) ** -power) @ v.T).to(dtype).to(dev.torch_device)
    _close(dev.newton_schulz([g])[0], _polar64(g), dtype, full_rank=False)
    _close(dev.newton_schulz([g.T.contiguous()])[0], _polar64(g.T), dtype, full_rank=False)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (7, 5), (100, 300), (300, 300), (260, 2100)])
def test_zeros_and_values_that_are_not_finite(dev, rows, cols, dtype):
    zero = torch.zeros((rows, cols), dtype=dtype, device=dev.torch_device)
    assert not dev.newton_schulz([zero])[0].any()
    good = _gradient(50, 70, 3).to(dtype).to(dev.torch_device)
    clean = dev.newton_schulz([good, _gradient(rows, cols, 1).to(dtype).to(dev.torch_device), zero])
    _close(clean[0], _polar64(good), dtype)
    for bad in (float("nan"), float("inf"), -float("inf")):
        g = _gradient(rows, cols, 1).to(dtype).to(dev.torch_device)
        g[rows // 2, cols - 1] = bad
        o = dev.newton_schulz([good, g, zero])
        assert torch.equal(o[0], clean[0]) and o[1].isnan().all() and not o[2].any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(60, 40), (300, 300), (128, 1024)])
@pytest.mark.parametrize("exponent", [-120, -60, 40, 120])
def test_scale_does_not_matter(dev, rows, cols, dtype, exponent):
    """A power of two on the gradient changes nothing: sums of squares neither overflow nor vanish."""
    g = _gradient(rows, cols, 9).to(dtype).to(dev.torch_device)
    small = torch.where(g.abs() < 2.0 ** -6, torch.zeros_like(g), g)   # keeps every scaled value a normal number
    a, b = dev.newton_schulz([small, small * 2.0 ** exponent])
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(33, 20), (300, 257), (100, 1500), (1500, 100)])
def test_strides_alignment_and_in_place(dev, rows, cols, dtype):
    g = _gradient(rows, cols, 2).to(dtype).to(dev.torch_device)
    want, = dev.newton_schulz([g])
    assert torch.equal(dev.newton_schulz([g.T.contiguous().T])[0], want)
    flat = torch.empty(rows * cols + 1, dtype=dtype, device=g.device)
    flat[1:] = g.reshape(-1)
    off = flat[1:].view(rows, cols)
    assert torch.equal(dev.newton_schulz([off])[0], want)
    m = ag._capi.PolarMatrix(off.data_ptr(), off.data_ptr(), rows, cols)
    code = ag._capi.AG_F32 if dtype == F32 else ag._capi.AG_BF16
    ag._capi.check(ag.lib().ag_newton_schulz(dev._h, code, 1, m, 5))
    assert torch.equal(off, want)
    # filter banks are [outputs, rest]
    if cols == 20:
        assert torch.equal(dev.newton_schulz([g.view(33, 5, 2, 2)])[0].view(33, 20), want)


# ---- Muon ------------------------------------------------------------------------------------------


def _muon64(w, g, v, lr, momentum, nesterov, decay, steps, scale):
    v = momentum * v.double() + g.double()
    u = g.double() + momentum * v if nesterov else v
    return (1 - lr * decay) * w.double() - lr * scale * _polar64(u, steps), v


def _muon_case(dev, sizes, dtype, seed=0):
    w = [_rand(s, seed + i, 0.05).to(dtype).to(dev.torch_device) for i, s in enumerate(sizes)]
    g = [_gradient(*s, seed + 50 + i).to(dtype).to(dev.torch_device) for i, s in enumerate(sizes)]
    v = [(_gradient(*s, seed + 90 + i) * 5).float().to(dev.torch_device) for i, s in enumerate(sizes)]
    return w, g, v


def _check_muon(w, v, want_w, want_v, lr, scale, dtype):
    """v: one rounding of the product and one of the sum, u of each; w: half a step, and the update's own error."""
    assert ((v.double() - want_v).abs() <= 2 * U * want_v.abs() + 4 * U * want_v.abs().max()).all()
    update = lr * scale * _tol(F32 if dtype == F32 else BF16)
    half = U if dtype == F32 else 2.0 ** -8
    size = math.sqrt(want_w.numel())
    # 2-norms: what the update may be off (its norm is at most 1.21 sqrt(min(rows, cols))), the rounding of w
    off = update * 1.21 * math.sqrt(min(want_w.shape)) + 3 * half * want_w.norm() + 1e-30 * size
    assert (w.double() - want_w).norm() <= off


MUON_SIZES = [(6, 25), (16, 150), (256, 128), (128, 84), (84, 10), (1, 40), (512, 10), (300, 520), (64, 1200)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("momentum,decay,steps", [(0.95, 0.1, 5), (0.0, 0.0, 5), (0.9, 0.0, 3)])
def test_muon(dev, dtype, nesterov, momentum, decay, steps):
    w, g, v = _muon_case(dev, MUON_SIZES, dtype)
    scales = [math.sqrt(max(1.0, c / r)) for r, c in MUON_SIZES]
    lr = 0.02
    for _ in range(2):   # the second call works with the first one's state
        want = [_muon64(*t, lr, momentum, nesterov, decay, steps, s) for *t, s in zip(w, g, v, scales)]
        before = [t.clone() for t in g]
        dev.muon_update(w, g, v, lr, momentum=momentum, nesterov=nesterov, weight_decay=decay, steps=steps, scales=scales)
        assert all(torch.equal(a, b) for a, b in zip(g, before))
        for wi, vi, (ww, wv), s in zip(w, v, want, scales):
            _check_muon(wi, vi, ww, wv, lr, s, dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_muon_of_zeros_and_nothing(dev, dtype):
    w, g, v = _muon_case(dev, [(40, 60), (300, 200)], dtype)
    for t in (*g, *v):
        t.zero_()
    want = [t.clone() for t in w]
    dev.muon_update(w, g, v, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(w, want)) and not any(t.any() for t in v)
    dev.muon_update(w, g, v, 0.5, weight_decay=1.0)   # decay alone: w halves, exactly
    assert all(torch.equal(a, b / 2) for a, b in zip(w, want))
    assert dev.muon_update([], [], [], 0.1) == ([], [])


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_muon_of_filter_banks_is_that_of_their_matrices(dev, dtype):
    w, g, v = _muon_case(dev, [(16, 150)], dtype)
    bank = [t[0].clone().view(16, 6, 5, 5) for t in (w, g, v)]
    dev.muon_update(w, g, v, 0.02)
    dev.muon_update(*[[t] for t in bank], 0.02)
    assert torch.equal(bank[0].view(16, 150), w[0]) and torch.equal(bank[2].view(16, 150), v[0])


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_same_bits_again_from_a_graph_and_another_stream(dev, dtype):
    dev.set_guards(False)
    sizes = [(84, 10), (300, 520), (700, 700), (260, 2200)]
    w, g, v = _muon_case(dev, sizes, dtype, seed=4)
    torch.cuda.synchronize()
    state = [[t.clone() for t in ts] for ts in (w, v)]

    def reset():
        for ts, olds in zip((w, v), state):
            for t, old in zip(ts, olds):
                t.copy_(old)
    results = []
    for _ in range(3):
        reset()
        dev.muon_update(w, g, v, 0.02)
        results.append([t.clone() for t in (*w, *v)])
    side = torch.cuda.Stream()
    side.wait_stream(dev.stream)
    with torch.cuda.stream(side):
        reset()
        dev.muon_update(w, g, v, 0.02)
    torch.cuda.synchronize()
    torch.cuda.set_stream(dev.stream)
    results.append([t.clone() for t in (*w, *v)])
    graph = torch.cuda.CUDAGraph()
    dev.wait()
    with torch.cuda.graph(graph, stream=dev.stream):
        dev.muon_update(w, g, v, 0.02)
    big = _gradient(1100, 1300, 1).to(dtype).to(dev.torch_device)
    for _ in range(2):
        dev.newton_schulz([big])   # grows and fills the workspace between the graph's capture and its replays
        reset()
        graph.replay()
        dev.wait()
        results.append([t.clone() for t in (*w, *v)])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    del graph


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_norms_losses_and_muon_train_together(dev, dtype):
    """A small classifier whose hidden layer is normalised, stepped by Muon through the operators: gradients as in 64 bits."""
    r = np.random.default_rng(0)
    to = lambda a: torch.from_numpy(a).to(dtype).to(dev.torch_device)
    x, t = to(r.standard_normal((64, 40))), torch.from_numpy(r.integers(0, 10, 64).astype(np.uint8)).to(dev.torch_device)
    w1, w2 = to(r.standard_normal((40, 96)) * 0.2), to(r.standard_normal((96, 10)) * 0.2)
    gain, shift = to(1 + 0.1 * r.standard_normal(96)), to(0.1 * r.standard_normal(96))
    v = [torch.zeros(w.shape, device=dev.torch_device) for w in (w1, w2)]
    for _ in range(3):
        h = dev.dot(x, w1)
        y, mean, rstd = dev.layer_norm_keep(h, gain, shift)
        a = dev.relu(y)
        z = dev.dot(a, w2)
        loss, dz = dev.cross_entropy_loss_with_grad(z, t)
        dw2 = dev.dot(a.t(), dz)
        dy = dev.relu_backward(y, dev.dot(dz, w2.t()))
        dh, dgain, dshift = dev.layer_norm_backward(h, dy, mean, rstd, gain, has_bias=True)
        dw1 = dev.dot(x.t(), dh)
        p = [q.double().requires_grad_() for q in (w1, gain, shift, w2)]
        hh = x.double() @ p[0]
        hat = (hh - hh.mean(1, keepdim=True)) / torch.sqrt(hh.var(1, correction=0, keepdim=True) + 1e-5)
        logits = torch.relu(hat * p[1] + p[2]) @ p[3]
        torch.nn.functional.cross_entropy(logits, t.long()).backward()
        # f32: products of length 96 and sums of 64 rows; bf16: a dozen roundings of half a step between layers, and gates
        # that turn where a rounded activation changes its sign
        tol = 1e-4 if dtype == F32 else 0.08
        for got, want in zip((dw1, dgain, dshift, dw2), p):
            assert (got.double() - want.grad).norm() <= tol * want.grad.norm()
        want = [_muon64(w, g, m, 0.02, 0.95, True, 0.0, 5, 1.0) for w, g, m in zip((w1, w2), (dw1, dw2), v)]
        dev.muon_update([w1, w2], [dw1, dw2], v, 0.02)
        for w, m, (ww, wv) in zip((w1, w2), v, want):
            _check_muon(w, m, ww, wv, 0.02, 1.0, dtype)


@gpu
def test_refusals(dev):
    d = dev.torch_device
    m = torch.ones((4, 6), device=d)
    other = lambda: torch.ones((4, 6), device=d)
    inv, shape, dt, lim = ag._capi.AG_ERR_INVALID, ag._capi.AG_ERR_SHAPE, ag._capi.AG_ERR_DTYPE, ag._capi.AG_ERR_LIMIT
    w, v = other(), other()
    cases = [
        (shape, lambda: dev.newton_schulz([m[0]])),
        (shape, lambda: dev.newton_schulz([m[:0]])),
        (shape, lambda: dev.newton_schulz([m[:, :0]])),
        (dt, lambda: dev.newton_schulz([m, m.bfloat16()])),
        (dt, lambda: dev.newton_schulz([m.half()])),
        (dt, lambda: dev.newton_schulz([m.double()])),
        (inv, lambda: dev.newton_schulz([m], steps=0)),
        (inv, lambda: dev.newton_schulz([m], steps=21)),
        (inv, lambda: dev.newton_schulz([m.cpu()])),
        (lim, lambda: dev.newton_schulz([m] * 4097)),
        (shape, lambda: dev.muon_update([w], [m], [], 0.1)),
        (shape, lambda: dev.muon_update([w], [m[:2]], [v], 0.1)),
        (shape, lambda: dev.muon_update([w], [m], [v[:2]], 0.1)),
        (shape, lambda: dev.muon_update([w], [m], [v], 0.1, scales=[1.0, 2.0])),
        (dt, lambda: dev.muon_update([w], [m.bfloat16()], [v], 0.1)),
        (dt, lambda: dev.muon_update([w.bfloat16()], [m.bfloat16()], [v.bfloat16()], 0.1)),
        (inv, lambda: dev.muon_update([w], [m], [v], 0.1, momentum=-0.5)),
        (inv, lambda: dev.muon_update([w], [m], [v], 0.1, momentum=float("nan"))),
        (inv, lambda: dev.muon_update([w], [m], [w], 0.1)),
        (inv, lambda: dev.muon_update([w], [w], [v], 0.1)),
        (inv, lambda: dev.muon_update([w], [v], [v], 0.1)),
        (inv, lambda: dev.muon_update([w, w], [m, m], [v, other()], 0.1)),
        (inv, lambda: dev.muon_update([w, other()], [m, m], [v, v], 0.1)),
        (inv, lambda: dev.muon_update([torch.ones((6, 4), device=d).T], [m], [v], 0.1)),
        (inv, lambda: dev.muon_update([w.cpu()], [m], [v], 0.1)),
    ]
    for status, call in cases:
        with pytest.raises(ag.AgError) as err:
            call()
        assert err.value.status == status
    assert (w == 1).all() and (v == 1).all()
    # one gradient for two parameters is fine: it is only read
    dev.muon_update([w, other()], [m, m], [v, other()], 0.1)
    f, p = ag.lib().ag_newton_schulz, lambda *a: ag._capi.PolarMatrix(*a)
    g, o = m.data_ptr(), v.data_ptr()
    assert f(dev._h, 0, -1, p(g, o, 4, 6), 5) == inv
    assert f(dev._h, 0, 1, None, 5) == inv
    assert f(dev._h, 0, 1, p(None, o, 4, 6), 5) == inv
    assert f(dev._h, 0, 1, p(g, None, 4, 6), 5) == inv
    assert f(dev._h, 0, 1, p(g, g + 4, 4, 5), 5) == inv
    assert f(dev._h, 0, 1, p(g, o, 0, 6), 5) == shape
    assert f(dev._h, 0, 1, p(g, o, 4, -6), 5) == shape
    assert f(dev._h, 0, 1, p(g, o, 16385, 16385), 5) == lim
    assert f(dev._h, 0, 1, p(g, o, 4, (1 << 20) + 1), 5) == lim
    assert f(dev._h, 0, 1, p(g, o, 1 << 62, 1 << 62), 5) == lim
    assert f(dev._h, 2, 1, p(g, o, 4, 6), 5) == dt
    two = (ag._capi.PolarMatrix * 2)(p(g, o, 4, 6), p(g, o, 4, 6))
    assert f(dev._h, 0, 2, two, 5) == inv


def test_refusals_without_a_device():
    m = ag._capi.PolarMatrix(None, None, 4, 6)
    assert ag.lib().ag_newton_schulz(None, 0, 1, m, 5) == ag._capi.AG_ERR_INVALID
    u = ag._capi.MuonMatrix(None, None, None, 4, 6, 1.0)
    assert ag.lib().ag_muon_update(None, 0, 1, u, 0.1, 0.9, 1, 0.0, 5) == ag._capi.AG_ERR_INVALID
