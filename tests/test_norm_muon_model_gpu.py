"""Models with LayerNorm layers and models trained by Muon, against the same network and update in 64 bits."""
import json
import math

import numpy as np
import pytest
import torch

import autograph_b200 as ag

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
DTYPES, IDS = [F32, BF16], ["f32", "bf16"]

# image [1, 12, 12] -> conv 5x5 (8) -> norm over [8, 8, 8] -> pool -> norm over the rows -> dense -> norm -> dense
NORM_SPEC = [("conv", 1, 8, (5, 5), True), ("layer_norm", 8 * 8 * 8, True), ("relu",), ("pool", (2, 2)), ("flatten",),
             ("layer_norm", 128, False), ("dense", 128, 40, True), ("layer_norm", 40, True), ("relu",),
             ("dense", 40, 10, True)]
NAMES = ["conv", "norm1", "relu1", "pool", "flatten", "norm2", "dense1", "norm3", "relu2", "dense2"]
SHAPES = [(8, 1, 5, 5), (8,), (512,), (512,), (128,), (128, 40), (40,), (40,), (40,), (40, 10), (10,)]


def _norm(x, w, b, cols):
    shape = x.shape
    x = x.reshape(-1, cols)
    hat = (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, correction=0, keepdim=True) + 1e-5)
    return (hat * w + (0 if b is None else b)).reshape(shape)


def _forward64(p, x):
    f = torch.nn.functional
    h = f.conv2d(x.double(), p[0], p[1])
    h = torch.relu(_norm(h, p[2], p[3], 512))
    h = f.max_pool2d(h, 2).flatten(1)
    h = _norm(h, p[4], None, 128) @ p[5] + p[6]
    h = torch.relu(_norm(h, p[7], p[8], 40))
    return h @ p[9] + p[10]


def _model(dev, dtype, spec=NORM_SPEC, shapes=SHAPES, seed=3):
    m = ag.Model(dev, spec, dtype, seed=seed)
    assert m.parameter_lens == [math.prod(s) for s in shapes]
    return m


def _params(m, shapes):
    return [torch.from_numpy(m.get_parameter(i).reshape(s)).double() for i, s in enumerate(shapes)]


def _batch(bs, dtype, seed=0, image=(1, 12, 12)):
    r = np.random.default_rng(seed)
    x = torch.from_numpy(r.standard_normal((bs, *image))).to(dtype)
    return x.pin_memory(), torch.from_numpy(r.integers(0, 10, bs).astype(np.uint8)).pin_memory()


def _shake(m, shapes, dtype):
    """Parameters away from their start, so that weights of ones and biases of zeros hide nothing."""
    r = np.random.default_rng(9)
    m.set_parameters([(m.get_parameter(i) + 0.1 * r.standard_normal(m.parameter_lens[i])).astype(np.float32)
                      for i in range(len(shapes))])


def test_a_norm_starts_as_one(dev):
    m = _model(dev, F32)
    assert (m.get_parameter(2) == 1).all() and (m.get_parameter(3) == 0).all() and (m.get_parameter(4) == 1).all()
    # and draws nothing: the layers around it start as they would without it
    plain = ag.Model(dev, [l for l in NORM_SPEC if l[0] != "layer_norm"], F32, seed=3)
    for i, k in enumerate([0, 1, 5, 6, 9, 10]):
        assert (plain.get_parameter(i) == m.get_parameter(k)).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("bs", [1, 7, 64])
def test_inference_and_gradients(dev, dtype, bs):
    m = _model(dev, dtype)
    _shake(m, SHAPES, dtype)
    x, t = _batch(bs, dtype)
    p = [q.requires_grad_() for q in _params(m, SHAPES)]
    logits = _forward64(p, x)
    torch.nn.functional.cross_entropy(logits, t.long()).backward()
    # f32: sums of up to 512 products, five layers deep.  bf16: some ten roundings of half a step, 2^-8, between layers, whose
    # norms keep them at that size; in the gradients also gates that turn with a rounded activation's sign
    tol, grad_tol = (1e-4, 1e-4) if dtype == F32 else (0.04, 0.15)
    for _ in range(3):   # eager, captured, replayed
        got = m.infer(x).double()
        assert (got - logits).norm() <= tol * logits.norm()
    for _ in range(3):
        m.train_forward_backward(x.to(dev.torch_device), t.to(dev.torch_device))
        for i, q in enumerate(p):
            g = torch.from_numpy(m.get_gradient(i)).double().reshape(q.shape)
            assert (g - q.grad).norm() <= grad_tol * q.grad.norm() + 1e-12, i


def test_sizes_that_no_trailing_dimensions_have(dev):
    x, _ = _batch(2, F32)
    for size in (7, 24, 5):
        with pytest.raises(ag.AgError) as err:
            ag.Model(dev, [("layer_norm", size, True), ("flatten",), ("dense", 144, 10, True)]).infer(x)
        assert err.value.status == ag._capi.AG_ERR_SHAPE
    for size in (12, 144):
        ag.Model(dev, [("layer_norm", size, False), ("flatten",), ("dense", 144, 10, True)]).infer(x)
    with pytest.raises(ag.AgError):
        ag.Model(dev, [("layer_norm", 0, True), ("flatten",), ("dense", 144, 10, True)])


def test_a_norm_of_one_value_a_row(dev):
    """It takes inputs whose last dimension is one, and gives the bias; others have rows of more than one value."""
    x, _ = _batch(2, F32)
    with pytest.raises(ag.AgError) as err:
        ag.Model(dev, [("layer_norm", 1, True), ("flatten",), ("dense", 144, 10, True)]).infer(x)
    assert err.value.status == ag._capi.AG_ERR_SHAPE
    with pytest.raises(ag.AgError) as err:
        ag.Model(dev, [("flatten",), ("dense", 144, 10, True), ("layer_norm", 1, True)]).infer(x)
    assert err.value.status == ag._capi.AG_ERR_SHAPE
    m = ag.Model(dev, [("flatten",), ("dense", 144, 1, True), ("layer_norm", 1, True), ("dense", 1, 10, True)])
    bias = np.float32(0.25)
    m.set_parameters([m.get_parameter(0), m.get_parameter(1), np.ones(1, np.float32), np.full(1, bias), m.get_parameter(4),
                      m.get_parameter(5)])
    want = bias * m.get_parameter(4) + m.get_parameter(5)
    assert np.abs(m.infer(x).numpy() - want).max() <= 4 * 2.0 ** -24 * (np.abs(m.get_parameter(4)).max() + 1)


def _polar64(g, steps):
    x = g / g.norm() if g.norm() > 0 else g
    flip = g.shape[0] > g.shape[1]
    x = x.T if flip else x
    for _ in range(steps):
        a = x @ x.T
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
    return x.T if flip else x


class Muon64:
    def __init__(self, momentum, nesterov, decay, steps, vector_scale):
        self.args = momentum, nesterov, decay, steps, vector_scale
        self.v = {}

    def step(self, params, grads, lr):
        momentum, nesterov, decay, steps, vector_scale = self.args
        out = []
        for i, (w, g) in enumerate(zip(params, grads)):
            v = self.v[i] = momentum * self.v.get(i, torch.zeros_like(g)) + g
            if w.dim() < 2:
                out.append(w - lr * vector_scale * v)
                continue
            u = (g + momentum * v if nesterov else v).reshape(w.shape[0], -1)
            ins, outs = (w.shape[0], w.shape[1]) if w.dim() == 2 else (w[0].numel(), w.shape[0])
            o = _polar64(u, steps).reshape(w.shape)
            out.append((1 - lr * decay) * w - lr * math.sqrt(max(1, outs / ins)) * o)
        return out


LENET_SHAPES = [(6, 1, 5, 5), (16, 6, 5, 5), (256, 128), (128, 84), (84, 10), (10,)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("net", ["lenet5", "norm"])
@pytest.mark.parametrize("host", [True, False], ids=["host", "device"])
def test_muon_steps(dev, dtype, net, host):
    """Each step's update is the formula's on the gradients that the step computed: eager steps, captured and replayed ones,
    two learning rates, and the split form."""
    dev.set_guards(False)
    spec, shapes, image = (ag.LENET5_SPEC, LENET_SHAPES, (1, 28, 28)) if net == "lenet5" else (NORM_SPEC, SHAPES, (1, 12, 12))
    m = _model(dev, dtype, spec, shapes)
    setting = dict(momentum=0.9, nesterov=True, weight_decay=0.05, steps=5, vector_scale=0.5)
    m.set_muon(**setting)
    ref = Muon64(0.9, True, 0.05, 5, 0.5)
    for i, lr in enumerate([0.02, 0.02, 0.02, 0.02, 0.01, 0.01, 0.02]):
        x, t = _batch(20, dtype, seed=i, image=image)
        before = _params(m, shapes)
        if host:
            m.train_step(x, t, lr)
        else:
            m.train_forward_backward(x.to(dev.torch_device), t.to(dev.torch_device), sync=False)
            m.apply_update(lr)
            m.last_loss()
        grads = [torch.from_numpy(m.get_gradient(k).reshape(s)).double() for k, s in enumerate(shapes)]
        want = ref.step(before, grads, lr)
        half = 2.0 ** -24 if dtype == F32 else 2.0 ** -8
        for k, (w0, w1) in enumerate(zip(before, want)):
            got = torch.from_numpy(m.get_parameter(k).reshape(shapes[k])).double()
            # the batches' gradients have few large singular values: 1.2e-4 of the update in f32, one and a half steps in
            # bf16, and the roundings of w (those of a vector's velocity, in the model's type, add up over the steps)
            off = (2e-4 if dtype == F32 else 1.5 * 2.0 ** -8) * (w1 - w0).norm() + 3 * half * w1.norm()
            if w1.dim() < 2:
                off = off + 20 * half * (w1 - w0).norm()
            assert (got - w1).norm() <= off, (i, k)
            v = torch.from_numpy(m.get_momentum(k)).double().reshape(shapes[k])
            tol_v = 1e-6 if dtype == F32 or w1.dim() >= 2 else 20 * half
            assert (v - ref.v[k]).norm() <= tol_v * ref.v[k].norm() + 1e-30


def test_muon_and_sgd_take_turns(dev):
    """set_muon and set_sgd switch, clear the momenta, and no captured step of the other is replayed."""
    dev.set_guards(False)
    x, t = _batch(16, F32)
    a, b = _model(dev, F32), _model(dev, F32)
    for m in (a, b):
        m.set_sgd(0.9)
        for _ in range(3):
            m.train_step(x, t, 0.01)
    a.set_muon()
    for _ in range(3):
        a.train_step(x, t, 0.01)
    assert any((a.get_parameter(i) != b.get_parameter(i)).any() for i in range(len(SHAPES)))
    a.set_parameters([b.get_parameter(i) for i in range(len(SHAPES))])
    for m in (a, b):
        m.set_sgd(0.9)
        for _ in range(3):
            m.train_step(x, t, 0.01)
    for i in range(len(SHAPES)):
        assert (a.get_parameter(i) == b.get_parameter(i)).all()
        assert (a.get_velocity(i) == b.get_velocity(i)).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_muon_continues_from_a_checkpoint(dev, dtype):
    dev.set_guards(False)
    a, b = _model(dev, dtype), _model(dev, dtype, seed=8)
    a.set_muon(momentum=0.9)
    for i in range(3):
        a.train_step(*_batch(16, dtype, seed=i), 0.02)
    text = a.to_serde_json(NAMES)
    state = json.loads(text)["dense1"]["weight"]["optim_state"]
    assert state["name"] == "Muon" and state["key_values"][0][0] == "velocity"
    b.set_muon(momentum=0.9)
    b.load_serde_json(text)
    for i in range(3, 6):
        assert a.train_step(*_batch(16, dtype, seed=i), 0.02) == b.train_step(*_batch(16, dtype, seed=i), 0.02)
    for i in range(len(SHAPES)):
        assert (a.get_parameter(i) == b.get_parameter(i)).all() and (a.get_momentum(i) == b.get_momentum(i)).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("to_muon", [True, False], ids=["sgd_to_muon", "muon_to_sgd"])
def test_another_optimizers_checkpoint(dev, dtype, to_muon):
    """The parameters load; the state is not the model's own, so that its momenta start at zero, as set_muon and set_sgd leave
    them."""
    dev.set_guards(False)
    a, b, c = (_model(dev, dtype, seed=s) for s in (3, 8, 9))
    set_other, set_own = (lambda m: m.set_sgd(0.9)), (lambda m: m.set_muon(momentum=0.9))
    if not to_muon:
        set_other, set_own = set_own, set_other
    set_other(a), set_own(b), set_own(c)
    for m in (a, b):
        m.train_step(*_batch(16, dtype), 0.02)
    b.load_serde_json(a.to_serde_json(NAMES))
    c.set_parameters([a.get_parameter(i) for i in range(len(SHAPES))])
    for i in range(len(SHAPES)):
        assert (b.get_parameter(i) == a.get_parameter(i)).all() and not b.get_momentum(i).any()
    for m in (b, c):
        m.train_step(*_batch(16, dtype, seed=1), 0.02)
    for i in range(len(SHAPES)):
        assert (b.get_parameter(i) == c.get_parameter(i)).all()


def test_refusals(dev):
    m = _model(dev, F32)
    inv, uns = ag._capi.AG_ERR_INVALID, ag._capi.AG_ERR_UNSUPPORTED
    for kw in (dict(momentum=-1.0), dict(momentum=float("nan")), dict(steps=0), dict(steps=21),
               dict(weight_decay=float("nan")), dict(vector_scale=float("nan"))):
        with pytest.raises(ag.AgError) as err:
            m.set_muon(**kw)
        assert err.value.status == inv
    m.set_muon()
    for call in (lambda: m.get_velocity(0), lambda: m.set_velocities([np.zeros(200, np.float32)])):
        with pytest.raises(ag.AgError) as err:
            call()
        assert err.value.status == uns
    m.get_velocity(1)   # a vector's is SGD's
    lib, p = ag.lib(), np.zeros(600, np.float32).ctypes.data
    assert lib.ag_model_get_momentum(m._h, 99, p) == inv and lib.ag_model_get_momentum(m._h, 0, None) == inv
    assert lib.ag_model_set_muon(None, 0.9, 1, 0.0, 5, 1.0) == inv


def test_parameters_beyond_the_limits_are_refused_at_set_muon(dev):
    """At once, not by every step after its vectors have moved: a longer side above 2^20."""
    m = ag.Model(dev, [("flatten",), ("dense", 1, (1 << 20) + 1, True)], F32, seed=1)
    m.set_sgd(0.5)
    m.set_velocities([np.ones(n, np.float32) for n in m.parameter_lens])
    with pytest.raises(ag.AgError) as err:
        m.set_muon()
    assert err.value.status == ag._capi.AG_ERR_LIMIT
    # the model keeps its optimizer and that one's state
    assert m.muon is None and m.momentum == 0.5
    assert all((m.get_velocity(i) == 1).all() for i in range(2))


def test_set_muon_takes_the_updates_workspace(dev):
    """No step fails for want of memory after some of it: where there is none for the workspace, set_muon says so."""
    dev.set_guards(False)
    own = ag.Device(0)
    torch.cuda.set_stream(own.stream)
    hog = []
    try:
        m = ag.Model(own, [("flatten",), ("dense", 8192, 8192, False)], BF16, seed=1)   # planes of 1.07 GB
        own.wait()
        # room for the momenta of 268 MB alone
        hog.append(torch.empty(torch.cuda.mem_get_info()[0] - (1 << 30), dtype=torch.uint8, device=own.torch_device))
        with pytest.raises(ag.AgError) as err:
            m.set_muon()
        assert err.value.status == ag._capi.AG_ERR_OOM
    finally:
        hog.clear()
        torch.cuda.empty_cache()
        torch.cuda.set_stream(dev.stream)
    m.set_muon()


def test_two_models_on_two_devices_of_one_gpu(dev):
    """Two threads, each with a device of its own: kernels that need the whole GPU do not wait for each other's halves."""
    import threading
    dev.set_guards(False)
    want, got, errors = {}, {}, []

    def work(k, out):
        try:
            d = ag.Device(0)
            m = ag.Model(d, NORM_SPEC, F32, seed=k)
            m.set_muon()
            for i in range(30):
                m.train_step(*_batch(16, F32, seed=i), 0.02)
            out[k] = [m.get_parameter(i) for i in range(len(SHAPES))]
            m.close()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    for k in (1, 2):
        work(k, want)
    threads = [threading.Thread(target=work, args=(k, got)) for k in (1, 2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.set_stream(dev.stream)
    assert not errors, errors
    for k in (1, 2):
        assert all((a == b).all() for a, b in zip(want[k], got[k]))
