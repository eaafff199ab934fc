"""Operators of training that users of this library call next to its layers and its SGD, as cases that can be timed and compared.

Four kinds, all through the public Python front end:

* ``norm``      layer norm over the trailing values of each row, for a pass that records gradients
                (``Device.layer_norm_keep``): the normalised rows, their means and reciprocal deviations;
* ``norm_back`` its backward pass (``Device.layer_norm_backward``): the gradients of input, weight and bias;
* ``polar``     Newton-Schulz orthogonalisation of gradient matrices (``Device.newton_schulz``);
* ``muon``      the optimiser step around it over the matrices of a network (``Device.muon_update``):
                momentum, orthogonalisation, decoupled weight decay and update.
"""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
_EPS = 1e-5
_STEPS = 5
_A, _B, _C = 3.4445, -4.7750, 2.0315
_LR, _MOMENTUM, _DECAY = 0.02, 0.95, 0.01

_MOST_VALUES = 1 << 26      # of a drawn case's rows
_MOST_FLOPS = 20 * 4096**3  # of a drawn case's products


def listed():
    return [
        # The last hidden activations of LeNet5 at the training benchmark's batch: one small launch.
        dict(name="norm_f32_100x84", kind="norm", dtype="f32", rows=100, cols=84),
        # A whole dataset's batch through a wide layer: streams through memory.
        dict(name="norm_bf16_65536x1024", kind="norm", dtype="bf16", rows=65536, cols=1024),
        # The flattened features of the wide conv stack: few rows, each too long for one thread block's registers.
        dict(name="norm_f32_256x25088", kind="norm", dtype="f32", rows=256, cols=25088),
        # The same small layer's gradients: latency.
        dict(name="norm_back_f32_100x128", kind="norm_back", dtype="f32", rows=100, cols=128),
        # Gradients of the large batch, the weight's sum over all of its rows.
        dict(name="norm_back_bf16_65536x1024", kind="norm_back", dtype="bf16", rows=65536, cols=1024),
        # Sizes as data brings them: no row starts on a 16-byte boundary but the first.
        dict(name="norm_back_f32_4093x2011", kind="norm_back", dtype="f32", rows=4093, cols=2011),
        # One hidden layer's gradient, larger than one thread block takes at once.
        dict(name="polar_f32_1024x1024", kind="polar", dtype="f32", matrices="1024x1024"),
        # The largest products of this library's benchmark as the gradients of one layer.
        dict(name="polar_bf16_4096x4096", kind="polar", dtype="bf16", matrices="4096x4096"),
        # Layers of unequal sizes, taller than wide and wider than tall, none a multiple of anything.
        dict(name="polar_f32_ragged", kind="polar", dtype="f32", matrices="509x1531,1531x509,777x1009"),
        # Every weight of LeNet5: a step's worth of small matrices.
        dict(name="muon_f32_lenet5", kind="muon", dtype="f32", matrices="6x25,16x150,256x128,128x84,84x10"),
        # Every weight of the wide conv stack, one of them very tall.
        dict(name="muon_bf16_wide", kind="muon", dtype="bf16", matrices="64x27,128x576,25088x512,512x10"),
        # A deep stack of equal hidden layers.
        dict(name="muon_bf16_8x1024", kind="muon", dtype="bf16", matrices=",".join(["1024x1024"] * 8)),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_back", "polar", "muon"])
    dtype = rng.choice(["f32", "bf16"])
    if kind in ("norm", "norm_back"):
        cols = _log_uniform(rng, 1, 32768)
        rows = _log_uniform(rng, 1, min(65536, _MOST_VALUES // cols))
        if rng.random() < 0.5:   # as designers of networks pick them
            cols = max(8, cols // 8 * 8)
        return dict(kind=kind, dtype=dtype, rows=rows, cols=cols)
    left, sizes = _MOST_FLOPS, []
    for _ in range(rng.choice([1, 2, 3, 5, 8])):
        rows, cols = _log_uniform(rng, 4, 4096), _log_uniform(rng, 4, 4096)
        if rng.random() < 0.5:
            rows, cols = max(8, rows // 8 * 8), max(8, cols // 8 * 8)
        if _matrix_work(rows, cols) <= left:
            left -= _matrix_work(rows, cols)
            sizes.append("%dx%d" % (rows, cols))
    return dict(kind=kind, dtype=dtype, matrices=",".join(sizes))


def _sizes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["matrices"].split(",")]


def _gradient(rows, cols, gen):
    """What a Dense layer's weight gradient looks like when it is summed over several batches: activations behind a Relu, whose
    mean makes one singular value stand out, times gradients whose outputs have unequal sizes."""
    batch = 4 * min(rows, cols) + 32
    x = torch.randn((batch, rows), generator=gen, device="cuda").relu_()
    dy = torch.randn((batch, cols), generator=gen, device="cuda")
    dy *= torch.rand((cols,), generator=gen, device="cuda") + 0.5
    return x.T @ dy / batch


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = _DTYPE[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    state = {"kind": case["kind"]}
    if case["kind"] in ("norm", "norm_back"):
        rows, cols = case["rows"], case["cols"]
        x = randn(rows, cols).mul_(1.5).add_(0.5 * randn(cols)).add_(0.3 * randn(rows, 1)).to(dt)
        state.update(x=x, weight=(1 + 0.1 * randn(cols)).to(dt), bias=(0.1 * randn(cols)).to(dt))
        if case["kind"] == "norm_back":
            _, mean, rstd = _norm(x, state["weight"], state["bias"])   # what the forward pass kept
            state.update(dy=randn(rows, cols).div_(rows).to(dt), mean=mean, rstd=rstd)
        return state
    sizes = _sizes(case)
    state["g"] = [_gradient(r, c, gen).to(dt) for r, c in sizes]
    if case["kind"] == "muon":
        state["w"] = [(0.05 * randn(r, c)).to(dt) for r, c in sizes]
        state["v"] = [(10 * _gradient(r, c, gen)).float() for r, c in sizes]
        # each Dense weight is [inputs, outputs]
        state["scales"] = [math.sqrt(max(1.0, c / r)) for r, c in sizes]
    return state


# ---- plain forms -----------------------------------------------------------------------------------


def _norm(x, weight, bias):
    v = x.float()
    mean = v.mean(1, keepdim=True)
    centred = v - mean
    rstd = 1 / torch.sqrt(centred.square().mean(1, keepdim=True) + _EPS)
    y = centred * rstd * weight.float() + bias.float()
    return y.to(x.dtype), mean[:, 0], rstd[:, 0]


def _norm_back(x, dy, mean, rstd, weight):
    scale = rstd[:, None]
    hat = (x.float() - mean[:, None]) * scale
    d = dy.float()
    dhat = d * weight.float()
    dx = scale * (dhat - dhat.mean(1, keepdim=True) - hat * (dhat * hat).mean(1, keepdim=True))
    return dx.to(x.dtype), (d * hat).sum(0).to(x.dtype), d.sum(0).to(x.dtype)


def _polar(g):
    x = g.T if g.shape[0] > g.shape[1] else g
    x = x.float()
    x = x / x.norm()
    for _ in range(_STEPS):
        a = x @ x.T
        x = _A * x + (_B * a + _C * (a @ a)) @ x
    return x.T if g.shape[0] > g.shape[1] else x


def _muon(w, g, v, scale):
    v.mul_(_MOMENTUM).add_(g.float())
    o = _polar(g.float() + _MOMENTUM * v)
    w.copy_(((1 - _LR * _DECAY) * w.float() - _LR * scale * o).to(w.dtype))


# ---- the library's own -----------------------------------------------------------------------------

_handle = None


def _device():
    global _handle
    if _handle is None:
        import autograph_b200 as ag
        _handle = ag.Device(torch.cuda.current_device())
    return _handle


def run(state):
    kind = state["kind"]
    if kind == "norm":
        x, weight, bias = state["x"], state["weight"], state["bias"]
        y, mean, rstd = _device().layer_norm_keep(x, weight, bias, eps=_EPS) if own else _norm(x, weight, bias)
        return {"y": y, "mean": mean, "rstd": rstd}
    if kind == "norm_back":
        x, dy, mean, rstd, weight = state["x"], state["dy"], state["mean"], state["rstd"], state["weight"]
        dx, dweight, dbias = (_device().layer_norm_backward(x, dy, mean, rstd, weight, has_bias=True) if own
                              else _norm_back(x, dy, mean, rstd, weight))
        return {"dx": dx, "dweight": dweight, "dbias": dbias}
    if kind == "polar":
        g = state["g"]
        return {"o": _device().newton_schulz(g, steps=_STEPS) if own else [_polar(m).contiguous().to(m.dtype) for m in g]}
    w, g, v, scales = state["w"], state["g"], state["v"], state["scales"]
    if own:
        _device().muon_update(w, g, v, lr=_LR, momentum=_MOMENTUM, nesterov=True, weight_decay=_DECAY, steps=_STEPS,
                              scales=scales)
    else:
        [_muon(*args) for args in zip(w, g, v, scales)]
    return {"w": w, "v": v}


# ---- work and 64-bit values --------------------------------------------------------------------------


def _matrix_work(rows, cols):
    """Fewest operations of the steps on one matrix with n <= m.  Two of the three products of a step are symmetric: half of
    each is the other half's mirror.  Where m is much longer than n, the steps on the n x n matrix x x^T alone (four
    symmetric products each) with one product with x at the end are fewer."""
    n, m = min(rows, cols), max(rows, cols)
    direct = _STEPS * (n * n * m + n**3 + 2 * n * n * m)
    small = n * n * m + (4 * _STEPS - 4) * n**3 + 2 * n * n * m
    return min(direct, small)


def work(case):
    es = _SIZE[case["dtype"]]
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * es * n + 2 * es * case["cols"] + 8 * case["rows"], "flops": 8 * n}
    if case["kind"] == "norm_back":
        n = case["rows"] * case["cols"]
        return {"bytes": 3 * es * n + 3 * es * case["cols"] + 8 * case["rows"], "flops": 14 * n}
    values = sum(r * c for r, c in _sizes(case))
    # polar: gradients in, results out; muon: gradients in, weights and momenta in and out
    return {"bytes": values * (2 * es if case["kind"] == "polar" else 3 * es + 8),
            "flops": sum(_matrix_work(r, c) for r, c in _sizes(case))}


def _polar64(g):
    """By the singular values: with x = u diag(s) v^T a step is u diag(a s + b s^3 + c s^5) v^T, and the steps' odd
    polynomial p of s gives u diag(p(s) / s) u^T x, from the eigenvectors of x x^T."""
    x = g if g.shape[0] <= g.shape[1] else g.mT
    x = x / torch.linalg.vector_norm(x)
    lam, u = torch.linalg.eigh(x.matmul(x.mT))
    s2 = lam.clamp(min=0)
    gain = torch.ones_like(s2)   # p(s) / s
    for _ in range(_STEPS):
        t = s2 * gain.square()
        gain = gain * (_A + t * (_B + t * _C))
    o = u.matmul((u * gain).mT.matmul(x))
    return o if g.shape[0] <= g.shape[1] else o.mT.contiguous()


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        x, weight, bias = (state[k].double() for k in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, dim=-1, correction=0)
        rstd = torch.rsqrt(var + _EPS)
        y = torch.addcmul(bias, (x - mean.unsqueeze(-1)) * rstd.unsqueeze(-1), weight)
        return {"y": y, "mean": mean, "rstd": rstd}
    if case["kind"] == "norm_back":
        x, dy, mean, rstd, weight = (state[k].double() for k in ("x", "dy", "mean", "rstd", "weight"))
        hat = torch.einsum("rc,r->rc", x - mean.unsqueeze(-1), rstd)
        cols = case["cols"]
        along, across = torch.einsum("rc,c->r", dy, weight) / cols, torch.einsum("rc,rc,c->r", dy, hat, weight) / cols
        dx = rstd.unsqueeze(-1) * (dy * weight - along.unsqueeze(-1) - hat * across.unsqueeze(-1))
        return {"dx": dx, "dweight": torch.einsum("rc,rc->c", dy, hat), "dbias": dy.sum(0)}
    if case["kind"] == "polar":
        return {"o": [_polar64(g.double()) for g in state["g"]]}
    w, v = [], []
    for weight, g, old, scale in zip(state["w"], state["g"], state["v"], state["scales"]):
        g = g.double()
        v.append(torch.add(g, old.double(), alpha=_MOMENTUM))
        o = _polar64(torch.add(g, v[-1], alpha=_MOMENTUM))
        w.append(weight.double() * (1 - _LR * _DECAY) - _LR * scale * o)
    return {"w": w, "v": v}
