"""The 8-bit operators as programs call them: what is timed, in its plain form and through the framework.

A row is one particle's (or token's) vector.  Its 8-bit form is one scale and one code a value:

    m = max(max |x|, 2^-100)    scale = m / 127    code = round(x * (127 / m))     value = code * scale

in float32 steps, rounding to the nearest code and ties to the even one; a row that holds a NaN or an
infinity has a NaN for its scale and zeros for codes.

* ``save``         activations kept in 8 bits between forward and backward, and read back.
* ``weight_grad``  a linear layer's input kept in 8 bits, and the layer's weight and bias gradients taken
                   from the codes.
* ``mlp_train``    the automaton's MLP (Linear, ReLU, Linear over one row per particle) in training, with
                   its input kept in 8 bits: the forward from the input itself, the backward from the
                   codes, whose hidden values it computes again.
* ``mlp_serve``    the same MLP in inference, both layers as products of 8-bit integers.
* ``linear``       one linear layer in inference: 8-bit integers with a scale for each row of the input and
                   each channel of the weights, which were laid out once.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
HIDDEN = 128  # the automaton's hidden units
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # perception features of a growing 3D cloud (32 states) kept for the backward of one rollout step
        dict(name="save_features", kind="save", rows=65536, cols=163, dtype="float32"),
        # activations of a wide layer, odd in both sizes
        dict(name="save_wide_odd", kind="save", rows=8191, cols=4097, dtype="bfloat16"),
        # the first layer's gradient over a million particles: a tiny output, a long sum
        dict(name="weight_grad_particles", kind="weight_grad", rows=1048576, cols=83, outs=128, dtype="float32"),
        # a wide layer over a batch of tokens
        dict(name="weight_grad_wide", kind="weight_grad", rows=8192, cols=2048, outs=2048, dtype="float32"),
        # one training step's MLP of the 2D growing model: latency-bound
        dict(name="mlp_train_2d", kind="mlp_train", rows=4096, cols=66, outs=18),
        # wide states (32), the 3D growth cloud, a ragged number of rows
        dict(name="mlp_train_growth", kind="mlp_train", rows=65521, cols=163, outs=35),
        # one training step's MLP of the million-particle model
        dict(name="mlp_train_stress", kind="mlp_train", rows=1048576, cols=83, outs=19),
        # the viewer's cloud, stepped forever
        dict(name="mlp_serve_2d", kind="mlp_serve", rows=4096, cols=66, outs=18),
        # a million particles rolled out
        dict(name="mlp_serve_stress", kind="mlp_serve", rows=1048576, cols=83, outs=19),
        # a single token through a wide layer: the weights are read once, latency counts
        dict(name="linear_token", kind="linear", rows=1, cols=4096, outs=4096, dtype="bfloat16"),
        # a handful of sequences decoded together, odd sizes
        dict(name="linear_decode_odd", kind="linear", rows=37, cols=2049, outs=8190, dtype="float16"),
        # a long prompt through a wide layer
        dict(name="linear_prompt", kind="linear", rows=8192, cols=4096, outs=8192, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["save", "weight_grad", "mlp_train", "mlp_serve", "linear", "linear"])
    if kind == "save":
        cols = _log(rng, 1, 16384)
        return dict(kind=kind, rows=_log(rng, 1, max(1, min(1 << 20, (1 << 25) // cols))), cols=cols,
                    dtype=rng.choice(sorted(DTYPES)))
    if kind == "weight_grad":
        cols, outs = _log(rng, 4, 4096), _log(rng, 4, 4096)
        return dict(kind=kind, rows=_log(rng, 64, min(1 << 20, (1 << 36) // (cols * outs), (1 << 27) // (cols + outs))),
                    cols=cols, outs=outs, dtype="float32")
    if kind == "linear":
        cols, outs = _log(rng, 16, 8192), _log(rng, 16, 8192)
        rows = rng.choice([_log(rng, 1, 64), _log(rng, 64, 8192)])
        return dict(kind=kind, rows=max(1, min(rows, (1 << 38) // (cols * outs))), cols=cols, outs=outs,
                    dtype=rng.choice(sorted(DTYPES)))
    return dict(kind=kind, rows=_log(rng, 1, 1 << 20), cols=rng.randint(4, 168), outs=rng.randint(4, 64))


def work(case):
    rows, cols, kind = case["rows"], case["cols"], case["kind"]
    size = 4 if case.get("dtype", "float32") == "float32" else 2
    kept = rows * (cols + 4)  # codes and scales
    if kind == "save":
        return {"bytes": 2 * rows * cols * size + 2 * kept, "flops": 5 * rows * cols}
    outs = case["outs"]
    if kind == "weight_grad":
        return {"bytes": rows * (cols + outs) * 4 + 2 * kept + (cols + 1) * outs * 4, "flops": 2 * rows * cols * outs}
    if kind == "linear":
        return {"bytes": rows * (cols + outs) * size + outs * (cols + 8), "flops": 2 * rows * cols * outs}
    weights = HIDDEN * (cols + outs + 1) + outs
    if kind == "mlp_serve":
        return {"bytes": rows * (cols + outs) * 4 + weights, "flops": 2 * rows * HIDDEN * (cols + outs)}
    return {"bytes": rows * (2 * cols + 2 * outs) * 4 + 2 * kept + 2 * weights * 4,
            "flops": 2 * rows * HIDDEN * (4 * cols + 3 * outs)}


# ------------------------------------------------------------------ inputs

def _rows_of(gen, rows, cols, dtype):
    """Normal values whose columns differ in size, a few of them by much, as features and activations do."""
    size = torch.exp(0.5 * torch.randn(cols, device=DEVICE, generator=gen))
    size = torch.where(torch.rand(cols, device=DEVICE, generator=gen) < 0.01, 10 * size, size)
    return (torch.randn(rows, cols, device=DEVICE, generator=gen) * size).to(DTYPES[dtype])


def _weight(gen, outs, cols):
    return torch.randn(outs, cols, device=DEVICE, generator=gen) / math.sqrt(cols)


def _laid_out(weight):
    """A weight's codes, each row padded with zeros to a multiple of 16, and its scales: laid out once."""
    codes, scale = _quantize(weight)
    pad = -weight.shape[1] % 16
    return torch.nn.functional.pad(codes.to(torch.int8), (0, pad)).contiguous(), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, rows, cols, dtype = case["kind"], case["rows"], case["cols"], case.get("dtype", "float32")
    s = dict(case, x=_rows_of(gen, rows, cols, dtype))
    if kind == "save":
        return s
    outs = case["outs"]
    if kind == "weight_grad":
        s["dy"] = torch.randn(rows, outs, device=DEVICE, generator=gen) / rows
        return s
    if kind == "linear":
        s["codes"], s["scale"] = _laid_out(_weight(gen, outs, cols))
        s["bias"] = 0.1 * torch.randn(outs, device=DEVICE, generator=gen)
        return s
    w1, w2 = _weight(gen, HIDDEN, cols), _weight(gen, outs, HIDDEN)
    b1, b2 = (0.1 * torch.randn(n, device=DEVICE, generator=gen) for n in (HIDDEN, outs))
    if kind == "mlp_serve":
        s["codes1"], s["scale1"] = _laid_out(w1)
        s["codes2"], s["scale2"] = _laid_out(w2)
        s["b1"], s["b2"] = b1, b2
        return s
    # Rows with a hidden value within rounding of the ReLU's kink, where either side's gradient is right,
    # get no upstream.
    net = torch.nn.Sequential(torch.nn.Linear(cols, HIDDEN), torch.nn.ReLU(), torch.nn.Linear(HIDDEN, outs)).to(DEVICE)
    with torch.no_grad():
        for p, v in zip(net.parameters(), (w1, b1, w2, b2)):
            p.copy_(v)
    codes, scale = _quantize(s["x"])
    kept = codes * scale[:, None]
    near = (cols + 3) * 2.0 ** -23 * (kept.abs() @ w1.abs().T + b1.abs())
    dy = torch.randn(rows, outs, device=DEVICE, generator=gen) / rows
    s["dy"] = torch.where(((kept @ w1.T + b1).abs() <= near).any(1, keepdim=True), torch.zeros_like(dy), dy)
    s["net"], s["x"] = net, s["x"].requires_grad_(True)
    return s


# ------------------------------------------------------------------ the plain forms

def _quantize(x):
    """Codes (whole numbers in float32) and scales of the rows of x."""
    v = x.float()
    m = v.abs().amax(-1)
    fine = torch.isfinite(m)
    m = m.clamp_min(2.0 ** -100)
    top = torch.full_like(m, 127.0)
    codes = torch.where(fine[..., None], torch.round(v * (top / m)[..., None]), torch.zeros_like(v))
    return codes, torch.where(fine, m / top, torch.full_like(m, math.nan))


def _integer_layer(codes, scale, w_codes, w_scale, bias):
    total = codes @ w_codes[:, :codes.shape[1]].float().T
    return total * (scale[:, None] * w_scale) + bias


def _plain(s):
    kind, x = s["kind"], s["x"].detach()
    if kind == "mlp_train":
        w1, b1, w2, b2 = (p.detach() for p in s["net"].parameters())
        y = torch.relu(x @ w1.T + b1) @ w2.T + b2
    codes, scale = _quantize(x)
    if kind == "save":
        return scale, (codes * scale[:, None]).to(x.dtype)
    if kind == "linear":
        return _integer_layer(codes, scale, s["codes"], s["scale"], s["bias"]).to(x.dtype)
    if kind == "mlp_serve":
        hidden = torch.relu(_integer_layer(codes, scale, s["codes1"], s["scale1"], s["b1"]))
        return _integer_layer(*_quantize(hidden), s["codes2"], s["scale2"], s["b2"])
    kept, dy = codes * scale[:, None], s["dy"]
    if kind == "weight_grad":
        return dy.T @ kept, dy.sum(0)
    a = kept @ w1.T + b1
    da = torch.where(a > 0, dy @ w2, torch.zeros_like(a))
    return y, da @ w1, da.T @ kept, da.sum(0), dy.T @ torch.relu(a), dy.sum(0)


def run(state):
    s = state
    if not own:
        with torch.no_grad():
            return _plain(s)
    from npa_amd import int8, mlp
    kind, x = s["kind"], s["x"]
    if kind == "save":
        r = int8.quantize_rows(x)
        return r.scale, int8.restore_rows(r, x.dtype)
    if kind == "weight_grad":
        return int8.weight_grad(int8.quantize_rows(x), s["dy"])
    if kind == "linear":
        return int8.linear(x, int8.Rows8(s["codes"], s["scale"], (s["outs"], s["cols"])), s["bias"])
    if kind == "mlp_serve":
        return int8.mlp(x, int8.Rows8(s["codes1"], s["scale1"], (HIDDEN, s["cols"])), s["b1"],
                        int8.Rows8(s["codes2"], s["scale2"], (s["outs"], HIDDEN)), s["b2"])
    y = mlp.mlp(s["net"], x, checkpoint="int8")
    return (y.detach(), *torch.autograd.grad(y, [x, *s["net"].parameters()], s["dy"]))


# ------------------------------------------------------------------ 64 bits

def _exact_codes(x):
    """The codes by their definition (float32 steps: they are whole numbers, the same for everybody) and the
    scales in 64 bits."""
    v = x.detach().float()
    m = torch.maximum(v.abs().max(dim=-1).values, torch.tensor(2.0 ** -100, device=v.device))
    step = torch.from_numpy(np.float32(127) / m.cpu().numpy()).to(v.device)
    return torch.round(v * step[:, None]).double(), m.double() / 127


def exact(case, seed):
    s = prepare(case, seed)
    kind, x = s["kind"], s["x"].detach()
    q, scale = _exact_codes(x)
    if kind == "save":
        return scale, q * scale[:, None]
    if kind == "weight_grad":
        dy = s["dy"].double()
        return torch.mm(dy.t(), q * scale[:, None]), dy.sum(dim=0)
    if kind == "linear":
        total = torch.mm(q, s["codes"][:, :case["cols"]].double().t())
        return total * scale[:, None] * s["scale"].double() + s["bias"].double()
    if kind == "mlp_serve":
        # the hidden codes follow from float32 values by definition; the second layer is in 64 bits
        w1, w2 = s["codes1"][:, :case["cols"]].double(), s["codes2"].double()
        unit = torch.from_numpy(scale.float().cpu().numpy()[:, None] * s["scale1"].cpu().numpy()).to(x.device)
        h = torch.mm(q, w1.t()).float() * unit
        h = (h + s["b1"]).clamp(min=0)
        qh, scale_h = _exact_codes(h)
        return torch.mm(qh, w2.t()) * scale_h[:, None] * s["scale2"].double() + s["b2"].double()
    w1, b1, w2, b2 = (p.detach().double() for p in s["net"].parameters())
    y = torch.addmm(b2, torch.addmm(b1, x.double(), w1.t()).clamp(min=0), w2.t())
    kept, dy = q * scale[:, None], s["dy"].double()
    a = torch.addmm(b1, kept, w1.t())
    da = torch.mm(dy, w2) * (a > 0)
    return (y, torch.mm(da, w1), torch.mm(da.t(), kept), da.sum(dim=0), torch.mm(dy.t(), a.clamp(min=0)),
            dy.sum(dim=0))
