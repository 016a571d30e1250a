"""Layer norm and mixtures of experts as programs call them: what is timed, in its plain form and through the
framework.

A row is one particle's (or token's) vector.

* ``norm``    y = (x - mean) / sqrt(mean of (x - mean)^2 + eps) * w + b over each row; in training also dx, dw and db.
* ``sort``    rows sorted by expert and back: each of a row's k entries names an expert, or none (any number outside
  0 .. experts - 1).  A stable sort puts the entries into places, expert after expert, those without one behind the last:
  ``offsets[e]`` is expert e's first place, ``slot`` each entry's place (~place for an entry without an expert) and
  ``source`` each place's entry.  The rows are copied into their places (zeros behind the last), and the experts' results
  come back as the sum over a row's entries of weight times result; in training also the gradients of both.
* ``linear``  one linear layer for each expert over rows sorted that way: y = x W_e^T + b_e for the rows of expert e,
  zeros behind the last; in training also dx, dW and db.
* ``mlp``     Linear, ReLU, Linear of each expert, the automaton's update rule, in training.
"""
import math

import torch

own = False
DEVICE = "cuda"
EPS = 1e-5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # a single token's normalisation in a wide layer: latency counts
        dict(name="norm_token", kind="norm", rows=1, cols=4096, dtype="bfloat16", train=False),
        # perception features of a million particles in front of the automaton's MLP
        dict(name="norm_particles", kind="norm", rows=1048576, cols=83, dtype="float32", train=True),
        # activations of a wide layer, odd in both sizes
        dict(name="norm_wide_odd", kind="norm", rows=8191, cols=4097, dtype="bfloat16", train=True),
        # a handful of sequences decoded together, two experts each
        dict(name="sort_decode", kind="sort", rows=16, choices=2, experts=8, cols=4096, dtype="bfloat16", train=False),
        # a million particles of four kinds, some of no kind, and the gradients back to them
        dict(name="sort_particles", kind="sort", rows=1048576, choices=1, experts=4, cols=83, dtype="float32", train=True),
        # a long prompt's tokens over many experts, in training
        dict(name="sort_prompt", kind="sort", rows=8192, choices=2, experts=64, cols=4096, dtype="bfloat16", train=True),
        # a handful of decoded tokens through the experts they chose: the weights are read once, latency counts
        dict(name="linear_decode", kind="linear", slots=32, experts=16, cols=4096, outs=2048, dtype="bfloat16", train=False),
        # odd sizes and few rows an expert
        dict(name="linear_odd", kind="linear", slots=1023, experts=7, cols=2049, outs=1030, dtype="float16", train=False),
        # a long prompt's tokens, two experts each, in training
        dict(name="linear_prompt", kind="linear", slots=16384, experts=8, cols=2048, outs=4096, dtype="bfloat16", train=True),
        # a wide layer kept in float32
        dict(name="linear_float32", kind="linear", slots=8192, experts=4, cols=1024, outs=2048, dtype="float32", train=True),
        # one training step's update rules of the 2D growing model, four kinds of cells: latency counts
        dict(name="mlp_2d", kind="mlp", slots=4096, experts=4, cols=66, hidden=128, outs=18, dtype="float32", train=True),
        # one training step's update rules of the million-particle model
        dict(name="mlp_particles", kind="mlp", slots=1048576, experts=8, cols=83, hidden=128, outs=19, dtype="float32",
             train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "sort", "linear", "linear", "mlp"])
    case = dict(kind=kind, dtype=rng.choice(sorted(DTYPES)), train=rng.random() < 0.5)
    if kind == "norm":
        cols = _log(rng, 1, 16384)
        return dict(case, rows=_log(rng, 1, max(1, min(1 << 20, (1 << 26) // cols))), cols=cols)
    if kind == "sort":
        cols, choices = _log(rng, 1, 8192), rng.randint(1, 8)
        return dict(case, rows=_log(rng, 1, max(1, min(1 << 20, (1 << 26) // (cols * choices)))), choices=choices,
                    experts=_log(rng, 1, 256), cols=cols)
    if kind == "mlp":
        return dict(case, dtype="float32", train=True, slots=_log(rng, 1, 1 << 20), experts=_log(rng, 1, 32),
                    cols=rng.randint(4, 168), hidden=128, outs=rng.randint(4, 64))
    cols, outs = _log(rng, 4, 8192), _log(rng, 4, 8192)
    slots = rng.choice([_log(rng, 1, 256), _log(rng, 256, 1 << 18)])
    size = 1 << (35 if case["dtype"] == "float32" else 36)
    return dict(case, slots=max(1, min(slots, size // (cols * outs), (1 << 27) // (cols + outs))),
                experts=_log(rng, 1, max(1, min(64, (1 << 28) // (cols * outs)))), cols=cols, outs=outs)


def work(case):
    kind, train, cols = case["kind"], case["train"], case["cols"]
    size = 4 if case["dtype"] == "float32" else 2
    if kind == "norm":
        return {"bytes": (4 if train else 2) * case["rows"] * cols * size + (4 if train else 2) * cols * 4,
                "flops": (16 if train else 7) * case["rows"] * cols}
    if kind == "sort":
        rows, n = case["rows"], case["rows"] * case["choices"]
        once = 2 * (rows + n) * cols * size  # x and y; the sorted rows and the experts' results
        return {"bytes": (2 if train else 1) * once + (16 + (8 if train else 4)) * n,
                "flops": (7 if train else 2) * n * cols}
    slots, experts, outs = case["slots"], case["experts"], case["outs"]
    held = min(experts, slots)  # experts whose weights have to be read
    if kind == "mlp":
        hidden = case["hidden"]
        weights = hidden * (cols + outs + 1) + outs
        return {"bytes": (slots * 2 * (cols + outs) + (held + experts) * weights) * 4,
                "flops": 6 * slots * hidden * (cols + outs)}
    weights = outs * (cols + 1)
    if train:
        return {"bytes": (slots * 2 * (cols + outs) + (held + experts) * weights) * size, "flops": 6 * slots * cols * outs}
    return {"bytes": (slots * (cols + outs) + held * weights) * size, "flops": 2 * slots * cols * outs}


# ------------------------------------------------------------------ inputs

def _randn(gen, *shape):
    return torch.randn(*shape, device=DEVICE, generator=gen)


def _rows_of(gen, rows, cols, dtype):
    """Normal values whose columns differ in size, a few of them by much, as features and activations do."""
    size = torch.exp(0.5 * _randn(gen, cols))
    size = torch.where(torch.rand(cols, device=DEVICE, generator=gen) < 0.01, 10 * size, size)
    return (_randn(gen, rows, cols) * size).to(dtype)


def _choices(gen, rows, choices, experts):
    """Each entry's expert: some experts are asked for far more than others, one entry in 50 has none (-1)."""
    liked = torch.softmax(_randn(gen, experts), 0).cumsum(0)
    index = torch.searchsorted(liked, torch.rand(rows, choices, device=DEVICE, generator=gen)).clamp_max(experts - 1)
    return torch.where(torch.rand(rows, choices, device=DEVICE, generator=gen) < 0.02, torch.full_like(index, -1), index)


def _count(index, experts):
    """The entries of experts below e, for e = 0 .. experts."""
    place = torch.sort(torch.where((index < 0) | (index >= experts), torch.full_like(index, experts), index).flatten())[0]
    return torch.searchsorted(place, torch.arange(experts + 1, device=DEVICE)).to(torch.int32)


def _stack(gen, experts, outs, cols, dtype):
    """Weights and biases of one layer of every expert."""
    weight = (_randn(gen, experts, outs, cols) / math.sqrt(cols)).to(dtype)
    return weight, (0.1 * _randn(gen, experts, outs)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, cols, train, dtype = case["kind"], case["cols"], case["train"], DTYPES[case["dtype"]]
    if kind == "norm":
        rows = case["rows"]
        x = (_rows_of(gen, rows, cols, torch.float32) + 0.5 * _randn(gen, rows, 1)).to(dtype)
        s = dict(case, x=x, w=1 + 0.2 * _randn(gen, cols), b=0.1 * _randn(gen, cols))
        wanted = ("x", "w", "b")
        if train:
            s["dy"] = _randn(gen, rows, cols).to(dtype)
    elif kind == "sort":
        rows, choices = case["rows"], case["choices"]
        s = dict(case, x=_rows_of(gen, rows, cols, dtype), index=_choices(gen, rows, choices, case["experts"]),
                 results=_rows_of(gen, rows * choices, cols, dtype),
                 weight=torch.sigmoid(_randn(gen, rows, choices)))
        wanted = ("x", "results", "weight")
        if train:
            s["dy"] = _randn(gen, rows, cols).to(dtype)
            s["d_sorted"] = _randn(gen, rows * choices, cols).to(dtype)
    else:
        slots, experts, outs = case["slots"], case["experts"], case["outs"]
        s = dict(case, x=_rows_of(gen, slots, cols, dtype),
                 offsets=_count(_choices(gen, slots, 1, experts), experts))
        s["w1"], s["b1"] = _stack(gen, experts, outs if kind == "linear" else case["hidden"], cols, dtype)
        wanted = ("x", "w1", "b1")
        if train:
            s["dy"] = (_randn(gen, slots, outs) / math.sqrt(slots)).to(dtype)
        if kind == "mlp":
            s["w2"], s["b2"] = _stack(gen, experts, outs, case["hidden"], dtype)
            wanted += ("w2", "b2")
            # Rows with a hidden value within rounding of the ReLU's kink, where either side's gradient is right, get no
            # upstream.
            for e, lo, hi in _spans(s["offsets"]):
                x, w, b = s["x"][lo:hi], s["w1"][e], s["b1"][e]
                near = (cols + 3) * 2.0 ** -23 * (x.abs() @ w.abs().T + b.abs())
                s["dy"][lo:hi] *= ~((x @ w.T + b).abs() <= near).any(1, keepdim=True)
    s["leaves"] = [s[n].requires_grad_(train) for n in wanted]
    return s


# ------------------------------------------------------------------ the plain forms

def _spans(offsets):
    """(expert, first place, place past the last) of the experts that have rows."""
    at = offsets.tolist()
    return [(e, at[e], at[e + 1]) for e in range(len(at) - 1) if at[e + 1] > at[e]]


def _plain_norm(s):
    x, w, b = s["x"].float(), s["w"], s["b"]
    d = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    h = d * r
    y = (h * w + b).to(s["x"].dtype)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return y, dx.to(y.dtype), (dy * h).sum(0), dy.sum(0)


def _plain_sort(s):
    index, experts, dtype = s["index"], s["experts"], s["x"].dtype
    rows, choices = index.shape
    has = (index >= 0) & (index < experts)
    place, source = torch.sort(torch.where(has, index, torch.full_like(index, experts)).flatten(), stable=True)
    offsets = torch.searchsorted(place, torch.arange(experts + 1, device=DEVICE))
    slot = torch.empty_like(source)
    slot[source] = torch.arange(rows * choices, device=DEVICE)
    slot = slot.view(rows, choices)
    of, behind = source // choices, (place == experts)[:, None]  # the row that each place comes from
    x_sorted = s["x"][of].masked_fill(behind, 0)
    results, weight = s["results"].float(), torch.where(has, s["weight"], torch.zeros_like(s["weight"]))
    y = sum(weight[:, j, None] * torch.where(has[:, j, None], results[slot[:, j]], torch.zeros((), device=DEVICE))
            for j in range(choices))
    out = [a.to(torch.int32) for a in (offsets, torch.where(has, slot, ~slot), source)] + [x_sorted, y.to(dtype)]
    if not s["train"]:
        return out
    dy, d_sorted = s["dy"].float(), s["d_sorted"].float()
    dx = sum(torch.where(has[:, j, None], d_sorted[slot[:, j]], torch.zeros((), device=DEVICE)) for j in range(choices))
    d_results = weight.flatten()[source][:, None] * dy[of]
    d_weight = torch.where(has, (results[slot.flatten()] * dy.repeat_interleave(choices, 0)).sum(-1).view(rows, choices),
                           torch.zeros_like(weight))
    return out + [dx.to(dtype), d_results.to(dtype), d_weight]


def _plain_layers(s):
    x, offsets, dtype = s["x"].float(), s["offsets"], s["x"].dtype
    layers = [(s["w1"], s["b1"])] + ([(s["w2"], s["b2"])] if s["kind"] == "mlp" else [])
    y = torch.zeros(len(x), layers[-1][0].shape[1], device=DEVICE)
    if s["train"]:
        dx, dy = torch.zeros_like(x), s["dy"].float()
        grads = [torch.zeros(p.shape, device=DEVICE) for layer in layers for p in layer]
    for e, lo, hi in _spans(offsets):
        inputs = [x[lo:hi]]
        for i, (w, b) in enumerate(layers):
            out = inputs[i] @ w[e].float().T + b[e].float()
            inputs.append(torch.relu(out) if i + 1 < len(layers) else out)
        y[lo:hi] = inputs[-1]
        if s["train"]:
            d = dy[lo:hi]
            for i in reversed(range(len(layers))):
                grads[2 * i][e], grads[2 * i + 1][e] = d.T @ inputs[i], d.sum(0)
                d = d @ layers[i][0][e].float()
                if i:
                    d = torch.where(inputs[i] > 0, d, torch.zeros_like(d))
            dx[lo:hi] = d
    if not s["train"]:
        return y.to(dtype)
    return tuple(t.to(dtype) for t in (y, dx, *grads))


def run(state):
    s = state
    kind, train = s["kind"], s["train"]
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "sort": _plain_sort}.get(kind, _plain_layers)(s)
    from npa_amd import experts, norm
    if kind == "norm":
        y = norm.layer_norm(s["x"], s["w"], s["b"], EPS)
    elif kind == "linear":
        y = experts.linear(s["x"], s["w1"], s["b1"], s["offsets"])
    elif kind == "mlp":
        y = experts.mlp(s["x"], s["w1"], s["b1"], s["w2"], s["b2"], s["offsets"])
    else:
        routing = experts.sort_rows(s["index"], s["experts"])
        x_sorted = experts.dispatch(s["x"], routing)
        y = experts.combine(s["results"], s["weight"], routing)
        out = (routing.offsets, routing.slot, routing.source, x_sorted.detach(), y.detach())
        if not train:
            return out
        return (*out, *torch.autograd.grad([x_sorted, y], s["leaves"], [s["d_sorted"], s["dy"]]))
    return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])) if train else y


# ------------------------------------------------------------------ 64 bits

def _exact_norm(s):
    x, w, b, n = s["x"].double(), s["w"].double(), s["b"].double(), s["cols"]
    mean = x.sum(1) / n
    square = torch.einsum("rc,rc->r", x - mean[:, None], x - mean[:, None]) / n
    h = (x - mean[:, None]) * (square + EPS).pow(-0.5)[:, None]
    y = torch.addcmul(b, h, w)
    if not s["train"]:
        return y
    dy = s["dy"].double()
    inner = (dy @ w / n)[:, None] + h * (torch.einsum("rc,rc->r", dy * h, w.expand_as(h)) / n)[:, None]
    return y, (dy * w - inner) * (square + EPS).pow(-0.5)[:, None], torch.einsum("rc,rc->c", dy, h), dy.sum(dim=0)


def _exact_sort(s):
    index, experts = s["index"], s["experts"]
    rows, choices = index.shape
    flat = index.flatten()
    key = torch.where((flat < 0) | (flat >= experts), experts, flat)
    # places by counting: expert after expert, each one's entries in their order
    source = torch.cat([torch.nonzero(key == e).flatten() for e in range(experts + 1)])
    sizes = torch.bincount(key, minlength=experts + 1)
    offsets = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)[:experts]])
    slot = torch.argsort(source)
    live = int(offsets[-1])
    row = source[:live] // choices
    x_sorted = torch.zeros(rows * choices, s["cols"], dtype=torch.float64, device=DEVICE)
    x_sorted[:live] = s["x"].double()[row]
    weight, results = s["weight"].double().flatten(), s["results"].double()
    y = torch.zeros(rows, s["cols"], dtype=torch.float64, device=DEVICE)
    y.index_add_(0, row, results[:live] * weight[source[:live], None])
    out = (offsets.int(), torch.where(key == experts, -1 - slot, slot).view(rows, choices).int(), source.int(), x_sorted, y)
    if not s["train"]:
        return out
    dy = s["dy"].double()
    dx = torch.zeros_like(y).index_add_(0, row, s["d_sorted"].double()[:live])
    d_results = torch.zeros_like(results)
    d_results[:live] = dy[row] * weight[source[:live], None]
    d_weight = torch.zeros_like(weight)
    d_weight[source[:live]] = torch.einsum("pc,pc->p", results[:live], dy[row])
    return (*out, dx, d_results, d_weight.view(rows, choices))


def _exact_layers(s):
    names = ["x", "w1", "b1"] + (["w2", "b2"] if s["kind"] == "mlp" else [])
    x, w1, b1, *last = (s[n].detach().double() for n in names)
    at = s["offsets"].cpu().numpy()
    y = x.new_zeros(len(x), s["outs"])
    outs = [y]
    if s["train"]:
        outs += [torch.zeros_like(t) for t in (x, w1, b1, *last)]
    for e in range(len(at) - 1):
        rows = slice(int(at[e]), int(at[e + 1]))
        a = torch.addmm(b1[e], x[rows], w1[e].t())
        h = a.clamp(min=0)
        y[rows] = torch.addmm(last[1][e], h, last[0][e].t()) if last else a
        if s["train"]:
            da = s["dy"].double()[rows]
            if last:
                outs[4][e], outs[5][e] = torch.mm(da.t(), h), da.sum(dim=0)
                da = torch.mm(da, last[0][e]) * (a > 0)
            outs[1][rows], outs[2][e], outs[3][e] = torch.mm(da, w1[e]), torch.mm(da.t(), x[rows]), da.sum(dim=0)
    return tuple(outs) if s["train"] else y


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        for leaf in s["leaves"]:
            leaf.requires_grad_(False)
        return {"norm": _exact_norm, "sort": _exact_sort}.get(case["kind"], _exact_layers)(s)
