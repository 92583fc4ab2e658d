"""The operators around a quantised projection when one model serves many requests, as cases to be timed.

Two operators of the package's public entry points:

    adapters   `forward_adapters`: layers that share their input, with a low-rank adapter for each request of the batch
    block      `block_norm` (16- and 32-bit results) and `forward_block_norm` (results that go straight into projections):
               the norm behind a block, its gate and residual scale, and the norm and modulation in front of the next one

    listed()          the named cases
    draw(rng)         one more case of the same ranges
    prepare(case, s)  what a program holds before the call: layers, adapters, activations, vectors
    run(state)        one pass: the package's operators where `own` is true, elementary torch operations else
    work(case)        bytes and operations the pass cannot do without
    exact(case, s)    the results in 64 bits
"""
from __future__ import annotations

import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SMALL_BATCH = 16   # rows up to which a layer multiplies its activations unquantised


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # Four requests that generate one token each, every one with an adapter of its own: the smallest call.
        {"name": "adapters_4x4096_4096_tokens", "kind": "adapters", "rows": 4, "width": 4096, "outs": "4096", "requests": 4, "count": 8,
         "ranks": "16", "dtype": "bf16", "rotate": False, "bias": False},
        # A full batch of single tokens through separate q, k and v projections, adapters of mixed ranks out of a stock of 32.
        {"name": "adapters_64x4096_qkv_tokens", "kind": "adapters", "rows": 64, "width": 4096, "outs": "4096 1024 1024", "requests": 64,
         "count": 32, "ranks": "8 16 32 64", "dtype": "bf16", "rotate": False, "bias": False},
        # Seven requests of unequal lengths packed into one batch, rotated weights, some requests without an adapter.
        {"name": "adapters_1357x2560_6912_packed", "kind": "adapters", "rows": 1357, "width": 2560, "outs": "6912", "requests": 7,
         "count": 5, "ranks": "4 16 48", "dtype": "fp16", "rotate": True, "bias": True},
        # Widths that fit no tile and ranks that are no multiple of anything: pruned layers.
        {"name": "adapters_333x1160_1001_odd", "kind": "adapters", "rows": 333, "width": 1160, "outs": "1001", "requests": 5, "count": 3,
         "ranks": "5 13", "dtype": "bf16", "rotate": False, "bias": True},
        # Four images of 1024 tokens, an adapter of rank 32 for each, through separate q, k and v projections.
        {"name": "adapters_4096x3840_qkv_images", "kind": "adapters", "rows": 4096, "width": 3840, "outs": "3840 3840 3840", "requests": 4,
         "count": 6, "ranks": "32", "dtype": "bf16", "rotate": False, "bias": False},
        # The up projection of a feed-forward on a batch of eight larger images, adapters of rank 64 and 128: the largest call.
        {"name": "adapters_9216x3840_15360_images", "kind": "adapters", "rows": 9216, "width": 3840, "outs": "15360", "requests": 8,
         "count": 8, "ranks": "64 128", "dtype": "bf16", "rotate": False, "bias": True},
        # One generated token for each of two requests between two blocks.
        {"name": "block_2x4096_tokens", "kind": "block", "rows": 2, "width": 4096, "vectors": 0, "post": "rms", "pre": "rms", "gate": "",
         "scale": False, "shift": False, "residual_scale": 1.0, "branch_scale": 0.22, "dtype": "bf16"},
        # Two images of 1024 tokens between a block's attention and its feed-forward: tanh gate and scale of each image.
        {"name": "block_2048x3840_images", "kind": "block", "rows": 2048, "width": 3840, "vectors": 2, "post": "rms", "pre": "rms",
         "gate": "tanh", "scale": True, "shift": False, "residual_scale": 1.0, "branch_scale": 1.0, "dtype": "bf16"},
        # A width that fits no vector load, with layer norms and their biases.
        {"name": "block_777x1001_odd", "kind": "block", "rows": 777, "width": 1001, "vectors": 7, "post": "layer", "pre": "layer",
         "gate": "plain", "scale": True, "shift": True, "residual_scale": 0.8, "branch_scale": 1.0, "dtype": "fp16"},
        # A residual stream kept in 32 bits.
        {"name": "block_4096x2048_fp32", "kind": "block", "rows": 4096, "width": 2048, "vectors": 4, "post": "rms", "pre": "layer",
         "gate": "plain", "scale": True, "shift": True, "residual_scale": 1.0, "branch_scale": 1.0, "dtype": "fp32"},
        # A long batch through a wide model.
        {"name": "block_16384x5120", "kind": "block", "rows": 16384, "width": 5120, "vectors": 8, "post": "rms", "pre": "rms",
         "gate": "tanh", "scale": True, "shift": False, "residual_scale": 1.0, "branch_scale": 1.0, "dtype": "bf16"},
        # The same step in front of the two up projections of a gated feed-forward, quantised on the way.
        {"name": "block_4096x3840_into_2x10240", "kind": "projected", "rows": 4096, "width": 3840, "outs": "10240 10240", "vectors": 4,
         "post": "rms", "pre": "rms", "gate": "tanh", "scale": True, "shift": False, "residual_scale": 1.0, "branch_scale": 1.0,
         "dtype": "bf16", "rotate": False, "bias": False},
    ]


def _ints(text):
    return [int(v) for v in text.split()]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi // step * step, max(-(-lo // step) * step, round(v / step) * step))


def _cost(case):
    """Seconds of a pass at rates near the card's (layers of odd widths are slower), to keep drawn cases within the largest listed one."""
    w = work(case)
    odd = "outs" in case and (case["width"] % 16 or any(n % 8 for n in _ints(case["outs"])))
    return w["flops"] / (3e13 if odd else 2e15) + w["bytes"] / 4e12


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        case = _draw_one(rng)
        if _cost(case) <= limit:
            return case


def _draw_one(rng):
    kind = rng.choice(["adapters", "adapters", "adapters", "block", "block", "projected"])
    rotate = rng.random() < 0.25
    odd = rng.random() < 0.25
    step = 128 if rotate else 1 if odd else 16
    if kind == "adapters":
        requests = _log_int(rng, 1, 128)
        rows = requests * 1 if rng.random() < 0.4 else max(requests, _log_int(rng, 1, 8192))
        ranks = " ".join(str(_log_int(rng, 1, 128)) for _ in range(rng.randint(1, 4)))
        outs = " ".join(str(_log_int(rng, 256, 8192, 1 if odd else 8)) for _ in range(rng.choice([1, 1, 2, 3])))
        return {"kind": kind, "rows": rows, "width": _log_int(rng, 256, 6144, step), "outs": outs, "requests": requests,
                "count": _log_int(rng, 1, 32), "ranks": ranks, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "rotate": rotate,
                "bias": rng.random() < 0.4}
    vectors = rng.choice([0, 1, 2, 4, 8])
    rows = max(1, vectors) * _log_int(rng, 1, 2048)
    case = {"kind": kind, "rows": rows, "vectors": vectors, "post": rng.choice(["rms", "rms", "layer", ""]), "pre": rng.choice(["rms", "rms", "layer"]),
            "gate": rng.choice(["tanh", "plain", ""]) if vectors else "", "scale": vectors > 0 and rng.random() < 0.7,
            "shift": vectors > 0 and rng.random() < 0.4, "residual_scale": rng.choice([1.0, 1.0, 0.8]), "branch_scale": rng.choice([1.0, 1.0, 0.22])}
    if kind == "block":
        return {**case, "width": _log_int(rng, 64, 8192, 1 if odd else 16), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    outs = " ".join(str(_log_int(rng, 256, 10240, 8)) for _ in range(rng.choice([1, 2, 3])))
    return {**case, "width": _log_int(rng, 256, 6144, 128 if rotate else 16), "outs": outs, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "rotate": rotate, "bias": rng.random() < 0.4}


# --------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *size, std=1.0, dtype=torch.float32):
    return (torch.randn(*size, generator=g, device="cuda") * std).to(dtype)


def _activations(g, rows, width, dtype):
    """Tokens as they come out of a block: a few channels far larger than the others."""
    x = _normal(g, rows, width)
    x[:, torch.randperm(width, generator=g, device="cuda")[: max(1, width // 500)]] *= 12
    return x.to(dtype)


def _layers(case, g):
    """Weights of the projections as a checkpoint holds them: int8 with one scale per row, and a bias."""
    dtype, width = DTYPES[case["dtype"]], case["width"]
    layers = []
    for n in _ints(case["outs"]):
        weight = torch.clamp(torch.round(_normal(g, n, width, std=31.0)), -127, 127).to(torch.int8)
        scale = (torch.rand(n, 1, generator=g, device="cuda") + 0.5) / (31.0 * width ** 0.5)
        layers.append({"weight": weight, "scale": scale, "bias": _normal(g, n, std=0.1, dtype=dtype) if case["bias"] else None})
    return layers


def _requests(case, seed):
    """Rows of each request (they fill the batch) and the adapter of each, -1 for none."""
    rng = random.Random(seed)
    rows, n = case["rows"], case["requests"]
    weights = [rng.uniform(0.3, 1.0) for _ in range(n)]
    lengths = [1 + int((rows - n) * w / sum(weights)) for w in weights]
    lengths[0] += rows - sum(lengths)
    return lengths, [rng.randrange(case["count"]) if rng.random() > 0.1 else -1 for _ in range(n)]


def _adapters(case, seed):
    """(down, up, scale) of every adapter for every layer; their ranks repeat those of the case."""
    g, dtype, width = _generator(seed), DTYPES[case["dtype"]], case["width"]
    ranks = _ints(case["ranks"])
    return [[(_normal(g, ranks[i % len(ranks)], width, std=width ** -0.5, dtype=dtype),
              _normal(g, n, ranks[i % len(ranks)], std=0.3 * ranks[i % len(ranks)] ** -0.5, dtype=dtype), 0.5 + 0.25 * (i % 4))
             for i in range(case["count"])] for n in _ints(case["outs"])]


def _vectors(case, seed):
    """The operands of a block's norms, gate and modulation."""
    g, dtype, width, v = _generator(seed), DTYPES[case["dtype"]], case["width"], case["vectors"]
    weight = lambda: (1.0 + _normal(g, width, std=0.2)).to(dtype)  # noqa: E731
    state = {"y": _activations(g, case["rows"], width, dtype), "residual": _activations(g, case["rows"], width, dtype)}
    state["post_weight"] = weight() if case["post"] else None
    state["post_bias"] = _normal(g, width, std=0.2, dtype=dtype) if case["post"] == "layer" else None
    state["pre_weight"] = weight()
    state["pre_bias"] = _normal(g, width, std=0.2, dtype=dtype) if case["pre"] == "layer" else None
    state["gate"] = _normal(g, v, 1, width, std=0.7, dtype=dtype) if case["gate"] else None
    state["mod_scale"] = _normal(g, v, 1, width, std=0.3, dtype=dtype) if case["scale"] else None
    state["mod_shift"] = _normal(g, v, 1, width, std=0.3, dtype=dtype) if case["shift"] else None
    if v:   # a batch of v images
        state["y"], state["residual"] = (state[k].view(v, -1, width) for k in ("y", "residual"))
    return state


def prepare(case, seed):
    state = {"case": dict(case)}
    if case["kind"] == "adapters":
        lengths, which = _requests(case, seed)
        ids = torch.tensor([a for a, n in zip(which, lengths) for _ in range(n)], dtype=torch.int32)
        state["ids"] = ids.to("cuda")
        state["x"] = _activations(_generator(seed), case["rows"], case["width"], DTYPES[case["dtype"]])
        adapters = _adapters(case, seed + 1)
    else:
        state.update(_vectors(case, seed))
    if "outs" in case:
        layers = _layers(case, _generator(seed + 2))
        if not own:
            state["layers"] = layers
        else:
            state["layers"] = [_linear(case, p) for p in layers]
    if case["kind"] == "adapters":
        if own:
            state["banks"] = [_package().AdapterBank(a) for a in adapters]
        else:   # the factors of a layer's adapters side by side, and which adapter each of their columns belongs to
            state["banks"] = [(torch.cat([down.float() * s for down, _, s in a]), torch.cat([up.float() for _, up, _ in a], 1),
                               torch.cat([torch.full((down.shape[0],), i, device="cuda") for i, (down, _, _) in enumerate(a)])) for a in adapters]
    return state


def _package():
    from __graft_entry__ import load_package

    return load_package()


def _linear(case, p):
    layer = _package().Int8TensorwiseOps.Linear(case["width"], p["weight"].shape[0], bias=case["bias"], device="meta")
    state = {"weight": p["weight"], "weight_scale": p["scale"]}
    if case["bias"]:
        state["bias"] = p["bias"]
    layer._load_from_state_dict(state, "", {}, True, [], [], [])
    layer._use_quarot = case["rotate"]
    return layer


# --------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["kind"] == "adapters":
        return _run_adapters(state)
    options = {k: state[k] for k in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias", "mod_scale", "mod_shift")}
    options.update(post_norm=case["post"] or None, pre_norm=case["pre"], gate_tanh=case["gate"] == "tanh",
                   residual_scale=case["residual_scale"], branch_scale=case["branch_scale"])
    if own:
        if case["kind"] == "block":
            return _package().block_norm(state["y"], state["residual"], **options)
        return _package().forward_block_norm(state["layers"], state["y"], state["residual"], **options)
    dtype = state["y"].dtype
    x, h = _block_norm(state["y"], state["residual"], **options)
    if case["kind"] == "block":
        return x.to(dtype), h.to(dtype)
    h = h.to(dtype)
    quantised = _quantise(h.reshape(-1, h.shape[-1]), case["rotate"]) if case["rows"] > SMALL_BATCH else None
    return x.to(dtype), [_project(h, quantised, p, case["rotate"]).to(dtype) for p in state["layers"]]


def _run_adapters(state):
    x, ids, rotate = state["x"], state["ids"], state["case"]["rotate"]
    if own:
        return _package().forward_adapters(state["layers"], x, state["banks"], ids)
    quantised = _quantise(x, rotate) if x.shape[0] > SMALL_BATCH else None
    outs = []
    for layer, (down, up, owner) in zip(state["layers"], state["banks"]):
        t = (x.float() @ down.t()) * (ids[:, None] == owner)
        outs.append((_project(x, quantised, layer, rotate) + t @ up.t()).to(x.dtype))
    return outs


def _hadamard():
    h = torch.ones(1, 1, device="cuda")
    while h.shape[0] < 128:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return h


def _rotated(x):
    """Every 128 values of a row times the normalised Hadamard matrix of their type (181 / 2048 in 16 bits), rounded to it."""
    return ((x.float().view(x.shape[0], -1, 128) @ _hadamard()) * 0.08837890625).view(x.shape).to(x.dtype)


def _quantise(x, rotate):
    x = (_rotated(x) if rotate else x).float()
    scale = torch.clamp(x.abs().amax(1, keepdim=True) / 127.0, min=1e-30)
    return torch.round(x * (1.0 / scale)), scale


def _project(x, quantised, p, rotate):
    """A layer's product in 32 bits: of int8 rows, or of up to 16 rows as they are with the weight widened to their type."""
    if quantised is None:
        rows = x.reshape(-1, x.shape[-1])
        weight = (p["weight"].float() * p["scale"]).to(x.dtype).float()
        y = (_rotated(rows) if rotate else rows).float() @ weight.t()
    else:
        q, scale = quantised
        y = (q @ p["weight"].float().t()) * (scale * p["scale"].view(1, -1))
    y = y if p["bias"] is None else y + p["bias"].float()
    return y.view(*x.shape[:-1], -1)


def _norm(x, kind, weight, bias, eps=1e-6):
    if kind is None:
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    x = x if weight is None else x * weight.float()
    return x if bias is None else x + bias.float()


def _block_norm(y, residual, *, post_norm, post_weight, post_bias, gate, gate_tanh, residual_scale, branch_scale, pre_norm, pre_weight, pre_bias,
                mod_scale, mod_shift):
    branch = _norm(y.float(), post_norm, post_weight, post_bias) * branch_scale
    if gate is not None:
        branch = branch * (torch.tanh(gate.float()) if gate_tanh else gate.float())
    x = residual.float() * residual_scale + branch
    h = _norm(x, pre_norm, pre_weight, pre_bias)
    h = h if mod_scale is None else h * (1.0 + mod_scale.float())
    return x, h if mod_shift is None else h + mod_shift.float()


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    rows, width, size = case["rows"], case["width"], 4 if case["dtype"] == "fp32" else 2
    nbytes = flops = 0
    if "outs" in case:
        for n in _ints(case["outs"]):
            nbytes += n * width + 4 * n + rows * n * 2 + (2 * n if case["bias"] else 0)
            flops += 2 * rows * n * width
    if case["kind"] == "adapters":
        nbytes += rows * width * 2 + 4 * rows
        lengths, which = _requests(case, 0)
        ranks = _ints(case["ranks"])
        for n in _ints(case["outs"]):
            nbytes += sum(2 * ranks[a % len(ranks)] * (width + n) for a in set(which) - {-1})
            flops += sum(2 * length * ranks[a % len(ranks)] * (width + n) for length, a in zip(lengths, which) if a >= 0)
    else:
        streams = 4 if case["kind"] == "block" else 3   # two read, x and h written; h goes no further than the projections
        vectors = case["vectors"] * sum(bool(case[k]) for k in ("gate", "scale", "shift")) + 4
        nbytes += (streams * rows + vectors) * width * size
        flops += 25 * rows * width
    return {"bytes": nbytes, "flops": flops}


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The same results from the formulas, row blocks and requests one by one, in 64 bits.  (An int8 row is what the layers'
    quantiser defines, in the 32-bit operations that it is defined by.)"""
    if case["kind"] == "adapters":
        return _exact_adapters(case, seed)
    v = _vectors(case, seed)
    width = case["width"]
    flat = {k: t.double().reshape(-1, width) for k, t in v.items() if t is not None}

    def norm(z, kind, name):
        if not kind:
            return z
        mean = z.sum(1, keepdim=True) / width if kind == "layer" else torch.zeros_like(z[:, :1])
        z = (z - mean) / (((z - mean) ** 2).sum(1, keepdim=True) / width + 1e-6).sqrt()
        if name + "_weight" in flat:
            z = z * flat[name + "_weight"]
        return z + flat[name + "_bias"] if name + "_bias" in flat else z

    per = case["rows"] // max(1, case["vectors"])
    xs, hs = [], []
    for i in range(max(1, case["vectors"])):
        part = slice(i * per, (i + 1) * per)
        branch = case["branch_scale"] * norm(flat["y"][part], case["post"], "post")
        if case["gate"]:
            branch = branch * (flat["gate"][i].tanh() if case["gate"] == "tanh" else flat["gate"][i])
        x = case["residual_scale"] * flat["residual"][part] + branch
        h = norm(x, case["pre"], "pre")
        if case["scale"]:
            h = h + h * flat["mod_scale"][i]
        if case["shift"]:
            h = h + flat["mod_shift"][i]
        xs.append(x)
        hs.append(h)
    x, h = torch.cat(xs), torch.cat(hs)
    if case["kind"] == "block":
        return x.view(v["y"].shape), h.view(v["y"].shape)
    rows = h.to(DTYPES[case["dtype"]])
    return x.view(v["y"].shape), [_exact_layer(rows, p, case).view(*v["y"].shape[:-1], -1) for p in _layers(case, _generator(seed + 2))]


def _exact_layer(rows, p, case):
    if case["rotate"]:
        order = torch.arange(128, device="cuda")
        bits = sum(((order[:, None] & order) >> b) & 1 for b in range(7))
        sign = 1.0 - 2.0 * (bits % 2).double()
        rows = torch.cat([(part.double() @ sign) * (181 / 2048) for part in rows.split(128, 1)], 1).to(rows.dtype)
    weight = p["weight"].double()
    if rows.shape[0] <= SMALL_BATCH:
        out = rows.double() @ (p["weight"].float() * p["scale"]).to(rows.dtype).double().t()
    else:
        top = rows.abs().amax(1).float() / torch.tensor(127.0, device="cuda")
        top = torch.where(top < 1e-30, torch.full_like(top, 1e-30), top)
        q = (rows.float() * top.reciprocal()[:, None]).round().double()
        out = (q @ weight.t()) * top.double()[:, None] * p["scale"].double().view(1, -1)
    return out if p["bias"] is None else out + p["bias"].double()


def _exact_adapters(case, seed):
    lengths, which = _requests(case, seed)
    x = _activations(_generator(seed), case["rows"], case["width"], DTYPES[case["dtype"]])
    outs = []
    for p, bank in zip(_layers(case, _generator(seed + 2)), _adapters(case, seed + 1)):
        out, at = _exact_layer(x, p, case), 0
        for length, a in zip(lengths, which):
            if a >= 0:
                down, up, s = bank[a]
                out[at:at + length] += s * ((x[at:at + length].double() @ down.double().t()) @ up.double().t())
            at += length
        outs.append(out)
    return outs
