"""The operators between the projections of an attention block, as cases to be timed.

Three operators of the package's public entry points:

    norm      `norm_heads`: the RMS norm of every head of queries and keys, with the rotation by their positions in the same pass
    rotate    `rotate_heads`: the rotation alone, over one to four position axes
    attend    `cross_attention`: queries over the keys and values of an encoder's states, another number of them and padded

    listed()          the named cases
    draw(rng)         one more case of the same ranges
    prepare(case, s)  what a program holds before the call: heads as the projections leave them, positions, lengths, masks
    run(state)        one pass: the package's operators where `own` is true, elementary torch operations else
    work(case)        bytes and operations the pass cannot do without
    exact(case, s)    the results in 64 bits
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # One new token for each of two requests, queries and fewer keys: the smallest call.
        {"name": "norm_2x1_32_8x128", "kind": "norm", "batch": 2, "tokens": 1, "heads": "32 8", "width": 128, "axes": "16 56 56", "theta": 10000.0,
         "pairs": "neighbours", "positions": "grid", "fused": False, "dtype": "bf16"},
        # Four images of 1024 tokens, queries and keys as views of one q, k, v projection.
        {"name": "norm_4x1024_30_30x128", "kind": "norm", "batch": 4, "tokens": 1024, "heads": "30 30", "width": 128, "axes": "32 48 48", "theta": 256.0,
         "pairs": "neighbours", "positions": "grid", "fused": True, "dtype": "bf16"},
        # A ragged batch of narrow heads, half of each rotated, pairs that lie apart.
        {"name": "norm_3x1357_16x72_apart", "kind": "norm", "batch": 3, "tokens": 1357, "heads": "16", "width": 72, "axes": "16 20", "theta": 10000.0,
         "pairs": "apart", "positions": "centred", "fused": False, "dtype": "fp16"},
        # A video of 21 x 30 x 52 tokens through a wide model.
        {"name": "norm_32760_40_40x128_video", "kind": "norm", "batch": 1, "tokens": 32760, "heads": "40 40", "width": 128, "axes": "44 42 42", "theta": 10000.0,
         "pairs": "neighbours", "positions": "grid", "fused": False, "dtype": "bf16"},
        # A few tokens of heads whose width fits no vector load.
        {"name": "rotate_77_5x37", "kind": "rotate", "batch": 1, "tokens": 77, "heads": "5 5", "width": 37, "axes": "10 14", "theta": 10000.0,
         "pairs": "neighbours", "positions": "grid", "fused": False, "dtype": "bf16"},
        # Two clips with positions in seconds and pixels, far from the origin, in 32 bits.
        {"name": "rotate_2x4096_32x64_fp32", "kind": "rotate", "batch": 2, "tokens": 4096, "heads": "32", "width": 64, "axes": "20 22 22", "theta": 10000.0,
         "pairs": "apart", "positions": "fraction", "fused": False, "dtype": "fp32"},
        # A pooling query over the 257 states of an image encoder.
        {"name": "attend_4x1_257_16x64", "kind": "attend", "batch": 4, "queries": 1, "keys": 257, "heads": 16, "kv_heads": 16, "width": 64, "mask": "",
         "fused": False, "dtype": "bf16"},
        # One new token over long states, several query heads to one of the states'.
        {"name": "attend_1_65536_32_8x128", "kind": "attend", "batch": 1, "queries": 1, "keys": 65536, "heads": 32, "kv_heads": 8, "width": 128, "mask": "",
         "fused": False, "dtype": "bf16"},
        # A ragged batch over masked states, narrow heads.
        {"name": "attend_2x1357_333_10x72", "kind": "attend", "batch": 2, "queries": 1357, "keys": 333, "heads": 10, "kv_heads": 10, "width": 72,
         "mask": "bool", "fused": True, "dtype": "fp16"},
        # Four images of 1024 tokens over text states of up to 512.
        {"name": "attend_4x1024_512_30x128", "kind": "attend", "batch": 4, "queries": 1024, "keys": 512, "heads": 30, "kv_heads": 30, "width": 128,
         "mask": "lengths", "fused": True, "dtype": "bf16"},
        # A video of 32760 tokens over 512 text states.
        {"name": "attend_32760_512_40x128", "kind": "attend", "batch": 1, "queries": 32760, "keys": 512, "heads": 40, "kv_heads": 40, "width": 128,
         "mask": "", "fused": False, "dtype": "bf16"},
        # Tokens of an image and a text over all of them: the largest call.
        {"name": "attend_8192_8192_40x128", "kind": "attend", "batch": 1, "queries": 8192, "keys": 8192, "heads": 40, "kv_heads": 40, "width": 128,
         "mask": "", "fused": False, "dtype": "bf16"},
    ]


def _ints(text):
    return [int(v) for v in text.split()]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi // step * step, max(-(-lo // step) * step, round(v / step) * step))


def _cost(case):
    """Seconds of a pass at rates near the card's, to keep drawn cases within the largest listed one of their kind.  (The exponentials of
    narrow heads cost what the products of wide ones do.)"""
    w = work(case)
    return w["flops"] * max(1.0, 128 / case["width"]) / 1e15 + w["bytes"] / 4e12


def draw(rng):
    while True:
        case = _draw_attend(rng) if rng.random() < 0.5 else _draw_heads(rng)
        if _cost(case) <= max(_cost(c) for c in listed() if (c["kind"] == "attend") == (case["kind"] == "attend")):
            return case


def _draw_attend(rng):
    kv_heads = _log_int(rng, 1, 40)
    return {"kind": "attend", "batch": rng.choice([1, 1, 2, 3, 4]), "queries": rng.choice([1, _log_int(rng, 1, 32768), _log_int(rng, 1, 32768)]),
            "keys": _log_int(rng, 1, 32768), "heads": kv_heads * rng.choice([1, 1, 2, 4]), "kv_heads": kv_heads,
            "width": rng.choice([64, 128, 128, 8 * rng.randint(1, 32), rng.randint(1, 256)]), "mask": rng.choice(["", "", "lengths", "bool", "float"]),
            "fused": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "fp16"])}


def _draw_heads(rng):
    width = rng.choice([64, 128, 128, 8 * rng.randint(1, 32), rng.randint(2, 256)])
    rotated = width // 2 if rng.random() < 0.7 else rng.randint(1, width // 2)   # pairs
    axes = rng.randint(1, min(4, rotated))
    cuts = sorted(rng.sample(range(1, rotated), axes - 1)) if axes > 1 else []
    dims = " ".join(str(2 * (b - a)) for a, b in zip([0, *cuts], [*cuts, rotated]))
    heads = _log_int(rng, 1, 40)
    case = {"kind": rng.choice(["norm", "norm", "rotate"]), "batch": rng.choice([1, 1, 2, 4]), "tokens": _log_int(rng, 1, 32768),
            "heads": rng.choice([f"{heads}", f"{heads} {heads}", f"{4 * heads} {heads}"]), "width": width, "axes": dims,
            "theta": rng.choice([10000.0, 256.0, 2000.0]), "pairs": rng.choice(["neighbours", "apart"]),
            "positions": rng.choice(["grid", "grid", "centred", "fraction", "far"]), "fused": rng.random() < 0.4, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if case["kind"] == "norm" and rng.random() < 0.2:
        case["axes"] = ""   # the norm alone
    return case


# --------------------------------------------------------------------------- inputs
def _normal(g, *size, std=1.0, dtype=torch.float32):
    return (torch.randn(*size, generator=g, device="cuda") * std).to(dtype)


def _positions(case, seed):
    """[tokens, axes] (or [batch, tokens, axes] where the clips begin at other times) of the grid that the tokens lie on, the last axis fastest."""
    n, axes = case["tokens"], len(_ints(case["axes"]))
    side = max(1, round(n ** (1 / axes))) if axes else 1
    index = torch.arange(n, device="cuda")
    grid = torch.stack([index // side ** (axes - 1 - a) if a == 0 else index // side ** (axes - 1 - a) % side for a in range(axes)], 1) if axes else index[:, None][:, :0]
    if case["positions"] == "centred":      # around the middle of the image
        return (grid - side // 2).to(torch.int32)
    if case["positions"] == "far":          # late in a long stream
        return grid + 1000003 + seed % 1000
    if case["positions"] == "fraction":     # seconds and pixels, of clips that begin at other times
        start = torch.arange(case["batch"], device="cuda")[:, None, None] * 731.25 + seed % 100
        return (grid[None].float() * 0.3203125 + start).float()
    return grid


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and "positions" in state:
        state["rotary"] = _package().RotaryAxes(_ints(case["axes"]), case["theta"], interleaved=case["pairs"] == "neighbours")
    return state


def _inputs(case, seed):
    g, dtype = torch.Generator(device="cuda").manual_seed(seed), DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    batch, width = case["batch"], case["width"]
    if case["kind"] == "attend":
        heads, kv_heads, queries, keys = (case[k] for k in ("heads", "kv_heads", "queries", "keys"))
        state["q"] = _normal(g, batch, queries, heads, width, std=1.5, dtype=dtype)
        if case["fused"]:   # views of one projection
            both = _normal(g, batch, keys, 2, kv_heads, width, std=1.5, dtype=dtype)
            state["k"], state["v"] = both[:, :, 0], both[:, :, 1]
        else:
            state["k"], state["v"] = (_normal(g, batch, keys, kv_heads, width, std=1.5, dtype=dtype) for _ in range(2))
        state.update(_masks(case, seed))
        return state
    sizes = _ints(case["heads"])
    if case["fused"]:       # queries, keys and values of one projection
        whole = _normal(g, batch, case["tokens"], sum(sizes) + sizes[-1], width, std=2.0, dtype=dtype)
        state["xs"] = list(whole.split([*sizes, sizes[-1]], 2))[:-1]
    else:
        state["xs"] = [_normal(g, batch, case["tokens"], n, width, std=2.0, dtype=dtype) for n in sizes]
    if case["kind"] == "norm":
        state["weights"] = [(1.0 + _normal(g, width, std=0.2)).to(dtype) for _ in sizes]
    if case["axes"]:
        state["positions"] = _positions(case, seed)
    return state


def _masks(case, seed):
    batch, keys = case["batch"], case["keys"]
    if case["mask"] == "lengths":       # states of each text, padded to the longest
        return {"key_lengths": torch.tensor(_lengths(case, seed), dtype=torch.int32, device="cuda")}
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    if case["mask"] == "bool":          # states that count
        return {"key_mask": torch.rand(batch, keys, generator=g, device="cuda") < 0.8}
    if case["mask"] == "float":         # logarithms of weights of the states, the lowest value for those that do not count
        dtype = DTYPES[case["dtype"]]
        kept = torch.rand(batch, keys, generator=g, device="cuda") < 0.9
        return {"key_mask": torch.where(kept, _normal(g, batch, keys, std=0.5, dtype=dtype), torch.full((), torch.finfo(dtype).min, dtype=dtype, device="cuda"))}
    return {}


def _lengths(case, seed):
    rng = random.Random(seed)
    return [rng.randint(case["keys"] // 4, case["keys"]) for _ in range(case["batch"])]


def _package():
    from __graft_entry__ import load_package

    return load_package()


# --------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if kind == "attend":
        masks = {k: state[k] for k in ("key_lengths", "key_mask") if k in state}
        if own:
            return _package().cross_attention(state["q"], state["k"], state["v"], **masks)
        return _attend(state["q"], state["k"], state["v"], **masks)
    if own and kind == "norm":
        return _package().norm_heads(state["xs"], state["weights"], eps=EPS, rotary=state.get("rotary"), positions=state.get("positions"))
    if own:
        return _package().rotate_heads(state["xs"], state["rotary"], state["positions"])
    turn = _turns(state["positions"], state["case"]) if "positions" in state else None
    weights = state.get("weights", [None] * len(state["xs"]))
    return [_rotate(_norm(x.float(), w), turn, state["case"]).to(x.dtype) for x, w in zip(state["xs"], weights)]


def _norm(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _turns(positions, case):
    """Cosine and sine of every pair's angle, for all heads alike; the angles in 64 bits, since positions may lie far out."""
    angles = torch.cat([positions[..., a:a + 1].double() * case["theta"] ** (-torch.arange(0, n, 2, device="cuda", dtype=torch.float64) / n)
                        for a, n in enumerate(_ints(case["axes"]))], -1).unsqueeze(-2)
    return angles.cos().float(), angles.sin().float()


def _rotate(x, turn, case):
    if turn is None:
        return x
    cos, sin = turn
    rotated, rest = x[..., :2 * cos.shape[-1]], x[..., 2 * cos.shape[-1]:]
    if case["pairs"] == "neighbours":
        a, b = rotated[..., 0::2], rotated[..., 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)
    a, b = rotated.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)


def _attend(q, k, v, key_lengths=None, key_mask=None):
    """softmax(q k^T / sqrt(width) + mask) v over the states that count, zeros where none does."""
    dtype, share = q.dtype, q.shape[2] // k.shape[2]
    q, k, v = (t.float().transpose(1, 2) for t in (q, k, v))
    k, v = (t.repeat_interleave(share, 1).contiguous() if share > 1 else t.contiguous() for t in (k, v))
    scores = q @ k.transpose(2, 3) / math.sqrt(q.shape[-1])
    if key_lengths is not None:
        counts = torch.arange(k.shape[2], device=q.device) < key_lengths[:, None]
        scores = scores.masked_fill(~counts[:, None, None], -math.inf)
    if key_mask is not None and key_mask.dtype == torch.bool:
        scores = scores.masked_fill(~key_mask[:, None, None], -math.inf)
    elif key_mask is not None:
        scores = torch.where((key_mask > torch.finfo(key_mask.dtype).min)[:, None, None], scores + key_mask.float()[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return ((p @ v) / torch.where(total == 0, torch.ones_like(total), total)).transpose(1, 2).to(dtype)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "attend":
        states = sum(_lengths(case, 0)) if case["mask"] == "lengths" else case["batch"] * case["keys"]
        rows = case["batch"] * case["queries"] * case["heads"]
        masks = {"": 0, "lengths": 4 * case["batch"], "bool": states, "float": states * size}[case["mask"]]
        return {"bytes": (2 * rows + 2 * states * case["kv_heads"]) * case["width"] * size + masks,
                "flops": 4 * case["queries"] * case["heads"] * states * case["width"]}
    tokens = case["batch"] * case["tokens"]
    elements = tokens * sum(_ints(case["heads"])) * case["width"]
    positions = case["tokens"] * len(_ints(case["axes"])) * {"centred": 4, "fraction": 4 * case["batch"]}.get(case["positions"], 8)
    return {"bytes": 2 * elements * size + positions, "flops": (3 if case["axes"] else 0) * elements + (4 if case["kind"] == "norm" else 0) * elements}


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The same results from the formulas in 64 bits: every head by itself, the rotation as a product of complex numbers."""
    state = _inputs(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, state)
    outs = []
    for i, x in enumerate(state["xs"]):
        z = x.double()
        if case["kind"] == "norm":
            z = z / ((z * z).sum(-1, keepdim=True) / case["width"] + EPS).sqrt() * state["weights"][i].double()
        first = 0
        for a, n in enumerate(_ints(case["axes"])):
            pairs = torch.arange(first, first + n // 2, device="cuda")
            rate = torch.exp(-math.log(case["theta"]) * (pairs - first).double() * 2 / n)
            angle = state["positions"][..., a].double()[..., None, None] * rate
            half = sum(_ints(case["axes"])) // 2
            re, im = (2 * pairs, 2 * pairs + 1) if case["pairs"] == "neighbours" else (pairs, pairs + half)
            turned = torch.complex(z[..., re], z[..., im]) * torch.polar(torch.ones_like(angle), angle)
            z = z.index_copy(-1, re, turned.real).index_copy(-1, im, turned.imag)
            first += n // 2
        outs.append(z)
    return outs


def _exact_attend(case, state):
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        counts = torch.ones(case["keys"], dtype=torch.bool, device="cuda")
        added = torch.zeros(case["keys"], dtype=torch.float64, device="cuda")
        if "key_lengths" in state:
            counts[int(state["key_lengths"][b]):] = False
        if "key_mask" in state:
            mask = state["key_mask"][b]
            counts = mask if mask.dtype == torch.bool else mask != torch.finfo(mask.dtype).min
            added = added if mask.dtype == torch.bool else mask.double()
        if not bool(counts.any()):
            continue
        for h in range(case["heads"]):
            group = h // (case["heads"] // case["kv_heads"])
            k, v = (state[n][b, counts, group].double() for n in ("k", "v"))
            for at in range(0, case["queries"], 4096):
                q = state["q"][b, at:at + 4096, h].double()
                out[b, at:at + 4096, h] = torch.softmax(torch.mm(q, k.t()) * case["width"] ** -0.5 + added[counts], 1) @ v
    return out
