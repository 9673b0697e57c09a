"""The operators of blocks that mix tokens by a state instead of attention, and of their norm, as cases that can be timed and compared.

A case names its operator and sizes:

  norm   ``group_norm``: a group norm with its activation, over maps [images, channels, height, width] or rows of tokens, channels last
  conv   ``causal_conv``: the short convolution of every channel along the tokens of a ragged batch of sequences, and its activation
  scan   ``selective_scan``: the state space recurrence along the tokens, its skip and its gate

All numbers are float32.  Rows are tokens, one a row; the rows offsets[s] .. offsets[s + 1] - 1 are the new tokens of sequence s, lengths[s]
its tokens so far with the new ones.  What a sequence keeps between calls lies in a slot of a pool: the last width - 1 inputs [slots, width - 1,
channels] (oldest first), the scan's state [slots, channels, state].  A sequence reads slots[s] (unless it begins with the new
tokens) and leaves its state in out_slots[s]: here slots of their own, as a program does that keeps the state before the call.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # the smallest norm: the last map of a network for one 224 x 224 image
        _norm("norm_maps_1x512x7x7", images=1, channels=512, height=7, width=7, groups=32, rows=False, activation="silu"),
        # the first level of a U-Net on 512 x 512 images, a batch of 4: groups of half a million numbers, bound by memory
        _norm("norm_maps_4x64x512x512", images=4, channels=64, height=512, width=512, groups=32, rows=False, activation="relu"),
        # tokens of 64 images of 14 x 14, channels last, with a shift and a scale for every image
        _norm("norm_rows_64x196x768", images=64, channels=768, height=14, width=14, groups=32, rows=True, activation="silu", modulate=True),
        # odd sizes: 37 x 37 tokens, 330 channels in groups of 30
        _norm("norm_rows_3x1369x330", images=3, channels=330, height=37, width=37, groups=11, rows=True, activation="none"),
        # a serving step: one token of 32 sequences
        _conv("conv_32x1x1280", seqs=32, new=1, ragged=False, channels=1280, width=4, kept=True),
        # ragged prompts of eight sequences
        _conv("conv_8x2048x2048", seqs=8, new=2048, ragged=True, channels=2048, width=4, kept=True),
        # the smallest scan: one token of one sequence
        _scan("scan_1x1x384", seqs=1, new=1, ragged=False, channels=384, state=16, kept=True),
        # a serving step of a wide network: one token of 128 sequences, bound by the states' bytes
        _scan("scan_128x1x4096", seqs=128, new=1, ragged=False, channels=4096, state=16, kept=True),
        # whole images of 14 x 14 tokens, from the last token to the first: the backward half of a network that scans both ways
        _scan("scan_64x196x768_reverse", seqs=64, new=196, ragged=False, channels=768, state=16, kept=False, reverse=True),
        # a long prompt of one sequence of a wide network: the largest
        _scan("scan_1x8192x4096", seqs=1, new=8192, ragged=False, channels=4096, state=16, kept=True),
        # a video of 16 frames of 64 x 64 tokens through a narrow network: few channels, a long sequence, which has to be divided
        _scan("scan_1x65536x256", seqs=1, new=65536, ragged=False, channels=256, state=16, kept=False),
        # mixed work: ragged chunks, odd sizes, two groups of channels
        _scan("scan_7x301x1002_state12", seqs=7, new=301, ragged=True, channels=1002, state=12, kept=True, groups=2),
    ]


def _norm(name, images, channels, height, width, groups, rows, activation, modulate=False):
    return dict(name=name, op="norm", images=images, channels=channels, height=height, width=width, groups=groups, rows=rows, activation=activation, modulate=modulate)


def _conv(name, seqs, new, ragged, channels, width, kept, activation="silu", reverse=False):
    return dict(name=name, op="conv", seqs=seqs, new=new, ragged=ragged, channels=channels, width=width, kept=kept, activation=activation, reverse=reverse)


def _scan(name, seqs, new, ragged, channels, state, kept, groups=1, gate=True, softplus=True, reverse=False):
    return dict(name=name, op="scan", seqs=seqs, new=new, ragged=ragged, channels=channels, state=state, kept=kept, groups=groups, gate=gate, softplus=softplus,
                reverse=reverse)


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    op = rng.choice(("norm", "norm", "conv", "scan", "scan", "scan"))
    if op == "norm":
        groups = rng.choice((1, 2, 7, 8, 11, 16, 32, 32, 32))
        return _norm(None, _log(rng, 1, 64), groups * _log(rng, 1, 64), _log(rng, 1, 512), _log(rng, 1, 512), groups, rng.random() < 0.5, rng.choice(("none", "relu", "silu")),
                     rng.random() < 0.3)
    seqs, new, channels = _log(rng, 1, 128), rng.choice((1, _log(rng, 1, 16), _log(rng, 16, 8192), _log(rng, 64, 65536))), rng.choice((16 * _log(rng, 1, 320), _log(rng, 1, 5000)))
    ragged, kept, reverse = rng.random() < 0.5, rng.random() < 0.6, rng.random() < 0.3
    if op == "conv":
        return _conv(None, seqs, new, ragged, channels, rng.choice((2, 3, 4, 4, 4, 5, 8)), kept, rng.choice(("none", "silu", "silu")), reverse)
    groups = rng.choice((1, 1, 2, 4))
    return _scan(None, seqs, new, ragged, groups * -(-channels // groups), rng.choice((1, 4, 5, 8, 12, 16, 16, 16, 16, 24, 32, 64)), kept, groups, rng.random() < 0.8,
                 rng.random() < 0.8, reverse)


def draw(rng):
    while True:
        case = {k: v for k, v in _drawn(rng).items() if k != "name"}
        if case["op"] == "norm":
            if case["images"] * case["channels"] * case["height"] * case["width"] <= 6.7e7:
                return case
        elif case["seqs"] * case["new"] * case["channels"] * case.get("state", 16) <= 5.3e8 and case["seqs"] * case["channels"] * case.get("state", 1) <= 3.4e7:
            return case


# ------------------------------------------------------------------------------------------------- what a program has in hand
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _uniform(g, *shape):
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32)


def _news(case):
    """New tokens of every sequence: all alike, or spread up to the largest (the case's own, whatever the seed)."""
    n, new = case["seqs"], case["new"]
    news = np.full(n, new)
    if case["ragged"]:
        news = np.random.default_rng([n, new]).integers(1, new + 1, n)
        news[0] = new
    return news.astype(np.int32)


def _batch(case, seed):
    """Offsets, lengths and slots of the batch; every fourth sequence begins with its new tokens."""
    news, n = _news(case), case["seqs"]
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    order = np.random.default_rng(int(seed) + 1).permutation(2 * n)
    before = np.where(np.arange(n) % 4 == 3, 0, 100)
    return {"offsets": put(np.concatenate([[0], np.cumsum(news)])), "rows": int(news.sum()), "max_new": int(news.max()), "lengths": put(news + before),
            "slots": put(order[:n]), "out_slots": put(order[n:])}


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] == "norm":
        images, channels, pixels = case["images"], case["channels"], case["height"] * case["width"]
        offset, spread = 0.5 * _normal(g, 1, channels, 1), 0.5 + _uniform(g, 1, channels, 1)  # channels differ, as a convolution's do
        x = _normal(g, images, channels, pixels) * spread + offset
        x = x.transpose(1, 2).reshape(images * pixels, channels).contiguous() if case["rows"] else x.reshape(images, channels, case["height"], case["width"])
        state.update(x=x, out=torch.empty_like(x), weight=1.0 + 0.1 * _normal(g, channels), bias=0.1 * _normal(g, channels), mod=None, shift=None)
        if case["modulate"]:
            state.update(mod=0.2 * _normal(g, images, channels), shift=0.2 * _normal(g, images, channels))
        return state
    state.update(_batch(case, seed))
    rows, channels = state["rows"], case["channels"]
    xz = _normal(g, rows, 2 * channels)  # one dense layer brings the inputs of the convolution and the gate
    if case["op"] == "conv":
        state.update(xz=xz, out=torch.empty(rows, channels, device="cuda"), weight=_normal(g, channels, case["width"]) / math.sqrt(case["width"]),
                     bias=0.1 * _normal(g, channels), pool=_normal(g, 2 * case["seqs"], case["width"] - 1, channels) if case["kept"] else None)
        return state
    n, groups = case["state"], case["groups"]
    rank = -(-channels // 16)
    steps = torch.exp(_uniform(g, channels) * math.log(100.0) + math.log(0.001))  # time steps of 0.001 to 0.1
    state.update(
        xz=xz, x=torch.nn.functional.silu(_normal(g, rows, channels)), out=torch.empty(rows, channels, device="cuda"),
        proj=_normal(g, rows, rank + 2 * groups * n),  # one dense layer brings the low-rank time steps, the inputs' and the outputs' vectors
        dt=0.5 * _normal(g, rows, channels) if case["softplus"] else steps * torch.exp(0.3 * _normal(g, rows, channels)),
        dt_bias=steps + torch.log(-torch.expm1(-steps)) if case["softplus"] else None,
        A=-torch.arange(1, n + 1, device="cuda", dtype=torch.float32) * (0.8 + 0.4 * _uniform(g, channels, n)), skip=1.0 + 0.1 * _normal(g, channels),
        pool=_normal(g, 2 * case["seqs"], channels, n) if case["kept"] else None)
    return state


# ------------------------------------------------------------------------------------------------- the plain forms
def _activated(x, activation):
    return x if activation == "none" else x.clamp(min=0.0) if activation == "relu" else x / (1.0 + torch.exp(-x))


def _plain_norm(state):
    case, x = state["case"], state["x"]
    images, channels, groups, pixels = case["images"], case["channels"], case["groups"], case["height"] * case["width"]
    shape, over, each = ((images, pixels, groups, channels // groups), (1, 3), (-1, 1, groups, channels // groups)) if case["rows"] else \
        ((images, groups, channels // groups, pixels), (2, 3), (-1, groups, channels // groups, 1))
    x = x.reshape(shape)
    x = x - x.mean(over, keepdim=True)
    y = x / torch.sqrt((x * x).mean(over, keepdim=True) + 1e-5) * state["weight"].reshape(each) + state["bias"].reshape(each)
    if state["mod"] is not None:
        y = y * (1.0 + state["mod"].reshape(each)) + state["shift"].reshape(each)
    state["out"].copy_(_activated(y, case["activation"]).reshape(state["out"].shape))
    return state["out"]


def _places(state):
    """For every row its sequence and its number among the new tokens, in the order in which they are taken."""
    row = torch.arange(state["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(state["offsets"], row, right=True) - 1
    new = state["offsets"][1:] - state["offsets"][:-1]
    nth = row - state["offsets"][seq]
    return seq, new[seq] - 1 - nth if state["case"]["reverse"] else nth, new


def _before(state):
    """The states that the sequences continue, zeros for those that begin."""
    new = state["offsets"][1:] - state["offsets"][:-1]
    return state["pool"][state["slots"]] * (state["lengths"] > new)[:, None, None]


def _plain_conv(state):
    case = state["case"]
    seqs, channels, width = case["seqs"], case["channels"], case["width"]
    seq, nth, new = _places(state)
    x = torch.zeros(seqs, state["max_new"] + width - 1, channels, device="cuda")
    x[seq, nth + width - 1] = state["xz"][:, :channels]
    if case["kept"]:
        x[:, :width - 1] = _before(state)
    windows = x.unfold(1, width, 1)  # [seqs, new, channels, width]
    y = (windows * state["weight"]).sum(3) + state["bias"]
    state["out"].copy_(_activated(y, case["activation"])[seq, nth])
    if not case["kept"]:
        return state["out"]
    last = new[:, None] + torch.arange(width - 1, device="cuda")
    state["pool"][state["out_slots"]] = x.gather(1, last[:, :, None].expand(-1, -1, channels).long())
    return state["out"], state["pool"]


def _plain_scan(state):
    case = state["case"]
    seqs, channels, n, groups, new = case["seqs"], case["channels"], case["state"], case["groups"], state["max_new"]
    seq, nth, news = _places(state)
    rank = state["proj"].shape[1] - 2 * groups * n

    def padded(t):
        p = torch.zeros(seqs, new, t.shape[1], device="cuda")
        p[seq, nth] = t
        return p

    dt = state["dt"]
    if case["softplus"]:
        dt = dt + state["dt_bias"]
        dt = dt.clamp(min=0.0) + torch.log1p(torch.exp(-dt.abs()))
    dt, x = padded(dt), padded(state["x"])
    spread = lambda t: t.reshape(seqs, new, groups, 1, n).expand(-1, -1, -1, channels // groups, -1).reshape(seqs, new, channels, n)
    a = torch.exp(dt[..., None] * state["A"])
    h = spread(padded(state["proj"][:, rank:rank + groups * n])) * (dt * x)[..., None]
    if case["kept"]:
        h[:, 0].addcmul_(a[:, 0], _before(state))
    step = 1
    while step < new:  # after each step a place holds what the last 2 step tokens bring, and the factor of what came before
        h[:, step:] = torch.addcmul(h[:, step:], a[:, step:], h[:, :-step])
        if 2 * step < new:
            a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    y = (h * spread(padded(state["proj"][:, rank + groups * n:]))).sum(3)[seq, nth] + state["skip"] * state["x"]
    if case["gate"]:
        y = y * _activated(state["xz"][:, channels:], "silu")
    state["out"].copy_(y)
    if not case["kept"]:
        return state["out"]
    state["pool"][state["out_slots"]] = h[torch.arange(seqs, device="cuda"), news.long() - 1]
    return state["out"], state["pool"]


# ------------------------------------------------------------------------------------------------- the framework's calls
_device = None


def _handles(state):
    """The framework's view of what the program has in hand, made once."""
    global _device
    import eddl_amd
    from eddl_amd.state_space import StateBatch
    if _device is None:
        _device = eddl_amd.Backend(0)
    hip, case = _device, state["case"]
    wrap = lambda t: None if t is None else hip.wrap(t)
    h = {"hip": hip, "out": wrap(state["out"])}
    if case["op"] == "norm":
        h.update({k: wrap(state[k]) for k in ("x", "weight", "bias", "mod", "shift")})
        return h
    kept = {"lengths": wrap(state["lengths"]), "slots": wrap(state["slots"]), "out_slots": wrap(state["out_slots"])} if case["kept"] else {}
    channels, xz = case["channels"], wrap(state["xz"])
    h.update(batch=StateBatch(wrap(state["offsets"]), state["max_new"], **kept), pool=wrap(state["pool"]))
    if case["op"] == "conv":
        h.update(x=xz.columns(0, channels), weight=wrap(state["weight"]), bias=wrap(state["bias"]))
        return h
    proj, vectors = wrap(state["proj"]), case["groups"] * case["state"]
    rank = proj.shape[1] - 2 * vectors
    h.update({k: wrap(state[k]) for k in ("x", "dt", "A", "skip", "dt_bias")})
    h.update(B=proj.columns(rank, rank + vectors), C=proj.columns(rank + vectors, rank + 2 * vectors), gate=xz.columns(channels, 2 * channels) if case["gate"] else None)
    return h


def _run_own(state):
    case = state["case"]
    if "handles" not in state:
        state["handles"] = _handles(state)
    h = state["handles"]
    hip, activation = h["hip"], None if case.get("activation") == "none" else case.get("activation")
    if case["op"] == "norm":
        hip.group_norm(h["x"], h["out"], case["groups"], h["weight"], h["bias"], eps=1e-5, activation=activation, mod=h["mod"], shift=h["shift"],
                       image_rows=case["height"] * case["width"] if case["rows"] else None)
        return state["out"]
    if case["op"] == "conv":
        hip.causal_conv(h["x"], h["weight"], h["bias"], h["out"], h["batch"], states=h["pool"], activation=activation, reverse=case["reverse"])
    else:
        hip.selective_scan(h["x"], h["dt"], h["A"], h["B"], h["C"], h["out"], h["batch"], states=h["pool"], skip=h["skip"], gate=h["gate"], dt_bias=h["dt_bias"],
                           softplus=case["softplus"], reverse=case["reverse"])
    return (state["out"], state["pool"]) if case["kept"] else state["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _silu64(x):
    return x * torch.sigmoid(x)


def _exact_norm(state):
    case, w, b = state["case"], state["weight"].double(), state["bias"].double()
    channels, groups = case["channels"], case["groups"]
    x = state["x"].reshape(case["images"], -1, channels).movedim(2, 1) if case["rows"] else state["x"].flatten(2)
    out = []
    for i in range(case["images"]):
        image = x[i].double().reshape(groups, -1)
        var, mean = torch.var_mean(image, dim=1, unbiased=False, keepdim=True)
        y = ((image - mean) * torch.rsqrt(var + 1e-5)).reshape(channels, -1) * w[:, None] + b[:, None]
        if state["mod"] is not None:
            y = y + y * state["mod"][i].double()[:, None] + state["shift"][i].double()[:, None]
        out.append(torch.relu(y) if case["activation"] == "relu" else _silu64(y) if case["activation"] == "silu" else y)
    y = torch.stack(out)
    return y.movedim(1, 2).reshape(state["out"].shape) if case["rows"] else y.reshape(state["out"].shape)


def _sequences(state):
    """(first row, last row + 1, whether it continues a state, the slot read, the slot written) of every sequence."""
    at, length = state["offsets"].tolist(), state["lengths"].tolist()
    return [(at[s], at[s + 1], state["case"]["kept"] and length[s] > at[s + 1] - at[s], state["slots"][s].item(), state["out_slots"][s].item()) for s in range(len(length))]


def _exact_conv(state):
    case = state["case"]
    channels, width = case["channels"], case["width"]
    w, out = state["weight"].double(), torch.empty(state["rows"], channels, dtype=torch.float64, device="cuda")
    pool = state["pool"].double() if case["kept"] else None
    for first, last, continues, read, write in _sequences(state):
        x = state["xz"][first:last, :channels].double()
        if case["reverse"]:
            x = x.flip(0)
        x = torch.cat([pool[read] if continues else x.new_zeros(width - 1, channels), x])
        y = torch.conv1d(x.T[None], w[:, None], state["bias"].double(), groups=channels)[0].T
        y = _silu64(y) if case["activation"] == "silu" else y
        out[first:last] = y.flip(0) if case["reverse"] else y
        if case["kept"]:
            pool[write] = x[x.shape[0] - width + 1:]
    return (out, pool) if case["kept"] else out


def _exact_scan(state):
    """The recurrence itself, token by token, all sequences side by side."""
    case = state["case"]
    seqs, channels, n, per = case["seqs"], case["channels"], case["state"], case["channels"] // case["groups"]
    todo, A = _sequences(state), state["A"].double()
    h = torch.zeros(seqs, channels, n, dtype=torch.float64, device="cuda")
    for s, (_, _, continues, read, _) in enumerate(todo):
        if continues:
            h[s] = state["pool"][read]
    out = torch.empty(state["rows"], channels, dtype=torch.float64, device="cuda")
    longest = sorted(range(seqs), key=lambda s: todo[s][0] - todo[s][1])  # the sequences that still have tokens stand in front
    h = h[longest]
    dt = state["dt"].double()
    if case["softplus"]:
        dt = torch.logaddexp(dt + state["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    vectors = state["proj"][:, -2 * case["groups"] * n:].double().reshape(-1, 2, case["groups"], n)
    firsts, lasts = torch.tensor([todo[s][0] for s in longest], device="cuda"), torch.tensor([todo[s][1] for s in longest], device="cuda")
    counts = [todo[s][1] - todo[s][0] for s in longest]
    for t in range(counts[0]):
        live = sum(c > t for c in counts) if counts[-1] <= t else seqs
        rows = lasts[:live] - 1 - t if case["reverse"] else firsts[:live] + t
        d, v = dt[rows], vectors[rows].repeat_interleave(per, 2)
        h[:live] = torch.exp(d[:, :, None] * A) * h[:live] + (d * state["x"][rows].double())[:, :, None] * v[:, 0]
        out[rows] = (h[:live] * v[:, 1]).sum(2)
    out += state["x"].double() * state["skip"].double()
    if case["gate"]:
        out *= _silu64(state["xz"][:, channels:].double())
    if not case["kept"]:
        return out
    pool = state["pool"].double()
    for k, s in enumerate(longest):
        pool[todo[s][4]] = h[k]
    return out, pool


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](state)


# ------------------------------------------------------------------------------------------------- the work of a pass
def work(case):
    channels = case["channels"]
    if case["op"] == "norm":
        count = case["images"] * channels * case["height"] * case["width"]
        return {"bytes": 8.0 * count + 8.0 * channels * (1 + case["modulate"] * case["images"]), "flops": (9.0 + 2.0 * case["modulate"] + 4.0 * (case["activation"] == "silu")) * count}
    rows, seqs = float(_news(case).sum()), case["seqs"]
    kept = 2 * seqs - seqs // 4 if case["kept"] else 0  # states read and written; every fourth sequence begins
    if case["op"] == "conv":
        each = case["width"] - 1
        return {"bytes": 8.0 * rows * channels + 4.0 * channels * (case["width"] + 1) + 4.0 * kept * each * channels,
                "flops": (2.0 * case["width"] + 4.0 * (case["activation"] == "silu")) * rows * channels}
    n = case["state"]
    return {"bytes": 4.0 * rows * ((4.0 if case["gate"] else 3.0) * channels + 2.0 * case["groups"] * n) + 4.0 * channels * (n + 2) + 4.0 * kept * channels * n,
            "flops": rows * channels * (7.0 * n + 8.0 * case["softplus"] + 5.0 * case["gate"] + 3.0)}
