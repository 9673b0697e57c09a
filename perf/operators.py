"""The operators of an attention block on image and video tokens, as cases that can be timed and compared.

A case names its operator and sizes:

  attend   ``paged_attention``: new tokens of a batch of sequences over a paged cache that holds them and what came before
  append   ``paged_append``: rotary positions on queries and keys, keys and values written to their places in the cache
  rotate   ``rotary_axes``: rotary positions on the heads of a tensor of rows
  norm     ``norm_residual``: the norm behind a block, its gate, the residual sum and the norm before the next block

Activations are float32 rows [tokens, heads * head_dim]; queries, keys and values are columns of one tensor, as one dense layer
brings them.  The cache holds float32 or bfloat16 in pages of ``page`` tokens, in the order in which the framework keeps them:

  keys    [pages, kv_heads, page / 16, head_dim / 8, 16 tokens, 8 dimensions]
  values  [pages, kv_heads, page / 16, 2, head_dim, 8 tokens]

A batch is a table of pages [sequences, width], the rows' offsets [sequences + 1] and the lengths [sequences] of the sequences,
new tokens included.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the smallest call: one new token over the cached tokens of one 7 x 7 feature map and a class token
        _attend("attend_1x1_over_50_f32", seqs=1, new=1, length=50, ragged=False, heads=8, kv_heads=8, dim=64, page=16, type="f32"),
        # a serving batch of single tokens, each sequence with its own length: bound by the cache's bytes
        _attend("attend_32x1_over_4096_bf16", seqs=32, new=1, length=4096, ragged=True, heads=32, kv_heads=8, dim=128, page=64, type="bf16"),
        # one token of one very long sequence: the work has to be split over the cache's length
        _attend("attend_1x1_over_131072_bf16", seqs=1, new=1, length=131072, ragged=False, heads=32, kv_heads=8, dim=128, page=128, type="bf16"),
        # frames of 14 x 14 tokens of four videos, each over the frames before it; tokens of a frame see one another
        _attend("attend_4x196_over_1568_f32", seqs=4, new=196, length=1568, ragged=False, heads=8, kv_heads=8, dim=64, page=64, type="f32", causal=False),
        # a long prompt's chunk over what came before it: the largest, bound by the matrix instructions
        _attend("attend_1x2048_over_8192_bf16", seqs=1, new=2048, length=8192, ragged=False, heads=32, kv_heads=8, dim=128, page=64, type="bf16"),
        # mixed work: sequences of ragged chunks and lengths, a window, heads of 80
        _attend("attend_7x301_over_1777_window_f32", seqs=7, new=301, length=1777, ragged=True, heads=12, kv_heads=4, dim=80, page=32, type="f32", window=500),
        # a decoding step's keys and values of 32 sequences
        _append("append_32x1_bf16", seqs=32, new=1, length=700, ragged=True, heads=32, kv_heads=8, dim=128, page=64, type="bf16", axes=1, halves=True),
        # four clips of eight frames of 14 x 14 tokens, three axes
        _append("append_4x1568_f32", seqs=4, new=1568, length=1568, ragged=False, heads=16, kv_heads=16, dim=64, page=64, type="f32", axes=3, halves=False),
        # one frame of 7 x 7 tokens, rows and columns
        _rotate("rotate_49_2axes", tokens=49, heads=8, dim=64, axes=2, halves=True, rot=64),
        # a video of 16 frames of 28 x 28 tokens, time, rows and columns
        _rotate("rotate_12544_3axes", tokens=12544, heads=16, dim=128, axes=3, halves=False, rot=128),
        # one image's 7 x 7 tokens between two blocks of 512 channels: latency
        _norm("norm_49x512", tokens=49, cols=512, groups=1, post="none", pre="layer", modulate=False, gate="vector"),
        # 64 images of 14 x 14 tokens, 2048 channels, a gate, a shift and a scale for every image: bound by memory
        _norm("norm_12544x2048_gated", tokens=12544, cols=2048, groups=64, post="rms", pre="rms", modulate=True, gate="group"),
    ]


def _attend(name, seqs, new, length, ragged, heads, kv_heads, dim, page, type, causal=True, window=0):
    return dict(name=name, op="attend", seqs=seqs, new=new, length=length, ragged=ragged, heads=heads, kv_heads=kv_heads, dim=dim, page=page, type=type,
                causal=causal, window=window)


def _append(name, seqs, new, length, ragged, heads, kv_heads, dim, page, type, axes, halves):
    return dict(name=name, op="append", seqs=seqs, new=new, length=length, ragged=ragged, heads=heads, kv_heads=kv_heads, dim=dim, page=page, type=type,
                axes=axes, halves=halves, rot=dim)


def _rotate(name, tokens, heads, dim, axes, halves, rot):
    return dict(name=name, op="rotate", tokens=tokens, heads=heads, dim=dim, axes=axes, halves=halves, rot=rot)


def _norm(name, tokens, cols, groups, post, pre, modulate, gate):
    return dict(name=name, op="norm", tokens=tokens, cols=cols, groups=groups, post=post, pre=pre, modulate=modulate, gate=gate)


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    op = rng.choice(("attend", "attend", "attend", "append", "rotate", "norm"))
    dim, kv_heads, page = rng.choice((16, 48, 64, 64, 80, 96, 128, 128, 192, 256)), rng.choice((1, 2, 3, 4, 8, 8, 16)), rng.choice((16, 32, 64, 128, 256))
    heads, type, axes, halves = kv_heads * rng.choice((1, 1, 2, 4, 5, 8)), rng.choice(("f32", "bf16")), rng.choice((1, 2, 3)), rng.random() < 0.5
    if op == "attend":
        new = rng.choice((1, 1, _log(rng, 1, 16), _log(rng, 16, 2048)))
        length = new + _log(rng, 1, 8192 if new > 1 else 131072) - 1
        window = rng.choice((0, 0, 0, _log(rng, 1, 4096)))
        return _attend(None, _log(rng, 1, 64), new, length, rng.random() < 0.6, heads, kv_heads, dim, page, type, rng.random() < 0.7, window)
    if op == "append":
        new = rng.choice((1, _log(rng, 1, 2048)))
        case = _append(None, _log(rng, 1, 64), new, new + _log(rng, 1, 1024) - 1, rng.random() < 0.6, heads, kv_heads, dim, page, type, axes, halves)
        return dict(case, rot=rng.choice((dim, dim, dim // 2)))
    if op == "rotate":
        return _rotate(None, _log(rng, 1, 20000), heads, dim, axes, halves, rng.choice((dim, dim, dim // 2)))
    tokens = _log(rng, 1, 50000)
    return _norm(None, tokens, rng.choice((_log(rng, 1, 8192), 64 * _log(rng, 1, 128))), rng.choice((1, _log(rng, 1, min(tokens, 256)))),
                 rng.choice(("none", "layer", "rms")), rng.choice(("none", "layer", "rms")), rng.random() < 0.5, rng.choice(("none", "vector", "group")))


def _floats(case):
    """What the plain form and a cache of the case hold, in numbers."""
    if case["op"] in ("attend", "append"):
        cached = 2 * case["seqs"] * case["length"] * case["kv_heads"] * case["dim"]
        rows = case["seqs"] * case["new"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return cached + rows + (case["seqs"] * case["heads"] * case["new"] * case["length"] if case["op"] == "attend" else 0)
    return case["tokens"] * (case["heads"] * case["dim"] if case["op"] == "rotate" else case["cols"])


def draw(rng):
    while True:
        case = {k: v for k, v in _drawn(rng).items() if k != "name"}
        if case["op"] == "attend" and case["seqs"] * case["new"] * case["length"] * case["heads"] * case["dim"] > 6.8e10:
            continue
        if _floats(case) <= (5.4e8 if case["op"] == "attend" else 2.6e7):
            return case


# ------------------------------------------------------------------------------------------------- what a program has in hand
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _lengths(case):
    """New tokens and length of every sequence: all alike, or spread up to the largest (the case's own, whatever the seed)."""
    n, new, length = case["seqs"], case["new"], case["length"]
    rng = np.random.default_rng([n, new, length])
    news, before = np.full(n, new), np.full(n, length - new)
    if case["ragged"]:
        news, before = rng.integers(1, new + 1, n), rng.integers(0, length - new + 1, n)
        news[0], before[0] = new, length - new
    return news.astype(np.int32), (news + before).astype(np.int32)


def _batch(case, seed, g):
    """A cache whose sequences lie on shuffled pages, and the table, offsets and lengths of the batch."""
    news, lengths = _lengths(case)
    page, dim, kv_heads = case["page"], case["dim"], case["kv_heads"]
    counts = -(-lengths // page)
    width, pages = int(counts.max()), int(counts.sum()) + 3
    order = np.random.default_rng(seed + 1).permutation(pages)
    table, at = np.full((case["seqs"], width), -1, np.int32), 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c]
        at += c
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    kind = TYPES[case["type"]]
    return {"keys": _normal(g, pages, kv_heads, page // 16, dim // 8, 16, 8).to(kind), "values": _normal(g, pages, kv_heads, page // 16, 2, dim, 8).to(kind),
            "table": put(table), "offsets": put(np.concatenate([[0], np.cumsum(news)])), "lengths": put(lengths), "rows": int(news.sum()),
            "max_new": int(news.max()), "max_length": int(lengths.max())}


def _plan(case):
    """Axis and frequency of every pair of dimensions: the axes take turns, the frequencies fall from 1 to about 1e-4."""
    pairs = case["rot"] // 2
    return np.arange(pairs, dtype=np.int32) % case["axes"], 10000.0 ** (-np.arange(pairs, dtype=np.float64) / pairs)


def _positions(case, seed, rows):
    """Frame, row and column of tokens of clips of 14 x 14 tokens somewhere in a long video; a single axis counts the tokens."""
    first = int(np.random.default_rng(seed + 2).integers(0, 100000))
    n = np.arange(rows) + first
    p = {1: (n,), 2: (n // 14, n % 14), 3: (n // 196, n // 14 % 14, n % 14)}[case["axes"]]
    return torch.from_numpy(np.stack(p, 1).astype(np.float32)).cuda()


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] in ("attend", "append"):
        state.update(_batch(case, seed, g))
        qkv = _normal(g, state["rows"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"])
        state.update(qkv=qkv, out=torch.empty(state["rows"], case["heads"] * case["dim"], device="cuda"))
        if case["op"] == "append":
            state["axis"], state["freq"] = _plan(case)
            state["positions"] = _positions(case, seed, state["rows"])
    elif case["op"] == "rotate":
        x = _normal(g, case["tokens"], case["heads"] * case["dim"])
        state.update(x=x, out=torch.empty_like(x), positions=_positions(case, seed, case["tokens"]))
        state["axis"], state["freq"] = _plan(case)
    else:
        rows, cols, groups = case["tokens"], case["cols"], -(-case["tokens"] // -(-case["tokens"] // case["groups"]))
        weight = lambda: (1.0 + 0.1 * _normal(g, cols), 0.1 * _normal(g, cols))
        state.update(x=_normal(g, rows, cols), residual=2.0 * _normal(g, rows, cols), sum=torch.empty(rows, cols, device="cuda"),
                     normed=torch.empty(rows, cols, device="cuda"), each=-(-rows // case["groups"]), gate=None, mod=None, shift=None, post=(None, None), pre=(None, None))
        if case["post"] != "none":
            state["post"] = weight()
        if case["pre"] != "none":
            state["pre"] = weight()
            if case["modulate"]:
                state.update(mod=0.2 * _normal(g, groups, cols), shift=0.2 * _normal(g, groups, cols))
        if case["gate"] != "none":
            state["gate"] = 0.5 * _normal(g, groups if case["gate"] == "group" else 1, cols)
    return state


# ------------------------------------------------------------------------------------------------- the plain forms
def _columns(state):
    case, qkv = state["case"], state["qkv"]
    q, k = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    return qkv[:, :q], qkv[:, q:q + k], qkv[:, q + k:]


def _rows_of(state):
    """For every row: its sequence, and its place in the cache."""
    row = torch.arange(state["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(state["offsets"], row, right=True) - 1
    nth = row - state["offsets"][seq]
    new = state["offsets"][seq + 1] - state["offsets"][seq]
    return seq, nth, state["lengths"][seq] - new + nth


def _plain_attend(state):
    case = state["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    seqs, new = case["seqs"], state["max_new"]
    seq, nth, place = _rows_of(state)
    table = state["table"].clamp(min=0)
    width = table.shape[1] * page
    k = state["keys"][table].permute(0, 2, 1, 3, 5, 4, 6).reshape(seqs, kv_heads, 1, width, dim).float()
    v = state["values"][table].permute(0, 2, 1, 3, 4, 6, 5).reshape(seqs, kv_heads, 1, width, dim).float()
    q = torch.zeros(seqs, new, heads * dim, device="cuda")
    q[seq, nth] = _columns(state)[0]
    q = q.reshape(seqs, new, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(seqs, kv_heads, 1, (heads // kv_heads) * new, dim)
    scores = torch.matmul(q, k.transpose(3, 4)).mul_(1.0 / math.sqrt(dim)).reshape(seqs, heads, new, width)
    news = state["offsets"][1:] - state["offsets"][:-1]
    at = (state["lengths"] - news)[:, None] + torch.arange(new, device="cuda")
    j = torch.arange(width, device="cuda")
    seen = (j < state["lengths"][:, None, None]).expand(seqs, new, width)
    if case["causal"]:
        seen = seen & (j <= at[:, :, None])
    if case["window"]:
        seen = seen & (j > at[:, :, None] - case["window"])
    scores.masked_fill_(~seen[:, None], -math.inf)
    top = scores.amax(3, keepdim=True)
    weights = scores.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = weights.sum(3, keepdim=True)
    weights = weights.reshape(seqs, kv_heads, 1, (heads // kv_heads) * new, width)
    out = torch.matmul(weights, v).reshape(seqs, heads, new, dim) / torch.where(total > 0, total, 1.0)
    state["out"].copy_(out.permute(0, 2, 1, 3)[seq, nth].reshape(-1, heads * dim))
    return state["out"]


def _plain_rotate(x, positions, case, axis, freq):
    """x [rows, heads, dim]; the angles in 64 bits."""
    rot, angle = case["rot"], positions.double()[:, torch.from_numpy(axis).long().cuda()] * torch.from_numpy(freq).cuda()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.clone()
    if case["halves"]:
        a, b = x[:, :, :rot // 2], x[:, :, rot // 2:rot]
        y[:, :, :rot // 2], y[:, :, rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[:, :, 0:rot:2], x[:, :, 1:rot:2]
        y[:, :, 0:rot:2], y[:, :, 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return y


def _plain_append(state):
    case = state["case"]
    dim, page, kv_heads = case["dim"], case["page"], case["kv_heads"]
    q, k, v = _columns(state)
    q = _plain_rotate(q.reshape(-1, case["heads"], dim), state["positions"], case, state["axis"], state["freq"])
    k = _plain_rotate(k.reshape(-1, kv_heads, dim), state["positions"], case, state["axis"], state["freq"])
    seq, _, place = _rows_of(state)
    at, t = state["table"][seq, place // page].long(), place % page
    keys, values = state["keys"], state["values"]
    keys[at, :, t // 16, :, t % 16] = k.reshape(-1, kv_heads, dim // 8, 8).to(keys.dtype)
    values[at, :, t // 16, t % 16 // 8, :, t % 8] = v.reshape(-1, kv_heads, dim).to(values.dtype)
    state["out"].copy_(q.reshape(state["rows"], -1))
    return state["out"], keys, values


def _plain_normed(x, kind, weight, bias, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    return x / torch.sqrt((x * x).mean(1, keepdim=True) + eps) * weight + bias


def _plain_norm(state):
    case = state["case"]
    group = torch.arange(case["tokens"], device="cuda") // state["each"]
    n = _plain_normed(state["x"], case["post"], *state["post"], 1e-6)
    if state["gate"] is not None:
        n = n * (state["gate"][group] if case["gate"] == "group" else state["gate"])
    state["sum"].copy_(0.5 * state["residual"] + n)
    h = _plain_normed(state["sum"], case["pre"], *state["pre"], 1e-5)
    if state["mod"] is not None:
        h = h * (1.0 + state["mod"][group]) + state["shift"][group]
    state["normed"].copy_(h)
    return state["sum"], state["normed"]


# ------------------------------------------------------------------------------------------------- the framework's calls
_device = None


def _handles(state):
    """The framework's view of what the program has in hand, made once."""
    global _device
    import eddl_amd
    from eddl_amd.attention import PagedBatch, PagedCache, RotaryPlan
    if _device is None:
        _device = eddl_amd.Backend(0)
    hip, case = _device, state["case"]
    h = {"hip": hip}
    wrap = lambda t: None if t is None else hip.wrap(t)
    if case["op"] in ("attend", "append"):
        pages = lambda t: hip.wrap(t.view(torch.int16), dtype="bfloat16") if t.dtype == torch.bfloat16 else hip.wrap(t)
        h["cache"] = PagedCache(hip, state["keys"].shape[0], case["page"], case["kv_heads"], case["dim"], {"f32": "float32", "bf16": "bfloat16"}[case["type"]],
                                storage=(pages(state["keys"]), pages(state["values"])))
        h["batch"] = PagedBatch(wrap(state["table"]), wrap(state["offsets"]), wrap(state["lengths"]), state["max_new"], state["max_length"])
        qkv, q, k = wrap(state["qkv"]), case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
        h.update(q=qkv.columns(0, q), k=qkv.columns(q, q + k), v=qkv.columns(q + k, q + 2 * k), out=wrap(state["out"]))
    if case["op"] in ("append", "rotate"):
        h["plan"] = RotaryPlan(case["dim"], state["axis"], state["freq"], "halves" if case["halves"] else "adjacent")
        h["positions"] = wrap(state["positions"])
    if case["op"] == "rotate":
        h.update(x=wrap(state["x"]), out=wrap(state["out"]))
    if case["op"] == "norm":
        kinds = {"none": None, "layer": "layer", "rms": "rms"}
        h.update(x=wrap(state["x"]), residual=wrap(state["residual"]), sum=wrap(state["sum"]), normed=wrap(state["normed"]),
                 post=(kinds[case["post"]], wrap(state["post"][0]), wrap(state["post"][1]), 1e-6), pre=(kinds[case["pre"]], wrap(state["pre"][0]), wrap(state["pre"][1]), 1e-5),
                 gate=wrap(state["gate"]), mod=wrap(state["mod"]), shift=wrap(state["shift"]))
    return h


def _run_own(state):
    case = state["case"]
    if "handles" not in state:
        state["handles"] = _handles(state)
    h = state["handles"]
    hip = h["hip"]
    if case["op"] == "attend":
        hip.paged_attention(h["q"], h["out"], h["cache"], h["batch"], causal=case["causal"], window=case["window"])
        return state["out"]
    if case["op"] == "append":
        hip.paged_append(h["q"], h["k"], h["v"], h["out"], h["cache"], h["batch"], rotary=h["plan"], positions=h["positions"])
        return state["out"], state["keys"], state["values"]
    if case["op"] == "rotate":
        hip.rotary_axes(h["x"], h["out"], h["plan"], h["positions"])
        return state["out"]
    hip.norm_residual(h["x"], h["residual"], h["sum"], h["normed"], post=h["post"], pre=h["pre"], gate=h["gate"], residual_scale=0.5, mod=h["mod"], shift=h["shift"],
                      group_rows=state["each"])
    return state["sum"], state["normed"]


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _plain_attend, "append": _plain_append, "rotate": _plain_rotate_case, "norm": _plain_norm}[state["case"]["op"]](state)


def _plain_rotate_case(state):
    case, x = state["case"], state["x"]
    y = _plain_rotate(x.reshape(-1, case["heads"], case["dim"]), state["positions"], case, state["axis"], state["freq"])
    state["out"].copy_(y.reshape(x.shape))
    return state["out"]


# ------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _token64(state, s, length):
    """Keys and values [kv_heads, length, dim] of one sequence, page by page."""
    page, dim = state["case"]["page"], state["case"]["dim"]
    ks, vs = [], []
    for p in state["table"][s, :-(-length // page)].tolist():
        ks.append(torch.einsum("hbctd->hbtcd", state["keys"][p]).reshape(-1, page, dim).double())
        vs.append(torch.einsum("hbudt->hbutd", state["values"][p]).reshape(-1, page, dim).double())
    return torch.cat(ks, 1)[:, :length], torch.cat(vs, 1)[:, :length]


def _exact_attend(state):
    case = state["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    offsets, out = state["offsets"].tolist(), []
    q_all = state["qkv"][:, :heads * dim].double()
    for s, length in enumerate(state["lengths"].tolist()):
        k, v = _token64(state, s, length)
        q = q_all[offsets[s]:offsets[s + 1]].reshape(-1, heads, dim)
        new = q.shape[0]
        at = torch.arange(length - new, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        hidden = torch.zeros(new, length, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= j > at
        if case["window"] > 0:
            hidden |= at - j >= case["window"]
        rows = []
        for h in range(heads):
            w = (q[:, h] @ k[h * kv_heads // heads].T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
            rows.append(torch.softmax(w, 1) @ v[h * kv_heads // heads])
        out.append(torch.stack(rows, 1).reshape(new, heads * dim))
    return torch.cat(out)


def _exact_rotate(x, state, heads):
    case = state["case"]
    y = x.double().reshape(-1, heads, case["dim"]).clone()
    p = state["positions"].double()
    for i, (axis, freq) in enumerate(zip(state["axis"].tolist(), state["freq"].tolist())):
        a, b = (i, i + case["rot"] // 2) if case["halves"] else (2 * i, 2 * i + 1)
        turned = torch.complex(y[:, :, a], y[:, :, b]) * torch.exp(1j * p[:, axis] * freq)[:, None]
        y[:, :, a], y[:, :, b] = turned.real, turned.imag
    return y.reshape(x.shape[0], -1)


def _exact_append(state):
    case = state["case"]
    q, k, v = _columns(state)
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    k = _exact_rotate(k, state, kv).reshape(-1, kv, dim // 8, 8)
    v = v.double().reshape(-1, kv, dim)
    keys, values = state["keys"].double(), state["values"].double()
    offsets, lengths, table = state["offsets"].tolist(), state["lengths"].tolist(), state["table"].tolist()
    at = []
    for s in range(case["seqs"]):
        new = offsets[s + 1] - offsets[s]
        at += [(table[s][n // page], n % page) for n in range(lengths[s] - new, lengths[s])]
    pg, t = (torch.tensor(c, device="cuda") for c in zip(*at))
    keys.transpose(1, 2).transpose(2, 4)[pg, t // 16, t % 16] = k.transpose(1, 2)
    values.permute(0, 2, 3, 5, 1, 4)[pg, t // 16, t // 8 % 2, t % 8] = v
    return _exact_rotate(q, state, case["heads"]), keys, values


def _exact_norm(state):
    case = state["case"]
    n = torch.arange(case["tokens"], device="cuda").div(state["each"], rounding_mode="floor")

    def normed(x, kind, params, eps):
        if kind == "none":
            return x
        w, b = (t.double() for t in params)
        if kind == "layer":
            return (x - x.mean(1)[:, None]) * torch.rsqrt(x.var(1, unbiased=False) + eps)[:, None] * w + b
        return x * torch.rsqrt(x.square().mean(1) + eps)[:, None] * w + b

    y = normed(state["x"].double(), case["post"], state["post"], 1e-6)
    if case["gate"] != "none":
        y = y * state["gate"].double()[n if case["gate"] == "group" else n * 0]
    total = state["residual"].double() / 2 + y
    h = normed(total, case["pre"], state["pre"], 1e-5)
    if state["mod"] is not None:
        h = h + h * state["mod"].double()[n] + state["shift"].double()[n]
    return total, h


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(state)
    if case["op"] == "append":
        return _exact_append(state)
    if case["op"] == "rotate":
        return _exact_rotate(state["x"], state, case["heads"])
    return _exact_norm(state)


# ------------------------------------------------------------------------------------------------- the work of a pass
def _attend_work(case):
    news, lengths = (a.astype(np.float64) for a in _lengths(case))
    visible, read = lengths * news, lengths
    if case["window"]:  # a query sees at most the window's tokens up to itself, and what comes after it where it may
        later = np.zeros_like(news) if case["causal"] else (news - 1) / 2
        visible = news * np.minimum(case["window"] + later, lengths)
        read = np.minimum(lengths, news - 1 + case["window"])
    if case["causal"]:
        visible = np.minimum(visible, news * (lengths - (news - 1) / 2))
    size = 4 if case["type"] == "f32" else 2
    return {"bytes": 8.0 * news.sum() * case["heads"] * case["dim"] + 2.0 * size * read.sum() * case["kv_heads"] * case["dim"],
            "flops": 4.0 * visible.sum() * case["heads"] * case["dim"]}


def work(case):
    if case["op"] == "attend":
        return _attend_work(case)
    if case["op"] == "append":
        rows = float(_lengths(case)[0].sum())
        q, kv = rows * case["heads"] * case["dim"], 2 * rows * case["kv_heads"] * case["dim"]
        return {"bytes": 8.0 * q + (4.0 + (4 if case["type"] == "f32" else 2)) * kv + 4.0 * rows * case["axes"], "flops": 3.0 * (q + kv / 2)}
    if case["op"] == "rotate":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 8.0 * n + 4.0 * case["tokens"] * case["axes"], "flops": 3.0 * n}
    n, tables = case["tokens"] * case["cols"], (1 if case["gate"] == "vector" else 0) + 2 * ((case["post"] != "none") + (case["pre"] != "none"))
    grouped = (case["gate"] == "group") + 2 * (case["modulate"] and case["pre"] != "none")
    return {"bytes": 16.0 * n + 4.0 * case["cols"] * (tables + grouped * min(case["groups"], case["tokens"])), "flops": 12.0 * n}
