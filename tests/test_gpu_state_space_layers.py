"""Group norm, causal convolution and selective scan as layers: states that a plan keeps between its runs, plans that fold layers together."""
import numpy as np
import pytest

from state_space_ref import causal_conv, selective_scan
from test_gpu_state_space import _check

pytestmark = pytest.mark.gpu


class Blocks:
    """x -> convolution -> (two dense layers) -> scan, gated by x; a plan for every number of tokens, all of them on the same pools of states."""

    def __init__(self, hip, entries, cols, n, width, slots, reverse=False):
        rng = np.random.default_rng([entries, cols, n])
        self.hip, self.entries, self.cols, self.n, self.width, self.reverse = hip, entries, cols, n, width, reverse
        r = lambda *s: rng.standard_normal(s, dtype=np.float32)
        self.inputs, self.states = r(slots, width - 1, cols), r(slots, cols, n)
        self.P, self.S = hip.array(self.inputs), hip.array(self.states)
        self.weights = {"causal_conv": {"W": 0.5 * r(cols, width), "bias": 0.1 * r(cols)}, "steps": {"W": r(cols, cols) / np.float32(cols ** 0.5)},
                        "vectors": {"W": r(cols, 2 * n + 1) / np.float32(cols ** 0.5)},
                        "selective_scan": {"A": -np.exp(r(cols, n)), "skip": r(cols), "dt_bias": r(cols) - 2}}

    def plan(self, tokens, batch, fuse=True):
        from eddl_amd import net as L
        x = L.Input([tokens, self.cols], self.entries)
        u = L.CausalConvolution(x, self.width, reverse=self.reverse, batch=batch, states=self.P)
        dt, v = L.Dense(u, self.cols, use_bias=False, name="steps"), L.Dense(u, 2 * self.n + 1, use_bias=False, name="vectors")
        y = L.SelectiveScan(u, dt, v, self.n, gate=x, reverse=self.reverse, batch=batch, states=self.S)
        net = L.Net([x], [y, u, dt, v])
        for l in net.layers:
            for k, value in self.weights.get(l.kind if l.kind != "dense" else l.name, {}).items():
                l.params[k] = value.copy()
        return net.build(self.hip, fuse=fuse)

    def check(self, x, got, batch):
        """A run's outputs and the pools behind it against 64 bits, each layer on the inputs that it was given; what the pools hold then is what the next run continues."""
        y, u, dt, v = (t.reshape(-1, t.shape[2]) for t in got)
        x, w, s = x.reshape(-1, self.cols), self.weights["causal_conv"], self.weights["selective_scan"]
        want, err, after = causal_conv(x, w["W"], w["bias"], kind="silu", reverse=self.reverse, pool=self.inputs, **batch)
        _check(u, want, err, "convolution")
        self.inputs = self.P.numpy()
        assert np.array_equal(self.inputs, after)
        want, err, after, after_err = selective_scan(u, dt, s["A"], v[:, 1:1 + self.n], v[:, 1 + self.n:], skip=s["skip"], gate=x, dt_bias=s["dt_bias"], reverse=self.reverse, pool=self.states,
                                                     **batch)
        rows = np.isfinite(want[:, 0])
        _check(y[rows], want[rows], err[rows], "scan")
        self.states = self.S.numpy()
        _check(self.states, after, after_err, "states")
        untouched = np.setdiff1d(np.arange(len(after)), batch["out_slots"])
        assert np.array_equal(self.states[untouched], after[untouched].astype(np.float32))


def _on(hip, batch, max_new, apart=True):
    from eddl_amd.state_space import StateBatch
    i = lambda t: hip.array(np.asarray(t), "int32")
    return StateBatch(i(batch["offsets"]), max_new, i(batch["lengths"]), i(batch["slots"]), i(batch["out_slots"]) if apart else None)


@pytest.mark.parametrize("cols, n, reverse", [(24, 16, False), (19, 5, False), (40, 16, True)])
def test_layers_continue_their_states(hip, cols, n, reverse):
    """Ragged prompts, then single tokens, then ragged pieces: three plans, whose layers read and write the slots of the same two pools."""
    rng = np.random.default_rng([cols, n, 3])
    blocks = Blocks(hip, 3, cols, n, 4, 8, reverse)
    slots = np.array([5, 0, 3], np.int32)
    for tokens, news, others, lengths in ((9, [11, 3, 9], [1, 6, 7], [11, 8, 9]), (1, [1, 1, 1], [1, 6, 7], [12, 9, 10]), (40, [40, 0, 75], [2, 4, 0], [52, 9, 85])):
        batch = dict(offsets=np.concatenate([[0], np.cumsum(news)]), lengths=np.array(lengths), slots=slots, out_slots=np.array(others))
        x = rng.standard_normal((3, tokens, cols), dtype=np.float32)
        net = blocks.plan(tokens, _on(hip, batch, tokens))
        before = blocks.P.numpy(), blocks.S.numpy()
        got = net.predict(x)
        blocks.check(x, got, batch)
        after = blocks.P.numpy(), blocks.S.numpy()
        blocks.P.copy_from(before[0])
        blocks.S.copy_from(before[1])
        walk = blocks.plan(tokens, _on(hip, batch, tokens), fuse=False).predict(x)
        there = int(batch["offsets"][-1])
        for a, b in zip(got, walk):  # (rows of no sequence hold what the memory held)
            assert np.array_equal(a.reshape(3 * tokens, -1)[:there], b.reshape(3 * tokens, -1)[:there])
        assert np.array_equal(after[0], blocks.P.numpy()) and np.array_equal(after[1], blocks.S.numpy())
        slots = batch["out_slots"]


@pytest.mark.parametrize("tokens", [1, 30, 600])
def test_capture_leaves_the_states(hip, tokens):
    """A captured plan takes its first step when it is replayed: capturing it moves no state, and replays continue one another as runs of the plan do."""
    rng = np.random.default_rng([tokens, 4])
    blocks = Blocks(hip, 2, 32, 16, 4, 3)
    batch = dict(offsets=np.array([0, tokens, 2 * tokens]), lengths=np.array([tokens + 4, tokens + 9]), slots=np.array([2, 0]), out_slots=np.array([2, 0]))
    net = blocks.plan(tokens, _on(hip, batch, tokens, apart=False))
    xs = rng.standard_normal((3, 2, tokens, 32), dtype=np.float32)
    before = blocks.P.numpy(), blocks.S.numpy()
    want = [(net.predict(x), blocks.P.numpy(), blocks.S.numpy()) for x in xs]
    blocks.P.copy_from(before[0])
    blocks.S.copy_from(before[1])
    net.input_tensor().copy_from(xs[0])
    net.capture()
    assert np.array_equal(blocks.P.numpy(), before[0]) and np.array_equal(blocks.S.numpy(), before[1])
    for x, (outs, inputs, states) in zip(xs, want):
        net.input_tensor().copy_from(x)
        net.run_graph()
        for o, w in zip(net.lout, outs):
            assert np.array_equal(net.output_of(o).numpy(), w)
        assert np.array_equal(blocks.P.numpy(), inputs) and np.array_equal(blocks.S.numpy(), states)
    net.input_tensor().copy_from(xs[0])  # and capturing it again, between two steps
    net.capture()
    assert np.array_equal(blocks.P.numpy(), want[-1][1]) and np.array_equal(blocks.S.numpy(), want[-1][2])


@pytest.mark.parametrize("maps", [True, False])
def test_a_relu_behind_a_group_norm_is_the_relu_layer(hip, maps):
    """A plan that folds a ReLU layer into the norm before it gives that layer's bits, for groups that are NaN too (the layer makes 0 of a NaN); a norm whose own activation is a
    ReLU leaves NaN as it is."""
    from eddl_amd import net as L
    rng = np.random.default_rng(6)
    shape, at = ([6, 5, 7], (1, 4, 3, 2)) if maps else ([35, 6], (1, 17, 4))
    x = rng.standard_normal([3] + shape, dtype=np.float32)
    x[at], x[2][tuple(np.array(at[1:]) // 2)] = np.nan, np.inf
    outs = []
    for fuse in (True, False):
        i = L.Input(shape, 3)
        net = L.Net([i], [L.ReLu(L.GroupNormalization(i, 3)), L.GroupNormalization(i, 3, activation="relu")]).build(hip, fuse=fuse)
        assert sum(op.kind == "relu" for op in net.ops) == (0 if fuse else 1)
        outs.append(net.predict(x))
    assert not np.any(np.isnan(outs[1][0])) and np.isnan(outs[1][1]).sum() == 2 * 2 * 35
    for a, b in zip(*outs):
        assert np.array_equal(a, b, equal_nan=True)
    fine = ~np.isnan(outs[0][1])
    assert np.array_equal(outs[0][0][fine], outs[0][1][fine])


@pytest.mark.parametrize("channels, pixels, groups", [(6, 35, 3), (8, 20000, 2), (30, 1500, 2), (96, 400, 2), (4, 3000, 2)])
def test_relu_layer_of_a_norm_is_the_relu(hip, channels, pixels, groups):
    """The "relu_layer" is the norm without an activation and ``Backend.relu`` behind it, bit for bit; NaN among the numbers, groups whole and divided, maps and rows."""
    rng = np.random.default_rng([channels, pixels])
    x = rng.standard_normal((2, channels, pixels), dtype=np.float32)
    x[1, 0, pixels // 2] = np.nan
    w, b = (hip.array(rng.standard_normal(channels, dtype=np.float32)) for _ in range(2))
    for t, tokens in ((x.reshape(2, channels, pixels, 1), None), (x.transpose(0, 2, 1).reshape(-1, channels), pixels)):
        X = hip.array(t)
        plain, want, got, kept = (hip.full(t.shape, -7.0) for _ in range(4))
        hip.group_norm(X, plain, groups, w, b, image_rows=tokens)
        hip.relu(plain, want)
        hip.group_norm(X, got, groups, w, b, activation="relu_layer", image_rows=tokens)
        hip.group_norm(X, kept, groups, w, b, activation="relu", image_rows=tokens)
        n, k = plain.numpy(), kept.numpy()
        assert np.isnan(n).sum() == channels // groups * pixels
        assert np.array_equal(got.numpy(), want.numpy()) and np.array_equal(np.isnan(k), np.isnan(n)) and np.array_equal(np.nan_to_num(k), want.numpy())
