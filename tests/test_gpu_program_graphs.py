"""Graphs that the program captures by itself, of calls that take the library's workspace."""
import ctypes

import numpy as np
import pytest

from test_gpu_state_space import Ragged, _scan_case

pytestmark = pytest.mark.gpu


class Program:
    """A stream of the program's, on which it captures the library's calls; ``launch`` replays them on the null stream."""

    def __init__(self, hip, fn):
        self.lib, self.stream, self.graph, self.exe = hip.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        assert self.lib.hipStreamCreateWithFlags(ctypes.byref(self.stream), 1) == 0
        self.error = None
        assert self.lib.hipStreamBeginCapture(self.stream, 1) == 0  # (thread-local)
        hip._check(self.lib.eddlhip_set_stream(hip.dev, self.stream))
        try:
            fn()
        except Exception as e:
            self.error = str(e)
        set_back = self.lib.eddlhip_set_stream(hip.dev, None)
        assert self.lib.hipStreamEndCapture(self.stream, ctypes.byref(self.graph)) == 0 and set_back == 0
        if not self.error:
            assert self.lib.hipGraphInstantiate(ctypes.byref(self.exe), self.graph, None, None, ctypes.c_size_t(0)) == 0

    def launch(self):
        assert self.lib.hipGraphLaunch(self.exe, None) == 0

    def close(self):
        if self.exe:
            self.lib.hipGraphExecDestroy(self.exe)
        self.lib.hipGraphDestroy(self.graph)
        self.lib.hipStreamDestroy(self.stream)


def _step(hip, tokens, pixels):
    """A divided scan and a divided norm: (the step, what it writes, its inputs)."""
    rng = np.random.default_rng([tokens, pixels])
    batch = Ragged(rng, [tokens], before=0, behind=0, kept=False)
    case, b = _scan_case(rng, batch, 16, 16, 1), batch.on(hip)
    X, dt, A, B, C = (hip.array(case[k]) for k in ("x", "dt", "A", "B", "C"))
    M = hip.array(rng.standard_normal((1, 4, pixels, 1), dtype=np.float32))
    Y, N = hip.full(X.shape, -7.0), hip.full(M.shape, -7.0)

    def step():
        hip.selective_scan(X, dt, A, B, C, Y, b)
        hip.group_norm(M, N, 2)

    return step, (Y, N), (X, M)


def test_a_programs_graph_outlives_the_workspace_that_it_names(hip):
    """Replays between eager calls, behind a call that needs a larger workspace and behind a trim give the bits of the eager step."""
    step, outs, ins = _step(hip, 2000, 40000)
    large, large_outs, _ = _step(hip, 60000, 60000)
    hip.workspace_trim()
    step()
    small_bytes = hip.workspace_bytes()
    assert small_bytes > 0
    program = Program(hip, step)
    try:
        assert program.error is None
        host = [t.numpy() for t in ins]
        for turn, between in enumerate((lambda: None, step, large, large, hip.workspace_trim, step)):
            between()
            if turn == 2:
                assert hip.workspace_bytes() > small_bytes
            for t, h in zip(ins, host):
                t.copy_from(h * np.float32(1 + turn))
            for t in outs:
                hip.fill_(t, float(turn))
            program.launch()
            got = [t.numpy() for t in outs]
            step()
            assert all(np.array_equal(g, t.numpy()) for g, t in zip(got, outs)), turn
    finally:
        program.close()
    large()
    want = [t.numpy() for t in large_outs]
    large()
    assert all(np.array_equal(w, t.numpy()) for w, t in zip(want, large_outs))


def test_a_workspace_that_would_grow_while_the_program_captures_is_refused(hip):
    """The capture stays whole, and the same step is captured once it has run."""
    step, outs, _ = _step(hip, 3000, 50000)
    hip.workspace_trim()
    refused = Program(hip, step)
    refused.close()
    assert refused.error is not None and "before recording" in refused.error
    step()
    want = [t.numpy() for t in outs]
    program = Program(hip, step)
    try:
        assert program.error is None
        for _ in range(3):
            for t in outs:
                hip.fill_(t, 0.5)
            program.launch()
            assert all(np.array_equal(w, t.numpy()) for w, t in zip(want, outs))
    finally:
        program.close()
