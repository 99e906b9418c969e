"""The operators together, as a training step uses them: a language model of one table, tied at both ends.

    h0 = dropout(sqrt(D) table[tokens])      h1 = h0 + dropout(h0)      loss = cross entropy(h1 table^T, targets)

and back: d h1 and d table from the loss, d h0 = d h1 + dropout(d h1), d table += the lookup's gradient of d h0; then the
mixed-precision step.  Gradients against the formula in 64 bits and against differences of the loss; the step against the CPU
oracle; the whole on a caller's stream, captured into a graph and replayed."""
import ctypes

import numpy as np
import pytest

from operator_lib import F16, F32, HALF_STEP, TINY, Buffers, mask, numpy_type, to_bits, to_float
from oracle_lib import oracle

pytestmark = pytest.mark.gpu
IGNORE, EMBED_P, BLOCK_P = -100, 0.1, 0.2
STATE = (2024, 7, 1, 0)


class Model:
    """Buffers and calls of the model for n tokens of a vocabulary of v words."""

    def __init__(self, b, t, n, v, d, table, tokens, targets):
        self.b, self.t, self.n, self.v, self.d = b, t, n, v, d
        kind = numpy_type(t)
        self.table, self.tokens, self.targets = b.put(table), b.put(tokens), b.put(targets)
        self.h0, self.h1, self.g1, self.g0 = (b.empty((n, d), kind) for _ in range(4))
        self.grad = b.empty((v, d), kind)
        self.losses, self.loss = b.empty(n, np.float32), b.empty(2, np.float32)
        self.loss_bytes = b.lib.gm_linear_cross_entropy_workspace(n, v, d, self.table, d, t, t, 1)
        self.table_bytes = b.lib.gm_embedding_gradient_workspace(n, v, d)
        self.loss_space, self.table_space = b.space(self.loss_bytes), b.space(self.table_bytes)

    def forward_and_back(self, rng, queue=0, amp=0, scale=1.0):
        b, n, v, d, t = self.b, self.n, self.v, self.d, self.t
        b.check(b.lib.execute_embedding_lookup(b.device, queue, self.table, self.tokens, self.h0, n, v, d, d, d, t, d ** 0.5, EMBED_P, rng, 0))
        b.check(b.lib.execute_dropout(b.device, queue, self.h0, self.h0, self.h1, n * d, t, BLOCK_P, rng, 1))
        b.check(b.lib.execute_linear_cross_entropy(b.device, queue, self.h1, self.table, self.targets, self.losses, self.loss, self.g1, self.grad, n, v,
                                                   d, d, d, d, d, t, t, IGNORE, 1, scale, amp, 0, self.loss_space, self.loss_bytes))
        b.check(b.lib.execute_dropout(b.device, queue, self.g1, self.g1, self.g0, n * d, t, BLOCK_P, rng, 1))
        b.check(b.lib.execute_embedding_gradient(b.device, queue, self.g0, self.tokens, self.grad, n, v, d, d, d, t, t, d ** 0.5, -1, 1, EMBED_P, rng, 0,
                                                 self.table_space, self.table_bytes))

    def results(self):
        get = self.b.get
        return {"losses": get(self.losses, (self.n,), np.float32), "loss": get(self.loss, (2,), np.float32),
                "grad": get(self.grad, (self.v, self.d), numpy_type(self.t))}


def data(t, n, v, d, seed):
    rng = np.random.default_rng(seed)
    table = to_bits(rng.normal(size=(v, d)) * 0.3 * d ** -0.5, t)
    tokens = rng.integers(0, v, n).astype(np.int32)
    targets = np.roll(tokens, -1)
    targets[-1] = IGNORE
    tokens[n // 3], targets[n // 3], targets[n // 3 - 1] = -1, IGNORE, IGNORE      # padding
    return table, tokens, targets


def formula(table, tokens, targets, state, t=F32, move=None):
    """In 64 bits: the mean loss, d table, how far the operators' may be from both, and (move: a direction of the table) the second
    and third derivatives' bounds along it.

    r is half a step of the type that tensors are stored in, u of fp32, in which sums are made.  h is rounded twice on its way (and
    made by three products in fp32); a logit is off by what that does to it and by (D + 8) u of its terms' magnitudes (D); a
    softmax entry p by that, twice, by the exponential's (4 R + 210) u and (16-bit types) by 3 r, and the slope by r more (fp32: operands and slopes are two parts of fp16,
    12 u a product more and 4 u for the slope).  Every
    gradient that is stored is rounded once, the table's a second time when the lookup's is added."""
    v, d = table.shape
    n = tokens.size
    r, u = HALF_STEP[t], 2.0 ** -24
    e = table.astype(np.float64)
    fine = tokens >= 0
    keep0, by0 = mask(n * d, EMBED_P, state, 0)
    keep1, by1 = mask(n * d, BLOCK_P, state, 1)
    m = keep0.reshape(n, d) * np.float64(by0) * fine[:, None] * np.sqrt(d) * (1.0 + keep1.reshape(n, d) * np.float64(by1))
    h = e[np.where(fine, tokens, 0)] * m
    rows = np.nonzero(targets >= 0)[0]
    c = 1.0 / rows.size
    s = h[rows] @ e.T
    top = s.max(1, keepdims=True)
    p = np.exp(s - top)
    total = p.sum(1, keepdims=True)
    p /= total
    at = (np.arange(rows.size), targets[rows])
    losses = (np.log(total) + top)[:, 0] - s[at]
    ds = p.copy()
    ds[at] -= 1.0
    err_h = np.abs(h) * (2 * r + 4 * u)
    # (what the parts' least steps, 2^-40 and 2^-39 of a row's largest, add is below the 1 % that errors are taken larger at the end)
    delta = (err_h[rows] @ np.abs(e).T + (d + (8 if t != F32 else 20)) * u * (np.abs(h[rows]) @ np.abs(e).T)).max(1)
    off = 2 * delta + (4 * (top - s).max(1) + 210) * u + 2 * u * np.abs(top[:, 0] + np.log(v))
    err_ds = p * (off[:, None] + 3 * r) + np.abs(ds) * (r + 30 * u) + (2.0 ** -37 if t != F32 else 0.0)
    grad = c * (ds.T @ h[rows])
    err = c * (err_ds.T @ np.abs(h[rows]) + np.abs(ds).T @ err_h[rows] + n * u * (np.abs(ds).T @ np.abs(h[rows]))) + r * np.abs(grad)
    back, err_back = np.zeros((n, d)), np.zeros((n, d))
    back[rows] = c * (ds @ e)
    err_back[rows] = c * (err_ds @ np.abs(e) + v * u * (np.abs(ds) @ np.abs(e)))
    err_back = (err_back + np.abs(back) * (2 * r + 6 * u)) * 1.01      # (1.01: products of errors)
    np.add.at(grad, tokens[fine], (back * m)[fine])
    np.add.at(err, tokens[fine], ((err_back + n * u * np.abs(back)) * np.abs(m))[fine])
    out = {"loss": losses.mean(), "loss_off": off.mean() + 2 * u * losses.mean(), "grad": grad, "off": err * 1.01 + r * np.abs(grad) + TINY[t]}
    if move is not None:
        # logits are s + a x + b x^2 along the direction: the loss's third derivative is the third central moment of their
        # slope, at most its spread cubed, and three covariances with 2 b, each at most a quarter of both spreads' product
        hd = move[np.where(fine, tokens, 0)] * m
        a, b = hd[rows] @ e.T + h[rows] @ move.T, hd[rows] @ move.T
        spread = lambda x: (x.max(1) - x.min(1)).max()
        out["third"] = lambda step: (spread(a) + 2 * step * spread(b)) ** 3 + 3 * (spread(a) + 2 * step * spread(b)) * 2 * spread(b) / 4
    return out


def test_gradient_against_the_formula_and_differences():
    n, v, d = 150, 90, 64
    table, tokens, targets = data(F32, n, v, d, 5)
    want = formula(table, tokens, targets, STATE)
    with Buffers() as b:
        model = Model(b, F32, n, v, d, table, tokens, targets)
        model.forward_and_back(b.state(STATE))
        got = model.results()
        assert abs(got["loss"][0] - want["loss"]) <= want["loss_off"]
        assert np.all(np.abs(got["grad"] - want["grad"]) <= want["off"])
        g = got["grad"].astype(np.float64)
        direction, step, losses = g / np.linalg.norm(g), 0.01, []
        for sign in (1, -1):
            moved = Model(b, F32, n, v, d, (table + sign * step * direction).astype(np.float32), tokens, targets)
            moved.forward_and_back(b.state(STATE))
            losses.append(moved.results()["losses"].astype(np.float64).sum() / got["loss"][1])
        third = formula(table, tokens, targets, STATE, move=direction)["third"](step)
        noise = (want["loss_off"] + 2.0 ** -24 * np.abs(table).max() * np.abs(g).sum()) / step      # the losses', the moved tables' rounding
        assert abs((losses[0] - losses[1]) / (2 * step) - np.linalg.norm(g)) <= step * step / 6 * third + noise + (want["off"] * np.abs(direction)).sum()


def test_steps_follow_the_oracle():
    """fp16: three mixed-precision steps on the table, the second overflowing.  The gradient that the operators leave is what the
    oracle is given; weights, copy, moments, scale and counters come out bit for bit."""
    n, v, d = 200, 300, 72
    table, tokens, targets = data(F16, n, v, d, 6)
    from __graft_entry__ import load_package
    pkg = load_package()
    o = oracle()
    hyper = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=1e-3)
    with Buffers() as b:
        amp = b.lib.gm_amp_state_create(b.device, 1024.0, 2.0, 0.5, 1)
        st = o.amp_state()
        st.scale, st.growth_interval = 1024.0, 1
        master = table.astype(np.float32).reshape(-1)
        m, va, copy = np.zeros_like(master), np.zeros_like(master), table.reshape(-1).view(np.uint16).copy()
        dev = [b.put(master), b.put(m), b.put(va)]
        model = Model(b, F16, n, v, d, table, tokens, targets)
        rng = b.state(STATE)
        one = lambda a: pkg.handle_array([a])
        try:
            for step, scale in enumerate((1.0, 1e9, 1.0)):
                model.forward_and_back(rng, amp=amp, scale=scale)
                b.check(b.lib.gm_rng_state_advance(b.device, 0, rng))
                grad = model.results()["grad"]
                assert np.isfinite(to_float(grad, F16)).all() == (scale == 1.0)
                skipped, out_scale, tracker = ctypes.c_int(-1), ctypes.c_float(), ctypes.c_int()
                b.check(b.lib.execute_adam_amp_step(b.device, one(dev[0]), one(model.grad), one(dev[1]), one(dev[2]), one(model.table), 1,
                                                    pkg.int_array([4 * v * d]), hyper["lr"], hyper["beta1"], hyper["beta2"], hyper["eps"],
                                                    hyper["weight_decay"], int(st.step_count) + 1, amp, ctypes.byref(skipped), ctypes.byref(out_scale),
                                                    ctypes.byref(tracker)))
                want = o.adam_amp([master], [grad.reshape(-1).view(np.uint16).copy()], [m], [va], [copy], state=st, **hyper)
                assert skipped.value == want == int(scale != 1.0) and out_scale.value == st.scale
                for h, host in zip(dev, (master, m, va)):
                    assert np.array_equal(b.get(h, (v * d,), np.float32).view(np.uint32), host.view(np.uint32)), step
                assert np.array_equal(b.get(model.table, (v * d,), np.uint16), copy)
            want = formula(to_float(copy.view(np.float16).reshape(v, d), F16), tokens, targets, (STATE[0], STATE[1], STATE[2] + 3, 0), F16)
            model.forward_and_back(rng, amp=amp)
            got = model.results()
            assert abs(got["loss"][0] - want["loss"]) <= want["loss_off"]
            assert np.all(np.abs(to_float(got["grad"], F16).astype(np.float64) / st.scale - want["grad"]) <= want["off"])
        finally:
            b.dev.synchronize()
            b.lib.gm_amp_state_destroy(amp)


@pytest.fixture()
def hip():
    lib = ctypes.CDLL("/opt/rocm/lib/libamdhip64.so")
    p, vp = ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p
    lib.hipStreamCreateWithFlags.argtypes = [p, ctypes.c_uint]
    lib.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    lib.hipStreamEndCapture.argtypes = [vp, p]
    lib.hipGraphInstantiate.argtypes = [p, vp, vp, vp, ctypes.c_size_t]
    lib.hipGraphLaunch.argtypes = [vp, vp]
    for name in ("hipStreamSynchronize", "hipStreamDestroy", "hipGraphDestroy", "hipGraphExecDestroy"):
        getattr(lib, name).argtypes = [vp]
    return lib


@pytest.mark.parametrize("n, v", [(70, 400), (9000, 200)])
def test_captured_step_on_a_callers_stream(hip, n, v):
    """The step captured on a stream of the caller's and replayed, eager work of the library and changes of the loss scale between
    the replays: each replay draws the next step's masks, takes the scale as of then, and gives the eager step's bits."""
    d = 48
    table, tokens, targets = data(F16, n, v, d, 8)
    stream, graph, program = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
    with Buffers() as b:
        amp = b.lib.gm_amp_state_create(b.device, 64.0, 2.0, 0.5, 1000)
        queue = b.lib.gm_command_queue_for_stream(b.device, stream)
        assert queue
        captured, eager = Model(b, F16, n, v, d, table, tokens, targets), Model(b, F16, n, v, d, table, tokens, targets)
        rng, rng_eager = b.state(STATE), b.state(STATE)
        b.dev.synchronize()
        try:
            assert hip.hipStreamBeginCapture(stream, 0) == 0
            b.check(b.lib.gm_rng_state_advance(b.device, queue, rng))
            captured.forward_and_back(rng, queue=queue, amp=amp)
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
            assert hip.hipGraphInstantiate(ctypes.byref(program), graph, None, None, 0) == 0
            before = None
            for replay in range(4):
                assert b.lib.gm_amp_state_set(amp, 64.0 * 2 ** replay, 0) == 0
                assert hip.hipGraphLaunch(program, stream) == 0
                if replay == 2:
                    assert hip.hipStreamSynchronize(stream) == 0
                b.check(b.lib.gm_rng_state_advance(b.device, 0, rng_eager))
                eager.forward_and_back(rng_eager, amp=amp)
                b.dev.synchronize()
                assert hip.hipStreamSynchronize(stream) == 0
                got, want = captured.results(), eager.results()
                for name in want:
                    assert np.array_equal(got[name].view(np.uint8), want[name].view(np.uint8)), (replay, name)
                assert before is None or not np.array_equal(before, got["grad"])
                before = got["grad"]
        finally:
            hip.hipStreamSynchronize(stream)
            b.dev.synchronize()
            if program.value:
                hip.hipGraphExecDestroy(program)
            if graph.value:
                hip.hipGraphDestroy(graph)
            b.lib.release_command_queue(queue)
            hip.hipStreamDestroy(stream)
            b.lib.gm_amp_state_destroy(amp)


def test_two_calls_at_once(hip):
    """The same operators on two streams, a workspace each, at the same time: each its own results."""
    n, v, d = 600, 900, 128
    streams, queues, models, want = [], [], [], []
    with Buffers() as b:
        rng = b.state(STATE)
        for k in range(2):
            table, tokens, targets = data(F16, n, v, d, 20 + k)
            models.append(Model(b, F16, n, v, d, table, tokens, targets))
            models[k].forward_and_back(rng)
            want.append(models[k].results())
            streams.append(ctypes.c_void_p())
            assert hip.hipStreamCreateWithFlags(ctypes.byref(streams[k]), 1) == 0
            queues.append(b.lib.gm_command_queue_for_stream(b.device, streams[k]))
        try:
            for _ in range(5):
                for k in range(2):
                    models[k].forward_and_back(rng, queue=queues[k])
            for k in range(2):
                assert hip.hipStreamSynchronize(streams[k]) == 0
                got = models[k].results()
                for name in got:
                    assert np.array_equal(got[name].view(np.uint8), want[k][name].view(np.uint8)), (k, name)
        finally:
            for k in range(2):
                hip.hipStreamSynchronize(streams[k])
                b.lib.release_command_queue(queues[k])
                hip.hipStreamDestroy(streams[k])


def test_workspaces_and_queues():
    with Buffers() as b:
        h = b.lib.gm_allocate_workspace(b.device, 3_000_000_001)      # above what allocate_metal_buffer can name
        assert h and h % 256 == 0 and b.lib.gm_buffer_length(h) == 3_000_000_256
        b.lib.deallocate_metal_buffer(h)
        assert b.lib.gm_buffer_length(h) == 0
        x = b.put(np.ones(64, np.float32))
        own = b.lib.create_command_queue(b.device)
        b.check(b.lib.execute_dropout(b.device, own, x, 0, x, 64, F32, 0.0, 0, 0))
        assert b.lib.execute_dropout(b.device, b.put(np.zeros(64, np.uint8)), x, 0, x, 64, F32, 0.0, 0, 0) == -2      # not a queue
        b.lib.release_command_queue(own)
