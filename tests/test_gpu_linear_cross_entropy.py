"""The linear cross entropy against its formula in 64 bits.

Bounds, in half steps u = 2^-24 of fp32.  A logit is a sum of D exact products in fp32: its error is at most
delta = (D + 8) u sum |x w|.  fp32 operands are two parts of fp16, the second rounded to 2^-22 of the element or, with
the row's largest below 2^e, 2^(e - 40), whichever is more; that, for both operands, and the product of the second parts, 2^-22 again,
are 12 u of the same sum more, and 2^(e - 40) of each operand's row with the other's magnitudes.  An
exponential's relative error is its argument's, (|s| u) for the difference and as much for the change of base, and a few
u of its own; the sum over the vocabulary adds at most 200 u (no lane adds more than 128 terms in a row, trees the rest).
So a loss is off by at most 2 delta + (4 R + 210) u + 2 u |lse|, R the largest |s - max|.  An entry p of the softmax is off by that much relative to p, plus
what rounding takes: twice the half step of fp16 where exponentials are kept in it, and the half step of the type the
slope is carried in; as two parts of fp16, 2^-22.  The products sum V (or N) terms in fp32, and the result is rounded once.
Where the slope's parts carry a row's power of two their least error is 2^-39 of the largest row's other operand."""
import numpy as np
import pytest

from operator_lib import ALL_TYPES, BF16, F16, F32, HALF_STEP, TINY, Buffers, loss_reference, numpy_type, to_bits, to_float

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
IGNORE = -100


def data(t, n, v, d, ignored=0.2, seed=0, lean=6.0):
    rng = np.random.default_rng(seed + n * 31 + v + d)
    w = to_bits(rng.normal(size=(v, d)) * d ** -0.5, t)
    targets = rng.integers(0, v, n).astype(np.int32)
    x = rng.normal(size=(n, d)) + lean * rng.uniform(size=(n, 1)) * to_float(w, t)[targets]
    targets[rng.uniform(size=n) < ignored] = IGNORE
    return to_bits(x, t), w, targets


def run(b, t, o, x, w, targets, mean=1, scale=1.0, amp=0, dx=True, dw=True, add=None, pad=0, shift=0, least=False, queue=0):
    n, d = x.shape
    v = w.shape[0]
    hx, hw, ht = b.put(x, shift, d + pad), b.put(w, shift, d + pad), b.put(targets)
    losses, loss = b.empty(max(n, 1), np.float32), b.empty(2, np.float32)
    gx = b.empty((max(n, 1), d), numpy_type(t), shift, d + pad) if dx else 0
    gw = (b.put(add, shift, d + pad) if add is not None else b.empty((v, d), numpy_type(o), shift, d + pad)) if dw else 0
    ask = b.lib.gm_linear_cross_entropy_least_workspace if least else b.lib.gm_linear_cross_entropy_workspace
    need = ask(n, v, d, hw, d + pad, t, o, int(dx or dw))
    assert need > 0
    b.check(b.lib.execute_linear_cross_entropy(b.device, queue, hx, hw, ht, losses, loss, gx, gw, n, v, d, d + pad, d + pad, d + pad, d + pad, t, o,
                                               IGNORE, mean, scale, amp, int(add is not None), b.space(need), need))
    out = {"losses": b.get(losses, (max(n, 1),), np.float32)[:n], "loss": b.get(loss, (2,), np.float32)}
    if dx:
        out["dx"] = b.get(gx, (max(n, 1), d), numpy_type(t), d + pad)[:n]
    if dw:
        out["dw"] = b.get(gw, (v, d), numpy_type(o), d + pad)
    return out


def check(got, t, o, x, w, targets, mean=1, scale=1.0, add=None):
    n, d = x.shape
    v = w.shape[0]
    fx, fw = to_float(x, t).astype(np.float64), to_float(w, t).astype(np.float64)
    losses, loss, count, dx, dw, ds = loss_reference(fx, fw, targets, IGNORE, mean, scale)
    counts = (targets != IGNORE) & (targets >= 0) & (targets < v)
    fx = np.where(counts[:, None], fx, 0.0)
    s = fx @ fw.T
    top = s.max(1, keepdims=True)
    delta = (d + (20 if t == F32 else 8)) * U * (np.abs(fx) @ np.abs(fw).T).max(1)
    reach = lambda m: 2 * np.abs(m).max(initial=0.0)      # of 2^e, over all rows
    if t == F32:
        delta = delta + 2.0 ** -40 * (reach(fx) * np.abs(fw).sum(1).max() + reach(fw) * np.abs(fx).sum(1))
    off = 2 * delta + (4 * (top - s).max(1) + 210) * U + 2 * U * np.abs(top[:, 0] + np.log(v))      # per token
    assert np.all(np.abs(got["losses"] - losses) <= np.where(counts, off, 0.0))
    assert got["loss"][1] == count
    assert abs(got["loss"][0] - loss) <= (off[counts].sum() / (max(1, count) if mean else 1)) + 2 * U * abs(loss)
    c = abs(scale) / max(1, count) if mean else abs(scale)
    p = np.where(ds < 0, 1 + ds, ds)      # the target's entry is p - 1
    p = np.clip(p, 0, 1)
    kept = 2 * HALF_STEP[F16] if o != F32 else 0.0
    # least values: fp16 keeps exponentials down to 2^-39 of their tile's largest and slopes down to 2^-38
    floor = 2.0 ** -37 if t != F32 else 0.0
    for name, kind, value, right, over in (("dx", t, dx, lambda a: a @ np.abs(fw), v), ("dw", o, dw, lambda a: a.T @ np.abs(fx), n)):
        if name not in got:
            continue
        parts = t == F32 or (name == "dw" and o == F32)
        slope = 2.0 ** -22 if parts else HALF_STEP[t]
        err = np.where(counts[:, None], p * (off[:, None] + (kept + 4 * U) * (ds > 0)) + np.abs(ds) * (slope + (over + 22) * U) + floor, 0.0)
        if name == "dw" and add is not None:
            value = value + to_float(add, o)
        other = fw if name == "dx" else fx
        least = (over * 2.0 ** -39 + np.abs(ds).sum(1 if name == "dx" else 0)[:, None] * 2.0 ** -40) * reach(other) if parts else 0.0
        bound = c * (right(err) + least) + HALF_STEP[kind] * np.abs(value) * (1 + 2.0 ** -7) + TINY[kind] + 4 * U * np.abs(value)
        diff = np.abs(to_float(got[name], kind).astype(np.float64) - value)
        assert np.all(diff <= bound), (name, (diff / bound).max())


PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]


@pytest.mark.parametrize("t, o", PAIRS)
@pytest.mark.parametrize("n, v, d", [(1, 1, 1), (1, 300, 64), (3, 65, 128), (32, 128, 64), (33, 129, 65), (65, 1000, 192), (130, 257, 100)])
def test_small(t, o, n, v, d):
    x, w, targets = data(t, n, v, d, ignored=0.2 if n > 3 else 0.0)
    scale = 64.0
    with Buffers() as b:
        check(run(b, t, o, x, w, targets, scale=scale), t, o, x, w, targets, scale=scale)


@pytest.mark.parametrize("t, o", PAIRS)
def test_wide_tiles(t, o):
    """Enough tiles for the largest shape in all three products, ragged at every edge; sums split and whole."""
    n, v, d = 300, 4099, 4096 + 64 if t != F32 else 320
    x, w, targets = data(t, n, v, d)
    with Buffers() as b:
        check(run(b, t, o, x, w, targets, mean=0, scale=0.5), t, o, x, w, targets, mean=0, scale=0.5)


@pytest.mark.parametrize("t, o", [(F16, F16), (BF16, F32)])
def test_many_tokens(t, o):
    n, v, d = 4100, 4300, 192
    x, w, targets = data(t, n, v, d)
    with Buffers() as b:
        check(run(b, t, o, x, w, targets, scale=1024.0), t, o, x, w, targets, scale=1024.0)


@pytest.mark.parametrize("t, o", PAIRS)
@pytest.mark.parametrize("add", [False, True])
def test_split_sums_of_the_weight_gradient(t, o, add):
    """Few words and many tokens: the sum over the tokens is cut into parts, more of them than a batch of which few count fills."""
    v, d = 130, 70
    for n, ignored in ((2500, 0.1), (2500, 0.99)):
        x, w, targets = data(t, n, v, d, ignored=ignored)
        before = to_bits(np.random.default_rng(2).normal(size=(v, d)), o) if add else None
        with Buffers() as b:
            check(run(b, t, o, x, w, targets, scale=8.0, add=before), t, o, x, w, targets, scale=8.0, add=before)


def test_wide_tiles_of_the_hidden_gradient():
    n, v, d = 4097, 300, 4100
    x, w, targets = data(BF16, n, v, d)
    with Buffers() as b:
        check(run(b, BF16, BF16, x, w, targets), BF16, BF16, x, w, targets)


@pytest.mark.parametrize("t, o", PAIRS)
def test_tokens_in_parts(t, o):
    """The least workspace: 256 tokens at a time, the last part of them without one that counts; with and without adding."""
    n, v, d = 700, 500, 96
    x, w, targets = data(t, n, v, d, ignored=0.4)
    with Buffers() as b:
        check(run(b, t, o, x, w, targets, scale=32.0, least=True), t, o, x, w, targets, scale=32.0)
        add = to_bits(np.random.default_rng(1).normal(size=(v, d)), o)
        check(run(b, t, o, x, w, targets, scale=32.0, least=True, add=add), t, o, x, w, targets, scale=32.0, add=add)


@pytest.mark.parametrize("t, o", PAIRS)
@pytest.mark.parametrize("d, pad, shift", [(65, 3, 4), (64, 8, 16), (64, 1, 0), (64, 0, 4), (63, 0, 0)])
def test_strides_and_alignment(t, o, d, pad, shift):
    x, w, targets = data(t, 70, 300, d)
    with Buffers() as b:
        check(run(b, t, o, x, w, targets, pad=pad, shift=shift), t, o, x, w, targets)


@pytest.mark.parametrize("t, o", PAIRS)
def test_each_output_alone(t, o):
    """The loss alone, either gradient alone: the same values, bit for bit, as all together."""
    x, w, targets = data(t, 50, 400, 128)
    with Buffers() as b:
        every = run(b, t, o, x, w, targets)
        for dx, dw in ((False, False), (True, False), (False, True)):
            got = run(b, t, o, x, w, targets, dx=dx, dw=dw)
            for name in got:
                if name.startswith("loss") and not (dx or dw):      # (the exponentials are made another way: the bound holds)
                    continue
                assert np.array_equal(got[name].view(np.uint8), every[name].view(np.uint8)), name
        check(run(b, t, o, x, w, targets, dx=False, dw=False), t, o, x, w, targets)


@pytest.mark.parametrize("t, o", PAIRS)
def test_tokens_that_do_not_count_reach_nothing(t, o):
    """NaN and inf in the rows of ignored tokens, of targets outside the vocabulary too."""
    n, v, d = 90, 200, 64
    x, w, targets = data(t, n, v, d, ignored=0.0)
    targets[::4], targets[1::9], targets[2::9] = IGNORE, v, -1
    out = ~((targets >= 0) & (targets < v))
    bad = to_float(x, t).copy()
    bad[out] = np.array([np.nan, np.inf, -np.inf, 1.0], np.float32)[np.arange(d) % 4]
    with Buffers() as b:
        clean, got = run(b, t, o, x, w, targets), run(b, t, o, to_bits(bad, t), w, targets)
        for name in clean:
            assert np.array_equal(got[name].view(np.uint8), clean[name].view(np.uint8)), name
        assert np.all(got["losses"][out] == 0) and np.all(to_float(got["dx"], t)[out] == 0)
        check(got, t, o, x, w, targets)


@pytest.mark.parametrize("t, o", PAIRS)
@pytest.mark.parametrize("n", [0, 1, 100])
def test_no_token_counts(t, o, n):
    x, w, targets = data(t, max(n, 1), 130, 64, ignored=0.0)
    x, targets = x[:n], np.full(n, IGNORE, np.int32)
    with Buffers() as b:
        got = run(b, t, o, x, w, targets) if n else None
        if n == 0:
            hx, hw, losses, loss, gw = b.put(w), b.put(w), b.empty(1, np.float32), b.empty(2, np.float32), b.empty(w.shape, numpy_type(o))
            need = b.lib.gm_linear_cross_entropy_workspace(0, 130, 64, hw, 64, t, o, 1)
            b.check(b.lib.execute_linear_cross_entropy(b.device, 0, hx, hw, losses, losses, loss, 0, gw, 0, 130, 64, 64, 64, 64, 64, t, o, IGNORE, 1,
                                                       1.0, 0, 0, b.space(need), need))
            got = {"losses": np.zeros(0), "loss": b.get(loss, (2,), np.float32), "dx": np.zeros(0, numpy_type(t)),
                   "dw": b.get(gw, w.shape, numpy_type(o))}
        assert np.all(got["losses"] == 0) and np.array_equal(got["loss"], [0, 0])
        assert np.all(to_float(got["dx"], t) == 0) and np.all(to_float(got["dw"], o) == 0)


@pytest.mark.parametrize("t", ALL_TYPES)
def test_certain_and_hopeless_tokens(t):
    """Logits of hundreds: losses near 0, whose slopes are p - 1 of p near 1, and losses of hundreds; no overflow."""
    n, v, d = 40, 300, 64
    rng = np.random.default_rng(4)
    w = to_bits(rng.normal(size=(v, d)) * 0.5, t)
    targets = rng.integers(0, v, n).astype(np.int32)
    # a lean of 0.1 to 30 times the target's row, for half of them away from it
    lean = np.geomspace(0.1, 30, n) * np.where(np.arange(n) % 2, 1, -1)
    x = to_bits(lean[:, None] * to_float(w, t)[targets], t)
    with Buffers() as b:
        check(run(b, t, t, x, w, targets, scale=16.0), t, t, x, w, targets, scale=16.0)


@pytest.mark.parametrize("t", [F32, BF16])
def test_rows_of_very_different_size(t):
    """Rows of both operands between 2^-40 and 2^20 times the others (and rows of zeros): the rows' powers of two are undone
    exactly, and what a sum leaves out of a small row stays below its largest term's error."""
    n, v, d = 70, 200, 96
    x, w, targets = data(t, n, v, d)
    rng = np.random.default_rng(12)
    fx = to_float(x, t) * np.exp2(rng.integers(-40, 3, (n, 1))).astype(np.float32)
    fw = to_float(w, t) * np.exp2(rng.integers(-40, 3, (v, 1))).astype(np.float32)
    fx[5], fw[7] = 0.0, 0.0
    small = to_bits(fx * np.float32(2.0 ** 20), t), to_bits(fw * np.float32(2.0 ** -20), t)
    for x, w in ((to_bits(fx, t), to_bits(fw, t)), small):
        with Buffers() as b:
            check(run(b, t, F32, x, w, targets, scale=4.0), t, F32, x, w, targets, scale=4.0)


def test_overflow_is_inf_and_nan_spreads_as_in_the_formula():
    """fp16 gradients that pass 65504 are inf (the mixed-precision step drops them); a NaN in a token that counts makes its
    loss NaN and no other token's."""
    n, v, d = 20, 100, 64
    x, w, targets = data(F16, n, v, d, ignored=0.0)
    with Buffers() as b:
        got = run(b, F16, F16, x, w, targets, mean=0, scale=3e7)
        assert np.isinf(to_float(got["dw"], F16)).any() and not np.isnan(to_float(got["dw"], F16)).any()
        x[3, 5] = np.nan
        got = run(b, F16, F16, x, w, targets)
        assert np.isnan(got["losses"][3]) and np.isnan(got["losses"]).sum() == 1 and np.isnan(got["loss"][0]) and got["loss"][1] == n
        assert np.isnan(to_float(got["dx"], F16)[3]).all() and not np.isnan(np.delete(to_float(got["dx"], F16), 3, 0)).any()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_row_of_fp32_that_is_not_finite(bad):
    """It has no power of two; its own loss and slopes are NaN, and what other tokens give is what it was, bit for bit."""
    n, v, d = 30, 200, 96
    x, w, targets = data(F32, n, v, d, ignored=0.0)
    with Buffers() as b:
        clean = run(b, F32, F32, x, w, targets)
        x[4, 7] = bad
        got = run(b, F32, F32, x, w, targets)
        assert np.isnan(got["losses"][4]) and np.isnan(got["dx"][4]).all() and np.isnan(got["loss"][0])
        for name in ("losses", "dx"):
            assert np.array_equal(np.delete(got[name], 4, 0).view(np.uint8), np.delete(clean[name], 4, 0).view(np.uint8)), name


@pytest.mark.parametrize("t, o", PAIRS)
def test_results_repeat(t, o):
    x, w, targets = data(t, 400, 3001, 320)
    with Buffers() as b:
        one, two = run(b, t, o, x, w, targets), run(b, t, o, x, w, targets)
        for name in one:
            assert np.array_equal(one[name].view(np.uint8), two[name].view(np.uint8)), name


def test_gradients_against_differences():
    """The losses' change along the gradient's direction, from the same kernels in fp32.  The third derivative of a token's
    loss along a direction is a third central moment of the logits' change: at most 2 R^3, R its largest change."""
    n, v, d = 60, 150, 96
    x, w, targets = data(F32, n, v, d)
    with Buffers() as b:
        base = run(b, F32, F32, x, w, targets)
        for name, h in (("dx", 0.05), ("dw", 0.02)):
            g = base[name].astype(np.float64)
            direction = g / np.linalg.norm(g)
            a = []
            for sign in (1, -1):
                step = (sign * h * direction).astype(np.float32)
                got = run(b, F32, F32, x + step, w, targets, dx=False, dw=False) if name == "dx" else run(b, F32, F32, x, w + step, targets,
                                                                                                      dx=False, dw=False)
                a.append(got["losses"].astype(np.float64).sum() / base["loss"][1])
            change = np.abs((direction if name == "dx" else x) @ (w if name == "dx" else direction).T).max() * 2
            noise = 2 * ((d + 8) * U * (np.abs(x) @ np.abs(w).T).max() + 300 * U) / (2 * h) + 4 * U * np.abs(x).max() * np.abs(w).max() * d / h
            assert abs((a[0] - a[1]) / (2 * h) - (g * direction).sum()) <= h * h / 6 * 2 * change ** 3 + noise + 1e-5 * np.linalg.norm(g)


def test_the_loss_scale_is_read_on_the_device():
    """amp_state multiplies the gradients by the scale as of now, whichever of its two records holds it."""
    x, w, targets = data(F16, 30, 200, 64)
    with Buffers() as b:
        amp = b.lib.gm_amp_state_create(b.device, 1024.0, 2.0, 0.5, 1)
        assert amp
        for k in range(3):
            got, want = run(b, F16, F16, x, w, targets, amp=amp, scale=0.5), run(b, F16, F16, x, w, targets, scale=0.5 * 1024.0 * 2 ** k)
            for name in want:
                assert np.array_equal(got[name].view(np.uint8), want[name].view(np.uint8)), (k, name)
            # a clean step over one element doubles the scale (interval 1) and swaps the records
            h = [b.put(np.ones(4, np.float32)) for _ in range(3)]
            g16, w16 = b.put(np.ones(4, np.float16)), b.put(np.ones(4, np.float16))
            from __graft_entry__ import load_package
            pkg = load_package()
            import ctypes
            skipped = ctypes.c_int(-1)
            one = lambda a: pkg.handle_array([a])
            b.check(b.lib.execute_adam_amp_step(b.device, one(h[0]), one(g16), one(h[1]), one(h[2]), one(w16), 1, pkg.int_array([16]), 1e-3, 0.9,
                                                0.999, 1e-8, 0.0, k + 1, amp, ctypes.byref(skipped), None, None))
            assert skipped.value == 0
        assert b.lib.execute_linear_cross_entropy(b.device, 0, *([b.put(x)] * 5), 0, 0, 1, 1, 1, 1, 1, 1, 1, F16, F16, IGNORE, 1, 1.0,
                                                  b.put(np.zeros(64, np.uint8)), 0, b.space(1 << 20), 1 << 20) == -16
        b.lib.gm_amp_state_destroy(amp)
