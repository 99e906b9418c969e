"""Embedding lookup and its gradient by sorted tokens.  The lookup is exact (one fp32 product, one more under dropout, one
rounding).  A row of the gradient is a sum of c terms in fp32: its error is at most c half steps of fp32 of the sum of
the terms' magnitudes, three more for the dropout factor, the scale and the addition to what was there, and one half
step of the type it is written in."""
import numpy as np
import pytest

from operator_lib import ALL_TYPES, BF16, F16, F32, HALF_STEP, TINY, Buffers, mask, numpy_type, same, size_of, to_bits, to_float

pytestmark = pytest.mark.gpu
STATE = (77, 3, 9, 0)


def tokens_for(kind, n, vocab, rng):
    if kind == "one word":
        return np.full(n, vocab - 1, np.int32)
    if kind == "all padding":
        return np.full(n, -1, np.int32)
    ids = np.minimum(np.exp(rng.uniform(0, np.log(vocab + 1), n)).astype(np.int64) - 1, vocab - 1).astype(np.int32)
    if kind == "padded":
        ids[rng.uniform(size=n) < 0.2] = -1
        ids[rng.uniform(size=n) < 0.1] = vocab
        ids[rng.uniform(size=n) < 0.05] = np.iinfo(np.int32).min
        ids[rng.uniform(size=n) < 0.05] = np.iinfo(np.int32).max
    return ids


@pytest.mark.parametrize("t", ALL_TYPES)
@pytest.mark.parametrize("n, vocab, dim, pad, shift", [(1, 1, 1, 0, 0), (1, 50, 4096, 0, 0), (5, 11, 8, 0, 0), (129, 1000, 100, 4, 4),
                                                       (64, 77, 65, 7, 4), (300, 333, 256, 8, 16), (33, 20, 7, 0, 4)])
def test_lookup(t, n, vocab, dim, pad, shift):
    rng = np.random.default_rng(n + dim)
    table, ids = to_bits(rng.normal(size=(vocab, dim)), t), tokens_for("padded" if n > 1 else "plain", n, vocab, rng)
    scale = np.float32(dim ** 0.5)
    fine = (ids >= 0) & (ids < vocab)
    y = np.where(fine[:, None], to_float(table, t)[np.where(fine, ids, 0)] * scale, np.float32(0))
    with Buffers() as b:
        ht, hi, s = b.put(table, shift, dim + pad), b.put(ids), b.state(STATE)
        for p in (0.0, 0.2):
            want = y
            if p:
                keep, by = mask(n * dim, p, STATE, 4)
                want = np.where(keep.reshape(n, dim), y * by, np.float32(0))
            out = b.empty((n, dim), numpy_type(t), shift, dim + pad)
            b.check(b.lib.execute_embedding_lookup(b.device, 0, ht, hi, out, n, vocab, dim, dim + pad, dim + pad, t, float(scale), p, s, 4))
            assert same(b.get(out, (n, dim), numpy_type(t), dim + pad), to_bits(want, t), t), p


def gradient_case(t, o, n, vocab, dim, kind, pad=0, shift=0, p=0.0, add=False, padding=-1, scale=1.0, twice=False):
    rng = np.random.default_rng(n * 7 + vocab + dim)
    ids = tokens_for(kind, n, vocab, rng)
    dy = to_bits(rng.normal(size=(n, dim)), t)
    before = to_bits(rng.normal(size=(vocab, dim)), o)
    terms = to_float(dy, t).astype(np.float64) * scale
    if p:
        keep, by = mask(n * dim, p, STATE, 4)
        terms = np.where(keep.reshape(n, dim), terms * np.float64(by), 0.0)
    fine = (ids >= 0) & (ids < vocab) & (ids != padding)
    total, size = np.zeros((vocab, dim)), np.zeros((vocab, dim))
    np.add.at(total, ids[fine], terms[fine])
    np.add.at(size, ids[fine], np.abs(terms[fine]))
    count = np.bincount(ids[fine], minlength=vocab)[:vocab, None]
    if add:
        total, size = total + to_float(before, o), size + np.abs(to_float(before, o))
    bound = (count + 3) * 2.0 ** -24 * size + HALF_STEP[o] * np.abs(total) * (1 + 2.0 ** -8) + TINY[o]
    with Buffers() as b:
        hy, hi, s = b.put(dy, shift, dim + pad), b.put(ids), b.state(STATE)
        out = b.put(before, shift, dim + pad) if add else b.empty((vocab, dim), numpy_type(o), shift, dim + pad)
        need = b.lib.gm_embedding_gradient_workspace(n, vocab, dim)
        space = b.space(need) if need else 0
        args = (b.device, 0, hy, hi, out, n, vocab, dim, dim + pad, dim + pad, t, o, scale, padding, int(add), p, s, 4, space, need)
        b.check(b.lib.execute_embedding_gradient(*args))
        got = b.get(out, (vocab, dim), numpy_type(o), dim + pad)
        if twice:      # the same again, bit for bit
            b.check(b.lib.execute_embedding_gradient(*args))
            assert np.array_equal(b.get(out, (vocab, dim), numpy_type(o), dim + pad).view(np.uint8), got.view(np.uint8))
    if add:
        untouched = count[:, 0] == 0
        assert np.array_equal(got[untouched], before[untouched])
    err = np.abs(to_float(got, o).astype(np.float64) - total)
    assert np.all(err <= bound), (err - bound).max()


@pytest.mark.parametrize("t, o", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("n, vocab, dim, kind", [(1, 1, 1, "plain"), (1, 100, 512, "plain"), (31, 7, 9, "padded"), (32, 500, 64, "plain"),
                                                 (33, 5, 520, "one word"), (1000, 300, 100, "padded"), (777, 90, 33, "all padding")])
def test_gradient(t, o, n, vocab, dim, kind):
    gradient_case(t, o, n, vocab, dim, kind)


@pytest.mark.parametrize("n, vocab, dim, kind", [(8191, 1000, 16, "padded"), (8192, 40, 24, "plain"), (8193, 2000, 8, "padded"),
                                                 (20000, 3000, 16, "padded"), (65536, 900, 4, "padded"), (65537, 2000, 8, "padded"), (70000, 600_000, 4, "padded"), (40000, 7, 8, "plain"), (16384, 9, 8, "one word"), (9000, 600_000, 4, "padded"),
                                                 (9000, 524_287, 4, "padded"), (9000, 524_286, 4, "padded"), (300, 600_000, 5, "padded")])
def test_gradient_of_long_lists(n, vocab, dim, kind):
    """Across the borders of the sort's chunks, and words whose occurrences fill many pieces."""
    gradient_case(F32, F32, n, vocab, dim, kind, twice=True)


@pytest.mark.parametrize("t, o", [(F32, F32), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("add", [False, True])
def test_gradient_with_everything(t, o, add):
    """Dropout, scale, a padding word inside the vocabulary, strides and odd alignment together."""
    gradient_case(t, o, 500, 120, 65, "padded", pad=3, shift=4, p=0.25, add=add, padding=3, scale=0.5)
    gradient_case(t, o, 500, 120, 64, "padded", pad=8, shift=16, p=0.25, add=add, padding=3, scale=8.0)


def test_gradient_without_tokens():
    with Buffers() as b:
        g, x = b.put(np.ones((10, 8), np.float32)), b.put(np.zeros(8, np.float32))
        args = (b.device, 0, x, x, g, 0, 10, 8, 8, 8, F32, F32, 1.0, -1)
        b.check(b.lib.execute_embedding_gradient(*args, 1, 0.0, 0, 0, 0, 0))
        assert np.all(b.get(g, (10, 8), np.float32) == 1)
        b.check(b.lib.execute_embedding_gradient(*args, 0, 0.0, 0, 0, 0, 0))
        assert np.all(b.get(g, (10, 8), np.float32) == 0)


def test_values_behind_padding_reach_nothing():
    """NaN and inf in the gradient rows of padded positions."""
    n, vocab, dim = 100, 20, 40
    rng = np.random.default_rng(3)
    ids = rng.integers(0, vocab, n).astype(np.int32)
    ids[::3] = -1
    dy = rng.normal(size=(n, dim)).astype(np.float32)
    dy[::6], dy[3::6] = np.nan, np.inf
    want = np.zeros((vocab, dim))
    np.add.at(want, ids[ids >= 0], dy[ids >= 0].astype(np.float64))
    with Buffers() as b:
        out = b.empty((vocab, dim), np.float32)
        need = b.lib.gm_embedding_gradient_workspace(n, vocab, dim)
        b.check(b.lib.execute_embedding_gradient(b.device, 0, b.put(dy), b.put(ids), out, n, vocab, dim, dim, dim, F32, F32, 1.0, -1, 0, 0.0,
                                                 0, 0, b.space(need), need))
        assert np.allclose(b.get(out, (vocab, dim), np.float32), want, rtol=0, atol=n * 2.0 ** -24 * 5 * n)
