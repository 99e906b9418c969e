"""Dropout from a counter-based generator against the formula: masks and values bit for bit (each output is one or two fp32
operations and one rounding)."""
import numpy as np
import pytest

from operator_lib import ALL_TYPES, BF16, F16, F32, Buffers, mask, numpy_type, same, size_of, to_bits, to_float

pytestmark = pytest.mark.gpu
STATE = (1234567, 0x89ABCDEF, 3, 0)


def expected(x, r, t, p, state, site):
    keep, by = mask(x.size, p, state, site)
    y = np.where(keep, to_float(x, t) * by, np.float32(0))
    return to_bits(y + to_float(r, t) if r is not None else y, t)


@pytest.mark.parametrize("t", ALL_TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2048, 2049, 100003])
@pytest.mark.parametrize("shift", [0, 4])
def test_values_and_mask(t, n, shift):
    rng = np.random.default_rng(n)
    x, r = to_bits(rng.normal(size=n), t), to_bits(rng.normal(size=n), t)
    with Buffers() as b:
        s, hx, hr = b.state(STATE), b.put(x, shift), b.put(r, shift)
        for p, residual in ((0.1, 0), (0.5, hr), (0.0, hr), (1.0, hr), (1e-6, 0)):
            y = b.empty(n, numpy_type(t), shift)
            b.check(b.lib.execute_dropout(b.device, 0, hx, residual, y, n, t, p, s, 7))
            got = b.get(y, (n,), numpy_type(t))
            assert same(got, expected(x, r if residual else None, t, p, STATE, 7), t), (p, residual)


@pytest.mark.parametrize("t", ALL_TYPES)
def test_dropped_elements_are_zero_whatever_they_were(t):
    n = 4096
    x = to_bits(np.tile([np.nan, np.inf, -np.inf, 65504.0], n // 4), t)
    with Buffers() as b:
        s, hx, y = b.state(STATE), b.put(x), b.empty(n, numpy_type(t))
        b.check(b.lib.execute_dropout(b.device, 0, hx, 0, y, n, t, 0.5, s, 1))
        got = b.get(y, (n,), numpy_type(t))
        keep, _ = mask(n, 0.5, STATE, 1)
        assert np.all(to_float(got, t)[~keep] == 0) and same(got, expected(x, None, t, 0.5, STATE, 1), t)


def test_in_place_and_backward():
    """The mask of the backward pass is the forward one's; output may be the input or the residual."""
    n, t = 10007, F16
    rng = np.random.default_rng(5)
    x, r = to_bits(rng.normal(size=n), t), to_bits(rng.normal(size=n), t)
    with Buffers() as b:
        s = b.state(STATE)
        hx, hr, ones = b.put(x), b.put(r), b.put(to_bits(np.ones(n), t))
        b.check(b.lib.execute_dropout(b.device, 0, hx, hr, hr, n, t, 0.3, s, 2))
        b.check(b.lib.execute_dropout(b.device, 0, hx, 0, hx, n, t, 0.3, s, 2))
        b.check(b.lib.execute_dropout(b.device, 0, ones, 0, ones, n, t, 0.3, s, 2))
        assert same(b.get(hr, (n,), np.float16), expected(x, r, t, 0.3, STATE, 2), t)
        assert same(b.get(hx, (n,), np.float16), expected(x, None, t, 0.3, STATE, 2), t)
        keep, by = mask(n, 0.3, STATE, 2)
        assert np.array_equal(b.get(ones, (n,), np.float16), np.where(keep, np.float16(by), np.float16(0)))


def test_sites_steps_and_seeds_give_masks_of_their_own():
    n = 1 << 16
    masks = {}
    with Buffers() as b:
        ones, y = b.put(np.ones(n, np.float32)), b.empty(n, np.float32)
        for words, site in ((STATE, 0), (STATE, 1), ((1234567, 0x89ABCDEF, 4, 0), 0), ((1234568, 0x89ABCDEF, 3, 0), 0), ((1234567, 1, 3, 0), 0)):
            b.check(b.lib.execute_dropout(b.device, 0, ones, 0, y, n, F32, 0.25, b.state(words), site))
            masks[words, site] = b.get(y, (n,), np.float32) != 0
        # advancing the state on the device is the next step's mask
        s = b.state(STATE)
        b.check(b.lib.gm_rng_state_advance(b.device, 0, s))
        b.check(b.lib.execute_dropout(b.device, 0, ones, 0, y, n, F32, 0.25, s, 0))
        assert np.array_equal(b.get(y, (n,), np.float32) != 0, masks[(1234567, 0x89ABCDEF, 4, 0), 0])
        assert np.array_equal(b.get(s, (4,), np.uint32), np.array((1234567, 0x89ABCDEF, 4, 0), np.uint32))
    every = list(masks.values())
    sigma = (0.25 * 0.75 / n) ** 0.5
    for i, a in enumerate(every):
        assert abs(a.mean() - 0.75) < 6 * sigma
        for c in every[:i]:      # two independent masks agree where both keep or both drop: 0.625 of the places
            assert abs((a == c).mean() - 0.625) < 6 * (0.625 * 0.375 / n) ** 0.5


def test_a_buffer_that_is_too_short_is_refused():
    with Buffers() as b:
        h = b.dev.alloc(1024)
        s = b.state()
        assert b.lib.execute_dropout(b.device, 0, h, 0, h, 256, F32, 0.0, s, 0) == 0
        assert b.lib.execute_dropout(b.device, 0, h, 0, h, 257, F32, 0.0, s, 0) == -5
        assert b.lib.execute_dropout(b.device, 0, h, 0, h, 0, F32, 0.5, s, 0) == 0
        b.dev.free(h)


def test_known_counters():
    """Philox4x32-10's published test vector for a counter and a key of zeros: block 0, site 0, step 0 and seeds 0; its words'
    halves decide elements 0 to 7."""
    words = (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    bits = [h for w in words for h in (w & 0xFFFF, w >> 16)]
    with Buffers() as b:
        s, ones, y = b.state((0, 0, 0, 0)), b.put(np.ones(8, np.float32)), b.empty(8, np.float32)
        for p in (0.1, 0.3, 0.5, 0.7, 0.9):
            b.check(b.lib.execute_dropout(b.device, 0, ones, 0, y, 8, F32, p, s, 0))
            border = int(np.float64(np.float32(p)) * 65536 + 0.5)
            assert [bool(v) for v in b.get(y, (8,), np.float32)] == [x >= border for x in bits]
