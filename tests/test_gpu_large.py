"""The language-model operators at their largest: as many tokens as they offer, more than one launch can address, buffers whose
offsets pass 2^32 bytes.

Large operands are made on the device by the lookup itself, out of a few rows.  Where a loss is checked most tokens' rows are 0, so
that a weight gradient is a sum of a few hundred terms whatever the number of tokens, and tokens of one target all have the same
loss and gradient, bit for bit; the others and some of these are checked as a batch of their own."""
import ctypes

import numpy as np
import pytest

from __graft_entry__ import load_package
from operator_lib import BF16, F16, F32, Buffers, numpy_type, size_of, to_bits
from test_gpu_linear_cross_entropy import IGNORE, check

pytestmark = pytest.mark.gpu


class Large(Buffers):
    """Buffers of any length, without canaries, besides the others."""

    def __enter__(self):
        self.large = []
        return self

    def __exit__(self, *exc):
        self.dev.synchronize()
        for h in self.large:
            self.lib.deallocate_metal_buffer(h)
        super().__exit__(*exc)

    def room(self, nbytes):
        h = self.lib.gm_allocate_workspace(self.device, nbytes)
        assert h, self.lib.gm_last_error()
        self.large.append(h)
        return h

    def rows(self, pattern, ids, t):
        """Row i is row ids[i] of the pattern, or zeros."""
        n, (count, d) = ids.size, pattern.shape
        out = self.room(n * d * size_of(t))
        self.check(self.lib.execute_embedding_lookup(self.device, 0, self.put(pattern), self.put(ids), out, n, count, d, d, d, t, 1.0, 0.0, 0, 0))
        return out

    def read(self, base, first, rows, d, t):
        return self.dev.to_numpy(base + first * d * size_of(t), rows * d, numpy_type(t)).reshape(rows, d)


def loss_of_many_tokens(t, o, n, v, d, marks, gradients):
    """`marks`: tokens whose rows are not 0."""
    rng = np.random.default_rng(n % 1000 + v)
    w = to_bits(rng.normal(size=(v, d)) * d ** -0.5, t)
    pattern = to_bits(rng.normal(size=(len(marks), d)), t)
    ids = np.full(n, -1, np.int32)
    ids[marks] = np.arange(len(marks))
    some = np.linspace(0, v - 1, 16).astype(np.int32)
    targets = some[np.arange(n) % 16]
    targets[marks] = rng.integers(0, v, len(marks))
    with Large() as b:
        x, hw, ht = b.rows(pattern, ids, t), b.put(w), b.put(targets)
        losses, loss = b.room(4 * n), b.empty(2, np.float32)
        gx, gw = (b.room(n * d * size_of(t)), b.empty((v, d), numpy_type(o))) if gradients else (0, 0)
        need = b.lib.gm_linear_cross_entropy_workspace(n, v, d, hw, d, t, o, int(gradients))
        b.check(b.lib.execute_linear_cross_entropy(b.device, 0, x, hw, ht, losses, loss, gx, gw, n, v, d, d, d, d, d, t, o, IGNORE, 0, 1.0, 0, 0,
                                                   b.room(need), need))
        all_losses = b.dev.to_numpy(losses, n)
        total, count = b.get(loss, (2,), np.float32)
        assert count == n and abs(total - all_losses.astype(np.float64).sum()) <= 2.0 ** -24 * abs(total)
        all_dx = b.read(gx, 0, n, d, t) if gradients else None
        batch = np.unique(np.concatenate([marks, np.arange(64), n - 1 - np.arange(64)]))
        rest = np.ones(n, bool)
        rest[marks] = False
        for k in range(16):
            same = rest & (np.arange(n) % 16 == k)
            first = np.nonzero(same)[0][0]
            assert first < 64 and np.all(all_losses[same] == all_losses[first])
            if gradients:
                assert np.array_equal(all_dx[same].view(np.uint8), np.broadcast_to(all_dx[first], (same.sum(), d)).copy().view(np.uint8))
        fx = np.zeros((batch.size, d), numpy_type(t))
        here = ids[batch] >= 0
        fx[here] = pattern[ids[batch][here]]
        got = {"losses": all_losses[batch], "loss": np.array([all_losses[batch].astype(np.float64).sum(), batch.size])}
        if gradients:
            got["dx"], got["dw"] = all_dx[batch], b.get(gw, (v, d), numpy_type(o))
        check(got, t, o, fx, w, targets[batch], mean=0)


@pytest.mark.parametrize("gradients", [False, True])
@pytest.mark.parametrize("n", [1 << 23, (1 << 24) - 65, 1 << 24])
def test_as_many_tokens_as_there_may_be(n, gradients):
    marks = np.unique(np.concatenate([np.arange(40), n - 1 - np.arange(40), *(k * (n >> 4) + np.array([-1, 0, 1]) for k in range(1, 16))]))
    loss_of_many_tokens(F16, F16, n, 16, 8, marks, gradients)


def kept_at(first, count, p, state, site):
    """Dropout's mask of `count` elements from the first-th on (a multiple of eight), and a kept element's factor, in whole numbers."""
    border = int(np.float64(np.float32(p)) * 65536 + 0.5)
    keep = np.zeros(count, bool)
    for at in range(0, count, 8):
        block = (first + at) // 8
        c, k = [block & 0xFFFFFFFF, block >> 32, site, state[2]], [state[0], state[1]]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        for e in range(min(8, count - at)):
            keep[at + e] = (c[e // 2] >> (16 * (e % 2)) & 0xFFFF) >= border
    return keep, np.float32(65536.0 / (65536 - border))


def test_a_lookup_of_more_than_one_launch_can_address():
    """2^32 vectors and some: 69 GB, in three launches, the generator's blocks past 2^32."""
    n, d, v, t, state = (1 << 23) + 5, 4096, 3, F16, (11, 22, 33, 0)
    rng = np.random.default_rng(2)
    table = rng.normal(size=(v, d)).astype(np.float16)
    ids = (np.arange(n) % 4).astype(np.int32)      # the last of four is padding
    with Large() as b:
        hi, ht, s, out = b.put(ids), b.put(table), b.state(state), b.room(n * d * 2)
        b.check(b.lib.execute_embedding_lookup(b.device, 0, ht, hi, out, n, v, d, d, d, t, 2.0, 0.25, s, 6))
        for first in (0, (1 << 22) - 1, 1 << 22, (1 << 23) - 1, 1 << 23, n - 1):
            keep, by = kept_at(first * d, d, 0.25, state, 6)
            row = table[ids[first]].astype(np.float32) * np.float32(2) if ids[first] < v else np.zeros(d, np.float32)
            assert np.array_equal(b.read(out, first, 1, d, t)[0], np.where(keep, row * by, np.float32(0)).astype(np.float16)), first


@pytest.mark.parametrize("t, o, n", [(F16, F16, 17000), (BF16, BF16, 16500), (F16, F32, 4000), (BF16, F32, 3500), (F32, F32, 3000)])
def test_more_tokens_than_four_gib_hold(t, o, n):
    """Two chunks without a small workspace: what is kept of a chunk's logits fills 4 GiB, the weight gradient is a sum of both."""
    v, d = 131072, 64
    plan = (ctypes.c_int * 7)()
    assert load_package().load_library().gm_linear_cross_entropy_plan(n, v, d, 0, d, t, o, 1, 1 << 62, plan) == 0 and plan[0] < n < 2 * plan[0]
    marks = np.unique(np.concatenate([np.arange(0, n, n // 60), n - 1 - np.arange(40)]))
    loss_of_many_tokens(t, o, n, v, d, marks, True)


def test_weights_of_more_than_four_gib():
    """The weights, their gradient and the fp16 rows of both, offsets past 2^32 bytes; words repeat with a period of 1000."""
    n, v, d, t = 5, 131072, 257 * 64, F16
    rng = np.random.default_rng(8)
    pattern = to_bits(rng.normal(size=(1000, d)) * d ** -0.5, t)
    x = to_bits(rng.normal(size=(n, d)), t)
    ids = (np.arange(v) % 1000).astype(np.int32)
    targets = np.array([0, v - 1, (1 << 32) // (2 * d) + 1, 70000, IGNORE], np.int32)
    fx, fp = x.astype(np.float64), pattern.astype(np.float64)
    counts = targets >= 0
    fx[~counts] = 0
    s = (fx @ fp.T)[:, ids]
    top = s.max(1, keepdims=True)
    lse = (np.log(np.exp(s - top).sum(1, keepdims=True)) + top)[:, 0]
    at = (np.arange(n), np.maximum(targets, 0))
    want = np.where(counts, lse - s[at], 0)
    ds = np.exp(s - lse[:, None])
    ds[at] -= 1
    ds[~counts] = 0
    u, half = 2.0 ** -24, 2.0 ** -11
    # a logit, a loss and a slope, as in the bounds of the other sizes: exponentials and slopes are in fp16 each, the sums in fp32
    off = 2 * (d + 8) * u * (np.abs(fx) @ np.abs(fp).T).max(1) + (4 * (top - s).max(1) + 210) * u + 2 * u * np.abs(lse)
    err = np.where(ds > 0, ds, 1 + ds) * (off[:, None] + 2 * half + 4 * u) + np.abs(ds) * (half + 30 * u) + 2.0 ** -37
    with Large() as b:
        w, hx, ht = b.rows(pattern, ids, t), b.put(x), b.put(targets)
        losses, loss, gx, gw = b.empty(n, np.float32), b.empty(2, np.float32), b.empty((n, d), np.float16), b.room(v * d * 2)
        need = b.lib.gm_linear_cross_entropy_workspace(n, v, d, w, d, t, t, 1)
        b.check(b.lib.execute_linear_cross_entropy(b.device, 0, hx, w, ht, losses, loss, gx, gw, n, v, d, d, d, d, d, t, t, IGNORE, 0, 1024.0, 0, 0,
                                                   b.room(need), need))
        assert np.all(np.abs(b.get(losses, (n,), np.float32) - want) <= np.where(counts, off, 0))
        by_class = lambda a: np.stack([a[:, k::1000].sum(1) for k in range(1000)], 1)
        dx = by_class(ds) @ fp
        bound = by_class(np.where(counts[:, None], err + v * u * np.abs(ds), 0)) @ np.abs(fp) + half * np.abs(dx)
        assert np.all(np.abs(b.get(gx, (n, d), np.float16).astype(np.float64) - 1024 * dx) <= 1024 * bound + 2.0 ** -24)
        for first in (0, 69990, (1 << 32) // (2 * d) - 10, v - 40):
            here = slice(first, first + 40)
            dw = ds[:, here].T @ fx
            bound = err[:, here].T @ np.abs(fx) + (half + n * u) * np.abs(ds[:, here]).T @ np.abs(fx)
            got = b.read(gw, first, 40, d, t).astype(np.float64)
            assert np.all(np.abs(got - 1024 * dw) <= 1024 * bound + 2.0 ** -24), first


def test_a_table_gradient_of_more_than_four_gib():
    """Output gradients and a table past 2^32 bytes: every position's row is one of 50, a word's sum their multiples."""
    n, v, d, t = 131072 + 700, 131072 + 100, 257 * 64, BF16
    rng = np.random.default_rng(9)
    pattern = to_bits(rng.normal(size=(50, d)), t)
    ids = rng.integers(0, 50, n).astype(np.int32)
    words = np.array([0, 1, 70000, (1 << 32) // (2 * d), v - 2, v - 1])
    tokens = words[rng.integers(0, words.size, n)].astype(np.int32)
    tokens[::11] = -1
    with Large() as b:
        dy, out = b.rows(pattern, ids, t), b.room(v * d * 2)
        need = b.lib.gm_embedding_gradient_workspace(n, v, d)
        b.check(b.lib.execute_embedding_gradient(b.device, 0, dy, b.put(tokens), out, n, v, d, d, d, t, t, 0.5, -1, 0, 0.0, 0, 0, b.room(need), need))
        f = (pattern.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        for word in (*words, 2, 69999, v - 3):
            count = np.bincount(ids[tokens == word], minlength=50)
            want, size = 0.5 * (count @ f), 0.5 * (count @ np.abs(f))
            got = (b.read(out, int(word), 1, d, t)[0].astype(np.uint32) << 16).view(np.float32).astype(np.float64)
            assert np.all(np.abs(got - want) <= (count.sum() + 3) * 2.0 ** -24 * size + 2.0 ** -8 * 1.01 * np.abs(want)), word


def test_dropout_of_more_than_four_gib():
    n, state = 2 ** 31 - 1, (5, 6, 7, 0)
    with Large() as b:
        ones = np.ones((1, 1 << 20), np.float32)
        x = b.rows(ones, np.zeros(2048, np.int32), F32)
        y = b.room(4 * n + 4)
        b.check(b.lib.execute_dropout(b.device, 0, x, x, y, n, F32, 0.3, b.state(state), 9))
        for first in (0, (1 << 30) - 512, (1 << 30) + 8, n - 1023):
            keep, by = kept_at(first // 8 * 8, 1024, 0.3, state, 9)
            got = b.dev.to_numpy(y + first // 8 * 8 * 4, min(1024, n - first // 8 * 8))
            assert np.array_equal(got, np.where(keep, by + np.float32(1), np.float32(1))[:got.size]), first
