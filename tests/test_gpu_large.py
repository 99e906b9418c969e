"""The language-model operators at their largest: as many tokens as they offer, more than one launch can address, buffers whose
offsets pass 2^32 bytes.

Large operands are made on the device by the lookup itself, out of a few rows.  Where a loss is checked most tokens' rows are 0, so
that a weight gradient is a sum of a few hundred terms whatever the number of tokens, and tokens of one target all have the same
loss and gradient, bit for bit; the others and some of these are checked as a batch of their own."""
import numpy as np
import pytest

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
