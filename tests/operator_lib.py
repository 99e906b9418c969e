"""What the tests of the language-model operators share: 16-bit types in numpy, dropout's generator, the formulas in
64 bits, and buffers placed at any alignment and stride."""
import ctypes

import numpy as np

from harness import gpu_device

F32, F16, BF16 = 0, 2, 4
ALL_TYPES = (F32, F16, BF16)
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}      # largest rounding error relative to the value
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}        # smallest subnormal


def to_bits(x, t):
    """fp32 values rounded to type t, as the array a buffer holds (bfloat16: its 16 bits)."""
    x = np.asarray(x, np.float32)
    if t == F32:
        return x.copy()
    if t == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    rounded = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), rounded)


def to_float(a, t):
    """What an array of type t holds, as fp32."""
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32)
    return a.astype(np.float32)


def numpy_type(t):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[t]


def size_of(t):
    return 4 if t == F32 else 2


def same(got, want, t):
    """Bit for bit, NaN for NaN."""
    g, w = to_float(got, t), to_float(want, t)
    return np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(g[~np.isnan(g)], w[~np.isnan(w)])


def mask(n, p, state, site):
    """Which of n elements dropout keeps, and the factor of a kept one."""
    border = int(np.floor(np.float64(np.float32(p)) * 65536.0 + 0.5))
    block = np.arange((n + 7) // 8, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    c = [block & low, block >> np.uint64(32), np.full_like(block, site & 0xFFFFFFFF), np.full_like(block, state[2])]
    k = [int(state[0]), int(state[1])]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    bits = np.stack([w >> np.uint64(s) & np.uint64(0xFFFF) for w in c for s in (0, 16)], 1).reshape(-1)[:n]
    return bits >= border, np.float32(65536.0 / (65536 - border)) if border < 65536 else np.float32(0.0)


class Buffers:
    """Device buffers of one test, freed at its end, every one with a border of canaries on either side."""

    BORDER = 4096

    def __init__(self):
        self.dev = gpu_device()
        assert self.dev is not None, "libgometal_hip.so or the GPU is missing: these operators have no fallback"
        self.lib, self.device = self.dev.lib, self.dev.handle
        self.owned, self.spaces = [], []

    def __enter__(self):
        return self

    def __exit__(self, kind, *exc):
        self.dev.synchronize()
        try:
            for at in self.spaces if kind is None else ():
                assert np.all(self.dev.to_numpy(at, self.BORDER, np.uint8) == 0xFF), "written outside the workspace"
        finally:
            for h, _, _ in self.owned:
                self.dev.free(h)

    def put(self, array, shift=0, stride=None):
        """The array's handle: its rows `stride` elements apart, its start `shift` bytes behind a 256-byte boundary."""
        a = np.ascontiguousarray(array)
        if stride is not None and a.ndim == 2 and stride != a.shape[1]:
            wide = np.zeros((a.shape[0], stride), a.dtype)
            wide.view(np.uint8)[:] = 0xA5
            wide[:, :a.shape[1]] = a
            a = wide
        raw = np.full(a.nbytes + 2 * self.BORDER + 256, 0xA5, np.uint8)
        raw[self.BORDER + shift:self.BORDER + shift + a.nbytes] = np.frombuffer(a.tobytes(), np.uint8)
        h = self.dev.from_numpy(raw)
        self.owned.append((h, raw.size, (self.BORDER + shift, a.nbytes)))
        return h + self.BORDER + shift

    def empty(self, shape, dtype, shift=0, stride=None):
        a = np.zeros(shape, dtype)
        a.reshape(-1).view(np.uint8)[:] = 0xA5
        return self.put(a, shift, stride)

    def get(self, address, shape, dtype, stride=None):
        """The array at that address; nothing around it, nor between its rows, has changed."""
        for h, size, (at, nbytes) in self.owned:
            if address == h + at:
                raw = self.dev.to_numpy(h, size, np.uint8)
                assert np.all(raw[:at] == 0xA5) and np.all(raw[at + nbytes:] == 0xA5), "written outside the buffer"
                data = raw[at:at + nbytes].view(dtype)
                if len(shape) == 2 and stride is not None and stride != shape[1]:
                    data = data.reshape(shape[0], stride)
                    assert np.all(np.ascontiguousarray(data[:, shape[1]:]).view(np.uint8) == 0xA5), "written between the rows"
                    data = data[:, :shape[1]]
                return data.reshape(shape).copy()
        raise KeyError(address)

    def state(self, words=(1234567, 0x89ABCDEF, 3, 0)):
        return self.put(np.array(words, np.uint32))

    def space(self, nbytes, align=256):
        """A workspace of exactly that many bytes, filled with NaN patterns."""
        raw = np.full(nbytes + 2 * self.BORDER, 0xFF, np.uint8)
        h = self.dev.from_numpy(raw)
        self.owned.append((h, raw.size, (0, raw.size)))
        assert h % align == 0
        self.spaces += [h, h + self.BORDER + nbytes]
        return h + self.BORDER

    def check(self, rc):
        assert rc == 0, (rc, self.lib.gm_last_error().decode())


def loss_reference(x, w, targets, ignore, mean, scale):
    """(losses, loss, count, dX, dW, dS / scale) of the linear cross entropy in 64 bits."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    n, v = x.shape[0], w.shape[0]
    counts = (targets != ignore) & (targets >= 0) & (targets < v)
    losses, ds = np.zeros(n), np.zeros((n, v))
    rows = np.nonzero(counts)[0]
    if rows.size:
        s = x[rows] @ w.T
        top = s.max(1, keepdims=True)
        lse = (top + np.log(np.exp(s - top).sum(1, keepdims=True)))[:, 0]
        at = s[np.arange(rows.size), targets[rows]]
        losses[rows] = lse - at
        p = np.exp(s - lse[:, None])
        p[np.arange(rows.size), targets[rows]] = np.expm1(at - lse)
        ds[rows] = p
    count = int(rows.size)
    c = scale / max(1, count) if mean else scale
    clean = np.where(counts[:, None], x, 0.0)      # a token that does not count reaches nothing
    return losses, losses.sum() / (max(1, count) if mean else 1), count, c * (ds @ w), c * (ds.T @ clean), ds


def pointer(array):
    return array.ctypes.data_as(ctypes.c_void_p)
