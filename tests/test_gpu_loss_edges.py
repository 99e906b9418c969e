"""The linear cross entropy at the edges of what its types hold, against the same bounds as elsewhere."""
import numpy as np
import pytest

from operator_lib import BF16, F32, Buffers, loss_reference, to_bits, to_float
from test_gpu_linear_cross_entropy import IGNORE, PAIRS, check, data, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n, v, d", [(40, 200, 96), (600, 200, 96), (300, 4099, 320)])
@pytest.mark.parametrize("x_power, w_power", [(100, -100), (-100, 100), (-60, -60), (100, -110), (60, -95)])
def test_operands_of_very_small_and_very_large_values(t, n, v, d, x_power, w_power):
    """Every gradient is a normal number, whatever the powers of two that are taken out of the operands' rows on the way: 2^-110
    times a slope above 2^-13 / n."""
    x, w, targets = data(t, n, v, d)
    x = to_bits(to_float(x, t) * np.float32(2.0 ** x_power), t)
    w = to_bits(to_float(w, t) * np.float32(2.0 ** w_power), t)
    with Buffers() as b:
        check(run(b, t, F32, x, w, targets, scale=1.0), t, F32, x, w, targets, scale=1.0)


def banned_words(t, n, v, d):
    """A vocabulary with words whose logit is -inf for every token: their rows hold -inf where every token's activation is 1."""
    x, w, targets = data(t, n, v, d)
    x, w = to_float(x, t).copy(), to_float(w, t).copy()
    x[:, 0] = 1.0
    banned = np.arange(v) % 7 == 3
    banned[-1] = True
    targets = np.where(banned[np.maximum(targets, 0)] & (targets >= 0), targets - 2, targets).astype(np.int32)      # (no two are neighbours but one)
    targets = np.where(banned[np.maximum(targets, 0)] & (targets >= 0), targets - 2, targets).astype(np.int32)
    assert not banned[targets[targets >= 0]].any()
    w[banned, 0] = -np.inf
    return to_bits(x, t), to_bits(w, t), targets, banned


@pytest.mark.parametrize("t, o", PAIRS)
@pytest.mark.parametrize("n, v, d", [(20, 100, 64), (100, 1000, 130), (600, 3000, 192)])
def test_words_whose_logit_is_minus_infinity(t, o, n, v, d):
    """They are as good as absent: losses and every gradient are those of the vocabulary without them, their own rows of the
    weight gradient are 0, and only the column that meets 0 times infinity in the hidden gradient is NaN, as in the formula."""
    x, w, targets, banned = banned_words(t, n, v, d)
    place = np.cumsum(~banned) - 1
    fewer = np.where(targets >= 0, place[np.maximum(targets, 0)], targets).astype(np.int32)
    counts = targets >= 0
    with Buffers() as b:
        got = run(b, t, o, x, w, targets, scale=8.0)
        assert np.all(to_float(got["dw"], o)[banned] == 0)
        assert np.isnan(to_float(got["dx"], t)[counts, 0]).all() and np.all(to_float(got["dx"], t)[~counts] == 0)
        got["dw"] = got["dw"][~banned]
        want = loss_reference(to_float(x, t), to_float(w, t)[~banned], fewer, IGNORE, 1, 8.0)[3]
        got["dx"][:, 0] = to_bits(want[:, 0], t)
        check(got, t, o, x, w[~banned], fewer, scale=8.0)


@pytest.mark.parametrize("t, o", PAIRS)
def test_a_target_whose_logit_is_minus_infinity(t, o):
    x, w, targets, banned = banned_words(t, 30, 200, 64)
    targets[:] = np.nonzero(~banned)[0][:30]
    with Buffers() as b:
        clean = run(b, t, o, x, w, targets, dx=False, dw=False)
        targets[4] = np.nonzero(banned)[0][0]
        got = run(b, t, o, x, w, targets, dx=False, dw=False)
        assert got["losses"][4] == np.inf and got["loss"][0] == np.inf
        assert np.array_equal(np.delete(got["losses"], 4), np.delete(clean["losses"], 4))
