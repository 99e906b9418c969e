"""The linear cross entropy at the edges of what its types hold, against the same bounds as elsewhere."""
import numpy as np
import pytest

from operator_lib import BF16, F32, Buffers, to_bits, to_float
from test_gpu_linear_cross_entropy import check, data, run

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
