"""Sizes whose launches HIP would refuse (2^32 lanes and more) are refused before anything is launched, with -5; sizes right
below are not.  No GPU is touched."""
import pytest

from test_operator_refusals import gradient, lib, no_gpu  # noqa: F401  (lib: the fixture)


@pytest.mark.parametrize("n, v, d, code", [
    (1, (1 << 26) - 17, 8192, -3),      # a workgroup of 64 lanes a row of 16 KiB to fill, 16 for the one token's sum
    (1, (1 << 26) - 16, 8192, -5),
    (1, (1 << 27), 8192, -5),
    (1 << 22, 10, 512 * 511, -3),      # 2^17 pieces of 511 columns of workgroups and a few for the rows of zeros
    (1 << 22, 10, 512 * 512, -5)])
def test_table_gradient(lib, n, v, d, code):  # noqa: F811
    if code == -3:
        no_gpu(lib)
    assert gradient(lib, n=n, v=v, d=d, ys=d, gs=d, size=1 << 62) == code
    if code == -5:
        assert b"launch" in lib.gm_last_error()
