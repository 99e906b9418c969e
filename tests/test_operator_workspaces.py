"""What the linear cross entropy's workspace queries promise, over types, few and many tokens, small and large vocabularies; the
sizes alone, no GPU is touched."""
import itertools

import pytest

from test_operator_refusals import A, lib, loss, no_gpu  # noqa: F401  (lib: the fixture)

PAIRS = [(0, 0), (2, 2), (4, 4), (2, 0), (4, 0)]
SIZES = [(n, v, d) for n, v, d in itertools.product((1, 100, 257, 300, 513, 2048, 4096, 70000), (50, 1500, 32000, 131072), (64, 1000, 4096))]


@pytest.mark.parametrize("t, o", PAIRS)
@pytest.mark.parametrize("gradients", [0, 1])
@pytest.mark.parametrize("weight", [0, A])
def test_the_least_workspace_is_no_larger_than_the_recommended_one(lib, t, o, gradients, weight):  # noqa: F811
    for n, v, d in SIZES:
        big = lib.gm_linear_cross_entropy_workspace(n, v, d, weight, d, t, o, gradients)
        small = lib.gm_linear_cross_entropy_least_workspace(n, v, d, weight, d, t, o, gradients)
        assert 0 < small <= big, (n, v, d, small, big)


@pytest.mark.parametrize("t, o", PAIRS)
def test_the_figure_that_a_refusal_reports_is_accepted(lib, t, o):  # noqa: F811
    no_gpu(lib)
    for n, v, d in SIZES:
        sizes = dict(n=n, v=v, d=d, xs=d, ws=d, dxs=d, dws=d, t=t, o=o)
        big = lib.gm_linear_cross_entropy_workspace(n, v, d, 0x20000, d, t, o, 1)
        small = lib.gm_linear_cross_entropy_least_workspace(n, v, d, 0x20000, d, t, o, 1)
        assert loss(lib, size=small - 1, **sizes) == -18 and b": at least %d are needed" % small in lib.gm_last_error(), (n, v, d)
        for size in (small, (small + big) // 2, big):
            assert loss(lib, size=size, **sizes) == -3, (n, v, d, size)


def test_sizes_that_are_not_offered(lib):  # noqa: F811
    ask, least = lib.gm_linear_cross_entropy_workspace, lib.gm_linear_cross_entropy_least_workspace
    for n, v, d, offered in ((1 << 24, 1 << 22, 1 << 15, True), (1 << 24, 1 << 22, (1 << 15) + 1, False), ((1 << 24) + 1, 10, 8, False),
                             (1, 1 << 17, 1 << 20, True), (1, (1 << 17) + 1, 1 << 20, False), (1, 10, (1 << 20) + 1, False)):
        for query in (ask, least):
            for gradients in (0, 1):
                assert (query(n, v, d, 0, d, 2, 2, gradients) > 0) == offered, (n, v, d)
        code = loss(lib, n=n, v=v, d=d, xs=d, ws=d, dxs=d, dws=d, size=1000)
        assert code == (-18 if offered else -5), (n, v, d)


@pytest.mark.parametrize("gradients", [0, 1])
def test_tokens_that_one_launch_cannot_take_are_taken_in_parts(lib, gradients):  # noqa: F811
    """What is kept of the logits does not grow with the tokens once they pass what a launch can address."""
    one, two = (lib.gm_linear_cross_entropy_workspace(n, 32000, 64, A, 64, 4, 4, gradients) for n in (1 << 23, 1 << 24))
    packed = 2 * 128 + 4 * 4      # bytes of a token's row with its skew, and of the lists
    assert abs(two - one - (packed << 23)) <= 4096
