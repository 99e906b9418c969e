"""Every shape that the linear cross entropy's products may take, for every pair of types: sizes chosen by the rule itself, which
is asked what it makes of them (so a change of the rule cannot leave a shape without a test)."""
import ctypes

import numpy as np
import pytest

from __graft_entry__ import load_package
from operator_lib import Buffers, to_bits
from test_gpu_linear_cross_entropy import PAIRS, check, data, run

WIDE, SQUARE, TALL, FLAT = range(4)      # tiles of 256 x 256, 128 x 128, 256 x 128 and 128 x 32
WHOLE, PARTS = False, True

# tokens, words, dimension: (logits, hidden gradient, its sums in parts, weight gradient, its sums in parts), the same for all types
CASES = {
    (20, 60, 64): (FLAT, FLAT, WHOLE, SQUARE, WHOLE),
    (20, 3001, 70): (FLAT, FLAT, PARTS, SQUARE, WHOLE),
    (100, 60, 64): (TALL, TALL, WHOLE, SQUARE, WHOLE),
    (100, 3001, 70): (TALL, TALL, PARTS, SQUARE, WHOLE),
    (200, 61, 65): (SQUARE, SQUARE, WHOLE, SQUARE, WHOLE),
    (300, 2003, 76): (SQUARE, SQUARE, PARTS, SQUARE, WHOLE),
    (2101, 61, 65): (SQUARE, SQUARE, WHOLE, SQUARE, PARTS),
    (138, 33786, 71): (WIDE, SQUARE, PARTS, SQUARE, WHOLE),
    (5400, 61, 1427): (SQUARE, WIDE, WHOLE, SQUARE, PARTS),
    (777, 3013, 4177): (SQUARE, WIDE, PARTS, WIDE, WHOLE),
    (4118, 519, 3870): (SQUARE, WIDE, WHOLE, WIDE, PARTS),
    (268, 25173, 799): (WIDE, WIDE, PARTS, WIDE, WHOLE),
}


def taken(lib, n, v, d, t, o, space=1 << 62):
    plan = (ctypes.c_int * 7)()
    assert lib.gm_linear_cross_entropy_plan(n, v, d, 0, d, t, o, 1, space, plan) == 0
    return tuple(plan)


@pytest.mark.parametrize("t, o", PAIRS)
def test_the_cases_take_the_shapes_they_are_here_for(t, o):
    lib = load_package().load_library()
    reached = set()
    for sizes in CASES:
        chunk, logits, dx, dx_parts, dw, dw_parts, sums = taken(lib, *sizes, t, o)
        assert (logits, dx, dx_parts > 1, dw, dw_parts > 1) == CASES[sizes], (sizes, logits, dx, dx_parts, dw, dw_parts)
        assert chunk == sizes[0] and not sums
        reached |= {("logits", logits), ("dx", dx, dx_parts > 1), ("dw", dw, dw_parts > 1)}
    assert reached == ({("logits", s) for s in range(4)} | {("dx", s, p) for s in range(4) for p in (WHOLE, PARTS)}
                       | {("dw", s, p) for s in (WIDE, SQUARE) for p in (WHOLE, PARTS)})


def test_plan_refusals():
    lib = load_package().load_library()
    ask, plan = lib.gm_linear_cross_entropy_plan, (ctypes.c_int * 7)()
    assert ask(10, 10, 8, 0, 8, 2, 2, 1, 1 << 40, None) == -4
    assert ask(10, 10, 8, 0, 7, 2, 2, 1, 1 << 40, plan) == -5 and ask(10, 0, 8, 0, 8, 2, 2, 1, 1 << 40, plan) == -5
    assert ask(10, 10, 8, 0, 8, 1, 2, 1, 1 << 40, plan) == -19 and ask(10, 10, 8, 0, 8, 2, 4, 1, 1 << 40, plan) == -19
    assert ask(10, 10, 8, 0, 8, 2, 2, 1, 100, plan) == -18


@pytest.mark.gpu
@pytest.mark.parametrize("t, o", PAIRS)
@pytest.mark.parametrize("sizes", list(CASES), ids=str)
@pytest.mark.parametrize("add", [False, True])
def test_against_the_formula(t, o, sizes, add):
    n, v, d = sizes
    x, w, targets = data(t, n, v, d)
    before = to_bits(np.random.default_rng(3).normal(size=(v, d)) * 0.01, o) if add else None
    with Buffers() as b:
        check(run(b, t, o, x, w, targets, scale=4.0, add=before), t, o, x, w, targets, scale=4.0, add=before)


class Sized:
    """The library with a workspace query that answers a size of the test's choice."""

    def __init__(self, lib, size):
        self.lib, self.gm_linear_cross_entropy_workspace = lib, lambda *_: size

    def __getattr__(self, name):
        return getattr(self.lib, name)


@pytest.mark.gpu
@pytest.mark.parametrize("t, o", PAIRS)
def test_workspaces_between_the_least_and_the_recommended(t, o):
    """Each number of tokens at a time that some workspace leads to."""
    n, v, d = 2100, 400, 96
    x, w, targets = data(t, n, v, d, ignored=0.3)
    with Buffers() as b:
        lib = b.lib
        big = lib.gm_linear_cross_entropy_workspace(n, v, d, 0, d, t, o, 1)
        small = lib.gm_linear_cross_entropy_least_workspace(n, v, d, 0, d, t, o, 1)
        forms = {}
        for size in np.linspace(small, big, 200).astype(np.int64) // 256 * 256:
            if size >= small:
                forms.setdefault(taken(lib, n, v, d, t, o, int(size))[0], int(size))
        assert len(forms) >= 3, forms
        for chunk, size in sorted(forms.items()):
            b.lib = Sized(lib, size)
            check(run(b, t, o, x, w, targets, scale=4.0), t, o, x, w, targets, scale=4.0)
        b.lib = lib
