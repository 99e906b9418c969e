"""What a HIP call that failed earlier on the thread leaves behind is not the operators' error: -6 is for a call's own launches."""
import ctypes

import numpy as np
import pytest

from operator_lib import F32, Buffers

pytestmark = pytest.mark.gpu
IGNORE = -100


def every_operator(b):
    """One small call of each: its name and code."""
    n, v, d = 4, 16, 8
    state, ids = b.state(), b.put(np.arange(n, dtype=np.int32))
    x, w = b.put(np.ones((n, d), np.float32)), b.put(np.ones((v, d), np.float32))
    y, g, losses, loss = b.empty((n, d), np.float32), b.empty((v, d), np.float32), b.empty(n, np.float32), b.empty(2, np.float32)
    need = b.lib.gm_linear_cross_entropy_workspace(n, v, d, w, d, F32, F32, 1)
    table = b.lib.gm_embedding_gradient_workspace(n, v, d)
    space, table_space = b.space(need), b.space(table)
    lib, device = b.lib, b.device
    return [
        ("dropout", lambda: lib.execute_dropout(device, 0, x, 0, y, n * d, F32, 0.5, state, 0)),
        ("advance", lambda: lib.gm_rng_state_advance(device, 0, state)),
        ("lookup", lambda: lib.execute_embedding_lookup(device, 0, w, ids, y, n, v, d, d, d, F32, 1.0, 0.0, 0, 0)),
        ("table gradient", lambda: lib.execute_embedding_gradient(device, 0, x, ids, g, n, v, d, d, d, F32, F32, 1.0, -1, 0, 0.0, 0, 0, table_space,
                                                                  table)),
        ("loss", lambda: lib.execute_linear_cross_entropy(device, 0, x, w, ids, losses, loss, y, g, n, v, d, d, d, d, d, F32, F32, IGNORE, 1, 1.0, 0, 0,
                                                          space, need)),
    ]


@pytest.mark.parametrize("which", range(5))
def test_after_a_workspace_that_was_refused(which):
    with Buffers() as b:
        name, call = every_operator(b)[which]
        assert b.lib.gm_allocate_workspace(b.device, 1 << 45) == 0 and b"workspace" in b.lib.gm_last_error()
        assert call() == 0, (name, b.lib.gm_last_error())


@pytest.mark.parametrize("which", range(5))
def test_after_a_failed_call_of_the_callers(which):
    hip = ctypes.CDLL("/opt/rocm/lib/libamdhip64.so")
    hip.hipMalloc.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t]
    with Buffers() as b:
        name, call = every_operator(b)[which]
        assert hip.hipMalloc(ctypes.byref(ctypes.c_void_p()), 1 << 45) != 0
        assert call() == 0, (name, b.lib.gm_last_error())
