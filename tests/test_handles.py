"""Handles of host objects (command queues, loss-scale states) are looked up, never read from the address that a caller passes:
any number is refused where it names none."""
import numpy as np
import pytest

from operator_lib import F32, Buffers

from __graft_entry__ import load_package

NOWHERE = [1, 8, 0xDEADBEEF, (1 << 47) - 64, 1 << 63]


@pytest.mark.parametrize("handle", NOWHERE)
def test_numbers_that_name_nothing(handle):
    lib = load_package().load_library()
    lib.release_command_queue(handle)
    lib.gm_amp_state_destroy(handle)
    assert lib.gm_amp_state_get(handle, None, None) == -16
    assert lib.gm_amp_state_set(handle, 1.0, 0) == -16


@pytest.mark.gpu
def test_operators_refuse_them():
    with Buffers() as b:
        x, w, y = b.put(np.ones((4, 8), np.float32)), b.put(np.ones((16, 8), np.float32)), b.empty((4, 8), np.float32)
        ids, losses, loss = b.put(np.arange(4, dtype=np.int32)), b.empty(4, np.float32), b.empty(2, np.float32)
        need = b.lib.gm_linear_cross_entropy_workspace(4, 16, 8, w, 8, F32, F32, 0)
        space = b.space(need)

        def drop(queue):
            return b.lib.execute_dropout(b.device, queue, x, 0, y, 32, F32, 0.0, 0, 0)

        def entropy(queue, amp):
            return b.lib.execute_linear_cross_entropy(b.device, queue, x, w, ids, losses, loss, 0, 0, 4, 16, 8, 8, 8, 8, 8, F32, F32, -100, 1, 1.0, amp, 0,
                                                      space, need)

        queue, amp = b.lib.create_command_queue(b.device), b.lib.gm_amp_state_create(b.device, 2.0, 2.0, 0.5, 10)
        assert drop(queue) == 0 and entropy(queue, amp) == 0
        for handle in NOWHERE + [x, amp, b.device]:      # of another kind, too
            assert drop(handle) == -2 and entropy(handle, 0) == -2
        for handle in NOWHERE + [x, queue, b.device]:
            assert entropy(0, handle) == -16
        for _ in range(2):      # what has been released is gone, and may be released again
            b.lib.release_command_queue(queue)
            b.dev.synchronize()
            b.lib.gm_amp_state_destroy(amp)
            assert drop(queue) == -2 and entropy(0, amp) == -16
