"""The language-model operators refuse what they cannot do, before they touch a GPU: every check of arguments here runs
without one (a call that passes all of them answers -3 here, "no GPU")."""
import pytest

from __graft_entry__ import load_package

A, B, C, D = 0x10000, 0x20000, 0x30000, 0x40000      # placeholders: no call below reaches them
DEVICE = 0x1000


@pytest.fixture(scope="module")
def lib():
    return load_package().load_library()


def no_gpu(lib):
    if lib.create_metal_device():
        pytest.skip("a GPU is here: placeholders must not reach it")


def dropout(lib, device=DEVICE, queue=0, x=A, r=0, y=B, n=64, t=2, p=0.5, state=C, site=0):
    return lib.execute_dropout(device, queue, x, r, y, n, t, p, state, site)


def lookup(lib, device=DEVICE, table=A, tokens=B, out=C, n=4, v=10, d=8, ts=8, os=8, t=2, p=0.0, state=0):
    return lib.execute_embedding_lookup(device, 0, table, tokens, out, n, v, d, ts, os, t, 1.0, p, state, 0)


def gradient(lib, device=DEVICE, dy=A, tokens=B, g=C, n=4, v=10, d=8, ys=8, gs=8, t=2, o=2, p=0.0, state=0, space=D, size=1 << 20):
    return lib.execute_embedding_gradient(device, 0, dy, tokens, g, n, v, d, ys, gs, t, o, 1.0, -1, 0, p, state, 0, space, size)


def loss(lib, device=DEVICE, x=A, w=B, target=C, losses=D, total=D, dx=0x50000, dw=0x60000, n=4, v=10, d=8, xs=8, ws=8, dxs=8, dws=8,
         t=2, o=2, amp=0, space=0x70000, size=1 << 30):
    return lib.execute_linear_cross_entropy(device, 0, x, w, target, losses, total, dx, dw, n, v, d, xs, ws, dxs, dws, t, o, -100, 1,
                                            1.0, amp, 0, space, size)


@pytest.mark.parametrize("change, code", [
    (dict(device=0), -1), (dict(x=0), -4), (dict(y=0), -4), (dict(state=0), -4), (dict(n=-1), -5), (dict(t=1), -19), (dict(t=3), -19),
    (dict(p=-0.1), -5), (dict(p=1.5), -5), (dict(p=float("nan")), -5), (dict(x=A + 1), -5), (dict(y=B + 1), -5), (dict(r=D + 1), -5),
    (dict(t=0, x=A + 2), -5), (dict(state=C + 4), -5)])
def test_dropout(lib, change, code):
    assert dropout(lib, **change) == code


def test_generator_state(lib):
    assert lib.gm_rng_state_advance(0, 0, A) == -1
    assert lib.gm_rng_state_advance(DEVICE, 0, 0) == -4
    assert lib.gm_rng_state_advance(DEVICE, 0, A + 4) == -5


@pytest.mark.parametrize("change, code", [
    (dict(device=0), -1), (dict(table=0), -4), (dict(tokens=0), -4), (dict(out=0), -4), (dict(n=-1), -5), (dict(v=0), -5), (dict(d=0), -5),
    (dict(ts=7), -5), (dict(os=7), -5), (dict(t=1), -19), (dict(p=0.1), -4), (dict(p=2.0), -5), (dict(tokens=B + 2), -5),
    (dict(table=A + 1), -5), (dict(out=C + 1), -5), (dict(n=2 ** 31 - 1, d=2 ** 20, ts=2 ** 20, os=2 ** 20), -5)])
def test_lookup(lib, change, code):
    assert lookup(lib, **change) == code


@pytest.mark.parametrize("change, code", [
    (dict(device=0), -1), (dict(dy=0), -4), (dict(tokens=0), -4), (dict(g=0), -4), (dict(n=-1), -5), (dict(v=-3), -5), (dict(d=0), -5),
    (dict(ys=7), -5), (dict(gs=7), -5), (dict(t=1), -19), (dict(t=2, o=4), -19), (dict(t=0, o=2), -19), (dict(p=0.5), -4),
    (dict(space=0), -18), (dict(space=D + 128), -18), (dict(size=0), -18), (dict(n=2 ** 22 + 1, size=1 << 62), -5)])
def test_table_gradient(lib, change, code):
    assert gradient(lib, **change) == code


def test_table_gradient_workspace(lib):
    assert lib.gm_embedding_gradient_workspace(-1, 10, 8) == 0 and lib.gm_embedding_gradient_workspace(4, 0, 8) == 0
    need = lib.gm_embedding_gradient_workspace(10000, 100, 1000)
    assert 4 * 4 * 10000 <= need <= 4 * 4 * 10000 + 10000 // 8 * 2 * 1000 * 4 + 5 * 256      # pieces of eight entries or more
    no_gpu(lib)
    assert gradient(lib, n=10000, d=1000, ys=1000, gs=1000, size=need - 1) == -18
    assert str(need).encode() in lib.gm_last_error()
    assert gradient(lib, n=10000, d=1000, ys=1000, gs=1000, size=need) == -3


@pytest.mark.parametrize("change, code", [
    (dict(device=0), -1), (dict(x=0), -4), (dict(w=0), -4), (dict(target=0), -4), (dict(losses=0), -4), (dict(total=0), -4),
    (dict(n=-1), -5), (dict(n=2 ** 24 + 1), -5), (dict(v=0), -5), (dict(v=2 ** 22 + 1), -5), (dict(d=0), -5), (dict(xs=7), -5),
    (dict(ws=7), -5), (dict(dxs=7), -5), (dict(dws=7), -5), (dict(t=1), -19), (dict(t=2, o=4), -19), (dict(t=0, o=2), -19),
    (dict(x=A + 1), -5), (dict(w=B + 1), -5), (dict(target=C + 2), -5), (dict(dx=0x50001), -5), (dict(dw=0x60001), -5),
    (dict(space=0), -18), (dict(space=0x70080), -18), (dict(size=1000), -18)])
def test_loss(lib, change, code):
    assert loss(lib, **change) == code


def test_loss_workspaces(lib):
    """The least workspace is less than the recommended one where tokens can be taken in parts, and both are refused one
    byte short; a copy of the weights is asked for only where they cannot be read as they lie."""
    ask, least = lib.gm_linear_cross_entropy_workspace, lib.gm_linear_cross_entropy_least_workspace
    assert ask(-1, 10, 8, 0, 8, 2, 2, 1) == 0 and ask(1, 10, 8, 0, 8, 1, 1, 1) == 0 and ask(1, 10, 8, 0, 8, 2, 4, 1) == 0
    for t, o in ((2, 2), (4, 4), (2, 0), (4, 0), (0, 0)):
        big, small = ask(4096, 32000, 1024, A, 1024, t, o, 1), least(4096, 32000, 1024, A, 1024, t, o, 1)
        assert 0 < small < big
        assert ask(4096, 32000, 1024, A, 1024, t, o, 0) < big
        assert ask(4096, 32000, 1024, 0, 1024, t, o, 1) >= big
    assert ask(64, 1000, 512, 0, 512, 2, 2, 1) - ask(64, 1000, 512, A, 512, 2, 2, 1) == 1000 * 512 * 2
    assert ask(64, 1000, 512, A + 2, 512, 2, 2, 1) == ask(64, 1000, 512, 0, 512, 2, 2, 1) == ask(64, 1000, 512, A, 513, 2, 2, 1)
    no_gpu(lib)
    need = least(4096, 32000, 1024, B, 1024, 2, 2, 1)
    sizes = dict(n=4096, v=32000, d=1024, xs=1024, ws=1024, dxs=1024, dws=1024)
    assert loss(lib, size=need - 1, **sizes) == -18 and str(need).encode() in lib.gm_last_error()
    assert loss(lib, size=need, **sizes) == -3


def test_queues_and_workspaces_without_a_device(lib):
    assert lib.gm_command_queue_for_stream(0, None) == 0
    assert lib.gm_allocate_workspace(0, 1024) == 0
    assert lib.gm_allocate_workspace(DEVICE, 0) == 0
