"""The Go wrappers of the language-model operators pass on what the library says of a refusal, and reach every call that a program
without HIP streams of its own has a use for."""
import os
import re

from test_go_integration_sources import GO, go_c_calls

PATH = os.path.join(GO, "cgo_bridge", "bridge_lm_linux.go")


def test_every_call_is_reached():
    called = {name for name, *_ in go_c_calls(PATH)}
    assert called >= {"execute_dropout", "gm_rng_state_advance", "execute_embedding_lookup", "execute_embedding_gradient",
                      "gm_embedding_gradient_workspace", "execute_linear_cross_entropy", "gm_linear_cross_entropy_workspace",
                      "gm_linear_cross_entropy_least_workspace", "gm_allocate_workspace", "gm_last_error"}


def test_errors_carry_the_librarys_message():
    """It belongs to the OS thread of the call, so the goroutine stays on it in between."""
    text = open(PATH).read()
    for name in ("lmCall", "AllocateWorkspace"):
        body = re.search(r"\nfunc %s\(.*?\n}\n" % name, text, re.S).group(0)
        assert body.index("runtime.LockOSThread()") < body.index("lastError()") and "defer runtime.UnlockOSThread()" in body
    for name, _, line, _ in go_c_calls(PATH):
        if name.startswith("execute_") or name == "gm_rng_state_advance":
            assert "lmCall(" in text.splitlines()[line - 2], name
