"""What the norms' C entry point reads, without a GPU."""

from __future__ import annotations

from torchure_amd import _native

FAKE = 0x1000


def test_what_each_gradient_needs():
    lib = _native.lib()
    need = lib.tm_norm_workspace_bytes(33, 40, 0, 0, 1)
    #       dx    dw    db    bf dy    yf lddy x    xf ldx rstd  mean  w     wf dwf layer rows cols ws
    good = [FAKE, FAKE, FAKE, 0, FAKE, 0, 40, FAKE, 0, 40, FAKE, FAKE, FAKE, 0, 0, 1, 33, 40, FAKE, need, None]
    for wanted in ((0,), (1,), (0, 1), (0, 2), (1, 2)):
        for at in (7, 10, 11):
            args = [None if i < 3 and i not in wanted else v for i, v in enumerate(good)]
            args[at] = None
            assert lib.tm_norm_backward(*args) < 0 and b"null input" in lib.tm_last_error(), (wanted, at)
    args = [None, None, *good[2:]]  # the bias's alone: its workspace is looked at, x is not
    args[7] = args[10] = args[11] = args[12] = None
    args[9], args[19] = 0, need - 1
    assert lib.tm_norm_backward(*args) < 0 and b"workspace" in lib.tm_last_error()
