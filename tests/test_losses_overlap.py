"""Where a gradient may be written: rows beside the logits' rows in one buffer
are no overlap (no GPU: a device that is not there answers what the checks let
through)."""
from __future__ import annotations

import ctypes as C

import pytest

pytest.importorskip("torch")

import distlr_amd as dlr  # noqa: E402
import distlr_amd.losses as L  # noqa: E402

BUF = (C.c_char * 65536)()
A = (C.addressof(BUF) + 255) // 256 * 256 + 16384
V = A + 16384  # vectors, out of the way
ROWS, VOCAB = 4, 8  # of 4 bytes: 32 a row


def answer(logits_stride, grad_at, grad_stride, rows=ROWS):
    x = L._Logits(A, V, rows, VOCAB, logits_stride, L.DTYPE_F32, 64, 1.0)
    p = L._Policy(V, None, V, None, 0.2, 0.2, 0.0)
    one = L.lib.dlr_token_logprob_grad(99, None, C.byref(x), V, V, A + grad_at, grad_stride)
    two = L.lib.dlr_policy_loss(99, None, C.byref(x), C.byref(p), None, 0, V, V, V, V, A + grad_at, grad_stride)
    assert one == two
    if one == dlr.E_ARG:
        assert "overlap" in L.lib.dlr_losses_last_error().decode()
    return one


@pytest.mark.parametrize("at,stride", [(32, 16), (48, 24), (32, 20), (-32, 16), (32 + 4 * 80, 20), (-80 * 2 + 32, 20),
                                       (80 * 3 - 32, 20)])
def test_rows_beside_the_logits_rows(at, stride):
    assert answer(stride, at, stride) == dlr.E_HIP


@pytest.mark.parametrize("at,stride,other", [
    (28, 16, 16),    # one element of the row before
    (36, 16, 16),    # and of the one behind
    (28, 20, 20), (52, 20, 20), (64 * 2 + 28, 16, 16), (80 * 2 - 28, 20, 20),
    (32, 16, 24),    # at another distance some rows meet
    (28, 0, 8),      # the logits' rows are one, of 32 bytes
])
def test_rows_that_meet(at, stride, other):
    assert answer(stride, at, other) == dlr.E_ARG


def test_behind_and_before():
    assert answer(16, 3 * 64 + 32, 8) == dlr.E_HIP and answer(16, -(3 * 32 + 32), 8) == dlr.E_HIP
    assert answer(16, 3 * 64 + 28, 8) == dlr.E_ARG and answer(16, -(3 * 32 + 28), 8) == dlr.E_ARG
    assert answer(8, 0, 8) == dlr.E_HIP  # the logits themselves
    assert answer(1 << 40, 32, 1 << 40, rows=1) == dlr.E_HIP and answer(1 << 40, 28, 1 << 40, rows=1) == dlr.E_ARG
