"""Workspaces of a draft model's operators: which sizes need one, which do not, and
that a call without it is refused before anything is launched."""

from __future__ import annotations

import pytest

from myelin_amd import _lib


def _refused(name, before, size, after=(None,)):
    """Without a workspace, with one too small, and with one that is not aligned."""

    for workspace, given, message in ((None, 0, "workspace of"), (16, size - 1, "workspace of"),
                                      (8, size, "16-byte aligned")):
        with pytest.raises(ValueError, match=message):
            _lib.call(name, *before, workspace, given, *after)


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("dtype", [0, 2])
def test_recurrence(dtype, backward):
    """Time is cut where channels are few and steps are more than one workgroup's."""

    need = _lib.load().myelin_gated_recurrence_workspace_elems
    for T, B, N in ((2**16, 1, 64), (513, 1, 1), (8192, 4, 2048)):
        n = need(dtype, T, B, N, backward)
        assert n > 0 and n % (2 * B * N) == 0
        args = ([16, 16, 16, dtype, 16, None, 16, None, 16, 16, 16] if backward else
                [16, 16, dtype, 16, None, None, 16, 16, None])
        name = "myelin_gated_recurrence_" + ("bwd" if backward else "fwd")
        strides = (_lib.ctypes.c_int64 * 6)(*[B * N, N] * 3)
        args[4 if backward else 3] = strides
        _refused(name, [*args, T, B, N], n)
    for T, B, N in ((256, 1, 64), (2048, 8, 2048), (1, 1, 1), (10**6, 1, 16384), (0, 1, 1), (100, 0, 5)):
        assert need(dtype, T, B, N, backward) == 0


def test_embedding():
    """Few tokens of a small table are not sorted."""

    need = _lib.load().myelin_token_embedding_bwd_workspace_bytes
    for M, V, D in ((100000, 1000, 64), (4097, 1, 1), (16384, 32768, 2048)):
        n = need(M, V, D)
        assert n >= 16 * M  # two pairs of keys and places
        _refused("myelin_token_embedding_bwd", [16, 16, 0, 16, M, V, D, 1.0, 0], n)
    for M, V, D in ((2048, 50, 128), (4096, 2048, 64), (1, 1, 1), (0, 1000, 64)):
        assert need(M, V, D) == 0


def test_distillation():
    """Long rows are split where they are few."""

    need = _lib.load().myelin_distillation_loss_workspace_bytes
    for R, V in ((1, 4097), (4, 100003), (256, 32768)):
        n = need(R, V)
        assert n > 0 and n % (8 * R) == 0
        _refused("myelin_distillation_loss", [16, 0, V, 16, 16, 1.0, 16, None, 16, R, V, 5], n)
    for R, V in ((1, 4096), (257, 32768), (10**6, 1000), (0, 100003)):
        assert need(R, V) == 0


def test_verification():
    need = _lib.load().myelin_verify_draft_workspace_bytes
    for B, V in ((1, 1), (1, 1025), (64, 100003)):
        n = need(B, V)
        assert n == B * -(-V // 1024) * 16
        _refused("myelin_verify_draft", [16, None, 0, 16, 16, 16, None, 16, 16, 3, B, V], n)
    assert need(0, 10) == 0 and need(3, 0) == 0


def test_embedding_of_few_positions():
    """A workgroup to a position needs nothing either; a wide row's slices count."""

    need = _lib.load().myelin_token_embedding_bwd_workspace_bytes
    for M, V, D in ((60, 5407, 26), (1024, 32000, 512), (2048, 100000, 1), (512, 150000, 2048)):
        assert need(M, V, D) == 0
    for M, V, D in ((2049, 100000, 1), (1025, 32000, 1024), (4096, 32000, 512)):
        n = need(M, V, D)
        assert n >= 16 * M
        _refused("myelin_token_embedding_bwd", [16, 16, 0, 16, M, V, D, 1.0, 0], n)
