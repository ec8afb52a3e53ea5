"""Memory that the operators around a recurrence ask for, as the library states it, against what their tensors take."""

import pytest

from mlstm_kernels_b200 import _lib


def padded(N):
    return next(n for n in (8, 16, 32, 64, 128) if N <= n)


@pytest.mark.parametrize("N", [1, 4, 16, 17, 32, 64, 100, 128])
@pytest.mark.parametrize("D", [64, 512, 2048, 4096, 8192])
@pytest.mark.parametrize("G", [1, 2, 8, 64])
@pytest.mark.parametrize("B,S", [(1, 2048), (4, 2048), (1, 16384)])
def test_backward_of_the_scan_takes_as_much_as_the_forward_kept(B, S, D, G, N):
    """Beside the segments' own states (up to 64 a sequence, twice: the adjoint's and da's) the partial sums of db and dc take 64 MB, or
    twice what the checkpoints take."""
    lib = _lib.load()
    kept = lib.mlstm_b200_ssm_checkpoint_bytes(B, S, D, N)
    assert kept == B * S // 16 * D * padded(N) * 4
    own = min(2 * kept, 2 * B * 64 * D * padded(N) * 4) + 2 * B * 64 * D * 4 + B * 64 * D * 4 + 5 * 256
    seams = B * 64 * 16 * G * min(64, -(-(D // G) * padded(N) // 1024)) * 2 * padded(N) * 4   # segments end between tiles of 16 tokens
    assert lib.mlstm_b200_ssm_workspace_bytes(B, S, D, N, G, 1) <= own + seams + max(64 << 20, 2 * kept)


def test_a_large_backward_of_many_states():
    """8 groups of 512 channels of 128 states, 4 x 2048 tokens: 4.3 GB of partial sums, were every tile of channels to write its own at once."""
    ws = _lib.load().mlstm_b200_ssm_workspace_bytes(4, 2048, 4096, 128, 8, 1)
    assert ws <= 2.25 * _lib.load().mlstm_b200_ssm_checkpoint_bytes(4, 2048, 4096, 128) < 2.5e9
