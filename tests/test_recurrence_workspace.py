"""The scan's workspace: its size for a descriptor is enough for every call of
no more rows and sequences, so that a program allocates once for its longest."""
import ctypes as C

import pytest

import native
from native import bh


def size(n_seqs, n_tokens, H, P, G, N):
    d = bh.Ssm(type=bh.F32, n_heads=H, head_dim=P, n_groups=G, d_state=N, n_seqs=n_seqs,
               n_tokens=n_tokens)
    return bh.lib().bm_hip_ssm_workspace_bytes(C.byref(d))


SHAPES = [(64, 64, 1, 128), (64, 64, 64, 1), (32, 64, 32, 1), (4, 16, 2, 8), (32, 64, 8, 64),
          (2, 32, 1, 24), (1, 1, 1, 1), (2000, 64, 1, 16), (4096, 64, 1, 2), (128, 128, 4, 256)]


@pytest.mark.parametrize("shape", SHAPES)
def test_size_never_falls_with_rows_or_sequences(shape):
    rows = sorted(set(list(range(0, 700)) + list(range(700, 70000, 31)) +
                      [1 << k for k in range(30)] + [(1 << k) + 1 for k in range(30)]))
    before = None
    for n in (1, 2, 3, 7, 16, 64, 1000, 1 << 16, 1 << 20):
        sizes = [size(n, t, *shape) for t in rows]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))
        if before is not None:
            assert all(a <= b for a, b in zip(before, sizes))
        before = sizes
    assert before[0] == 0


def test_sizes_that_once_fell():
    """Fewer rows in shorter units take more places."""
    assert size(1, 1920, 64, 64, 1, 128) <= size(1, 16384, 64, 64, 1, 128)
    assert size(1, 1024, 64, 64, 64, 1) <= size(1, 2049, 64, 64, 64, 1)
    assert size(1, 1024, 64, 64, 64, 1) > 0
