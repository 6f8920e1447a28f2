"""The largest token and rank counts of the 4-bit layer, without a device."""

import ctypes


def test_most_tokens_and_ranks(qb):
    """Counts whose padded values would leave 32 bits are refused before anything is
    launched."""
    lib = qb._lib.load()
    n = ctypes.c_size_t(0)
    P, A = None, 256  # A: a non-null address, never dereferenced
    for M, rank, want in ((2 ** 31 - 1024, 4, 0), (2 ** 31 - 1023, 4, 1), (2 ** 31 - 1, 0, 1), (2 ** 31, 0, 1),
                          (70, 2 ** 24, 0), (70, 2 ** 24 + 1, 1), (70, 2 ** 31 - 1, 1)):
        for size_of in (lib.qlin_mx_workspace_size, lib.qlin_mx_backward_workspace_size):
            for dtype in (0, 1, 2):
                assert size_of(dtype, M, 1, 1, rank, ctypes.byref(n)) == want, (M, rank)
        if want:
            assert lib.qlin_mx_forward(1, A, 4, A, P, A, A, rank, 1.0, A, 4, M, 1, 1, A, 2 ** 60, P) == 1
            assert lib.qlin_mx_backward(1, A, 4, A, 4, A, A, A, rank, 1.0, A, 4, P, P, P, M, 1, 1, A, 2 ** 60, P) == 1
