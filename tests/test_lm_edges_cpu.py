"""Edges of the operators around the attention layers that need no GPU."""

from selective_attention import _lib

A = 1 << 20   # an aligned address that nothing reads


def test_rows_of_probabilities_stay_within_a_tiles_offsets():
    """A piece of the vocabulary has as many words as a row of 2^22 bytes holds, however few the tokens: a tile's 256 rows of probabilities
    are then within 2^30 bytes. (The workspace: two pieces of one token's, and 64 parts of its fp32 sums of dX at the most.)"""
    lib = _lib.load()
    for dtype in (1, 2):
        for vocab in (1 << 26, 1 << 27, (1 << 28) - 1):
            size = lib.sa_linear_xent_backward_workspace_bytes(A, 64, 1, vocab, 64, 1, 1, dtype, dtype)
            assert 0 < size < 2 * (1 << 22) + 64 * 64 * 4 + (1 << 16), (dtype, vocab, size)
