"""Refusals of the kept rows' library entry: no GPU."""

from __future__ import annotations


def test_a_cache_beyond_one_launch_is_checked_before_the_first():
    """64 caches go in one launch: a 65th of another geometry, a null or a misaligned one refuses the call before
    any row has moved (on a machine without a GPU, a launch would be a CUDA error)."""
    from mlx_motif import _native as N

    structs = (N.motif_kv4_slots * 65)()
    for s in structs:
        for i in range(4):
            s.data[i] = s.scales[i] = s.biases[i] = 1 << 20
        s.bits, s.group_size, s.batch, s.heads, s.capacity, s.head_dim = 16, 64, 1, 2, 64, 128

    def call():
        return N.lib.motif_kv4_keep_rows(0, structs, 65, 1, 4, 1, 4, 0, None, 0, 64, None)

    structs[64].heads = 3
    assert call() == N.ERR_BAD_SHAPE and b"cache 64 differs" in N.lib.motif_last_error()
    structs[64].heads = 2
    structs[64].data[2] = None
    assert call() == N.ERR_NULL
    structs[64].data[2] = (1 << 20) + 1
    assert call() == N.ERR_BAD_CONTRACT and b"misaligned" in N.lib.motif_last_error()


def test_sizes_beyond_the_kernels_32_bits_are_refused():
    """Rows of a tree times bytes of a row are counted in 32 bits on the device."""
    from mlx_motif import _native as N

    s = N.motif_kv4_slots()
    for i in range(4):
        s.data[i] = s.scales[i] = s.biases[i] = 1 << 20
    s.bits, s.group_size, s.batch, s.heads, s.capacity = 16, 64, 1, 1, 1 << 30

    def call(head_dim, T, batch=1):
        s.head_dim, s.batch = head_dim, batch
        return N.lib.motif_kv4_keep_rows(0, s, 1, 1, T, 1, T, 0, None, 0, 1 << 30, None)

    assert call(1 << 12, 1 << 20) == N.ERR_BAD_SHAPE and call((1 << 32) + 128, 4) == N.ERR_BAD_SHAPE
    assert call(128, 4, batch=1 << 62) == N.ERR_BAD_SHAPE
