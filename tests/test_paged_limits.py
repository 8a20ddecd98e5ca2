"""What the paged attention takes and what it refuses as too large, without a device: sizes are
settled before anything is launched."""
from summa_amd import _lib

BF16, F8 = _lib.SM_BF16, _lib.SM_F8E4M3
D = 1 << 20  # a device pointer that is never dereferenced


def workspace(S, rows, most, H, KVH, hd=64, tokens=64):
    return _lib.lib().sm_paged_attention_workspace_bytes(S, rows, most, H, KVH, hd, tokens)


def attention(S, rows, most, H, KVH, hd=64, tokens=1 << 20):
    """Status and message of a call without a workspace, or with q over out where none is needed:
    refused at the latest there, so nothing is launched."""
    import ctypes
    c = _lib.PagedCache(D, D, D, D, 4, KVH, 32, hd, F8)
    st = _lib.lib().sm_paged_attention(ctypes.addressof(c), D, 4, D, D, S, rows, most, tokens, D, BF16,
                                       H * hd, H, D, None, None, 0, None)
    return st, _lib.lib().sm_last_error().decode()


def test_one_long_sequence_among_many_short_ones():
    """The longest sequence's rows count for every sequence in the grid, 128 to a workgroup, and
    not in a join that is not launched."""
    for S, most, H, KVH, hd in ((128, 32768, 16, 4, 128), (256, 4096, 64, 8, 128),
                                (1024, 32768, 16, 4, 64), (1024, 16384, 16, 16, 128)):
        rows = most + S - 1
        assert workspace(S, rows, most, H, KVH, hd, most) == 0
        st, err = attention(S, rows, most, H, KVH, hd, most)
        assert st == -1 and "out must not overlap q" in err, err


def test_what_no_grid_holds():
    for S, most, H, KVH, hd in ((1 << 14, 131072, 16, 1, 64),    # 2^28 tiles of 128 rows
                                (1 << 23, 2, 4, 2, 64),          # 2^24 workgroups of 16 rows
                                (1 << 30, 1, 65535, 65535, 64),  # no 64-bit product
                                (8192, 131072, 16, 8, 128),      # 2^26 tiles of 256 rows
                                (1024, 131072, 16, 8, 128)):     # 2^23 of them, of 512 threads
        rows = S * 2 if most == 2 else most + S - 1
        assert workspace(S, rows, most, H, KVH, hd, 1 << 20) == -1
        st, err = attention(S, rows, most, H, KVH, hd)
        assert st == -3 and "too large" in err, err
    assert workspace(1, (1 << 31) - 2, (1 << 31) - 2, 2, 1) == -1  # rows of a KV head past 32 bits
    assert workspace(1, (1 << 31) - 2, 1, 1024, 1) == -1           # 2^41 - 2^11 rows of all heads
