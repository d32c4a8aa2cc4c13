"""Calls of the 8-bit operators at the limits of what a launch takes: refused
before anything is queued, none cut short."""
from defer_amd import gpu as G
from defer_amd import q8

P = 4096  # an address that is aligned; nothing reads it on the host


def refused(name, *args):
    assert getattr(q8._lib(), "defer_gpu_q8_" + name)(*args) == G.E_INVALID, (name, args)
    return G.lib().defer_gpu_last_error().decode()


def test_attention_of_more_pairs_than_32_bits_count():
    """Rows times query heads that pass 2^32 by a little: once taken for that little."""
    pages = q8._CPages(P, P, P, P, P, 4, 1, 1, 2)
    for rows, heads in ((65538, 65535), (4194303, 1024), (131074, 32768), (4194303, 65535), (1 << 21, 2048)):
        r = q8._CRows(P, P, 1, rows, rows)
        assert "too many rows" in refused("attention", pages, r, 1, 1 << 40, heads, heads, 128, 1.0, None, 0, 0, 1 << 41, heads, 0, P,
                                          1 << 20, None), (rows, heads)
        assert q8._lib().defer_gpu_q8_attention_workspace(pages, r, heads, 128) == 0


def test_linear_of_more_channels_than_a_launch_has_threads_for():
    """16 channels are 256 threads, 32 channels 512, and a launch has fewer than 2^32."""
    for rows in (1, 17, 100):
        for m in (268435425, 268435441, 268435455):
            assert "268435424" in refused("linear", P, 32, P, P, 32, P, rows, m, 32, 0, P, m, None)
