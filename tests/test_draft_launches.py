"""Log probabilities at the limit of what a launch takes: refused before anything is queued."""
import pytest

from defer_amd import gpu as G
from defer_amd import q8

P = 1 << 20  # an address that is aligned; nothing reads it on the host


@pytest.mark.parametrize("rows,chunks", [(1813753, 37), (192289, 349), (2164802, 31), (1082401, 62)])
def test_log_probs_of_more_waves_than_a_launch_has_threads_for(rows, chunks):
    """Four waves, a chunk of 1,024 logits each, are 256 threads, and a launch has fewer than 2^32: 67,108,860 chunks."""
    n, most = 1024 * chunks, 67108860
    assert most < rows * chunks < 1 << 26
    for r in (rows, 4194303):
        assert q8._lib().defer_gpu_q8_log_probs(0, P, n, r, n, None, 1.0, 0, P, P, P, None, None, P, 1 << 40, None) == G.E_INVALID
        assert "too many rows" in G.lib().defer_gpu_last_error().decode()
