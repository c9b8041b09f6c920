"""The adapters' gradient workspace follows the batch, not the table of adapters."""
import pytest

from mxgg import _lib


def size(M, K, N, R, L, S):
    return _lib.load().mxgg_lora_mm_backward_workspace_size(M, K, N, R, L, S)


@pytest.mark.parametrize("M,K,N,R,S", [(1000, 8192, 8192, 64, 8), (1, 64, 128, 8, 1), (16384, 5120, 8192, 16, 8)])
def test_more_adapters_than_segments_take_no_more(M, K, N, R, S):
    want = size(M, K, N, R, S, S)
    assert want > 0
    for L in (S + 1, 64 * S, 65535):
        assert size(M, K, N, R, L, S) == want
    # the intermediate's gradient, and per column tile of 128 a partial for each segment, one more per CTA at most
    rp = (R + 15) // 16 * 16
    tiles = (K + 127) // 128 + (N + 127) // 128
    assert want <= 4 * M * rp + (tiles * S + 2 * 2 * 148) * 128 * rp * 4 + 3 * 256


def test_fewer_adapters_take_less():
    assert size(4096, 1024, 1024, 16, 2, 1000) < size(4096, 1024, 1024, 16, 1000, 1000)


def test_sizes_that_no_call_takes():
    assert size(8, 64, 64, 8, 2, 1025) == -1 and size(8, 1 << 30, 64, 8, 2, 2) == -1
