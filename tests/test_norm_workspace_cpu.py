"""Bytes of the norms' backward workspace: what the launches can use, not a row
of partial sums for every row of the batch."""
import pytest

from mhc_proj import capi


@pytest.mark.parametrize("size", [capi.layer_norm_backward_workspace, capi.stream_norm_n4_backward_workspace])
def test_workspace_is_what_the_launches_use(size):
    def rows(N, C):
        assert size(N, C) % (8 * C) == 0
        return size(N, C) // (8 * C)

    # rows wider than the rings hold: 64 chunks of rows at most, of eight rows at least
    assert rows(1024, 1 << 20) == 64 and rows(2048, 32768) == 64
    assert rows(256, 20001) == 32 and rows(3, 1 << 30) == 1
    # a row for each block, three for each of up to 160 SMs
    assert rows(65536, 4096) == rows((1 << 31) - 1, 64) == 480
    assert rows(3, 4096) == 16 and rows(300, 16384) == 300
