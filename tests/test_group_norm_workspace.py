"""How much room group norm asks for, on the host."""
import pytest


@pytest.mark.parametrize("batch,cells,channels,groups", [(1, 343, 256, 32), (1000000, 1, 256, 8), (1000, 343, 256, 32), (3, 1955, 60, 6), (2, 5000, 12, 2)])
def test_results_of_small_samples_need_none(batch, cells, channels, groups):
    from medvision_amd import _lib
    assert 0 < _lib.load().mv_group_norm_workspace_bytes(batch, cells, channels, groups) <= 16


@pytest.mark.parametrize("batch,cells,channels,groups", [(1, 343, 256, 32), (100000, 1, 256, 8), (3, 1955, 60, 6), (7, 2999, 3, 3)])
def test_gradients_of_small_samples_need_a_sum_per_channel(batch, cells, channels, groups):
    from medvision_amd import _lib
    assert 0 < _lib.load().mv_group_norm_backward_workspace_bytes(batch, cells, channels, groups) <= 8 * batch * channels


@pytest.mark.parametrize("batch,cells,channels,groups", [(2, 2097152, 32, 8), (2, 27648, 256, 32), (1, 6000, 128, 1), (4, 5001, 20, 5)])
def test_large_samples_need_a_share_of_themselves(batch, cells, channels, groups):
    """Sums of the chunks: less than the cells in 16 bits take."""
    from medvision_amd import _lib
    lib = _lib.load()
    for query in (lib.mv_group_norm_workspace_bytes, lib.mv_group_norm_backward_workspace_bytes):
        assert 8 * batch * channels <= query(batch, cells, channels, groups) < 2 * batch * cells * channels
