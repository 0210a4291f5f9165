"""Refusals of forks in pools that the call cannot copy in.  CPU only."""
import pytest

from test_paged_serving_args import IE_ERR_INVALID_ARG, fork, ints


@pytest.mark.parametrize("pos", [(64, 70), (127, 64), (1, 0), (70, 70)])
def test_forks_within_a_page_need_a_pool(hip, pos):
    assert fork(hip.lib, pages=None, pos=ints(*pos)) == IE_ERR_INVALID_ARG
    assert "pool" in hip.last_error()


def test_no_forks_need_no_pool(hip):
    assert fork(hip.lib, n=0, pages=None) == 0
