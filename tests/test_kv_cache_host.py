"""The host side of the cache's operators: reports and refusals that need no GPU."""
import pytest
import torch

from atlasinfer_b200 import _capi, build
from atlasinfer_b200.integration import atlas_wrappers


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


def test_report_of_a_wait_that_ran_out():
    """The status word is shared by the linears and the attention: the report names both."""
    cpu = torch.device("cpu")
    atlas_wrappers.check_status(cpu)
    atlas_wrappers.status_word(cpu).fill_(1)
    with pytest.raises(_capi.AtlasError, match="attention") as e:
        atlas_wrappers.check_status(cpu)
    assert e.value.status == _capi.ERR_TIMEOUT
    atlas_wrappers.check_status(cpu)   # cleared
