"""pcl_context_reserve of any size, then a launch that needs more."""
import numpy as np
import pytest

from test_paged import bits, torch  # noqa: F401
from test_paged_tree import TreeCache


@pytest.mark.gpu
@pytest.mark.parametrize("nbytes", [0, 1, 2, 3, 4, 5, 17])
def test_a_workspace_of_few_bytes(pcl, torch, nbytes):
    own = pcl.Context(0)
    own.reserve(nbytes)
    cache = TreeCache(pcl, torch, (4, 2, 64), [700, 40], [3, 3], 16, "f32", 22)
    q = cache.queries()
    out = cache.tree_attend(own, q)
    assert own.sync() == 0
    cache.check(own, q, out)
    again = cache.tree_attend(own, q)
    assert np.array_equal(bits(out), bits(again)) and own.sync() == 0
    own.close()
