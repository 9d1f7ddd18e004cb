"""The page planner and page ids that cannot be."""
import numpy as np
import pytest

from test_serve_gpu import check_plan

pytestmark = pytest.mark.gpu


def test_a_page_outside_the_pool_is_reported_where_it_is_given_back(ctx):
    """By the call that ends the request, and not by the one that takes the page: it goes into the ring as it stands."""
    from cyb_b200 import qeng
    i = lambda *v: np.array(v, np.int32)  # noqa: E731
    ends = np.array([0, 2], np.int64)
    for bad in (-1, 12, 2 ** 31 - 1, -2 ** 31):
        table = i(0, 1, 2, bad, 4, 5).reshape(3, 2)
        ring = i(10, 11, -7, -7, -7, -7)
        assert check_plan(ctx, i(5, 20, 32), i(0, -1, -1), None, table, ring, ends, 12, 4) == 0
        with pytest.raises(qeng.QengError, match="status 1"):
            ctx.device_status()
        # a page that a request keeps, or one behind its length, is none of the call's business
        assert check_plan(ctx, i(5, 16, 32), i(0, -1, -1), i(0, 0, 0), table, ring, ends, 12, 4) == 0
        assert check_plan(ctx, i(5, 20, 32), i(0, -1, -1), i(0, 2, 0), table, ring, ends, 12, 4) == 0
        ctx.device_status()
