"""Eviction by masses (trx_kv_evict) against a sort on the host, to the bit: what stays where more rows are at kept
positions than stay, and caches that the selecting kernel holds in LDS or reads again for every step."""

import numpy as np
import pytest

from test_kv_mass_gpu import Cache


@pytest.mark.gpu
def test_more_kept_positions_than_rows_stay_by_slot():
    """The largest masses do not decide among rows at kept positions; beyond them they do, an infinity no more than a row
    at a kept position."""
    c = Cache(1, 1, 64, 6, seed=31)
    c.positions[0] = [0, 1, 2, 3, 9, 8]
    c.mass[0] = [0.1, 0.9, 0.5, 0.7, 0.2, 0.3]
    c.check_evict(6, 10, 2, 4, 0)
    assert c.positions[0, :2].tolist() == [0, 1]
    c = Cache(1, 1, 64, 6, seed=31)
    c.positions[0] = [4, 5, 0, 6, 9, 8]
    c.mass[0] = [0.1, np.inf, 0.0, 0.7, np.nan, 0.3]
    c.check_evict(6, 10, 3, 1, 1)                                # positions 0 and 9 are kept
    assert sorted(c.positions[0, :3].tolist()) == [0, 5, 9]
