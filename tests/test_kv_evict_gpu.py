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


def check(c, count, keep, sinks, recent, on_device):
    """The cache stays as it was for the next one."""
    pos = 1 << 20
    got = c.evict(*((-1, -1) if on_device else (count, pos)), keep, sinks, recent, state=(count, pos) if on_device else None)
    for a, b, name in zip(got, c.evicted(count, pos, keep, sinks, recent), ("K", "V", "mass", "positions")):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), (name, np.argwhere(a != b)[:5].tolist())


def fill(m, what, rng):
    """Masses that make the steps of the cut hard: many alike, none alike, close ones, no numbers."""
    if what == "equal":
        m[:] = 0.25
    elif what == "zeros":
        m[:] = np.where(rng.random(m.shape) < 0.5, 0.0, -0.0)
    elif what == "few values":
        m[:] = rng.integers(0, 3, m.shape)
    elif what == "nan":
        m[rng.random(m.shape) < 0.4] = np.nan
        m[rng.random(m.shape) < 0.2] = -np.nan
    elif what == "inf":
        m[rng.random(m.shape) < 0.4] = np.inf
        m[rng.random(m.shape) < 0.1] = -np.inf
    else:
        m[:] = (np.float32(1.5).view(np.uint32) + rng.integers(0, 700, m.shape).astype(np.uint32)).view(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["equal", "zeros", "few values", "nan", "inf", "close"])
@pytest.mark.parametrize("count,slots", [(5000, 5050), (33000, 33100), (40000, 40001)])
def test_long_caches_of_every_mass(count, slots, what):
    """More rows than a block holds in LDS (32768) and fewer; few that go, few that stay, and in between; from the host's
    count, and from the device's with a grid for all slots."""
    c = Cache(2, 2, 64, slots, seed=32)
    fill(c.mass[:, :count], what, c.rng)
    for keep in (1, 90, 700, count // 2, count - 100, count - 2, count - 1):
        for sinks, recent in ((0, 0), (200000, 30000)):
            for on_device in (False, True):
                print(count, slots, what, keep, sinks, recent, on_device, flush=True)
                check(c, count, keep, sinks, recent, on_device)


@pytest.mark.gpu
@pytest.mark.parametrize("slots,counts", [(4096, (4096, 4095, 500, 65, 64)), (40000, (40000, 33000, 5000, 66, 65))])
def test_a_count_on_the_device_far_below_the_slots(slots, counts):
    """The launch is that of all slots, whatever the count: of many rows, of one more than stay, of none too many."""
    c = Cache(2, 2, 64, slots, seed=33)
    for count in counts:
        for keep in (1, 64, count - 1, count - 70):
            if 1 <= keep:
                print(slots, count, keep, flush=True)
                check(c, count, keep, 3, 20, True)
    before = [a.copy() for a in c.arrays()]
    for bad in ((slots + 1, 5), (-1, 5), (slots, -1), (0, 0)):
        assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(before, c.evict(-1, -1, 30, 0, 0, state=bad))), bad


@pytest.mark.gpu
def test_what_stays_was_there_once():
    """Of each kv head the positions after an eviction are some of those before it, none twice, at their own rows."""
    c = Cache(3, 3, 64, 600, seed=34)
    for g in range(3):
        c.positions[g, :500] = c.rng.permutation(500)
    K, positions = c.K.copy(), c.positions.copy()
    c.K, c.V, c.mass, c.positions = c.evict(500, 500, 300, 5, 40)
    for g in range(3):
        stays = c.positions[g, :300]
        assert np.unique(stays).size == 300 and np.isin(stays, positions[g, :500]).all()
        at = np.argsort(positions[g, :500])[stays]
        assert np.array_equal(c.K[g, :300].view(np.uint16), K[g, at].view(np.uint16))


@pytest.mark.gpu
def test_drafts_behind_a_cache_without_rows():
    """KVMass with nothing in it: an eviction that has nothing to do, no masses, drafts whose prefix is empty."""
    from trixium_amd.attention import KVMass, SharedPrefix
    m = KVMass(4, 2, 64, 16)
    m.evict(5)
    assert m.count == 0 and m.masses().shape == m.positions().shape == (2, 0) and m.rows()[0].shape == (2, 0, 64)
    none = np.zeros((2, 0, 64), np.float16)
    rng = np.random.default_rng(35)
    q, k, v = rng.standard_normal((3, 1, 4, 64)), rng.standard_normal((3, 1, 2, 64)), rng.standard_normal((3, 1, 2, 64))
    for d in (m.share(3, 4), SharedPrefix(4, 2, 64, none, none, 3, 4)):
        # One key: its value, whatever the score, but for the probability's planes (2^-22 of it) and what is rounded of
        # products, sum and reciprocal (2^-24 each, fewer than eight).
        want = np.repeat(v.astype(np.float16), 2, axis=2).astype(np.float64)
        assert (np.abs(d.attend(q, k, v) - want) <= np.abs(want) * 2.0**-20).all()
        assert np.array_equal(d.rows(-1)[0], k[2].astype(np.float16).transpose(1, 0, 2))
