"""CPU: the order of the paged attention kernels' roles (tests/paged_protocol.py)."""
from __future__ import annotations

import random

import pytest

from tests.paged_protocol import Cta, FewRows, random_items


@pytest.mark.parametrize("seed", range(6))
def test_roles_go_through_in_any_order(seed):
    """Every row of every item is stored, whatever the order of events."""
    rng = random.Random(seed)
    for _ in range(60):
        items = random_items(rng)
        cta = Cta(items, rng)
        assert not cta.run()
        assert cta.stored == {(i, s): t for i, (t, two) in enumerate(items) for s in range(1 + two)}


@pytest.mark.parametrize("seed", range(6))
def test_waits_that_run_out_leave_nothing_in_flight(seed):
    """Waits that give up anywhere: all roles end, copies and products have landed, and what is
    stored is complete."""
    rng = random.Random(100 + seed)
    gave_up = 0
    for _ in range(120):
        gave_up += Cta(random_items(rng), rng, give_up=rng.choice([0.002, 0.01, 0.05])).run()
    assert gave_up > 30


def test_a_copy_that_is_not_counted_is_found():
    """A producer that forgets a tile's K where the wait for V's place gave up."""
    rng = random.Random(7)
    found = 0
    for _ in range(400):
        try:
            Cta(random_items(rng), rng, give_up=0.02, forget_k=True).run()
        except AssertionError as e:
            # left early, or waiting for a phase that the forgotten copy has passed
            assert "in flight" in str(e) or "two phases apart" in str(e)
            found += 1
    assert found > 0


@pytest.mark.parametrize("seed", range(4))
def test_few_rows_go_through_in_any_order(seed):
    rng = random.Random(200 + seed)
    for _ in range(60):
        items = [rng.randint(1, 20) for _ in range(rng.randint(1, 4))]
        cta = FewRows(items, rng)
        assert not cta.run()
        assert cta.stored == dict(enumerate(items)) and not cta.kept


@pytest.mark.parametrize("seed", range(4))
def test_few_rows_keep_back_what_is_not_complete(seed):
    """Behind a wait that gave up, no warp stores rows that lack another's keys, and every item
    is stored or marked."""
    rng = random.Random(300 + seed)
    kept = 0
    for _ in range(120):
        items = [rng.randint(1, 20) for _ in range(rng.randint(1, 4))]
        cta = FewRows(items, rng, give_up=rng.choice([0.002, 0.01]))
        cta.run()
        assert set(cta.stored) | cta.kept == set(range(len(items))) and not set(cta.stored) & cta.kept
        kept += len(cta.kept)
    assert kept > 30


def test_a_warp_that_looks_at_its_own_wait_only_is_found():
    rng = random.Random(8)
    found = 0
    for _ in range(200):
        try:
            FewRows([rng.randint(1, 20) for _ in range(3)], rng, give_up=0.01, forget=True).run()
        except AssertionError as e:
            assert "without all of their keys" in str(e)
            found += 1
    assert found > 0
