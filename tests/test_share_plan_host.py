"""How calls are cut whose sequences share their first pages (kv8_device.h), as the host decides it."""

import ctypes as C
import itertools
import random

import pytest

from test_step_host import compiled


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    lib = compiled(tmp_path_factory.mktemp("plan"), '''
#include "kv8_device.h"
using namespace fortai_hip;
extern "C" void plan(int fp32, int head, int sequences, int groups, int kv, int64_t rows, int64_t group_rows, int64_t own, int64_t shared, int64_t *out) {
    const Kv8SharedPlan p = kv8_shared_plan(fp32 != 0, head, sequences, groups, kv, rows, group_rows, own, shared);
    const Kv8Plan q = kv8_plan(fp32 != 0, head, sequences, kv, rows, own + shared);
    const int64_t all[] = {p.shares, p.own.rows, p.own.row_tiles, p.own.splits, p.group.rows, p.group.row_tiles, p.group.splits, q.splits};
    for (int i = 0; i < 8; ++i) out[i] = all[i]; }''')
    lib.plan.argtypes = [C.c_int] * 5 + [C.c_int64] * 4 + [C.c_void_p]
    names = "shares own_rows own_tiles own_splits rows tiles splits plain_splits".split()

    def call(fp32, head, sequences, groups, kv, rows, group_rows, own, shared):
        out = (C.c_int64 * 8)()
        lib.plan(fp32, head, sequences, groups, kv, rows, group_rows, own, shared, out)
        return dict(zip(names, out[:]))

    return call


def test_few_rows_are_one_launch(plan):
    """16-bit groups of up to 16 rows of sequences of up to 8 go with these in one launch, in workgroups of 16 rows."""
    for rows, group_rows, shared in itertools.product((1, 4, 8), (9, 12, 16), (1000, 8000, 100000)):
        p = plan(0, 256, 4, 1, 4, rows, group_rows, 100, shared)
        assert p["own_rows"] == p["rows"] == 16, p
    assert plan(0, 256, 4, 1, 4, 2, 8, 100, 1000)["own_rows"] == 8
    assert plan(1, 256, 4, 1, 4, 4, 16, 100, 1000)["own_rows"] == 8  # fp32 has no others


def test_little_is_not_shared(plan):
    """Up to 256 shared tokens where the plain call is one launch: a second launch costs more than reading them again."""
    for fp32, (heads, kv), head, n, shared in itertools.product((0, 1), ((8, 2), (16, 4), (12, 1)), (64, 256), (2, 4, 31), (64, 128, 256)):
        rows = heads // kv
        p = plan(fp32, head, n, 1, kv, rows, n * rows, 8, shared)
        assert not p["shares"] or p["plain_splits"] > 1, (fp32, heads, head, n, shared)
    assert plan(1, 256, 4, 1, 4, 4, 16, 8, 1000)["shares"] and not plan(1, 256, 4, 1, 4, 4, 16, 1000, 32)["shares"]


def test_workgroups_fit_the_chip_where_they_are_many(plan):
    """Four sequences of 20 rows of 4 kv heads behind 24,000 tokens: 42 splits of 12 blocks, not 43."""
    assert plan(1, 256, 4, 1, 4, 20, 68, 150, 24000)["splits"] == 42
    rng = random.Random(3)
    many = 0
    for _ in range(4000):
        head, n, kv = rng.choice([64, 128, 256]), rng.randint(2, 40), rng.choice([1, 2, 3, 4, 8])
        groups, rows = rng.randint(1, min(3, n)), rng.randint(1, 80)
        p = plan(rng.randrange(2), head, n, groups, kv, rows, max(rows, rows * n // groups), rng.randint(1, 700), int(2 ** rng.uniform(6, 18)))
        blocks, chip = groups * p["tiles"] * kv, 512 * (256 // head)
        assert blocks * p["splits"] <= chip or p["splits"] == 1
        many += blocks * p["splits"] > chip // 2
    assert many > 200


def test_a_last_turn_of_little_is_saved(plan):
    """125 tiles of 64 in 16 splits of four waves are two turns, in 15 three; 375 in 47 two, in 43 three."""
    assert plan(1, 256, 4, 1, 2, 20, 68, 150, 8000)["splits"] == 16
    assert plan(0, 256, 2, 1, 2, 20, 36, 150, 24000)["splits"] == 47


def test_what_gains_is_shared_and_what_loses_is_not(plan):
    """Measured on both sides: fp32, 4 kv heads of 256."""
    for n, rows, shared in ((8, 4, 8000), (32, 4, 8000), (8, 4, 24000), (32, 4, 24000), (5, 20, 24000), (32, 20, 24000), (4, 4, 1000)):
        assert plan(1, 256, n, 1, 4, rows, n * rows, 150, shared)["shares"], (n, rows, shared)
    for n, rows, shared in ((2, 20, 24000), (2, 4, 192), (31, 4, 64)):
        assert not plan(1, 256, n, 1, 4, rows, n * rows, 150 if shared > 256 else 8, shared)["shares"], (n, rows, shared)
