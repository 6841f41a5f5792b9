"""How calls are cut whose sequences share their first pages (kv8_device.h), as the host decides it."""

import ctypes as C
import itertools

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
