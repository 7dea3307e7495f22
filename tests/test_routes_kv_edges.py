"""The rule of test_routes_kv.py at its edges, on the CPU: the forms that
tests/test_gpu_kv_edges.py names are those its sizes take, and calls of any size have a
bounded number of parts and workspace."""
import random

import pytest

from test_gpu_kv_edges import FORMS
from test_routes_kv import route  # noqa: F401 (a fixture)

WANT = {"one": (0, 1), "one in parts": (0, 2), "few": (0, 1), "few in parts": (0, 2), "many": (1, 1), "many in parts": (1, 2),
        "many rows joined": (1, 2)}


@pytest.mark.parametrize("dim", [64, 96, 128])
def test_forms(route, dim):  # noqa: F811
    for name, (lens, queries, heads, kv_heads) in FORMS.items():
        tokens = None if queries is None else sum(queries)
        per = None if tokens is None else tokens // len(lens)
        assert tokens is None or per * len(lens) == tokens
        got = route(per, 32 * -(-max(lens) // 32), kv_heads, heads // kv_heads, dim, len(lens))
        assert (got[0], min(got[2], 2)) == WANT[name], (name, got)
        rows = (tokens or len(lens)) * heads
        assert (got[2] <= 32 and rows >= 2048) == (name in ("many", "many rows joined")) or got[2] == 1, name


def bounds(got, queries, kv_heads, group, dim, batch, cus=256):
    """(workgroups, bytes of workspace) of a call of `queries` for each sequence."""
    _, rows, splits, _ = got
    tokens = batch * (queries or 1)
    tiles = batch * -(-group // rows) if queries is None else -(-tokens * group // rows) + batch
    return tiles * kv_heads * splits, 0 if splits == 1 else tokens * kv_heads * group * splits * (dim + 2) * 4


def test_large_calls_have_few_parts(route):  # noqa: F811
    # (sequences, queries, key heads, group, keys): parts of 1536 keys would be 86, 683, 86 and 683
    for batch, queries, kv_heads, group, keys in ((256, None, 8, 8, 131072), (512, None, 8, 8, 2 ** 20),
                                                  (1024, 8, 8, 8, 131072), (1024, None, 32, 1, 2 ** 20)):
        got = route(queries, keys, kv_heads, group, 128, batch)
        grid, workspace = bounds(got, queries, kv_heads, group, 128, batch)
        assert got[2] <= 4 and workspace <= 2 ** 27 and grid <= 2 ** 15, (batch, got, workspace)


def test_parts_and_workspace_are_bounded(route):  # noqa: F811
    rng = random.Random(7)
    log = lambda hi: int(2 ** rng.uniform(0, hi))
    for _ in range(4000):
        queries, keys, batch = rng.choice([None, None, log(13)]), log(30), log(14)
        kv_heads, group, dim, cus = log(6), log(6), 32 * rng.randint(1, 8), rng.choice([64, 256, 304])
        if batch * (queries or 1) * kv_heads * group > 2 ** 30:
            continue
        got = route(queries, keys, kv_heads, group, dim, batch, rng.choice([0, 0, log(20)]), cus)
        grid, workspace = bounds(got, queries, kv_heads, group, dim, batch)
        # 32 workgroups a CU, as many again for sequences' last tiles; 64 rows of 256 dims at most in each
        assert got[2] == 1 or (grid <= 2 * 32 * cus and workspace <= 32 * cus * 64 * 258 * 4), (got, grid, workspace)
