"""The forms that tests/test_gpu_kv_edges.py names are those its sizes take (on the CPU)."""
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
