"""How many tokens the routing entry points take, on the host: what the header
allows gets past the check of the sizes (to that of the NULL buffers), the rest
is refused."""
import pytest

import minirun_hip as M


@pytest.fixture(scope="module")
def calls():
    lib = M.load()
    return [
        lambda t, dim, k=1: lib.mr_expert_dispatch(None, M.BF16, t, dim, dim, None, k, None, dim, None),
        lambda t, dim, k=1: lib.mr_expert_combine(None, M.BF16, dim, dim, None, None, t, k, None, dim, None),
        lambda t, dim, k=1: lib.mr_expert_combine_backward(None, M.BF16, dim, dim, None, dim, None, None, t, k, 1 << 32, dim,
                                                           None, None),
    ]


@pytest.mark.parametrize("tokens,dim,fits", [
    (1 << 24, 1, True), (1 << 24, 8, True), (1 << 24, 512, True), (1 << 24, 2040, True), (1 << 24, 2041, False),
    (1 << 24, 2048, False), (1 << 23, 4080, True), (1 << 23, 4089, False), (1 << 22, 7168, True), (1 << 22, 8192, False),
    (1 << 11, 1 << 24, False), ((1 << 11) - 1, 1 << 24, True), (1, 1 << 24, True),
])
def test_tokens_and_row_widths(calls, tokens, dim, fits):
    assert fits == (tokens * max(64, -(-dim // 8)) < 1 << 32)
    for call in calls:
        status = call(tokens, dim)
        assert status == (M.INVALID_ARGUMENT if fits else M.INVALID_SHAPE), M.last_error()
        assert ("non-NULL" if fits else "one launch") in M.last_error()
