"""The many-rows kernel's work split, replayed on the host: its pieces cover all work once, and
the shapes that the GPU tests of pieces use have the transitions that they are about."""

import pytest

import paged_split as S
from test_paged_pieces_gpu import SHAPES


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_pieces_cover_every_step_once(name):
    queries, lens, hq, h, _ = SHAPES[name]
    most, room = max(queries), max(lens)
    got = {}
    for mine in S.pieces(queries, lens, hq, h, most, room):
        for r, head, tile, steps, two in mine:
            got[r, head, tile] = got.get((r, head, tile), 0) + steps
            assert two == (queries[r] * (hq // h) - 256 * tile > 128)
    want = {}
    for r, (n, length) in enumerate(zip(queries, lens)):
        rows = n * (hq // h)
        for tile in range(-(-rows // 256)):
            limit = length - n + (min(rows, 256 * tile + 256) - 1) // (hq // h) + 1
            want.update({(r, head, tile): -(-max(0, limit) // 128) for head in range(h)})
    assert got == want


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_shapes_skip_a_ring_of_steps(name):
    """Four steps and more of one-tile pieces in front of a two-tile piece: a ring's round, which
    a wait by parity alone cannot tell from none."""
    queries, lens, hq, h, _ = SHAPES[name]
    assert max(S.skipped(queries, lens, hq, h, max(queries), max(lens))) >= 4
