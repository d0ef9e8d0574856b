"""The waits of the 8-bit canvas kernel at head_dim 256, on a model of its barriers: how a softmax warp learns that a tile's scores
are there.

K units go through a ring of three stages, one unit of a cached tile, two of a canvas tile; a unit that has been used completes a
phase of its stage's barrier, in order.  The scores of a canvas tile also complete a phase of one of two barriers, by turns.  The
issuing warp may be one tile ahead of a softmax warp and no more: scores of tile n + 2 go where that warp's weights of tile n lie.
A wait for a parity is over while the barrier's phase has the other one, so a warp that looks late must not find a second phase."""
import pytest

STAGES = 3


def over(phases, parity):
    return phases % 2 != parity


def units(n, n_cached):
    return [n] if n < n_cached else [2 * n - n_cached, 2 * n - n_cached + 1]


def waits(n, n_cached):
    """What the warp waits for at tile n: (barrier, parity) in order."""
    if n < n_cached:
        return [(("stage", n % STAGES), n // STAGES % 2)]
    x = n - n_cached
    return [(("scores", x % 2), x // 2 % 2)]


def phases(barrier, used, n_cached):
    """Completed phases of a barrier when the first `used` units have been."""
    kind, i = barrier
    if kind == "stage":
        return sum(u % STAGES == i for u in range(used))
    return sum(2 * x + 1 + n_cached < used for x in range(i, 64, 2))


@pytest.mark.parametrize("n_cached", range(8))
@pytest.mark.parametrize("n_canvas", range(5))
def test_a_late_warp_still_finds_its_phase(n_cached, n_canvas):
    for n in range(n_cached + n_canvas):
        first, last = units(n, n_cached)[0], units(n, n_cached)[-1]
        ahead = units(n + 1, n_cached)[-1] if n + 1 < n_cached + n_canvas else last
        for used in range(first, ahead + 2):           # the warp has seen the tile before; one tile more may be done
            got = all(over(phases(b, used, n_cached), parity) for b, parity in waits(n, n_cached))
            assert got == (used > last), (n, used)


def test_the_units_of_canvas_tiles_would_not_do():
    """Waiting for both units of a canvas tile: the fourth unit from the first one is in the first one's stage."""
    n_cached, n = 0, 0
    both = [(("stage", u % STAGES), u // STAGES % 2) for u in units(n, n_cached)]
    assert not all(over(phases(b, units(n + 1, n_cached)[-1] + 1, n_cached), parity) for b, parity in both)
