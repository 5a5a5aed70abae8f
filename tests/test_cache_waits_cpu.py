"""The waits of the cache attention's tcgen05 kernels (csrc/cache_attn_tile.cu), as models that run on the CPU: a circle of waits ends on a GPU only when
the bounded waits run out, so it is looked for here.

1. The ring of piece notes.  The scout tells pieces and their units, converters finish a unit when the next one is told, softmax warps finish a piece
   when its units are finished, and a piece's note is told again when the piece PIECES before it is finished.
2. The row buffers of the weights kernel.  A waiter sees the parity of a barrier's phase only."""

import random

import pytest

PIECES, UNITS = 4, 8                    # notes that are kept


def finishes(counts):
    """True if all pieces (of counts[i] units) are finished.  Every step only enables others, so any order of steps ends at the same place.  (Pieces of more units than
    notes of units are kept are like longer ones.)"""
    counts = [min(count, UNITS + 3) for count in counts]
    units = sum(counts)
    told_pieces = told_units = converted = finished = 0
    end = [sum(counts[:i + 1]) for i in range(len(counts))]          # units before the end of piece i
    while True:
        before = (told_pieces, told_units, converted, finished)
        # the scout: all units of the pieces told so far, then the next piece (number len(counts): there is none any more), at last the unit that says so
        known = units + 1 if told_pieces > len(counts) else end[told_pieces - 1] if told_pieces else 0
        if told_units < known:
            if told_units < UNITS or converted > told_units - UNITS + 3:
                told_units += 1
        elif told_pieces <= len(counts) and (told_pieces < PIECES or finished > told_pieces - PIECES):
            told_pieces += 1
        if converted < units and told_units > converted + 1:         # its own note and the next one
            converted += 1
        if finished < len(counts) and told_pieces > finished and converted >= end[finished]:
            finished += 1
        if (told_pieces, told_units, converted, finished) == before:
            return finished == len(counts) and told_units == units + 1


def pieces(lens, new, heads, group, rows, blocks, extra, most, leave_out):
    """Units of the pieces of every block.  leave_out: tiles of rows that see nothing are no items."""
    items = []                                                       # (cost, units, units that some row sees)
    for length, n in zip(lens, new):
        units = -(-length // 128)
        first = max(n - length, 0) * group // rows if leave_out else 0
        for _ in range(heads if units else 0):
            for tile in range(first, -(-n * group // rows)):
                last = min(n - 1, (tile * rows + rows - 1) // group)
                items.append((units + extra, units, -(-max(length - n + last + 1, 0) // 128)))
    total = sum(cost for cost, _, _ in items)
    ranges = min(blocks, total)
    for i in range(ranges):
        lo, hi, at, counts = total * i // ranges, total * (i + 1) // ranges, 0, []
        for cost, units, seen in items:
            a, b = max(lo - at, 0), min(hi - at, cost)
            at += cost
            while a < b:
                stop = min(b, max(a, extra) + most)
                if stop - extra >= seen:
                    stop = b
                if stop > extra:
                    counts.append(max(min(seen, stop - extra) - max(a - extra, 0), 0))
                a = stop
        yield counts


def test_the_ring_stands_still_behind_four_pieces_without_units():
    assert finishes([]) and finishes([0]) and finishes([3, 1, 1, 1, 1, 1, 20, 1]) and finishes([0, 1, 1, 1, 1, 1])
    assert finishes([2, 0, 0, 1, 1]) and not finishes([2, 0, 0, 0, 1]) and not finishes([1, 0, 0, 0, 0, 0])


def test_no_division_of_the_work_has_them():
    """Random calls, most with more queries than tokens; with the empty tiles among the items many of them stood still."""
    rng, stood = random.Random(1), 0
    for _ in range(300):
        B, group, heads, rows = rng.randint(1, 4), rng.choice((1, 2, 4, 7)), rng.randint(1, 3), rng.choice((128, 256))
        T = rng.randint(33, 1000)
        lens = [rng.choice((0, rng.randint(0, 200), rng.randint(0, 3 * T), rng.randint(0, 40000))) for _ in range(B)]
        new = [rng.choice((T, rng.randint(0, T))) for _ in range(B)]
        for leave_out in (True, False):
            whole = list(pieces(lens, new, heads, group, rows, rng.choice((1, 4, 148)), 4, rng.choice((2, 128, 256)), leave_out))
            fine = [finishes(counts) for counts in whole]
            if leave_out:
                assert all(fine), (lens, new, heads, group, rows)
                assert all(0 not in counts[1:] for counts in whole)
            stood += not all(fine)
    assert stood > 20


# ------------------------------------------------------------------------------------------------------- rows of the weights kernel
def can_hang(tiles, own_barrier):
    """Whether some order of steps leaves the loader waiting for good.  The loader posts tile q's rows when the tile four before has been summed; the
    groups sum even and odd tiles.  Its wait reads a parity: `own_barrier` = that of the buffer, else that of the group, two phases back."""
    seen, todo = set(), [(0, 0, 0)]                                  # rows posted, tiles summed by the even and by the odd group
    while todo:
        posted, even, odd = state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        summed, steps = (even, odd), []
        if posted < tiles:
            free = True
            if posted >= 4:
                if own_barrier:
                    done = sum(1 for q in range(posted % 4, tiles, 4) if q // 2 < summed[q % 2])
                    phase = posted // 4 - 1
                else:
                    done, phase = summed[posted % 2], posted // 2 - 2
                free = done > phase and (done - phase) % 2 == 1      # the barrier is in phase `done`: its parity differs from that of `phase`
            if free:
                steps.append((posted + 1, even, odd))
        if 2 * even < posted:
            steps.append((posted, even + 1, odd))
        if 2 * odd + 1 < posted:
            steps.append((posted, even, odd + 1))
        if not steps and (posted, even, odd) != (tiles, (tiles + 1) // 2, tiles // 2):
            return True
        todo += steps
    return False


@pytest.mark.parametrize("tiles", [1, 4, 5, 8, 17])
def test_rows_are_posted_for_every_tile(tiles):
    assert not can_hang(tiles, True)
    assert can_hang(tiles, False) == (tiles > 4)
