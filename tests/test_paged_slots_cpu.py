"""How the rows kernel (csrc/paged_rows.cu) deals out its tiles by slots, restated: every tile has one slot, and one only."""
import random


def rows_of_slots(start, n_seq, rows, tokens):
    """The rows that each slot's tile begins and holds; slot u belongs to the last sequence s with start[s] // tokens + s <= u."""
    out = []
    for slot in range(rows // tokens + n_seq):
        seq, hi = 0, n_seq
        while hi - seq > 1:
            mid = (seq + hi) >> 1
            if start[mid] // tokens + mid <= slot:
                seq = mid
            else:
                hi = mid
        first = start[seq]
        row0 = first + (slot - first // tokens - seq) * tokens
        end = min(start[seq + 1], rows)
        if first <= row0 < end:
            out.append(range(row0, min(row0 + tokens, end)))
    return out


def test_every_tile_has_one_slot():
    for seed in range(4000):
        rng = random.Random(seed)
        tokens, n = rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.randint(1, 12)
        start = [rng.choice([0, 0, 7, rng.randint(0, 50)])]
        for _ in range(n):
            start.append(start[-1] + rng.choice([0, 0, 1, 2, rng.randint(0, 40)]))
        rows = max(0, start[-1] + rng.choice([0, 0, 3, -2, -9]))  # fewer than the offsets say, or padding behind them
        tiles = rows_of_slots(start, n, rows, tokens)
        want = [range(r, min(r + tokens, start[s + 1], rows)) for s in range(n) for r in range(start[s], min(start[s + 1], rows), tokens)]
        assert sorted(tiles, key=lambda t: t[0]) == want
