"""The many-rows kernel's work split, step by step on the host: which pieces each CTA takes."""

ROWS, TILE, OVER, LEAST, SMS = 256, 128, 2, 2, 148


def pieces(queries, lens, q_heads, heads, most, room):
    """Per CTA the list of (sequence, head, tile, steps, two) in order: ``two`` says whether the
    piece has more than 128 query rows.  ``queries`` / ``lens``: query rows and cached tokens of
    each sequence; ``most``: the call's max_query_len; ``room``: tokens that a table row has
    room for."""
    group = q_heads // heads
    unit = TILE * group

    def work(r):
        tiles = -(-queries[r] * group // ROWS)
        first = group * (OVER * TILE + max(lens[r] - queries[r], 0) + 1) + ROWS - 1
        return tiles, first

    def before(first, t):
        return t * first + ROWS * (t * (t - 1) // 2)

    items = []  # (begin, cost, r, h, tile)
    at = 0
    for r in range(len(lens)):
        tiles, first = work(r)
        for h in range(heads):
            for t in range(tiles):
                items.append((at + before(first, t), first + ROWS * t, r, h, t))
            at += before(first, tiles)
    total = at
    tiles = -(-most * group // ROWS)
    grid = min(SMS, max(1, len(lens) * heads * tiles * (-(-room // TILE) + OVER + 1)))
    least = LEAST * unit
    used = min(grid, -(-total // least))
    out = []
    i = 0
    for b in range(used):
        pos, end, mine = total * b // used, total * (b + 1) // used, []
        while i > 0 and items[i][0] > pos:
            i -= 1
        while items[i][0] + items[i][1] <= pos:
            i += 1
        while pos < end:
            begin, cost, r, h, t = items[i]
            nrows = queries[r] * group
            last = min(nrows, (t + 1) * ROWS) - 1
            limit = max(0, lens[r] - queries[r] + last // group + 1)
            steps = max(1, -(-limit // TILE))
            body, to = begin + OVER * unit, min(end, begin + cost)

            def step(x):
                return steps if x >= begin + cost else min(max(0, x - body) // unit, steps)
            u0, u1 = step(pos), step(to)
            if u0 < u1:
                stop = min(limit, u1 * TILE)
                mine.append((r, h, t, -(-max(0, stop - u0 * TILE) // TILE),
                             nrows - t * ROWS > 128))
            pos = to
            i += to == begin + cost
        out.append(mine)
    return out


def skipped(*call):
    """Steps of one-tile pieces in front of a two-tile piece in the same CTA, one number for each
    such place."""
    found = []
    for mine in pieces(*call):
        run = 0
        for _, _, _, steps, two in mine:
            if two and run:
                found.append(run)
            run = 0 if two else run + steps
    return found
