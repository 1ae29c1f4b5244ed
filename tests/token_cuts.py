"""How gated_recurrence cuts histories into pieces: the rule of recurrence.hip's split_of for histories of more
than 128 steps, said again, and the shapes that reach every way of walking the pieces."""

# (batch, steps, channels)
CUT_SHAPES = [(100, 1100, 5),     # two pieces of several tiles each
              (8, 4200, 200),     # the same with several slabs of channels
              (1, 8500, 3),       # more pieces than a workgroup scans at once, one tile each
              (1, 70000, 2)]      # both: several tiles a piece, several rounds over the pieces

TILE, SLAB = {"forward": 256, "backward": 128}, 64
AT_ONCE = {"forward": 32, "backward": 16}     # pieces that a workgroup scans in one round


def cut(b, t, d, direction):
    """(tiles, tiles per piece, pieces)"""
    assert t > 128
    tiles, groups = -(-t // TILE[direction]), b * -(-d // SLAB)
    pieces = 1 if groups > 128 or tiles <= 3 else min(256 // groups, tiles)
    per_piece = -(-tiles // pieces)
    return tiles, per_piece, -(-tiles // per_piece)
