"""Sizes that reach each kernel of the 4-bit products, for the GPU tests; the host's choice is held to them on the CPU."""

# (kernel, groups, rows, columns). The columns' tiles of 16 leave the last workgroup of 4 or 8 tiles with one, two, .. of
# them and its last tile with half; sizes on either side of each threshold.
CHOICES = [
    ("few16", 15, 15, 200),    # 4 x 15 workgroups of 64 columns, one short of the next
    ("few32", 15, 16, 200),    # 4 x 16
    ("few32", 15, 15, 968),    # 16 x 15
    ("few64", 15, 16, 968),    # 16 x 16
    ("few64", 48, 815, 904),   # 16 rows on average: 57 tiles
    ("rows", 48, 816, 904),    # 17
    ("few64", 32, 1008, 904),  # 8 x 95 / 2 workgroups of 128 columns
    ("rows", 32, 1024, 904),   # 8 x 96 / 2: just enough
    ("rows", 32, 1024, 944),   # 59 tiles
    ("rows", 32, 1100, 968),   # 61
    ("rows", 32, 1050, 1008),  # 63
    ("rows", 24, 960, 1192),   # 40 rows a group, 75 tiles, the last one half
    ("rows", 24, 961, 1216),   # 76: a workgroup's third and fourth waves without tiles
]

# Calls whose groups have more pieces of rows than the grid has workgroups for (some groups lie outside x), so that
# workgroups come back for another: (kernel, groups, rows, columns).
TRIPS = [
    ("few16", 200, 32, 24),
    ("few32", 200, 32, 136),
    ("few64", 200, 32, 520),
    ("rows", 40, 680, 1192),
]
