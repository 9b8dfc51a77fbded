"""Products of 8-bit rows that between them take every kernel a product can take, each with
more steps than its loads run ahead and with tiles that end past the last row and column."""

# (gated, tile of nitro_row8_tile): [(rows, n, d), ...].  A workgroup of 16 rows is another
# kernel for up to 8 rows.  In blocks of 32: a split kernel's waves take 4 at a time; the
# kernels for many rows 4 (tiles of 64 x 64) or 2 in a step, an odd number of steps and an
# even one, the last of them ragged.
CASES = {
    (False, (16, 16, 4)): [(5, 1184, 50), (9, 1184, 17), (2072, 2912, 34)],
    (False, (16, 16, 8)): [(3, 2592, 17), (9, 2592, 33)],
    (False, (16, 32, 4)): [(1, 1184, 12295), (2, 5312, 12608), (34, 160, 8188), (9, 1184, 12431)],
    (False, (16, 32, 8)): [(1, 544, 5049), (2, 2912, 4111), (17, 2592, 2058)],
    (False, (32, 32, 4)): [(55, 160, 6230), (17, 1184, 4583), (4151, 1184, 17)],
    (False, (32, 32, 8)): [(17, 2592, 4107), (4145, 2912, 17)],
    (False, (64, 64, 1)): [(6151, 288, 101), (10963, 416, 65)],
    (False, (64, 128, 1)): [(65, 160, 17046), (139, 224, 16655), (700, 96, 16000)],
    (False, (128, 128, 1)): [(2656, 96, 5418), (19640, 160, 645), (16612, 224, 775)],
    (False, (256, 128, 1)): [(8192, 96, 8192), (3211, 160, 19647), (16455, 224, 2712)],
    (True, (16, 32, 4)): [(1, 1184, 4108), (9, 1184, 4103)],
    (True, (16, 32, 8)): [(1, 2592, 17), (9, 2592, 17)],
    (True, (32, 32, 4)): [(17, 96, 6170), (17, 1184, 4103), (8259, 2592, 17)],
    (True, (32, 32, 8)): [(17, 2912, 2079), (2071, 2592, 17)],
    (True, (64, 64, 4)): [(35, 1152, 7912), (34, 2912, 6185), (12835, 1184, 17)],
    (True, (64, 128, 1)): [(66, 160, 5650), (65, 224, 5493)],
    (True, (128, 128, 1)): [(846, 96, 8274), (19386, 160, 321), (325, 224, 19903)],
    (True, (256, 128, 1)): [(4069, 96, 7786), (2201, 160, 13683), (1163, 224, 18214)],
}

# A model's wq, wk and wv in one launch, which takes the same kernels: (rows, dim, kv_dim,
# heads, kv heads) by tile, with kv_dims that end inside a tile of 64 or 128 columns.
GROUPS = {
    (16, 16, 4): [(5, 64, 32, 2, 1), (9, 64, 64, 1, 1)],
    (16, 16, 8): [(3, 576, 192, 3, 1), (9, 576, 64, 9, 1)],
    (16, 32, 4): [(565, 192, 192, 1, 1)],
    (16, 32, 8): [(1, 1600, 1600, 8, 8), (17, 704, 704, 4, 4)],
    (32, 32, 4): [(677, 192, 192, 1, 1)],
    (32, 32, 8): [(65, 576, 576, 3, 3)],
    (64, 64, 1): [(333, 768, 768, 8, 8), (2561, 64, 32, 2, 1)],
    (64, 128, 1): [(2210, 320, 320, 2, 2)],
    (128, 128, 1): [(2580, 832, 832, 4, 4)],
    (256, 128, 1): [(2897, 1472, 1472, 8, 8)],
}


def variant(gated, rows, tile):
    """What tells one product kernel from another."""
    return gated, tile, rows <= 8 and tile[0] == 16


def blocks_of_a_step(tile):
    """Of a wave's (split kernels) or a workgroup's; a split kernel's waves share the blocks."""
    rows, cols, split = tile
    if split > 1:
        return 4 * split
    return 4 if cols == 64 else 2
