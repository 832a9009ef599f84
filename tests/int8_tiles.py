"""Sizes at which the 8-bit projections run in each of their tiles: (rows and columns of the tile, SwiGLU, M, N, K).  Every
tile with several stages, so that its ring turns, with rows, columns and K that end within a tile and a group, and with whole ones."""

TILES = [
    (256, 256, False, 4000, 4096, 256), (256, 256, False, 3900, 4083, 600),
    (256, 256, True, 3000, 2051, 256), (256, 256, True, 3000, 2056, 1400),
    (192, 256, False, 2100, 2051, 384), (192, 256, False, 3000, 2056, 1400),
    (192, 256, True, 2100, 2051, 384), (192, 256, True, 2500, 2048, 600),
    (128, 128, False, 1500, 2100, 600), (128, 128, False, 20000, 70, 384),
    (128, 128, True, 1500, 1000, 384), (128, 128, True, 1500, 2099, 1400),
    (64, 128, False, 700, 2100, 384), (64, 128, False, 1000, 1030, 600),
    (64, 128, True, 1100, 300, 640), (64, 128, True, 20000, 71, 384),
    (64, 64, False, 1100, 300, 600), (64, 64, False, 2000, 69, 384),
    (64, 64, True, 1030, 200, 6100), (64, 64, True, 2000, 99, 6144),
]
