"""Shapes of the 4-bit linears and of the expert layer for a few tokens, each with the kernel that it is meant for on 256
compute units: test_fp4_plan.py holds them against the rules, the GPU tests run them."""

FEW, T64, T64X128, T128X192, T128X256, T192X256, T256 = range(7)

# steps of 256 columns: 1 to 5, the last of them cut short
KS = (32, 352, 736, 992, 1120)
# tokens, weight rows: no multiple of a tile's sides
TILES = {T64: (47, 90), T64X128: (195, 12300), T128X192: (325, 10925), T128X256: (390, 12310), T192X256: (645, 11915),
         T256: (1025, 10760)}
# M, K, N, tile: K split
SPLIT = [(52, 4448, 24, T64), (70, 8352, 3907, T64X128)]
# M, N, 16-row tiles of a workgroup; K is of one slice of 128 a wave, of many, of fewer than there are waves
ROWS16 = {(1, 40): 1, (5, 16300): 4, (16, 6000): 2, (16, 8300): 3, (17, 4000): 1, (32, 5000): 2, (31, 9000): 3, (20, 13000): 4}
ROWS16_K = (32, 160, 1056, 4128, 8480)

# experts' rows [sizes], rows behind the last one, K, N, tile
GROUPED = {
    "64": ([1, 0, 40, 64, 65, 3], 0, 992, 100, T64),
    "64-one-step": ([3, 0, 5], 4, 32, 90, T64),
    "64x128": ([1, 0, 2, 1, 1, 0, 1, 3, 1, 1], 2, 736, 5010, T64X128),
    "128x256": ([60, 1, 0, 33, 129, 30, 40, 2, 31, 50], 8, 352, 5900, T128X256),
    # several tiles for a workgroup, of one step to three
    "64-turns-1": ([7 * i % 10 for i in range(40)], 5, 32, 2200, T64),
    "64-turns-2": ([7 * i % 10 for i in range(40)], 0, 480, 2190, T64),
    "64-turns-3": ([7 * i % 10 for i in range(40)], 5, 544, 2210, T64),
    "64x128-turns-1": ([1 + 3 * i % 9 for i in range(64)], 3, 32, 1900, T64X128),
    "64x128-turns-3": ([1 + 3 * i % 9 for i in range(64)], 0, 608, 1890, T64X128),
    "256": ([140, 0, 257, 1, 256, 90, 255, 100, 200, 140], 9, 800, 5900, T256),
}

# experts' rows (whole blocks of 128), rows behind, N, K, tile of the weights' gradients
GRADS = {
    "64x128": ([128, 0, 256, 512], 128, 90, 71, T64X128),
    "64x128-one": ([896], 0, 330, 129, T64X128),
    "64x128-none": ([0, 0], 256, 40, 33, T64X128),
    "128x256": ([256, 128, 0, 512], 0, 2050, 1990, T128X256),
    "256": ([128, 0, 384, 256], 128, 1500, 2050, T256),
}

# T, H, I, E, top_k
LAYERS = [(8, 2080, 96, 4, 2), (33, 2080, 96, 4, 2), (64, 96, 128, 4, 2), (33, 160, 96, 4, 2), (9, 4128, 64, 4, 2),
          (3, 8320, 32, 2, 1), (8, 64, 2080, 4, 2), (16, 64, 2080, 4, 2), (33, 64, 2080, 4, 2), (8, 64, 4064, 16, 2),
          (16, 96, 4064, 4, 2), (16, 32, 5632, 4, 2), (1, 2048, 96, 8, 2), (2, 2080, 2080, 4, 2), (64, 32, 3104, 64, 64), (64, 4128, 32, 64, 64)]
# (steps, column tiles, slices > 1) of gate and up; (steps, column tiles) of down
GATE_UP = {(2, 1, False), (2, 2, False), (2, 3, False), (4, 1, False), (4, 2, False), (4, 1, True)}
DOWN = {(2, 1), (2, 2), (2, 3), (3, 1), (3, 2), (3, 3), (4, 1)}
