"""Shapes that reach each kernel of the 8-bit linears on a card of 256 compute units: (M, K, N, rows of b a scale covers,
8-bit pipe) and what frx_policy.hpp's rules make of them: the tile, whether K is split, and for few tokens the row tiles of a
workgroup. test_fp8_plan holds them to the rules on the CPU, the GPU tests run them.

Unless a kernel takes only short sums, every one has five whole blocks of 128 columns or more to a slice, so that the stages
of its pipeline are filled again while the products run, and ends in a part of a block."""

FEW, T128, RING256, RING192, RING128, T64 = 0, 1, 2, 3, 4, 5  # frx_policy.hpp's FP8_T_*

# name: (M, K, N, b_rows, pipe8), tile, split, row tiles of a workgroup
DENSE = {
    "few-1": ((1, 4112, 300, 128, 0), FEW, False, 1),
    "few-2": ((16, 4112, 8000, 128, 0), FEW, False, 2),
    "few-3": ((7, 4112, 12200, 128, 0), FEW, False, 3),
    "few-4": ((3, 4112, 16100, 128, 0), FEW, False, 4),
    "few32-1": ((20, 4112, 300, 128, 0), FEW, False, 1),
    "few32-2": ((32, 4112, 8000, 128, 0), FEW, False, 2),
    "few32-3": ((17, 2064, 12200, 128, 0), FEW, False, 3),
    "few32-4": ((31, 2064, 16100, 128, 0), FEW, False, 4),
    "few64-1": ((40, 4112, 300, 128, 0), FEW, False, 1),
    "few64-2": ((64, 4112, 8000, 128, 0), FEW, False, 2),
    "groups-of-64": ((200, 784, 1000, 128, 0), FEW, False, 1),
    "few-rows-1": ((5, 4112, 300, 1, 0), FEW, False, 1),
    "few-rows-3": ((7, 4112, 12200, 1, 0), FEW, False, 3),
    "few64-rows-2": ((64, 4112, 8000, 1, 0), FEW, False, 2),
    "ring128": ((190, 784, 3300, 128, 0), RING128, False, 0),
    "ring128-split": ((300, 4112, 1100, 128, 0), RING128, True, 0),
    "ring192": ((900, 784, 8200, 128, 0), RING192, False, 0),
    "ring192-split": ((129, 2832, 11000, 128, 0), RING192, True, 0),
    "128": ((16500, 784, 260, 128, 0), T128, False, 0),
    "128-split": ((2900, 2064, 260, 128, 0), T128, True, 0),
    "128-rows": ((257, 784, 3300, 1, 0), T128, False, 0),
    "128-rows-split": ((300, 4112, 1100, 1, 0), T128, True, 0),
    "pipe-ring128": ((65, 784, 4100, 128, 1), RING128, False, 0),
    "pipe-ring128-split": ((300, 4112, 1100, 128, 1), RING128, True, 0),
    "pipe-ring192": ((900, 784, 8200, 128, 1), RING192, False, 0),
    "pipe-ring192-split": ((129, 2832, 11000, 128, 1), RING192, True, 0),
    "pipe-ring256": ((1000, 784, 11000, 128, 1), RING256, False, 0),
    "pipe-ring256-split": ((200, 8208, 11000, 128, 1), RING256, True, 0),
    "pipe-128": ((16500, 784, 260, 128, 1), T128, False, 0),
    "pipe-128-split": ((3300, 8208, 260, 128, 1), T128, True, 0),
    "pipe-ring128-rows": ((65, 784, 4100, 1, 1), RING128, False, 0),
    "pipe-ring128-rows-split": ((300, 4112, 1100, 1, 1), RING128, True, 0),
    "pipe-128-rows": ((16500, 784, 260, 1, 1), T128, False, 0),
    "pipe-128-rows-split": ((3300, 8208, 260, 1, 1), T128, True, 0),
}

# name: (rows of each expert, rows behind them, K, N, 8-bit pipe), tile
GROUPED = {
    "few": (([1, 0, 3, 2], 9, 4112, 300, 0), FEW),
    "64": (([60, 0, 130, 5], 11, 784, 515, 0), T64),
    "64-long": (([700, 0, 1100, 1], 3, 784, 515, 0), T64),
    "pipe-ring128": (([300, 0, 700, 260], 5, 784, 515, 1), RING128),
    "pipe-ring256": (([1500, 701, 1300, 0], 7, 784, 3001, 1), RING256),
}
