"""Sizes at which each kernel of the 4-bit products runs: test_gpu_mx4_forms.py multiplies them, test_mx4_forms.py holds them to the
rules that choose the kernels."""

# (m, rows, k): whole tiles and ragged ones, K in several groups of scales
GEMMS = {"strip": [(16, 256, 1024), (40, 301, 1100)],
         "64x32": [(64, 4096, 1280), (33, 5003, 1100)],
         "64x64": [(512, 2048, 1280), (700, 2050, 1100)],
         "128x128": [(1024, 2560, 1280), (1000, 2501, 1100)],
         "256x256": [(4096, 4096, 2080), (3000, 5003, 2100)]}

# (m, slots, E, rows) by tile: entries, narrow or wide, weights past the caches' order (once) or not (again)
UP = {"32 narrow": (101, 2, 20, 67), "32 wide": (500, 4, 200, 131), "64 narrow": (640, 4, 64, 141), "64 wide": (640, 4, 64, 271),
      "128 narrow once": (900, 4, 64, 141), "128 narrow again": (900, 4, 16, 141), "128 wide once": (960, 4, 64, 351),
      "128 wide again": (1120, 4, 32, 461)}
DOWN = {"32 narrow": (101, 2, 20, 133), "32 wide": (500, 4, 200, 203), "64 narrow": (640, 4, 64, 301), "64 wide": (640, 4, 64, 531),
        "128 narrow once": (900, 4, 64, 301), "128 narrow again": (900, 4, 16, 301), "128 wide once": (960, 4, 64, 691),
        "128 wide again": (1120, 4, 32, 901)}

# (m, rows, k) whose rows a test sets too far apart for tiles, and would take them otherwise: of activations, of weights
FAR_X, FAR_W = (33, 5003, 300), (4096, 64, 300)
