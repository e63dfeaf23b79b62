"""Sizes at which linear_xent, linear_xent_bwd, dropout_add and dropout_add_bwd are
compared with their definitions on a GPU (test_gpu_xent_tiles.py), chosen so that
every kernel of theirs runs, the ones of large tiles with several tiles a workgroup
and many k tiles (test_xent_routes.py has that checked on the host)."""

# rows, width, vocab, type, dw's type, ignored labels
TILES = [
    # 256 x 256 tiles, two a workgroup, 13 k tiles; dx's runs before dw's tiles
    (2041, 776, 16379, "bf16", "bf16", False),
    (2041, 776, 16379, "f16", "f32", True),
    # three a workgroup; dw's tiles before dx's runs
    (3001, 776, 16379, "bf16", "f32", True),
    (3001, 776, 16379, "f16", "f16", False),
    # more than eight runs of dx's classes, of rows off the 16-byte boundaries
    (762, 177, 39915, "bf16", "bf16", True),
    (231, 173, 88327, "f16", "f16", False),
    # many rows of few classes: dw's rows in runs, of 256 x 256 tiles
    (50416, 709, 389, "f16", "f32", False),
    (50416, 709, 389, "bf16", "bf16", True),
    (24000, 1500, 512, "bf16", "f32", False),
    (24000, 1500, 512, "bf16", "bf16", True),
    (24000, 1500, 512, "f16", "f16", False),
    (44936, 960, 137, "f16", "f16", True),
    # g in two pieces of the vocabulary
    (9000, 200, 33000, "bf16", "f32", False),
    # 128 x 128 tiles
    (300, 520, 5003, "bf16", "bf16", True),
    (300, 520, 5003, "f16", "f16", False),
    (700, 264, 3001, "f32", "f32", True),
    (100, 768, 9001, "bf16", "f32", False),
    (40, 100, 90, "bf16", "bf16", False),
    (64, 40, 129, "f16", "f32", True),
    (130, 40, 200, "f16", "f16", False),
]
# weights past the workspace's share of them (copied piece by piece), and past 2^31 bytes where they lie
PIECES = [
    (40, 1025, 131101, "bf16", "f32", False),
    (40, 1025, 131101, "f16", "f16", True),
    (40, 1025, 131101, "f32", "f32", False),
    (80, 1025, 131101, "bf16", "bf16", True),
    (80, 1025, 131101, "f16", "f32", False),
    (65, 8456, 131072, "bf16", "f32", False),
    (33, 8456, 131072, "f16", "f16", False),
]
# the kernels of few rows, of many and of few classes
FEW = [
    (16, 768, 40001, "bf16", "bf16", False), (16, 768, 5003, "bf16", "f32", True),
    (31, 520, 40001, "f16", "f16", True), (7, 130, 999, "f16", "f32", False),
    (6, 200, 40001, "f32", "f32", False), (32, 100, 777, "f32", "f32", True),
]
# rows, cols, type
DROPS = [
    (3001, 4097, "f32"), (5001, 4097, "bf16"), (5001, 4097, "f16"),  # four rows of a thread in flight, and a remainder
    (3000, 2056, "bf16"), (3000, 2056, "f16"), (1500, 2056, "f32"),  # two
    (64, 768, "bf16"), (64, 769, "f16"), (64, 770, "f32"),
]
DROP_GRADS = [
    (40000, 768, "bf16"), (40001, 769, "f16"), (40001, 770, "f32"),  # eight rows and more
    (4001, 1001, "bf16"), (3000, 1001, "f16"), (1700, 1001, "f32"),
    (100, 768, "bf16"), (100, 769, "f16"), (100, 770, "f32"),
]
