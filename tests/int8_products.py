"""Products for each kernel that mk_gemm_int8 has, with remainders of rows, columns
and k: (kernel, rows, columns, k's, whether rows lie on the 16-byte grid).  The
kernels' names are those that tests/int8_routes_check.cc prints, which
test_int8_products.py holds the list against; test_gpu_int8_products.py checks
the results."""

BF16, F16, F32 = 13, 10, 11

# a k tile and less, whole ones, the pipelines' ends, one that each loop turns over often
KS = (100, 128, 131, 250, 384, 515, 1035, 2100)

TILED = [
    ("tiled<256, 256, true", 3167, 3954, KS[2:], True),
    ("tiled<128, 128, true", 1500, 4101, KS, True),
    ("tiled<64, 128, true", 75, 8501, KS, True),
    ("tiled<64, 64, true", 201, 2101, KS, True),
    ("tiled<64, 32, true", 201, 1901, KS, True),
    ("tiled<128, 128, false", 1500, 4101, KS, False),
    ("tiled<64, 64, false", 201, 2101, KS, False),
]

# At most 64 rows: columns a wave / 16, rows / 16, waves
FEW = [
    ("rows<1, 1, 8>", 7, 2305, (770,), True),
    ("rows<1, 1, 16>", 13, 4101, (4100,), True),
    ("rows<1, 2, 8>", 27, 8101, (1000,), True),
    ("rows<1, 2, 16>", 27, 4101, (2085,), True),
    ("rows<1, 4, 8>", 51, 4101, (2085,), False),
    ("rows<2, 1, 8>", 11, 8201, (1035,), True),
    ("rows<2, 2, 8>", 29, 9001, (1035,), False),
    ("rows<2, 4, 8>", 60, 9001, (4097,), False),
    ("rows<4, 1, 8>", 11, 12301, (2100,), True),
    ("rows<4, 2, 8>", 30, 12301, (2101,), False),
    ("rows<4, 4, 8>", 35, 12301, (2101,), False),
]

# 131071 deep, with a pitch of 131072
DEEP = [
    ("tiled<256, 256, true", 4000, 4001),
    ("tiled<128, 128, true", 1500, 2101),
    ("tiled<64, 128, true", 75, 8501),
    ("tiled<64, 64, true", 201, 2101),
    ("tiled<64, 32, true", 201, 1901),
]

# C of 192 MiB and more, its rows on the 128-byte lines: past the caches
STREAMED = [
    ("tiled<256, 256, true", BF16, 6669, 15440, 250),
    ("tiled<256, 256, true", F32, 8871, 6860, 515),
    ("tiled<128, 128, true", F32, 20502, 2926, 250),
    ("tiled<128, 128, false", BF16, 6669, 15440, 251),
]


def pitch(k, on_grid):
    """Elements from one operand row to the next."""
    return (k + 31) // 16 * 16 if on_grid else k | 1


def lines(columns):
    """Columns of C up to a whole number of 128-byte lines, of either type."""
    return (columns + 63) // 64 * 64
