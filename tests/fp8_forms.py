"""Sizes of gsp_matmul_batch_fp8 for each of its forms on 256 CUs, with what each is meant to reach.

(in_dim, out_dim, batch, form, ranges of K, units of 256 in a range).  tests/test_matmul_fp8_plan.py holds the planner
to them, so that a change of its model cannot leave a form without its tests.
"""
CUS = 256

TILES = [
    (1536, 2105, 1939, "wide", 1, 6),
    (3584, 1797, 1371, "wide", 2, 7),     # the second range starts at an odd unit
    (3328, 1554, 1287, "wide", 3, 5),     # and the last is shorter
    (2816, 1666, 1194, "wide", 3, 4),
    (6400, 787, 1176, "wide", 5, 5),
    (1344, 2089, 1963, "wide", 1, 6),     # K ends inside a unit
    (3136, 1154, 1608, "wide", 3, 5),
    (3392, 1798, 1303, "wide", 2, 7),
    (768, 778, 1263, "tile64", 1, 3),
    (3328, 1031, 580, "tile64", 2, 7),
    (2816, 417, 588, "tile64", 4, 3),
    (3200, 522, 1102, "tile64", 2, 7),
    (512, 17001, 50, "tile64", 1, 2),     # up to 64 rows: outputs that repay the conversion
    (768, 383, 66, "tile32", 1, 3),
    (1792, 334, 200, "tile32", 3, 3),
    (1664, 311, 152, "tile32", 3, 3),
    (8192, 201, 90, "tile32", 16, 2),
]
STREAMS = [
    (1024, 100, 1, "stream", 1, 4), (1024, 4501, 3, "stream", 1, 4), (768, 70, 7, "stream", 1, 3),
    (768, 5001, 8, "stream", 1, 3), (2816, 90, 15, "stream", 1, 11), (512, 5003, 12, "stream", 1, 2),
    (1280, 601, 40, "stream", 1, 5), (768, 4001, 37, "stream", 1, 3), (512, 16403, 20, "stream", 1, 2),
    (1024, 5001, 40, "stream", 1, 4),
]
# Weights of whole units at 16-byte addresses only.
STREAM32 = [(256, 4500, 32, "stream32", 1, 1), (256, 8001, 64, "stream32", 1, 1)]
# Ranges of K in a batch that goes piece by piece: 896 rows of converted activations at 2048 units.
PIECES = [(524096, 250, 1600, "wide", 16, 128), (524288, 300, 1100, "wide", 14, 147)]
