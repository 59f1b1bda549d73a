"""The sum of a group of 32 e4m3 codes, held as two fp16 numbers: the nearest one and what that leaves.

gsp_matmul_batch_fp8 multiplies the groups' minimums by these.  Codes are whole multiples of 2^-9 up to 448, so a sum is
one of 2^24 numbers: this takes them all."""
import numpy as np


def test_two_halves_hold_every_sum():
    most = 32 * 448 * 512
    assert most < 1 << 23  # and every partial sum is exact in fp32
    for lo in range(0, most + 1, 1 << 20):
        total = np.arange(lo, min(lo + (1 << 20), most + 1)).astype(np.float32) * np.float32(2.0 ** -9)
        first = total.astype(np.float16)
        rest = (total - first.astype(np.float32)).astype(np.float16)
        assert np.all(np.isfinite(first)) and np.array_equal(first.astype(np.float64) + rest, total.astype(np.float64))
