"""int8 codes of values that lie exactly between two: away from zero, whatever
the scale, on each of the ways that a row's codes are made."""
from fractions import Fraction

import numpy as np
import pytest

from test_rows_q8_gpu import rows_case

pytestmark = pytest.mark.gpu

# Scales that are no powers of two: 127 of them is a float, and so is each half.
SCALES = [49.0, 98.0 / 32, 103.0, 107.0 * 4, 161.0, 187.0 / 1024, 2047.0, 4999.0]


def tied_rows(batch, k):
    """Row b holds 127 s and the halves (j + 1/2) s of both signs, s = SCALES[b]."""
    x = np.zeros((batch, k), np.float32)
    for b in range(batch):
        s = SCALES[b % len(SCALES)]
        j = np.arange(k - 1) % 127
        x[b, 0] = 127.0 * s
        x[b, 1:] = (j + 0.5) * s * np.where(np.arange(k - 1) // 127 % 2, -1.0, 1.0)
        assert all(Fraction(float(v)) == Fraction(s) * (int(i) + Fraction(1, 2)) * (1 if v > 0 else -1)
                   for v, i in zip(x[b, 1:], j))
        assert Fraction(float(np.float32(float(x[b, 0]) / 127.0))) == Fraction(s)
    return x


@pytest.mark.parametrize("m,k,batch", [
    (70, 256, 1), (70, 1536, 1), (70, 4096, 1),      # one launch, one row
    (9000, 256, 1), (8300, 4096, 1),                 # the same, 32 weight rows a workgroup
    (70, 256, 2), (70, 768, 8), (70, 1280, 8),       # one launch, a wave a row
    (70, 256, 9), (70, 2048, 8), (70, 4096, 20), (70, 8192, 8), (300, 8208, 100), (70, 16400, 3)])  # two launches
def test_halves(gpu, xe, m, k, batch):
    rows_case(xe, gpu, m, k, batch, x=tied_rows(batch, k), want_sum=False)


@pytest.mark.parametrize("batch", [1, 8, 40])
def test_next_to_halves(gpu, xe, batch):
    """The floats beside each half: one step below is the lower code, one step
    above the higher one."""
    x = tied_rows(batch, 512)
    x[:, 1:256] = np.nextafter(x[:, 1:256], np.float32(0))
    x[:, 256:] = np.nextafter(x[:, 256:], np.copysign(np.float32(np.inf), x[:, 256:]))
    x[:, 1:] = np.clip(x[:, 1:], -x[:, :1], x[:, :1])
    rows_case(xe, gpu, 70, 512, batch, x=x, want_sum=False)
