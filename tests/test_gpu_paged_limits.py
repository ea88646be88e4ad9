"""The paged cache's attention where its numbers, lengths and grids reach their
limits, against the float64 definitions (paged_oracle)."""
import numpy as np
import pytest

from tests import paged_oracle as po

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llmoxide_amd as lmx  # noqa: E402
from tests.test_gpu_paged import check_attention, gpu, on_gpu, rows, say  # noqa: E402


# ------------------------------------------------------------ 8-bit V scales --
def quiet_and_loud(c, b, quiet, loud):
    """Sequence b's V rows: zeros where ``quiet``, a scale of 2^loud elsewhere."""
    for p in range(c.ctx[b]):
        pg, s = c.place(b, p)
        c.v_scale[pg, 0, s] = 0 if quiet(p) else np.float32(2.0 ** loud)
        if quiet(p):
            c.v[pg, 0, :, s] = 0


@pytest.mark.parametrize("loud", [20, 47, 100])
@pytest.mark.parametrize("quiet", ["first half", "every second", "all but one", "last half"])
@pytest.mark.parametrize("new", [[1, 3], [60, 130]])
@pytest.mark.parametrize("hd", [64, 512])
def test_zero_values_keep_their_share_beside_loud_ones(hd, new, quiet, loud):
    """Rows of zeros (scale 0) beside values up to 2^107: each key has its share of the
    softmax's sum, whichever comes first, in one walk and where several join."""
    say("zero values", hd, new, quiet, loud)
    c = po.PagedCase(60, new=new, ctx=[900, 140], page=16, kv=1, hd=hd, store="i8")
    for b in range(2):
        n = c.ctx[b]
        at = {"first half": lambda p: p < n // 2, "every second": lambda p: p % 2 == 0,
              "all but one": lambda p: p != 5, "last half": lambda p: p >= n // 2}[quiet]
        quiet_and_loud(c, b, at, loud)
    check_attention(c, 2, q16=False)
    check_attention(c, 2, q16=False, scale=0.0)  # a plain mean


def test_zero_values_of_half_precision_rows():
    for new in ([1, 3], [60, 130]):
        c = po.PagedCase(61, new=new, ctx=[900, 140], page=16, kv=1, hd=128, store="i8")
        for b in range(2):
            quiet_and_loud(c, b, lambda p: p % 3 != 0, 8)
        check_attention(c, 2, q16=True)


@pytest.mark.parametrize("new", [[2], [150]])
def test_small_values_beside_loud_ones(new):
    """Scales from 2^-80 to 2^100 along the keys, the loud ones at scores far below the
    others': a weight follows score and scale, the sum the score alone."""
    c = po.PagedCase(62, new=new, ctx=[700], page=16, kv=1, hd=64, store="i8")
    for p in range(700):
        pg, s = c.place(0, p)
        c.v_scale[pg, 0, s] = np.float32(2.0 ** (100 if p % 7 == 3 else -80 + p // 8))
        c.k_scale[pg, 0, s] *= np.float32(12 if p % 7 == 3 else 0.5)
    check_attention(c, 2, q16=False)
