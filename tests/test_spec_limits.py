"""Steps with drafted tokens on the CPU: calls that must not be made."""
import ctypes

import pytest

from llmoxide_amd import paged, spec
from tests.test_paged import FAKE, S, batch, pool
from tests.test_spec import BIG


# ------------------------------------------------------------------ keeping --
def layers(n, **kw):
    """8-bit pools whose arrays lie far apart; ``kw``: "2.k_scale": address, of the third."""
    out = []
    for i in range(n):
        d = {x: FAKE + (4 * i + j + 1) * BIG for j, x in enumerate(("k", "v", "k_scale", "v_scale"))}
        d.update({k.split(".")[1]: v for k, v in kw.items() if k.split(".")[0] == str(i)})
        out.append(pool(store=paged.STORE_I8, **d))
    return out


def keep(pools, path=FAKE + 2):
    """Behind the arrays of other pools the path's alignment refuses the call, so that
    none reaches the GPU."""
    at = (ctypes.c_void_p * len(pools))(*map(ctypes.addressof, pools))
    return spec.spec_lib().lmxs_keep(at, len(pools), ctypes.byref(batch()), path, 8, FAKE, None)


def test_layers_that_share_scales_are_refused():
    """The default pool has 8 pages of 2 heads and 16 positions of 128 dims: scales of 1024
    bytes, K and V of 32768."""
    a = layers(3)
    scales = [(i, w) for i in range(3) for w in ("k_scale", "v_scale")]
    for i, w in scales:
        for j, x in scales:
            if i == j:
                continue
            for off in (0, 16, 1008, -1008):
                assert keep(layers(3, **{f"{i}.{w}": getattr(a[j], x) + off})) == S.E_SHAPE, (i, w, j, x, off)
            assert keep(layers(3, **{f"{i}.{w}": getattr(a[j], x) + 1024})) == S.E_ALIGN
        # a scale in another layer's K or V
        for x in ("k", "v"):
            j = (i + 1) % 3
            assert keep(layers(3, **{f"{i}.{w}": getattr(a[j], x) + 32752})) == S.E_SHAPE
            assert keep(layers(3, **{f"{i}.{w}": getattr(a[j], x) - 1008})) == S.E_SHAPE
            assert keep(layers(3, **{f"{i}.{w}": getattr(a[j], x) + 32768})) == S.E_ALIGN


def test_a_layer_whose_arrays_overlap_is_refused():
    a = layers(2)
    for kw in ({"1.v_scale": a[1].k_scale}, {"0.v": a[0].k + 16}, {"0.k_scale": a[0].v + 32752}):
        assert keep(layers(2, **kw), path=FAKE) == S.E_SHAPE


@pytest.mark.parametrize("n", [1, 2, 70, 1024])
def test_the_most_layers_are_looked_through(n):
    p = layers(n)
    assert keep(p) == S.E_ALIGN
    if n > 1:
        p[n - 1].v_scale = p[n // 2 - 1].k_scale + 16
        assert keep(p) == S.E_SHAPE
