"""Steps with drafted tokens on the GPU at their limits: what a result's own rounding
leaves, full tables, many requests, and streams beside the current one."""
from types import SimpleNamespace

import numpy as np
import pytest

from tests import paged_oracle as po
from tests import spec_oracle as so

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llmoxide_amd as lmx  # noqa: E402
from tests.test_gpu_paged import gpu, on_gpu, rows, say  # noqa: E402
from tests.test_gpu_spec import ints, masks  # noqa: E402
from tests.test_spec_plan import requests  # noqa: E402


# ------------------------------------------------------------------ precision --
@pytest.mark.parametrize("new,ctx", [([1], [40]), ([4, 1, 3], [70, 5, 33]), ([20, 7], [60, 90]), ([70], [100])])
@pytest.mark.parametrize("hd,kv,heads,store", [(64, 2, 8, "f16"), (64, 2, 8, "i8"), (128, 2, 8, "f16"), (128, 2, 8, "i8"),
                                               (256, 1, 4, "i8"), (256, 1, 4, "f16"), (512, 1, 2, "f16"), (512, 1, 2, "i8")])
def test_f16_results_by_masks_are_off_by_their_own_rounding(new, ctx, hd, kv, heads, store):
    """With f16 q the weights have 22 bits, as with f32.  q has one element that is not 0
    in each row head, so that a score is one product (exact: 22 bits) and attend_bound's
    term of head_dim products is that of one.  What it then gives for f32 results, b, is
    some 1e-5 of the result; f16(y) is off from y by 2^-11 |y|, or 2^-25 where f16's
    steps are 2^-24: together (1 + 2^-11) b + 2^-11 |want| + 2^-25.  Weights of 11 bits
    would add 2^-12 of each weighted value or so, half of the last place."""
    say("f16 rounding", new, hd, store)
    c = po.PagedCase(101, new=new, ctx=ctx, page=16, kv=kv, hd=hd, store=store)
    cache, batch = on_gpu(c)
    rng = np.random.default_rng(102)
    q = np.zeros((c.tokens, heads, hd), np.float32)
    at = rng.integers(0, hd, (c.tokens, heads, 1))
    np.put_along_axis(q, at, (rng.standard_normal(at.shape) * 8).astype(np.float16).astype(np.float32), 2)
    sees = masks(c, 103, "tree")
    seen = gpu(np.concatenate([so.words_of(m, -(-max(new) // 64)) for m in sees]))
    got = lmx.spec_attention(gpu(q.reshape(c.tokens, -1)).half(), cache, batch, seen, n_heads=heads)
    want, mag, prod, top = so.attend(c, q, sees, heads=heads)
    b = po.attend_bound(SimpleNamespace(hd=1, store=store), mag, prod, top, max(ctx), f32=True)
    off = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    most = (1 + 2.0 ** -11) * b + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    assert np.all(off <= most), f"{(off > most).sum()} of {off.size} are off by up to {(off / most).max():.2f} times the bound"


# --------------------------------------------------------------- verification --
@pytest.mark.parametrize("vocab", [3, 700, 32768, 40000])
def test_a_test_beside_its_border_is_decided_in_64_bits(vocab):
    """The root's second child: a is 1, W = (3/8 - 2^-27) + (5/8 - 1/2) = 1/2 - 2^-27, and
    u W q = 1/2 W 1/2 = 1/8 - 2^-29 lies below w = 1/8.  With 3/8 - 2^-27 rounded to 24
    bits W is 1/2, and the child, for which 1/8 < 1/8 fails, is refused."""
    p, q = np.zeros((3, vocab), np.float32), np.zeros((3, vocab), np.float32)
    p[0, :3], q[0, :3] = (0, 3 / 8, 5 / 8), (0.5, 2.0 ** -27, 0.5)
    p[1:, 1] = q[1:, 1] = 1
    tokens, u, r, parent = [0, 0, 2], [0, 0.5, 0.5], [0.5], [-1, 0, 0]
    path, token = so.verify(p, tokens, u, r[0], parent, q)
    assert path == [0, 2] and token == 1  # child 1, of p 0, is refused and makes a 1
    got = lmx.spec_verify(gpu(p), ints(tokens), gpu(np.float32(u)), gpu(np.float32(r)), ints([0, 3]), max_new=3,
                          parent=ints(parent), q=gpu(q))
    assert got.path.tolist() == [[0, 2, -1]] and got.accepted.tolist() == [2] and got.token.tolist() == [1]


# ----------------------------------------------------------------------- plans --
@pytest.mark.parametrize("n_seq", [129, 160, 192, 257, 300, 448, 513, 700, 832, 960, 1024 + 160])
@pytest.mark.parametrize("trim", [False, True])
@pytest.mark.parametrize("extra", [1, 9000])
def test_plans_of_any_number_of_requests(n_seq, trim, extra):
    """Numbers of requests between a power of two and the next, rows mapped by either
    kernel; the tables lie among rows that have to stay as they are."""
    say("plan", n_seq, trim, extra)
    lens, new, table, held, free, n_free = requests(n_seq, n_seq, 16, 40)
    n = int(new.sum()) + extra
    wide = torch.full((3 * n_seq, table.shape[1]), 77, dtype=torch.int32, device="cuda")
    wide[n_seq:2 * n_seq] = ints(table)
    t = lmx.PageTables(wide[n_seq:2 * n_seq], ints(held), ints(free), ints(n_free), page_size=16)
    got = lmx.spec_plan(t, ints(lens), ints(new), n_tokens=n, trim=trim)
    want = so.plan(lens, new, table.astype(np.int32), held.astype(np.int32), free.astype(np.int32), n_free, page=16, n_tokens=n,
                   n_pages=len(free), trim=trim)
    for name, g, w in zip("table held free n_free cu ctx slots pos".split(), (t.page_table, t.held, t.free_pages, t.n_free, *got), want):
        assert np.array_equal(g.cpu().numpy(), w), name
    assert (wide[:n_seq] == 77).all() and (wide[2 * n_seq:] == 77).all()
