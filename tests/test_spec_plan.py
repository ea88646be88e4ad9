"""lmxs_plan's kernels on the CPU (hip_on_cpu.hpp), against the definition: whatever
number of requests, nothing outside the tables is written, and pages go where they
belong."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from llmoxide_amd import spec
from tests import spec_oracle as so

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "llmoxide_amd", "csrc")
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")

MORE = r"""
extern "C" int plan_on_cpu(const lmxs_plan_desc* d, const int32_t* lens, const int32_t* fresh, int32_t* table, int32_t* held,
                           int32_t* free_pages, int32_t* n_free, int32_t* cu, int32_t* ctx, int64_t* slots, int32_t* pos) {
    return lmx::spec_plan(d, lens, fresh, table, held, free_pages, n_free, cu, ctx, slots, pos, nullptr);
}
"""


@pytest.fixture(scope="module")
def on_cpu(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    shutil.copy(os.path.join(CSRC, "spec.hpp"), at / "spec.hpp")
    (at / "paged.hpp").write_text('#include "hip_on_cpu.hpp"\n')
    (at / "plan.cpp").write_text(open(os.path.join(CSRC, "spec_plan.hip")).read() + MORE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-I", str(at), "-I", os.path.join(ROOT, "tests"),
                    "-I", os.path.join(ROOT, "include"), "-I", CSRC, str(at / "plan.cpp"), "-o", str(at / "plan.so")], check=True)
    fn = ctypes.CDLL(str(at / "plan.so")).plan_on_cpu
    fn.argtypes = [ctypes.c_void_p] * 11
    return fn


class Guarded:
    """An array among others of its own kind, which have to stay as they are."""

    def __init__(self, x, guard):
        x = np.asarray(x)
        self.n, self.guard = x.size, guard
        self.all = np.full(x.size + 2 * guard, 0x5a5a5a, x.dtype)
        self.all[guard:guard + x.size] = x.ravel()
        self.shape = x.shape

    @property
    def at(self):
        return self.all.ctypes.data + self.guard * self.all.itemsize

    @property
    def x(self):
        return self.all[self.guard:self.guard + self.n].reshape(self.shape)

    def whole(self):
        return np.all(self.all[:self.guard] == 0x5a5a5a) and np.all(self.all[self.guard + self.n:] == 0x5a5a5a)


def run(fn, lens, new, table, held, free, n_free, *, page, n_tokens, trim, maps=True):
    """(page_table, held, free_pages, n_free, cu, ctx_lens, slots, pos) after a plan."""
    n_seq, entries = table.shape
    guard = 2 * n_seq * entries + 1024  # more than n_seq rounded up to a power of two reaches
    ins = [Guarded(np.asarray(x, np.int32), guard) for x in (lens, new)]
    outs = [Guarded(np.asarray(x, np.int32), guard) for x in (table, held, free, n_free)]
    outs += [Guarded(np.full(n, 77, t), guard) for n, t in ((n_seq + 1, np.int32), (n_seq, np.int32), (n_tokens, np.int64),
                                                            (n_tokens, np.int32))]
    d = spec.SpecPlanDesc(n_seq=n_seq, n_tokens=n_tokens, page_size=page, table_stride=entries, n_pages=len(free), trim=int(trim))
    ptrs = [g.at for g in ins + outs]
    if not maps:
        ptrs[-2:] = None, None
    assert fn(ctypes.byref(d), *ptrs) == 0
    for g, name in zip(ins + outs, "lens new_rows page_table held free_pages n_free cu ctx_lens slots pos".split()):
        assert g.whole(), f"written outside {name}"
    return [g.x for g in outs]


def requests(seed, n_seq, page, most):
    """Requests that stay, grow and leave; entries behind `held` hold anything."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, most, n_seq)
    held = -(-lens // page) + rng.integers(0, 3, n_seq)
    new = np.where(rng.random(n_seq) < 0.3, 0, rng.integers(0, most, n_seq))
    left = rng.random(n_seq) < 0.2
    lens, new = np.where(left, 0, lens), np.where(left, 0, new)
    n_pages = int(held.sum() - (-(lens + new) // page).sum() + 5)
    ids = rng.permutation(n_pages)
    table = rng.integers(-5, 1 << 30, (n_seq, 2 * most // page + 4))
    at = 0
    for b in range(n_seq):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    free = rng.integers(-5, 1 << 30, n_pages)
    free[:n_pages - at] = ids[at:]
    return lens, new, table, held, free, [n_pages - at, 7]


# whole waves of the workgroup lie between the requests and the power of two above them in
# 129-192, 257-448 and 513-960
COUNTS = [1, 2, 63, 64, 65, 128, 129, 160, 192, 193, 256, 257, 300, 320, 448, 449, 513, 600, 704, 769, 832, 960, 961, 1024,
          1025, 1200, 2048 + 160]


@pytest.mark.parametrize("n_seq", COUNTS)
@pytest.mark.parametrize("trim", [False, True])
def test_plans_of_any_number_of_requests(on_cpu, n_seq, trim):
    case = requests(n_seq, n_seq, 16, 40)
    for extra in (0, 9000) if n_seq in (160, 600) else (5,):  # rows mapped by either kernel
        n = int(case[1].sum()) + extra or 1
        got = run(on_cpu, *case, page=16, n_tokens=n, trim=trim)
        want = so.plan(case[0], case[1], case[2].astype(np.int32), case[3].astype(np.int32), case[4].astype(np.int32), case[5],
                       page=16, n_tokens=n, n_pages=len(case[4]), trim=trim)
        for name, g, w in zip("table held free n_free cu ctx slots pos".split(), got, want):
            assert np.array_equal(g, w), name



@pytest.mark.parametrize("seed", range(6))
def test_rows_stay_behind_the_cached_ones_where_a_table_ends(on_cpu, seed):
    """Requests at the end of their rows of the table: a row's position, counted back from
    ctx_lens, is that of the map, and not one that is cached.  (A request of more rows than
    the table has positions gets a length below its rows: no positions.)"""
    rng = np.random.default_rng(seed)
    n_seq, entries, page = 40, int(rng.integers(1, 5)), int(rng.choice([16, 32]))
    room = entries * page
    lens = rng.integers(0, room + 20, n_seq)
    lens[:3] = room, room - 1, (1 << 31) - 1
    new = rng.integers(0, 2 * room, n_seq)
    new[:3] = 1, 3, 5
    n = int(new.sum())
    _, held, _, n_free, cu, ctx, slots, pos = run(on_cpu, lens, new, np.full((n_seq, entries), -1), np.zeros(n_seq), np.arange(400),
                                                  [400, 0], page=page, n_tokens=n, trim=bool(seed & 1))
    assert cu.tolist() == [0, *np.cumsum(new)] and n_free[1] == 0
    for b in range(n_seq):
        assert held[b] == -(-min(lens[b] + new[b], room) // page)
        if new[b] > room:
            assert ctx[b] == room < new[b]
            continue
        assert int(ctx[b]) == min(lens[b] + new[b], (1 << 31) - 1)
        for j in range(new[b]):
            r, p = int(cu[b]) + j, int(ctx[b]) - int(new[b]) + j
            assert (slots[r] >= 0) == (p < room) and (pos[r] == p if b != 2 else pos[r] >= p)


def test_a_plan_reads_no_entry_behind_what_is_held(on_cpu):
    """Lengths that pass the 2^30 positions that lengths are counted to: the table has more
    entries, which hold anything, and no row is mapped by them."""
    entries = (1 << 22) + 100  # of 256 positions: 2^30 and 25600
    table = np.full((1, entries), 3, np.int32)
    table[0, :10] = -1
    lens = [(1 << 30) - 4]
    _, _, _, _, _, ctx, slots, pos = run(on_cpu, lens, [9], table, [entries], np.arange(8), [0, 0], page=256, n_tokens=9, trim=False)
    assert ctx[0] == lens[0] + 9 and pos.tolist() == [lens[0] + j for j in range(9)]
    assert slots.tolist() == [3 * 256 + 252 + j for j in range(3)] + [-1] * 6


@pytest.mark.parametrize("n_seq,n_tokens", [(1, 3), (5, 20), (70, 100), (300, 64)])
def test_rows_that_the_maps_have_no_place_for_move_no_others(on_cpu, n_seq, n_tokens):
    """More new rows than n_tokens, which a caller must not bring: the rows that are left
    still stand behind the cached ones, by the lengths as by the map."""
    rng = np.random.default_rng(n_seq)
    lens, new = rng.integers(0, 40, n_seq), rng.integers(1, 9, n_seq)
    new[-1] = 200  # more than the table has positions
    _, _, _, _, cu, ctx, slots, pos = run(on_cpu, lens, new, np.full((n_seq, 4), -1), np.zeros(n_seq), np.arange(4 * n_seq),
                                          [4 * n_seq, 0], page=16, n_tokens=n_tokens, trim=False)
    assert cu.tolist() == [0, *np.minimum(np.cumsum(np.minimum(new, n_tokens)), n_tokens)]
    for b in range(n_seq):
        n = int(cu[b + 1] - cu[b])
        assert ctx[b] == (64 if n > 64 else lens[b] + n)
        assert pos[cu[b]:cu[b + 1]].tolist() == [lens[b] + j for j in range(n)]
