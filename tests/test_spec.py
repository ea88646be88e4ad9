"""Steps with drafted tokens, on the CPU: the header and its mirrors, refusals (every
call here returns before anything is enqueued), and what pins the oracle."""
import ctypes
import math
import os
import random
import re
import subprocess

import numpy as np
import pytest

import llmoxide_amd as lmx
from llmoxide_amd import paged, spec
from tests import spec_oracle as so
from tests.test_paged import BAD_BATCHES, BAD_POOLS, FAKE, FAR, S, batch, pool
from tests.test_paged_workspace import SHAPES, rows as batch_of, wide

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "lmx", "spec.h")
RUST = os.path.join(ROOT, "rust", "llmoxide-hip-ffi", "src", "spec.rs")
BIG = 1 << 36  # between arrays that may not overlap


def header():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_header_compiles_as_c_and_cxx(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "lmx/spec.h"\nint main(void){lmxs_plan_desc p; return sizeof p == 0;}\n')
    for cc, extra in (("gcc", ["-std=c99"]), ("g++", ["-x", "c++", "-std=c++17"])):
        r = subprocess.run([cc, *extra, "-fsyntax-only", "-Wall", "-Werror", "-I",
                            os.path.join(ROOT, "include"), str(src)], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr


def test_library_exports_what_the_header_declares():
    names = set(re.findall(r"\b(lmxs_\w+)\s*\(", header()))
    assert names == set(spec.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", lmx.LIB_PATH], capture_output=True, text=True).stdout
    assert set(re.findall(r"\bT (lmxs_\w+)", out)) == names


C_TYPES = {"uint32_t": "u32", "uint64_t": "u64", "int64_t": "i64", "float": "f32", "int32_t": "i32", "void": "c_void",
           "lmx_dtype": "i32", "lmx_status": "i32", "lmx_stream": "HipStream", "size_t": "usize"}


def to_rust(ctype):
    const = "const" in ctype
    words = [w for w in re.findall(r"\w+|\*", ctype) if w != "const"]
    t = C_TYPES.get(words[0]) or "".join(p.capitalize() for p in words[0].split("_"))
    return ("*const " if const else "*mut ") * words.count("*") + t  # const: all of a pointer's levels


def test_rust_mirror_matches():
    src = re.sub(r"//[^\n]*", "", open(RUST).read())
    structs = {n: re.findall(r"pub (\w+): ([^,]+),", b) for n, b in re.findall(r"pub struct (\w+) \{(.*?)\}", src, flags=re.S)}
    for body, name in re.findall(r"typedef struct \{(.*?)\}\s*(\w+);", header(), flags=re.S):
        want = []
        for decl in body.split(";"):
            decl = " ".join(decl.split())
            if decl:
                kind, n = re.match(r"^(.*?)(\w+)$", decl).groups()
                want.append((n, to_rust(kind)))
        assert structs["".join(p.capitalize() for p in name.split("_"))] == want, name
    fns = {}
    for name, args, ret in re.findall(r"pub fn (lmxs_\w+)\((.*?)\)\s*->\s*([^;]+);", src, flags=re.S):
        fns[name] = ([tuple(x.strip() for x in a.split(":")) for a in args.split(",") if a.strip()], ret.strip())
    declared = re.findall(r"^(\w+) (lmxs_\w+)\(([^;]*?)\);", header(), flags=re.M | re.S)
    for ret, name, args in declared:
        want = []
        for a in " ".join(args.split()).split(","):
            kind, n = re.match(r"^(.*?)(\w+)$", a.strip()).groups()
            want.append((n, to_rust(kind)))
        assert fns[name] == (want, to_rust(ret)), name
    assert len(fns) == len(declared) == len(spec.SIGNATURES)
    assert "LMXS_MAX_ROWS: u32 = 1024;" in src and "#define LMXS_MAX_ROWS 1024" in header() and spec.MAX_ROWS == 1024


def test_python_structures_have_the_headers_sizes(tmp_path):
    pairs = [("lmxs_plan_desc", spec.SpecPlanDesc), ("lmxs_rope", spec.SpecRope), ("lmxs_verify_desc", spec.SpecVerifyDesc)]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "lmx/spec.h"\nint main(void) {\n' +
                   "".join(f'  printf("%zu\\n", sizeof({c}));\n' for c, _ in pairs) + "  return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(p) for _, p in pairs]


# ----------------------------------------------------------------- refusals --
def plan(lens=FAKE, new=FAKE + BIG, table=FAKE + 2 * BIG, held=FAKE + 3 * BIG, free=FAKE + 4 * BIG, n_free=FAKE + 5 * BIG,
         cu=FAKE + 6 * BIG, ctx=FAKE + 7 * BIG, slots=FAKE + 8 * BIG, pos=FAKE + 9 * BIG, **kw):
    d = dict(n_seq=4, n_tokens=100, page_size=16, table_stride=8, n_pages=32, trim=1)
    d.update(kw)
    return spec.spec_lib().lmxs_plan(ctypes.byref(spec.SpecPlanDesc(**d)), lens, new, table, held, free, n_free, cu, ctx,
                                     slots, pos, None)


@pytest.mark.parametrize("kw,code", [
    (dict(lens=None), S.E_NULL), (dict(new=None), S.E_NULL), (dict(table=None), S.E_NULL), (dict(held=None), S.E_NULL),
    (dict(free=None), S.E_NULL), (dict(n_free=None), S.E_NULL), (dict(cu=None), S.E_NULL), (dict(ctx=None), S.E_NULL),
    (dict(page_size=8), S.E_UNSUPPORTED), (dict(page_size=100), S.E_UNSUPPORTED), (dict(n_seq=0), S.E_SHAPE),
    (dict(n_seq=1 << 21), S.E_SHAPE), (dict(n_tokens=0), S.E_SHAPE), (dict(n_tokens=(1 << 28) + 1), S.E_SHAPE),
    (dict(table_stride=0), S.E_SHAPE), (dict(n_pages=0), S.E_SHAPE), (dict(n_pages=1 << 30), S.E_SHAPE),
    (dict(trim=2), S.E_SHAPE), (dict(n_seq=1 << 20, table_stride=257), S.E_SHAPE), (dict(lens=FAKE + 2), S.E_ALIGN),
    (dict(slots=FAKE + 8 * BIG + 4), S.E_ALIGN), (dict(pos=FAKE + 1), S.E_ALIGN),
    (dict(pos=FAKE + 8 * BIG + 796), S.E_SHAPE), (dict(cu=FAKE + 8), S.E_SHAPE), (dict(held=FAKE), S.E_SHAPE),
    (dict(ctx=FAKE + 6 * BIG + 16), S.E_SHAPE),
])
def test_bad_plans_are_refused(kw, code):
    assert plan(**kw) == code


def tree(b=None, parent=FAKE + BIG, words=1, window=0, pos=FAKE + 2 * BIG, seen=FAKE + 3 * BIG):
    return spec.spec_lib().lmxs_tree(ctypes.byref(b or batch()), parent, words, window, pos, seen, None)


@pytest.mark.parametrize("kw,code", [
    (dict(parent=None), S.E_NULL), (dict(pos=None, seen=None), S.E_NULL), (dict(words=0), S.E_SHAPE),
    (dict(words=17), S.E_SHAPE), (dict(b=batch(n_tokens=65, max_new=65)), S.E_SHAPE), (dict(window=1 << 30), S.E_SHAPE),
    (dict(parent=FAKE + 1), S.E_ALIGN), (dict(seen=FAKE + 3 * BIG + 4), S.E_ALIGN), (dict(pos=FAKE + BIG + 12), S.E_SHAPE),
    (dict(seen=FAKE), S.E_SHAPE), (dict(b=batch(cu=None)), S.E_NULL), (dict(b=batch(n_seq=0)), S.E_SHAPE),
    (dict(b=batch(max_new=5)), S.E_SHAPE), (dict(b=batch(ctx_lens=FAKE + 2)), S.E_ALIGN),
])
def test_bad_trees_are_refused(kw, code):
    assert tree(**kw) == code


def prologue(p=None, b=None, r=(0, 1.0), pos=FAKE + BIG, q=FAKE, k=FAKE, v=FAKE, qg=None, kg=None, rf=None, out=FAR,
             dt=lmx.F32, **kw):
    d = dict(n_heads=4, n_rot=128, v_norm=0, q_head_stride=0, q_row_stride=0, kv_row_stride=0, rms_eps=1e-6, rope_base=1e6)
    d.update(kw)
    rope = None if r is None else ctypes.byref(spec.SpecRope(*r))
    return spec.spec_lib().lmxs_prologue(ctypes.byref(p or pool()), ctypes.byref(b or batch()),
                                         ctypes.byref(paged.PagedPrologueDesc(**d)), rope, pos, q, k, v, qg, kg, rf, out,
                                         dt, None)


def attn(p=None, b=None, seen=FAKE + BIG, words=1, pos=FAKE + 2 * BIG, q=FAKE, out=FAR, dt=lmx.F32, ws=None, ws_bytes=0, **kw):
    d = dict(n_heads=4, window=0, q_head_stride=0, q_row_stride=0, scale=0.1)
    d.update(kw)
    return spec.spec_lib().lmxs_attn(ctypes.byref(p or pool()), ctypes.byref(b or batch()),
                                     ctypes.byref(paged.PagedAttnDesc(**d)), seen, words, pos, q, dt, out, ws, ws_bytes, None)


def keep(p=None, b=None, n=1, path=FAKE, stride=8, accepted=FAKE):
    p = p or pool()
    pools = (ctypes.c_void_p * max(1, min(n, 4)))(*[ctypes.addressof(p)] * max(1, min(n, 4)))
    return spec.spec_lib().lmxs_keep(pools, n, ctypes.byref(b or batch()), path, stride, accepted, None)


@pytest.mark.parametrize("call", [prologue, attn, keep])
@pytest.mark.parametrize("kw,code", BAD_POOLS)
def test_bad_pools_are_refused(call, kw, code):
    assert call(p=pool(**kw)) == code


@pytest.mark.parametrize("call", [prologue, attn, keep])
@pytest.mark.parametrize("kw,code", BAD_BATCHES)
def test_bad_batches_are_refused(call, kw, code):
    assert call(b=batch(**kw)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(r=None), S.E_NULL), (dict(r=(2, 1.0)), S.E_SHAPE), (dict(r=(0, math.inf)), S.E_SHAPE),
    (dict(r=(1, math.nan)), S.E_SHAPE), (dict(pos=FAKE + 2), S.E_ALIGN), (dict(pos=FAR + 64), S.E_SHAPE),
    (dict(n_rot=129), S.E_SHAPE), (dict(q=None), S.E_NULL), (dict(out=FAKE + 512), S.E_SHAPE), (dict(dt=7), S.E_UNSUPPORTED),
])
def test_bad_prologues_are_refused(kw, code):
    assert prologue(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(seen=None), S.E_NULL), (dict(pos=None, window=5), S.E_NULL), (dict(words=0), S.E_SHAPE), (dict(words=17), S.E_SHAPE),
    (dict(b=batch(n_tokens=70, max_new=70)), S.E_SHAPE), (dict(seen=FAKE + BIG + 4), S.E_ALIGN), (dict(pos=FAKE + 1), S.E_ALIGN),
    (dict(seen=FAR + 64), S.E_SHAPE), (dict(pos=FAR), S.E_SHAPE), (dict(q=None), S.E_NULL), (dict(n_heads=5), S.E_SHAPE),
    (dict(out=FAKE), S.E_SHAPE),
    (dict(b=batch(max_ctx=4096, table_stride=256)), S.E_WORKSPACE),
    (dict(b=batch(max_ctx=4096, table_stride=256), ws=FAKE + 8, ws_bytes=1 << 30), S.E_ALIGN),
])
def test_bad_attention_calls_are_refused(kw, code):
    assert attn(**kw) == code


def verify(cu=FAKE, tokens=FAKE + BIG, parent=FAKE + 2 * BIG, p=FAKE + 3 * BIG, q=FAKE + 4 * BIG, dt=lmx.F32,
           u=FAKE + 5 * BIG, r=FAKE + 6 * BIG, path=FAKE + 7 * BIG, accepted=FAKE + 8 * BIG, token=FAKE + 9 * BIG,
           lens=FAKE + 10 * BIG, ws=FAKE + 11 * BIG, ws_bytes=1 << 30, **kw):
    d = dict(n_seq=4, n_tokens=40, max_new=10, vocab=1000, p_stride=0, q_stride=0, greedy=0)
    d.update(kw)
    return spec.spec_lib().lmxs_verify(ctypes.byref(spec.SpecVerifyDesc(**d)), cu, tokens, parent, p, q, dt, u, r, path,
                                       accepted, token, lens, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(cu=None), S.E_NULL), (dict(tokens=None), S.E_NULL), (dict(p=None), S.E_NULL), (dict(u=None), S.E_NULL),
    (dict(r=None), S.E_NULL), (dict(path=None), S.E_NULL), (dict(accepted=None), S.E_NULL), (dict(token=None), S.E_NULL),
    (dict(dt=3), S.E_UNSUPPORTED), (dict(n_seq=0), S.E_SHAPE), (dict(n_tokens=0), S.E_SHAPE), (dict(max_new=0), S.E_SHAPE),
    (dict(max_new=41), S.E_SHAPE), (dict(n_tokens=5000, max_new=1025), S.E_SHAPE), (dict(vocab=0), S.E_SHAPE),
    (dict(vocab=(1 << 24) + 1), S.E_SHAPE), (dict(p_stride=999), S.E_SHAPE), (dict(q_stride=1), S.E_SHAPE),
    (dict(greedy=2), S.E_SHAPE), (dict(n_seq=1 << 20, vocab=1 << 20), S.E_SHAPE),
    (dict(ws=None, vocab=40000), S.E_WORKSPACE), (dict(ws_bytes=100, vocab=40000), S.E_WORKSPACE),
    (dict(ws=FAKE + 11 * BIG + 8, vocab=40000), S.E_ALIGN), (dict(p=FAKE + 3 * BIG + 2), S.E_ALIGN),
    (dict(lens=FAKE + 3), S.E_ALIGN), (dict(path=FAKE + 5 * BIG), S.E_SHAPE), (dict(lens=FAKE + 8 * BIG), S.E_SHAPE),
    (dict(token=FAKE + 3 * BIG + 159996), S.E_SHAPE), (dict(ws=FAKE + 9 * BIG, vocab=40000), S.E_SHAPE),
])
def test_bad_verifications_are_refused(kw, code):
    assert verify(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(path=None), S.E_NULL), (dict(accepted=None), S.E_NULL), (dict(n=0), S.E_SHAPE), (dict(n=65537), S.E_SHAPE),
    (dict(stride=2), S.E_SHAPE), (dict(path=FAKE + 2), S.E_ALIGN), (dict(accepted=FAKE + 1), S.E_ALIGN),
    (dict(b=batch(n_tokens=2000, max_new=1025)), S.E_SHAPE),
])
def test_bad_keepings_are_refused(kw, code):
    assert keep(**kw) == code


def test_layers_of_different_geometry_are_refused():
    for kw in (dict(n_pages=9), dict(page_size=32), dict(n_kv_heads=1), dict(head_dim=64),
               dict(store=paged.STORE_I8, k_scale=FAKE, v_scale=FAKE)):
        two = pool(), pool(**kw)
        pools = (ctypes.c_void_p * 2)(*map(ctypes.addressof, two))
        assert spec.spec_lib().lmxs_keep(pools, 2, ctypes.byref(batch()), FAKE, 8, FAKE, None) == S.E_SHAPE


def test_null_descriptions_are_refused():
    L = spec.spec_lib()
    assert L.lmxs_plan(None, *[FAKE] * 10, None) == S.E_NULL
    assert L.lmxs_tree(None, FAKE, 1, 0, FAKE, FAKE, None) == S.E_NULL
    assert L.lmxs_verify(None, *[FAKE] * 5, 0, *[FAKE] * 7, 0, None) == S.E_NULL
    assert L.lmxs_verify_workspace_bytes(None) == 0
    assert L.lmxs_keep(None, 1, ctypes.byref(batch()), FAKE, 8, FAKE, None) == S.E_NULL
    assert L.lmxs_keep((ctypes.c_void_p * 1)(None), 1, ctypes.byref(batch()), FAKE, 8, FAKE, None) == S.E_NULL


def test_verification_workspace():
    def need(**kw):
        d = dict(n_seq=4, n_tokens=40, max_new=10, vocab=1000, p_stride=0, q_stride=0, greedy=0)
        d.update(kw)
        return spec.spec_lib().lmxs_verify_workspace_bytes(ctypes.byref(spec.SpecVerifyDesc(**d)))
    assert need(greedy=1) == 0 and need(vocab=0) == 0
    assert need() == need(vocab=32768) == 0  # one workgroup a request
    assert 0 < need(vocab=32769) <= need(vocab=100000) <= need(vocab=100000, n_seq=8)


# -------------------------------------------------------------- the oracle --
def test_oracle_plan_by_hand():
    table = np.array([[7, 8, -1], [9, -1, -1], [3, 4, 5]], np.int32)
    held, free = np.array([2, 1, 3], np.int32), np.array([0, 1, 2] + [9] * 7, np.int32)
    got = so.plan([5, 16, 0], [4, 20, 0], table, held, free, [3, 0], page=16, n_tokens=26, n_pages=10, trim=True)
    # request 2 leaves: 5, 4, 3 go on the list; request 0 needs one page: 8 goes on it; request 1 takes 8 and 3... from the top
    assert got[0].tolist() == [[7, -1, -1], [9, 8, 3], [-1, -1, -1]]
    assert got[1].tolist() == [1, 3, 0] and got[3].tolist() == [5, 0] and got[2][:5].tolist() == [0, 1, 2, 5, 4]
    assert got[4].tolist() == [0, 4, 24, 24] and got[5].tolist() == [9, 36, 0]
    assert got[6].tolist() == [7 * 16 + i for i in range(5, 9)] + [8 * 16 + i for i in range(16)] + [48, 49, 50, 51] + [-1, -1]


def test_oracle_tree_by_hand():
    depth, sees = so.tree([-1, 0, 0, 1, 3, 9, -1])
    assert depth.tolist() == [0, 1, 1, 2, 3, 0, 0]
    assert [np.nonzero(r)[0].tolist() for r in sees] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [5], [6]]
    assert [np.nonzero(r)[0].tolist() for r in so.tree([-1, 0, 1, 2], 2)[1]] == [[0], [0, 1], [1, 2], [2, 3]]
    assert so.words_of(np.eye(65, dtype=bool)[63:], 2).tolist() == [[-1 << 63, 0], [0, 1]]


@pytest.mark.parametrize("q", [None, [0.5, 0.3, 0.2, 0.0]])
@pytest.mark.parametrize("children", [1, 2, 3])
def test_oracle_verification_gives_the_targets_distribution(q, children):
    """What comes first behind the root, summed over drafts and a fine grid of random
    numbers, is distributed as p: the midpoints of N cells a number are off by at most
    one cell at each border."""
    p = np.array([[0.1, 0.45, 0.2, 0.25]] + [[0.25] * 4] * children)
    N = 24
    grid = (np.arange(N) + 0.5) / N
    got = np.zeros(4)
    if q is None:
        drafts = [((1, 3, 2)[:children], 1.0)]
    else:
        drafts = [(d, float(np.prod([q[t] for t in d]))) for d in np.ndindex(*[4] * children)]
    for d, weight in drafts:
        if weight == 0:
            continue
        for us in np.ndindex(*[N] * min(children, 2)):
            u = [0.0] + [grid[i] for i in us] + [0.5] * (children - len(us))
            for r in grid[::3]:
                cells = N ** len(us) * len(grid[::3])
                path, token = so.verify(p, [0, *d], u, r, [-1] + [0] * children,
                                        None if q is None else np.array([q] * (children + 1)))
                first = d[path[1] - 1] if len(path) > 1 else token
                got[first] += weight / cells
    # a third child's number is one point here: its test is all or nothing, and only the sum below is checked
    assert abs(got.sum() - 1) < 1e-9
    if children < 3:
        assert np.abs(got - p[0]).max() < 0.06


def test_oracle_verification_of_a_draft_like_the_target_accepts_all():
    rng = np.random.default_rng(1)
    p = rng.dirichlet([1.0] * 9, 6)
    tok = [0, *(rng.integers(0, 9, 5))]
    path, _ = so.verify(p, tok, rng.random(6), 0.3, list(range(-1, 5)), p)
    assert path == list(range(6))


def test_oracle_keep_by_hand():
    from tests.paged_oracle import PagedCase
    c = PagedCase(1, new=[5], ctx=[21], page=16, kv=1, hd=64)
    k, v, _, _ = so.keep(c, np.array([[0, 2, 4, -1, -1]]), [3], [c.k, c.v, None, None])
    for j, src in ((17, 18), (18, 20)):
        (p1, s1), (p0, s0) = c.place(0, j), c.place(0, src)
        assert np.array_equal(k[p1, 0, s1], c.k[p0, 0, s0]) and np.array_equal(v[p1, 0, :, s1], c.v[p0, 0, :, s0])


def test_oracle_masked_attention_of_chains_is_the_causal_one():
    from tests import paged_oracle as po
    c = po.PagedCase(2, new=[4, 1], ctx=[20, 7], page=16, kv=2, hd=64)
    q = np.random.default_rng(3).standard_normal((c.tokens, 4, 64)).astype(np.float32)
    sees = [so.tree(np.arange(-1, n - 1))[1] for n in c.new]
    for window in (0, 3, 30):
        pos = [p for _, _, p, _ in c.row_places()]
        mine = [so.tree(np.arange(-1, n - 1), window)[1] for n in c.new]
        got = so.attend(c, q, mine if window else sees, heads=4, window=window, pos=pos)[0]
        assert np.allclose(got, po.attend(c, q, heads=4, window=window)[0], rtol=1e-12, atol=1e-12)


# ------------------------------------------------------------ rope scaling --
def test_rope_scaling():
    assert lmx.rope_scaling(8, kind="linear", factor=4) == ([4.0] * 4, 1.0)
    for kind in ("bands", "yarn"):
        f, m = lmx.rope_scaling(128, kind=kind, factor=8, rope_base=5e5, trained_ctx=8192, fast=4 if kind == "bands" else 32, slow=1)
        assert len(f) == 64 and f[0] == 1.0 and abs(f[-1] - 8) < 1e-12 and all(a <= b for a, b in zip(f, f[1:]))
        assert m == (1.0 if kind == "bands" else 0.1 * math.log(8) + 1)
    # bands, a pair in between by hand: 8192 positions, turns = 8192 / (2 pi base^(j/half))
    f, _ = lmx.rope_scaling(128, kind="bands", factor=8, rope_base=5e5, trained_ctx=8192, fast=4, slow=1)
    for j, x in enumerate(f):
        turns = 8192 / (2 * math.pi * 5e5 ** (j / 64))
        want = 1.0 if turns >= 4 else 8.0 if turns <= 1 else 1 / ((turns - 1) / 3 + (1 - (turns - 1) / 3) / 8)
        assert abs(x - want) < 1e-12
    for bad in (dict(kind="x", factor=2), dict(kind="linear", factor=0), dict(kind="yarn", factor=2),
                dict(kind="bands", factor=2, trained_ctx=10, fast=1, slow=2)):
        with pytest.raises(ValueError):
            lmx.rope_scaling(64, **bad)
    with pytest.raises(ValueError):
        lmx.rope_scaling(7, kind="linear", factor=2)


# -------------------------------------------------- what calls may rely on --
def test_a_pool_twice_among_the_layers_is_refused():
    """A layer's moves are ordered within one pool only."""
    far = dict(k=FAKE + BIG, v=FAKE + 2 * BIG)
    one = pool()

    def call(*pools):
        return spec.spec_lib().lmxs_keep((ctypes.c_void_p * len(pools))(*map(ctypes.addressof, pools)), len(pools),
                                         ctypes.byref(batch()), FAKE + 2, 8, FAKE, None)
    assert call(one, pool(**far)) == S.E_ALIGN  # the next check's
    for other in (one, pool(), pool(**dict(far, v=one.v)), pool(**dict(far, k=one.k)), pool(**dict(far, k=one.v)),
                  pool(**dict(far, v=one.k + 16))):
        assert call(one, pool(**far), other) == S.E_SHAPE


def seen_workspace(p, b, heads, window=0):
    d = paged.PagedAttnDesc(n_heads=heads, window=window, q_head_stride=0, q_row_stride=0, scale=0.1)
    return spec.spec_lib().lmxs_attn_workspace_bytes(ctypes.byref(p), ctypes.byref(b), ctypes.byref(d))


@pytest.mark.parametrize("kv,group,hd", SHAPES + [(2, 16, 512), (16, 1, 512), (1, 40, 64)])
@pytest.mark.parametrize("store", [paged.STORE_F16, paged.STORE_I8])
def test_the_workspace_of_a_batch_serves_every_smaller_one(kv, group, hd, store):
    rng = random.Random(kv * hd + store)
    p = wide(kv=kv, hd=hd, store=store)

    def most(hi):
        return max(1, min(hi, int(2 ** rng.uniform(0, 14))))
    for _ in range(400):
        tokens = most(1 << 14)
        big = (most(40), tokens, most(min(tokens, 1024)), most(1 << 14))
        tokens = most(tokens)
        small = (most(big[0]), tokens, most(min(tokens, big[2])), most(big[3]))
        window = rng.choice([0, 1, 100, 1 << 20])
        has = seen_workspace(p, batch_of(*big), kv * group)
        assert seen_workspace(p, batch_of(*small), kv * group, window) <= has, (small, big, window)


@pytest.mark.parametrize("hd,seqs,small", [
    (128, 1, (1, 1, 1)), (128, 1, (1, 6, 6)), (128, 1, (1, 300, 300)), (64, 40, (33, 544, 512)), (256, 40, (8, 64, 9)),
    (512, 1, (1, 4, 4)), (512, 9, (2, 40, 39)), (512, 9, (1, 2, 2)),
])
@pytest.mark.parametrize("store", [paged.STORE_F16, paged.STORE_I8])
@pytest.mark.parametrize("dt", [lmx.F32, lmx.F16])
@pytest.mark.parametrize("window", [0, 4000])
def test_calls_take_the_workspace_of_a_larger_batch(hd, seqs, small, store, dt, window):
    """Each small batch is cut between workgroups: its call needs a workspace, and goes on
    past its size to the next check (the alignment), which refuses it."""
    p = wide(kv=2, hd=hd, store=store)
    has = seen_workspace(p, batch_of(seqs, 1024, 1024, 32768), 8)
    call = dict(p=p, b=batch_of(*small, 8192), dt=dt, n_heads=8, window=window, words=16, out=FAR * 64, ws=FAKE + 8)
    assert attn(ws_bytes=0, **call) == S.E_WORKSPACE
    assert attn(ws_bytes=has, **call) == S.E_ALIGN


class Fake:
    """A tensor's looks, of device 0."""

    def __init__(self, *shape, dtype=None, at=0, contiguous=True):
        import torch
        self.shape, self.dtype, self.at, self.flat = shape, dtype or torch.int32, at, contiguous
        self.device = torch.device("cuda", at) if at >= 0 else torch.device("cpu")

    def dim(self):
        return len(self.shape)

    def numel(self):
        return math.prod(self.shape)

    def get_device(self):
        return self.at

    def is_contiguous(self):
        return self.flat

    def data_ptr(self):
        return FAKE

    def stride(self):
        return tuple(math.prod(self.shape[i + 1:]) for i in range(len(self.shape)))


def test_tensors_and_streams_of_another_device_are_refused(monkeypatch):
    """Stand-ins for what two GPUs would give: nothing but devices is read before the call."""
    pytest.importorskip("torch")

    class Stream:
        def __init__(self, at):
            self.device_index, self.cuda_stream = at, None

    def plan(at=0, lens=0, out=0, stream=None):
        tables = spec.PageTables(*[Fake(*s, at=at) for s in ((3, 5), (3,), (9,), (2,))], page_size=16)
        step = spec.StepPlan(Fake(4, at=out), Fake(3, at=out), None, Fake(7, at=out))
        return spec.spec_plan(tables, Fake(3, at=lens), Fake(3, at=at), out=step, stream=stream)
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    for kw in (dict(lens=1), dict(out=1), dict(at=1, lens=1, out=1), dict(stream=Stream(1)), dict(lens=-1)):
        with pytest.raises(ValueError):
            plan(**kw)

    def verify(cu=0, p=0, u=0, stream=None, workspace=None, out=None):
        import torch
        f32 = torch.float32
        return spec.spec_verify(Fake(7, 30, dtype=f32, at=p), Fake(7, at=p), Fake(7, dtype=f32, at=u), Fake(3, dtype=f32, at=p),
                                Fake(4, at=cu), max_new=4, out=out, stream=stream, workspace=workspace)

    def held(at):
        return spec.Verified(Fake(3, 4, at=at), Fake(3, at=at), Fake(3, at=at))
    for kw in (dict(cu=1, out=held(0)), dict(u=1, out=held(0)), dict(out=held(1)), dict(p=1, cu=1, u=1, out=held(1)),
               dict(stream=Stream(1), out=held(0)), dict(workspace=lmx.Workspace(device="cuda:1"), out=held(0))):
        with pytest.raises(ValueError):
            verify(**kw)


def test_python_tables_and_plans_refuse_what_does_not_fit():
    torch = pytest.importorskip("torch")

    def tables(**kw):  # name: shape, or looks
        shapes = dict(table=(3, 5), held=(3,), free=(9,), n_free=(2,))
        return spec.PageTables(*[Fake(*(kw[n] if isinstance(kw.get(n), tuple) else s),
                                      **(kw[n] if isinstance(kw.get(n), dict) else {})) for n, s in shapes.items()],
                               page_size=16)
    assert (tables().n_seq, tables().entries, tables().n_pages) == (3, 5, 9)
    for kw, error in ((dict(table=(15,)), ValueError), (dict(held=(4,)), ValueError), (dict(n_free=(1,)), ValueError),
                      (dict(free=dict(dtype=torch.int64)), TypeError), (dict(held=dict(at=1)), ValueError),
                      (dict(table=dict(at=-1)), ValueError), (dict(table=dict(contiguous=False)), ValueError)):
        with pytest.raises(error):
            tables(**kw)
    with pytest.raises(ValueError):
        spec.spec_plan(tables(), Fake(3), Fake(3))  # no rows given
    with pytest.raises(ValueError):
        spec.spec_keep([], None, None, None)
